"""CPU checks of ffn.block's place in torch's autograd, with its two passes replaced by plain torch (the kernels need a GPU)."""
import pytest
import torch

from chpl_b200 import _lib, ckpt8, ffn


class Passes:
    """Plain passes of Y = (X W1^T + b1)^3 W2^T + b2 [+ X] with the interface of ffn.forward and ffn.backward; what is
    held goes through as it is."""

    def __init__(self):
        self.calls = []

    def forward(self, x, w1, b1, w2, b2, *, act="gelu", residual=False, save=False, stream=None):
        assert x.dim() == 2
        self.calls.append(("forward", save))
        with torch.no_grad():
            z = x @ w1.t() + (0 if b1 is None else b1)
            y = z ** 3 @ w2.t() + (0 if b2 is None else b2) + (x if residual else 0)
            held = [ckpt8.Ckpt8(v.clone(), torch.zeros(v.shape[0], 1, dtype=torch.uint8), v.dtype) for v in (x, z)]
        return (y, ffn.Saved(*held, act, residual)) if save else y

    def backward(self, dy, saved, w1, w2, *, need_dx=True, need_dw1=True, need_dw2=True, need_db=True, grad_dtype=None, stream=None):
        assert dy.dim() == 2
        self.calls.append(("backward", need_dx, need_dw1, need_dw2, need_db))
        with torch.no_grad():
            x, z = saved.x.codes, saved.z.codes
            dz = (dy @ w2) * 3 * z ** 2
            dx = dz @ w1 + (dy if saved.residual else 0)
            return (dx if need_dx else None, dz.t() @ x if need_dw1 else None, dz.sum(0) if need_db else None,
                    dy.t() @ z ** 3 if need_dw2 else None, dy.sum(0) if need_db else None)


@pytest.fixture
def passes(monkeypatch):
    p = Passes()
    monkeypatch.setattr(ffn, "forward", p.forward)
    monkeypatch.setattr(ffn, "backward", p.backward)
    return p


def leaves(frozen=(), lead=(5,)):
    g = torch.Generator().manual_seed(1)
    t = {"x": torch.randn(*lead, 3, generator=g), "w1": torch.randn(4, 3, generator=g), "b1": torch.randn(4, generator=g),
         "w2": torch.randn(3, 4, generator=g), "b2": torch.randn(3, generator=g)}
    t = {name: v.double().requires_grad_(name not in frozen) for name, v in t.items()}
    return t


def plain(x, w1, b1, w2, b2):
    return (x @ w1.t() + b1) ** 3 @ w2.t() + b2 + x


def test_first_gradients(passes):
    t = leaves()
    dy = torch.randn(5, 3, dtype=torch.float64)
    want = torch.autograd.grad(plain(**t), list(t.values()), dy)
    got = torch.autograd.grad(ffn.block(*t.values(), "gelu", True), list(t.values()), dy)
    assert all(torch.allclose(a, b) for a, b in zip(got, want))


def test_a_second_differentiation_raises(passes):
    """The block's backward is not differentiable: a gradient penalty raises instead of losing the block's share, also
    where dy carries no graph of its own."""
    for weight in (1.0, torch.ones((), dtype=torch.float64, requires_grad=True)):
        t = leaves()
        y = ffn.block(*t.values(), "gelu", True)
        dx, = torch.autograd.grad((y * weight).sum() + (t["x"] ** 2).sum(), t["x"], create_graph=True)
        with pytest.raises(_lib.ChplError, match="differentiated again"):
            (y.sum() + dx.square().sum()).backward()
    # with the graph kept but no second differentiation, the gradients are those without
    t = leaves()
    dy = torch.randn(5, 3, dtype=torch.float64)
    y = ffn.block(*t.values(), "gelu", True)
    want = torch.autograd.grad(y, list(t.values()), dy, retain_graph=True)
    got = torch.autograd.grad(y, list(t.values()), dy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_frozen_weights_cost_no_product(passes):
    """Only the gradients that autograd asks for are formed; dW of a frozen weight is left out."""
    for frozen in (("w1",), ("w2",), ("w1", "w2"), ("x",), ("b1", "b2"), ("x", "w1", "b1", "w2")):
        t = leaves(frozen)
        dy = torch.randn(5, 3, dtype=torch.float64)
        wanted = [v for v in t.values() if v.requires_grad]
        want = torch.autograd.grad(plain(**t), wanted, dy)
        got = torch.autograd.grad(ffn.block(*t.values(), "gelu", True), wanted, dy)
        assert all(torch.allclose(a, b) for a, b in zip(got, want)), frozen
        _, dx, dw1, dw2, db = passes.calls[-1]
        assert (dx, dw1, dw2, db) == ("x" not in frozen, "w1" not in frozen, "w2" not in frozen, not {"b1", "b2"} <= set(frozen))


def test_nothing_is_held_where_nothing_is_differentiated(passes):
    t = leaves()
    with torch.no_grad():
        y = ffn.block(*t.values(), "gelu", True)
    assert passes.calls == [("forward", False)] and not y.requires_grad and torch.allclose(y, plain(**t))
    t = leaves(("x", "w1", "b1", "w2", "b2"))
    ffn.block(*t.values(), "gelu", True)
    assert passes.calls[1:] == [("forward", False)]


@pytest.mark.parametrize("lead", [(), (5,), (2, 3), (1, 1, 4), (0, 3)])
def test_leading_dimensions(passes, lead):
    """X of any leading dimensions, as batch x sequence x features; Y and dX have its shape."""
    t = leaves(lead=lead)
    y = ffn.block(*t.values(), "gelu", True)
    want = plain(**t)
    assert y.shape == want.shape and torch.allclose(y, want)
    dy = torch.randn(want.shape, dtype=torch.float64)
    for a, b in zip(torch.autograd.grad(y, list(t.values()), dy), torch.autograd.grad(want, list(t.values()), dy)):
        assert a.shape == b.shape and torch.allclose(a, b)
