"""ffn.block on the GPU under torch's autograd: the gradients of ffn.backward, whatever is frozen and however X is shaped."""
import pytest
import torch

from chpl_b200 import ChplError, ckpt8, ffn

pytestmark = pytest.mark.gpu


def leaves(dt, lead, d, h):
    g = torch.Generator(device="cuda")
    g.manual_seed(d + h)
    mk = lambda *s, scale=1.0: torch.empty(*s, dtype=dt, device="cuda").normal_(0.0, scale, generator=g)
    t = {"x": mk(*lead, d), "w1": mk(h, d, scale=d ** -0.5), "b1": mk(h), "w2": mk(d, h, scale=h ** -0.5), "b2": mk(d)}
    return t, mk(*lead, d, scale=0.1)


@pytest.mark.parametrize("lead", [(1,), (37,), (4, 25), (2, 3, 50), ()])
@pytest.mark.parametrize("frozen", [(), ("w1",), ("w2",), ("w1", "w2"), ("x",), ("b1",), ("b1", "b2"), ("x", "w1", "b1", "w2")])
def test_gradients(cuda, lead, frozen):
    t, dy = leaves(torch.bfloat16, lead, 96, 200)
    x2, dy2 = t["x"].reshape(-1, 96), dy.reshape(-1, 96)
    y, saved = ffn.forward(x2, t["w1"], t["b1"], t["w2"], t["b2"], act="silu", residual=True, save=True)
    want = dict(zip(("x", "w1", "b1", "w2", "b2"), ffn.backward(dy2, saved, t["w1"], t["w2"])))
    for name, v in t.items():
        v.requires_grad_(name not in frozen)
    got = ffn.block(*t.values(), "silu", True)
    assert got.shape == t["x"].shape and torch.equal(got.reshape(-1, 96), y)
    got.backward(dy)
    for name, v in t.items():
        assert (v.grad is None) == (name in frozen), name
        if v.grad is not None:
            assert v.grad.shape == v.shape and torch.equal(v.grad.reshape(want[name].shape), want[name]), name
    with torch.no_grad():
        free = ffn.block(*t.values(), "silu", True)
    assert not free.requires_grad and torch.equal(free, got)


def test_only_the_gradients_that_are_asked_for(cuda):
    t, dy = leaves(torch.float16, (130,), 64, 300)
    _, saved = ffn.forward(*t.values(), act="gelu", save=True)
    want = ffn.backward(dy, saved, t["w1"], t["w2"])
    for need in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 1, 0, 0), (0, 1, 1, 0), (0, 0, 1, 1), (0, 0, 0, 0)):
        dx, dw1, dw2, db = (bool(v) for v in need)
        got = ffn.backward(dy, saved, t["w1"], t["w2"], need_dx=dx, need_dw1=dw1, need_dw2=dw2, need_db=db)
        for v, w, there in zip(got, want, (dx, dw1, db, dw2, db)):
            assert (v is not None) == there and (v is None or torch.equal(v, w)), need


def test_a_second_differentiation_raises(cuda):
    t, _ = leaves(torch.bfloat16, (20,), 64, 128)
    for v in t.values():
        v.requires_grad_()
    y = ffn.block(*t.values(), "gelu", True)
    dx, = torch.autograd.grad(y.float().sum(), t["x"], create_graph=True)
    with pytest.raises(ChplError):
        (y.float().sum() + dx.float().square().sum()).backward()


def test_under_torchs_checkpointing(cuda):
    """Recomputed in the backward pass: the same gradients, and nothing held in between."""
    from torch.utils.checkpoint import checkpoint
    t, dy = leaves(torch.bfloat16, (3, 40), 128, 256)
    for v in t.values():
        v.requires_grad_()
    want = torch.autograd.grad(ffn.block(*t.values(), "gelu", True), list(t.values()), dy)
    got = torch.autograd.grad(checkpoint(ffn.block, *t.values(), "gelu", True, use_reentrant=False), list(t.values()), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert isinstance(ffn.forward(t["x"].detach()[0], *[v.detach() for v in list(t.values())[1:]], save=True)[1].x, ckpt8.Ckpt8)
