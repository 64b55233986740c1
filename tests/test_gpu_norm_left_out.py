"""Gradients of norms and joins where something is not there: no tokens, or inputs that no asked-for gradient uses."""
import pytest
import torch

from chpl_b200 import _lib, check_device, norm

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def mk(g, *s, dt=BF):
    return torch.empty(*s, device="cuda").normal_(generator=g).to(dt)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("matrix", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_no_tokens(cuda, dt, matrix, f32):
    """Sums over no tokens are 0 whatever the gate and the weights hold, and leave what is accumulated to as it is."""
    n = 70
    v = norm.Norm(torch.tensor([INF, NAN, -INF] + [1.0] * (n - 3), dtype=dt, device="cuda"), torch.full((n,), NAN, dtype=dt, device="cuda"), "layer")
    e, s = torch.empty(0, n, dtype=dt, device="cuda"), torch.empty(0, 2, device="cuda")
    gate = e if matrix else torch.full((n,), INF, dtype=dt, device="cuda")
    how = dict(post=v, gate=gate, pre=v, grad_dtype=torch.float32 if f32 else None)
    got = norm.join_backward(e, e, e, e, s, s, **how)
    want = torch.zeros(n, dtype=torch.float32 if f32 else dt, device="cuda")
    assert got.dx.shape == got.dy.shape == (0, n)
    sums = got[3:] if matrix else got[2:]
    assert all(torch.equal(t, want) for t in sums)
    into = norm.Joined(e, e, e if matrix else want + 3, *(want + i for i in range(4)))
    got = norm.join_backward(e, e, e, e, s, s, **how, into=into, accumulate=True)
    assert all(torch.equal(t, want + i) for i, t in enumerate(got[3:])) and (matrix or torch.equal(got.dgate, want + 3))
    _, dw, db = norm.backward(e, e, s, v, grad_dtype=how["grad_dtype"])
    assert torch.equal(dw, want) and torch.equal(db, want)
    check_device()


@pytest.mark.parametrize("T,n,pad", [(1, 64, 0), (300, 520, 0), (77, 1031, 1), (200, 4096, 0)])
@pytest.mark.parametrize("matrix", [False, True])
@pytest.mark.parametrize("pre", [False, True])
def test_frozen_gate_needs_no_y(cuda, T, n, pad, matrix, pre):
    """Without a norm of y and without the gate's gradient, dx, dy and the next norm's gradients are those of the whole call."""
    g = gen(n + T)
    x, y, dr, dh = (mk(g, T, n + pad)[:, :n] for _ in range(4))
    gate, v = mk(g, T, n) if matrix else mk(g, n), norm.Norm(mk(g, n), mk(g, n), "layer") if pre else None
    r, st = norm.join(x, y, gate=gate, scale=0.5, pre=v, save=True)[0::2 if pre else 1]
    how = dict(gate=gate, scale=0.5, residual_scale=0.75, pre=v)
    d = dh if pre else None
    want = norm.join_backward(dr, d, r, y, *st, **how)
    got = norm.join_backward(dr, d, r, None, *st, **how, need_dgate=False)
    assert want.dgate is not None and got.dgate is None
    for name, a, b in zip(norm.Joined._fields, got, want):
        assert name == "dgate" or a is b is None or torch.equal(a, b), name
    check_device()


def test_autograd_keeps_y_where_it_is_used(cuda):
    """joined holds y for a norm of it or for a gate that is trained, and not for a frozen gate."""
    g = gen(1)
    x, gate, v = mk(g, 30, 64), mk(g, 64), norm.Norm(mk(g, 64))
    d = mk(g, 30, 64)
    for post, trained in ((None, False), (None, True), (v, False)):
        y = mk(g, 30, 64).requires_grad_()
        gate = gate.detach().requires_grad_(trained)
        held = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t.data_ptr()) or t, lambda t: t):
            r, h = norm.joined(x, y, post=post, gate=gate, pre=v)
        assert (y.data_ptr() in held) == (post is not None or trained)
        leaves = [y, gate] if trained else [y]
        got = torch.autograd.grad((r, h), leaves, (d, d))
        r, h, st = norm.join(x, y.detach(), post=post, gate=gate.detach(), pre=v, save=True)
        want = norm.join_backward(d, d, r, y.detach(), *st, post=post, gate=gate.detach(), pre=v)
        assert torch.equal(got[0], want.dy) and (not trained or torch.equal(got[1], want.dgate))


def test_y_is_refused_missing_where_it_is_used(cuda):
    g = gen(2)
    dr, gate, v, s = mk(g, 3, 64), mk(g, 64), norm.Norm(mk(g, 64)), torch.ones(3, 2, device="cuda")
    for how in (dict(gate=gate), dict(post=v), dict(post=v, gate=gate, need_dgate=False)):
        with pytest.raises(_lib.ChplError) as err:
            norm.join_backward(dr, None, None, None, s, None, **how)
        assert err.value.code == _lib.CHPL_ERR_INVALID
