"""Gradients of norms and joins where something is not there: no tokens, or inputs that no asked-for gradient uses."""
import pytest
import torch

from chpl_b200 import check_device, norm

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
