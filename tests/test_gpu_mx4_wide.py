"""4-bit products of a few tokens on layers wider than 16384 features, where two CTAs share an SM and their rings are short: the
rows coded by the product itself, bit for bit those that are coded before, call after call."""
import pytest
import torch

import linear_ref as lin
import mx4_ref as ref
from chpl_b200 import check_device, ffn, mx4

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def mk(g, *s, dt=BF, scale=1.0):
    return torch.empty(*s, dtype=dt, device="cuda").normal_(0.0, scale, generator=g)


@pytest.mark.parametrize("n", [19000, 28672, 32000, 128256])
@pytest.mark.parametrize("k", [2560, 2816, 4096, 8192])
@pytest.mark.parametrize("dt", [BF, HF])
def test_few_tokens(cuda, n, k, dt):
    g = gen(n + k)
    w = mk(g, n, k, dt=dt, scale=k ** -0.5)
    w4 = mx4.pack(w)
    b, x8, r8 = mk(g, n, dt=dt), mk(g, 8, k, dt=dt), mk(g, 8, n, dt=dt)
    x8[:, 3::97] *= 8
    some = torch.cat([torch.arange(300), torch.arange(n - 300, n)]).cuda()
    for i, T in enumerate((1, 3, 4, 5, 8)):
        name, x, r = lin.ACTS[(i + k // 256) % 5], x8[:T], r8[:T] if i % 2 else None
        want = mx4.linear(mx4.pack(x), w4, b, residual=r, act=name)
        got = [mx4.linear(x, w4, b, residual=r, act=name) for _ in range(10)]
        assert all(torch.equal(y, want) for y in got), T
        y, z, size = lin.forward(ref.values(*ref.pack(x)), ref.values(*ref.pack(w[some])), b[some], None if r is None else r[:, some], name)
        # exact products, FP32 sums, the activation's and the addend's errors
        lin.check(want[:, some], y, dt, 1.2 * lin.add_error(k) * size + lin.ACT_ERROR * z.abs() + 2.0 ** -24 * y.abs(), f"{T} tokens")
    check_device()


@pytest.mark.parametrize("T", [1, 3, 8])
def test_block_of_28672(cuda, T):
    """A block's two products: 28672 features out, and 28672 contracted."""
    g = gen(T)
    c1, c2 = mx4.pack(mk(g, 28672, 4096, scale=4096 ** -0.5)), mx4.pack(mk(g, 4096, 28672, scale=28672 ** -0.5))
    b1, b2, x = mk(g, 28672), mk(g, 4096), mk(g, T, 4096)
    h = mx4.linear(mx4.pack(x), c1, b1, act="gelu")
    want = mx4.linear(mx4.pack(h), c2, b2, residual=x)
    for _ in range(10):
        assert torch.equal(ffn.forward(x, c1, b1, c2, b2, act="gelu", residual=True), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ffn.forward(x, c1, b1, c2, b2, act="gelu", residual=True)
    for _ in range(10):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    check_device()
