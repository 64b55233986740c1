"""4-bit coding of rows that lie apart, with NaN in the gaps; a row of a batch beside the same row alone."""
import pytest
import torch

import linear_ref as lin
import mx4_ref as ref
from chpl_b200 import check_device, mx4

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def apart(v, pad, off=0):
    """v's rows v.shape[1] + pad elements apart, from the off-th on, NaN in between."""
    T, n = v.shape
    full = torch.full((T * (n + pad) + off,), float("nan"), dtype=v.dtype, device="cuda")
    out = full[off:].view(T, n + pad)[:, :n]
    out.copy_(v)
    return out


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("T,n", [(3, 31), (7, 33), (5, 255), (5, 257), (129, 1000), (64, 4096), (1000, 259), (127, 2048), (9600, 1031), (2, 100003)])
@pytest.mark.parametrize("pad,off", [(1, 0), (8, 0), (5, 3), (0, 1)])
def test_rows_apart(cuda, T, n, dt, pad, off):
    g = gen(T + n)
    v = torch.empty(T, n, device="cuda").normal_(generator=g).to(dt) * torch.exp2(torch.randint(-6, 7, (T, n), device="cuda", generator=g).float()).to(dt)
    x = apart(v, pad, off)
    assert x.stride(0) == n + pad and torch.equal(x, v)
    code, scales = ref.pack(v)
    c = mx4.pack(x)
    got, s, tail, stail = ref.unpacked(c)
    assert torch.equal(got, code) and torch.equal(s, scales) and bool((tail == 0).all()) and bool((stail == 5).all())
    back = apart(torch.zeros_like(v), pad, off)
    mx4.unpack(c, out=back)
    assert torch.equal(back, ref.values(code, scales).to(FP).to(dt))
    gaps = back._base if back._base is not None else back
    assert int(torch.isnan(gaps).sum()) == T * pad + off  # left as they were


@pytest.mark.parametrize("T", [2, 5, 9, 40, 200, 700])
@pytest.mark.parametrize("dt", [BF, HF])
def test_a_row_alone_is_the_batchs(cuda, T, dt):
    """Q(x) does not depend on a row's neighbours; the products are exact, so a row alone and in a batch differ by the order of
    their FP32 sums and by one rounding each."""
    g = gen(T)
    k, n = 1000, 520
    x, w = torch.empty(T, k, device="cuda").normal_(generator=g).to(dt), torch.empty(n, k, device="cuda").normal_(0.0, k ** -0.5, generator=g).to(dt)
    w4 = mx4.pack(w)
    y = mx4.linear(x, w4, act="gelu")
    want, z, size = lin.forward(ref.values(*ref.pack(x)), ref.values(*ref.pack(w)), None, None, "gelu")
    slack = 1.2 * lin.add_error(k) * size + lin.ACT_ERROR * z.abs()
    for t in {0, T // 2, T - 1}:
        one = mx4.linear(x[t:t + 1], w4, act="gelu")
        lin.check(one, want[t:t + 1], dt, slack[t:t + 1], "alone")
        assert bool(((one.double() - y[t:t + 1].double()).abs() <= 2 * (lin.UNIT[dt] * want[t:t + 1].abs() + slack[t:t + 1] + lin.TINY[dt])).all())
    check_device()
