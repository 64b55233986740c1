"""4-bit floating point on the GPU: every code, scale and value against the FP64 restatement of the rule, and the products of
every kernel, tile and split against FP64."""
import pytest
import torch

import linear_ref as lin
import mx4_ref as ref
from chpl_b200 import _lib, check_device, ffn, linear, mx4

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows(g, T, width, dt, pad=0, scale=1.0):
    """T x width, rows width + pad apart, NaN between them."""
    full = torch.full((T, width + pad), float("nan"), dtype=dt, device="cuda")
    full[:, :width] = torch.empty(T, width, device="cuda").normal_(0.0, scale, generator=g).to(dt)
    return full[:, :width]


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("T,n", [(1, 1), (1, 32), (3, 31), (7, 33), (5, 255), (5, 257), (129, 1000), (64, 4096), (1000, 259), (127, 2048), (9600, 1031), (2, 100003)])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_codes_scales_and_values(cuda, T, n, dt, pad):
    g = gen(T + n)
    x = rows(g, T, n, dt, pad) * torch.exp2(torch.randint(-6, 7, (T, n), device="cuda", generator=g).float()).to(dt)
    if T > 2:
        x[1] = 0
    c = mx4.pack(x)
    code, scales = ref.pack(x)
    got, s, tail, stail = ref.unpacked(c)
    assert torch.equal(got, code) and torch.equal(s, scales)
    assert bool((tail == 0).all()) and bool((stail == 5).all())
    want = ref.values(code, scales)
    for to in (BF, HF, FP):
        assert torch.equal(mx4.unpack(c, to), want.to(FP).to(to))  # a code times its step is exact in FP32
    # into given memory: codes' rows apart, scales' bytes behind the last row left as they were
    ld = c.codes.shape[1] + 32
    full = torch.full((T, ld), 99, dtype=torch.uint8, device="cuda")
    out = mx4.Mx4(full[:, : c.codes.shape[1]], torch.full_like(c.scales, 77), n, dt)
    assert mx4.pack(x, out=out) is out
    got, s, tail, _ = ref.unpacked(out)
    assert torch.equal(got, code) and torch.equal(s, scales) and bool((full[:, c.codes.shape[1]:] == 99).all())
    if T % 128:
        written = torch.zeros(c.scales.numel(), dtype=torch.bool, device="cuda")
        t = torch.arange(T, device="cuda")[:, None]
        q = torch.arange(-(-n // 256) * 8, device="cuda")[None]
        written[((t // 128) * (2 * -(-n // 256)) + q // 4) * 512 + (t % 32) * 16 + (t % 128) // 32 * 4 + q % 4] = True
        assert bool((out.scales[~written] == 77).all())
    back = torch.full((T, n + pad + 1), 7.0, dtype=dt, device="cuda")
    mx4.unpack(out, out=back[:, :n])
    assert torch.equal(back[:, :n], want.to(FP).to(dt)) and bool((back[:, n:] == 7).all())


def test_every_tie_and_extreme(cuda):
    """Midpoints of all levels and their neighbours at several scales, the topmost values of a binade, magnitudes from the least
    to the largest, infinities and NaN."""
    inf, nan = float("inf"), float("nan")
    mid = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    near = [m * (1 + d * 2.0 ** -23) for m in mid for d in (-1, 0, 1)]
    groups = [[4.0] + near, [4.0] + [-v for v in near], [7.9999995] + near, [6.0, 5.0, -6.5, 7.5], [3.4e38, -1e38, 1e37], [1e-38, -2e-38], [1e-45, 3e-45],
              [0.0, -0.0], [inf, 1.0], [-inf, inf], [nan, 1.0], [1.0, nan, inf], [2.0 ** -126], [2.0 ** -120, 2.0 ** -123], [65504.0, 1.0]]
    groups += [[4.0 * 2.0 ** e] + [v * 2.0 ** e for v in near] for e in (-100, -20, 10, 100)]
    x = torch.zeros(1, 32 * len(groups), device="cuda")
    for i, v in enumerate(groups):
        x[0, 32 * i:32 * i + len(v)] = torch.tensor(v)
    for dt in (FP, BF, HF):
        y = x.to(dt)
        code, scales = ref.pack(y)
        got, s, _, _ = ref.unpacked(mx4.pack(y))
        assert torch.equal(got, code) and torch.equal(s, scales)
        back, want = mx4.unpack(mx4.pack(y), FP), ref.values(code, scales).to(FP)
        assert torch.equal(torch.isnan(back), torch.isnan(want)) and torch.equal(torch.nan_to_num(back, 0), torch.nan_to_num(want, 0))


def reference(x, w, b, r, name):
    """(Y, slack) from the coded operands: exact products, FP32 sums, the activation's and the addend's errors."""
    y, z, size = lin.forward(ref.values(*ref.pack(x)), ref.values(*ref.pack(w)), b, r, name)
    return y, 1.2 * lin.add_error(x.shape[1]) * size + lin.ACT_ERROR * z.abs() + 2.0 ** -24 * y.abs()


@pytest.mark.parametrize("T,n,k", ref.SIZES + ref.MORE)
@pytest.mark.parametrize("dt,pad", [(BF, 0), (HF, 1), (BF, 8)])
def test_linear(cuda, T, n, k, dt, pad):
    i = T + n + k + pad
    name, g = lin.ACTS[i % 5], gen(i)
    x, w = rows(g, T, k, dt, pad), rows(g, n, k, dt, pad, k ** -0.5)
    x[:, 3::97] *= 8
    b = rows(g, 1, n, dt)[0] if i % 3 else None
    r = rows(g, T, n, dt, pad) if i % 2 else None
    w4 = mx4.pack(w)
    full = torch.full((T + 1, n + pad), 7.0, dtype=dt, device="cuda")
    out = mx4.linear(x, w4, b, residual=r, act=name, out=full[:T, :n])
    y, slack = reference(x, w, b, r, name)
    lin.check(out, y, dt, slack, "y")
    assert bool((full[:T, n:] == 7).all()) and bool((full[T] == 7).all())
    # coded before: bit for bit the same (up to eight tokens the product codes X itself)
    assert torch.equal(mx4.linear(mx4.pack(x), w4, b, residual=r, act=name), out)
    if r is not None:  # in place of the addend
        z = rows(g, T, n, dt, pad)
        z.copy_(r)
        assert torch.equal(mx4.linear(x, w4, b, residual=z, act=name, out=z), out)


def test_sizes_reach_every_plan(cuda):
    """Kernels, tiles and splits of SIZES are all different, and every one that random layers meet is among them."""
    import math
    import random
    have = {ref.plan(*s) for s in ref.SIZES}
    assert len(have) == len(ref.SIZES)
    rng = random.Random(4)

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    met = {ref.plan(size(1, 8192), size(32, 16384), size(32, 16384)) for _ in range(50000)}
    assert met <= have, met - have


def test_groups_with_nan_spoil_their_rows_and_columns_only(cuda):
    g = gen(1)
    for T in (3, 40, 700):
        x, w = rows(g, T, 600, BF), rows(g, 500, 600, BF)
        want = mx4.linear(x, mx4.pack(w))
        x[1, 599] = float("inf")
        w[7, 3] = float("nan")
        got = mx4.linear(x, mx4.pack(w))
        spoilt = torch.zeros(T, 500, dtype=torch.bool, device="cuda")
        spoilt[1], spoilt[:, 7] = True, True
        assert torch.equal(torch.isnan(got), spoilt) and torch.equal(got[~spoilt], want[~spoilt])


def test_zero_and_empty(cuda):
    g = gen(2)
    w = mx4.pack(rows(g, 40, 96, BF))
    b, r = rows(g, 1, 40, BF)[0], rows(g, 5, 40, BF)
    assert mx4.linear(torch.empty(0, 96, dtype=BF, device="cuda"), w).shape == (0, 40)
    z = torch.zeros(5, 96, dtype=BF, device="cuda")
    assert torch.equal(mx4.linear(z, w, b, residual=r), (b.float() + r.float()).to(BF))
    none = mx4.pack(torch.empty(40, 0, dtype=BF, device="cuda"))
    assert torch.equal(mx4.linear(torch.empty(5, 0, dtype=BF, device="cuda"), none, b, residual=r), (b.float() + r.float()).to(BF))
    assert mx4.linear(z, mx4.pack(torch.empty(0, 96, dtype=BF, device="cuda"))).shape == (5, 0)
    e = mx4.pack(torch.empty(0, 40, device="cuda"))
    assert e.shape == (0, 40) and mx4.unpack(e).shape == (0, 40)


def test_streams_workspace_and_graphs(cuda):
    g = gen(3)
    w = [mx4.pack(rows(g, 700, 1000, HF)), mx4.pack(rows(g, 1000, 700, HF))]
    x = rows(g, 130, 1000, HF)
    want = mx4.linear(mx4.linear(x, w[0], act="silu"), w[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = mx4.linear(mx4.linear(x, w[0], act="silu", stream=side), w[1], stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    assert torch.equal(mx4.linear(mx4.linear(x, w[0], act="silu", work=work), w[1], work=work), want)
    for T in (1, 130):  # coded by the product, and before it
        a = x[:T].clone()
        graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
        for graph in graphs:
            with torch.cuda.graph(graph):
                outs.append(mx4.linear(mx4.linear(a, w[0], act="silu"), w[1]))
        for seed in (1, 2):
            a.copy_(rows(gen(seed), T, 1000, HF))
            for graph in graphs:
                graph.replay()
            want = mx4.linear(mx4.linear(a, w[0], act="silu"), w[1])
            assert all(torch.equal(o, want) for o in outs)
    check_device()


def test_ffn_from_4_bit_weights(cuda):
    """ffn.forward with coded weights is the two products; one coded and one not mix."""
    g = gen(4)
    x, w1, w2, b1, b2 = rows(g, 70, 256, BF), rows(g, 520, 256, BF, scale=0.06), rows(g, 256, 520, BF, scale=0.04), rows(g, 1, 520, BF)[0], rows(g, 1, 256, BF)[0]
    c1, c2 = mx4.pack(w1), mx4.pack(w2)
    got = ffn.forward(x, c1, b1, c2, b2, act="gelu", residual=True)
    assert torch.equal(got, mx4.linear(mx4.linear(x, c1, b1, act="gelu"), c2, b2, residual=x))
    assert torch.equal(ffn.forward(x, w1, b1, c2, b2), mx4.linear(linear.forward(x, w1, b1, act="gelu"), c2, b2))
    assert torch.equal(ffn.block(x, c1, b1, c2, b2, "gelu", True), got)
    for f in (lambda: ffn.forward(x, c1, b1, c2, b2, save=True), lambda: ffn.block(x.requires_grad_(), c1, b1, c2, b2)):
        with pytest.raises(_lib.ChplError) as err:
            f()
        assert err.value.code == _lib.CHPL_ERR_UNSUPPORTED


def test_refusals(cuda):
    x = torch.randn(4, 64, device="cuda", dtype=BF)
    c = mx4.pack(x)
    b = x[0, :4].contiguous()
    M = mx4.Mx4
    bad = [lambda: mx4.pack(x.double()), lambda: mx4.pack(x.t()), lambda: mx4.pack(x.cpu()), lambda: mx4.pack(x[0]), lambda: mx4.pack(x, out=mx4.pack(x[:3])),
           lambda: mx4.pack(x, out=M(c.codes, c.scales[:512], 64, BF)), lambda: mx4.pack(x, out=M(c.codes, c.scales, 65, BF)), lambda: mx4.unpack(c, torch.int8),
           lambda: mx4.unpack(M(c.codes.to(torch.int8), c.scales, 64, BF)), lambda: mx4.unpack(M(c.codes, c.scales, 97, BF)), lambda: mx4.unpack(M(c.codes, c.scales, -1, BF)),
           lambda: mx4.unpack(M(c.codes, c.scales[:-1], 64, BF)), lambda: mx4.unpack(c, out=x[:3]), lambda: mx4.linear(x, x), lambda: mx4.linear(x.float(), c),
           lambda: mx4.linear(x[:, :63], c), lambda: mx4.linear(x, c, act="tanh"), lambda: mx4.linear(x, c, b.half()), lambda: mx4.linear(x, c, b[:3]),
           lambda: mx4.linear(x, c, residual=x), lambda: mx4.linear(x, c, out=x), lambda: mx4.linear(M(c.codes, c.scales, 64, FP), c),
           lambda: mx4.linear(mx4.pack(x[:, :32].contiguous()), c), lambda: mx4.linear(x.cpu(), c),
           lambda: mx4.linear(x, M(torch.zeros(4, 41, dtype=torch.uint8, device="cuda")[:, 1:33], c.scales, 64, BF)),
           lambda: mx4.linear(x, M(c.codes, torch.zeros(1025, dtype=torch.uint8, device="cuda")[1:], 64, BF))]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.ChplError) as err:
            f()
        assert err.value.code == _lib.CHPL_ERR_INVALID, (i, err.value)
    big = torch.randn(20, 64, device="cuda", dtype=BF)
    with pytest.raises(_lib.ChplError) as err:
        mx4.linear(big, c, work=torch.empty(256, dtype=torch.uint8, device="cuda"))
    assert err.value.code == _lib.CHPL_ERR_WORKSPACE
    torch.cuda.synchronize()
