"""8-bit activation checkpoints on the GPU: every code, scale and value against the FP64 restatement of the rule."""
import pytest
import torch

import linear_ref as ref
from chpl_b200 import _lib, ckpt8, ffn

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("dt", [BF, HF, FP])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (7, 33), (5, 64), (129, 1000), (64, 4096), (1000, 259), (2, 100003)])
@pytest.mark.parametrize("pad", [0, 1, 8, 16])
def test_codes_and_values(cuda, rows, cols, dt, pad):
    g = gen(rows + cols)
    full = torch.empty(rows, cols + pad, device="cuda").normal_(generator=g)
    full *= torch.exp2(torch.randint(-12, 13, (rows, cols + pad), device="cuda", generator=g).float())  # 2^+-12: F16 holds it
    if rows > 2:
        full[1] = 0
    x = full.to(dt)[:, :cols]
    c = ckpt8.pack(x)
    codes, scales = ref.pack(x)
    assert torch.equal(c.codes, codes) and torch.equal(c.scales, scales)
    for to in (BF, HF, FP):
        want = ref.unpack(codes, scales).to(FP).to(to)  # a 7-bit code is exact in FP32
        assert torch.equal(ckpt8.unpack(c, to), want)
    # into given memory with row distances of its own
    out = ckpt8.Ckpt8(torch.full((rows, cols + 5), 99, dtype=torch.int8, device="cuda")[:, :cols],
                      torch.full((rows, -(-cols // 32) + 3), 99, dtype=torch.uint8, device="cuda")[:, : -(-cols // 32)], dt)
    ckpt8.pack(x, out=out)
    assert torch.equal(out.codes, codes) and torch.equal(out.scales, scales)
    back = torch.full((rows, cols + pad + 1), 7.0, dtype=dt, device="cuda")
    ckpt8.unpack(out, out=back[:, :cols])
    assert torch.equal(back[:, :cols], ref.unpack(codes, scales).to(FP).to(dt)) and bool((back[:, cols:] == 7).all())
    # error at most half a step (a whole one where the code is clamped)
    step = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 133).repeat_interleave(32, 1)[:, :cols]
    err = (ref.unpack(codes, scales) - x.double()).abs()
    assert bool((err <= torch.where(codes.abs() == 127, step, 0.5 * step)).all())


def test_extremes(cuda):
    """Ties, the topmost values of a binade, the largest and the least magnitudes, infinities and NaN."""
    inf, nan = float("inf"), float("nan")
    groups = [[1.0, 0.5 / 64, 1.5 / 64, 2.5 / 64, -0.5 / 64, 1.999, -1.999], [3.4e38, -3.4e38, 1e30], [1e-38, -1e-38, 2e-38],
              [1e-45, 3e-45], [0.0, -0.0], [inf, 1.0], [-inf, inf], [nan, 1.0], [1.0, nan, inf], [2.0 ** -126], [2.0 ** -120, 2.0 ** -126]]
    x = torch.zeros(1, 32 * len(groups), device="cuda")
    for i, v in enumerate(groups):
        x[0, 32 * i:32 * i + len(v)] = torch.tensor(v)
    for dt in (FP, BF):
        y = x.to(dt)
        c = ckpt8.pack(y)
        codes, scales = ref.pack(y)
        assert torch.equal(c.codes, codes) and torch.equal(c.scales, scales)
        got, want = ckpt8.unpack(c), ref.unpack(codes, scales).to(FP).to(dt)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got, 0), torch.nan_to_num(want, 0))


def test_empty_and_refusals(cuda):
    c = ckpt8.pack(torch.empty(0, 40, device="cuda"))
    assert c.codes.shape == (0, 40) and ckpt8.unpack(c).shape == (0, 40)
    c = ckpt8.pack(torch.empty(3, 0, device="cuda"))
    assert ckpt8.unpack(c).shape == (3, 0)
    x = torch.randn(4, 64, device="cuda")
    good = ckpt8.pack(x)
    bad = [lambda: ckpt8.pack(x.double()), lambda: ckpt8.pack(x.t()), lambda: ckpt8.pack(x.cpu()), lambda: ckpt8.pack(x[0]),
           lambda: ckpt8.pack(x, out=ckpt8.empty(4, 65, FP, "cuda")),
           lambda: ckpt8.unpack(good, torch.int8), lambda: ckpt8.unpack(ckpt8.Ckpt8(good.codes, good.codes, FP)),
           lambda: ckpt8.unpack(ckpt8.Ckpt8(good.codes, good.scales[:, :1], FP)),
           lambda: ckpt8.unpack(good, out=torch.empty(4, 63, device="cuda"))]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.ChplError) as err:
            f()
        assert err.value.code == _lib.CHPL_ERR_INVALID, i


def ffn_ref(x, w1, b1, w2, b2, dy, name, residual):
    """The block's outputs and gradients in FP64, at the checkpoints of X and of the FP64 Z."""
    x, w1, b1, w2, b2, dy = (v.double() for v in (x, w1, b1, w2, b2, dy))
    z = x @ w1.t() + b1
    y = ref.act(z, name) @ w2.t() + b2 + (x if residual else 0)
    x8, z8 = ref.unpack(*ref.pack(x)), ref.unpack(*ref.pack(z))
    dz = (dy @ w2) * ref.slope(z8, name)
    return (y, dz @ w1 + (dy if residual else 0), dz.t() @ x8, dz.sum(0), dy.t() @ ref.act(z8, name), dy.sum(0)), (z, z8)


@pytest.mark.parametrize("T,d,h", [(1, 64, 256), (50, 129, 515), (300, 256, 1024), (1100, 512, 768)])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("name,residual", [("gelu", True), ("relu", False), ("silu", True), ("gelu_tanh", False)])
def test_ffn_block(cuda, T, d, h, dt, name, residual):
    """The block's training step: 2-norm errors within the roundings that its products' operands and results take
    (at most three each of u, plus u for sums), plus the codes of Z that FP32's and FP64's Z round differently: at
    2^-22 sqrt(d) of |Z| from a tie, fewer than one in a thousand moves, by 2^-6 of its group's size."""
    g = gen(T + d)
    def mk(*s, scale=1.0):
        return torch.empty(*s, dtype=dt, device="cuda").normal_(0.0, scale, generator=g)
    x, w1, b1, w2, b2, dy = mk(T, d), mk(h, d, scale=d ** -0.5), mk(h), mk(d, h, scale=h ** -0.5), mk(d), mk(T, d, scale=0.1)
    y, saved = ffn.forward(x, w1, b1, w2, b2, act=name, residual=residual, save=True)
    assert torch.equal(y, ffn.forward(x, w1, b1, w2, b2, act=name, residual=residual))
    grads = ffn.backward(dy, saved, w1, w2)
    want, _ = ffn_ref(x, w1, b1, w2, b2, dy, name, residual)
    u = ref.UNIT[dt]
    for what, a, b in zip(("y", "dx", "dw1", "db1", "dw2", "db2"), (y, *grads), want):
        off = (a.double() - b).norm() / b.norm()
        assert off <= 4 * u + 0.001 ** 0.5 * 2.0 ** -6, f"{what}: {off}"
    # through autograd: the same gradients
    leaves = [v.clone().requires_grad_(True) for v in (x, w1, b1, w2, b2)]
    ffn.block(*leaves, name, residual).backward(dy)
    assert all(torch.equal(v.grad, a) for v, a in zip(leaves, grads))
