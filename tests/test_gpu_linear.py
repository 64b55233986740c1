"""Linear layers on the GPU (chpl_b200.linear) against their FP64 definitions."""
import pytest
import torch

import linear_ref as ref
from chpl_b200 import _lib, ckpt8, linear

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def rows(g, T, width, dt, pad=0, scale=1.0, shift=0):
    """T x width, rows width + pad apart, the first `shift` elements into its memory."""
    full = torch.empty(T * (width + pad) + shift, dtype=dt, device="cuda").normal_(0.0, scale, generator=g)
    return full[shift:].view(T, width + pad)[:, :width]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def out_like(T, width, dt, pad):
    """An output matrix inside a sea of a marker value, and the sea."""
    sea = torch.full((T, width + pad), 7.0, dtype=dt, device="cuda")
    return sea[:, :width], sea


SIZES = [(1, 1, 1), (1, 64, 32), (1, 1024, 1024), (2, 31, 33), (5, 4096, 40), (17, 129, 255), (24, 2048, 520), (64, 256, 128),
         (100, 8, 1000), (128, 128, 256), (130, 1000, 514), (257, 515, 1029), (300, 1024, 4096), (1000, 777, 300),
         (1024, 192, 2050), (2048, 264, 1160), (1500, 200, 3100), (4096, 1000, 1100)]


@pytest.mark.parametrize("T,k,n", SIZES)
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("pad", [0, 8, 1])
def test_forward(cuda, T, k, n, dt, pad):
    i = SIZES.index((T, k, n))
    name, g = ref.ACTS[(i + pad) % 5], gen(i)
    x, w = rows(g, T, k, dt, pad, shift=pad), rows(g, n, k, dt, pad, k ** -0.5)
    b = torch.empty(n, dtype=dt, device="cuda").normal_(generator=g) if i % 3 else None
    r = rows(g, T, n, dt, pad) if i % 2 else None
    y, z, size = ref.forward(x, w, b, r, name)
    acc = ref.add_error(k) * size
    out, sea = out_like(T, n, dt, pad)
    slack = 1.2 * acc + ref.ACT_ERROR * z.abs() + 2.0 ** -24 * y.abs()
    linear.forward(x, w, b, residual=r, act=name, out=out)
    ref.check(out, y, dt, slack, "y")
    assert bool((sea[:, n:] == 7).all()), "written past the row's end"
    # with the pre-activation kept: the same Y, and Z in 16 bits or coded within half a step of FP32's Z
    y2, z2 = linear.forward(x, w, b, residual=r, act=name, save="z")
    assert torch.equal(y2, out)
    ref.check(z2, z, dt, acc, "z")
    y3, z3 = linear.forward(x, w, b, residual=r, act=name, save="z8")
    assert torch.equal(y3, out)
    got, _ = ref.unpack(z3.codes, z3.scales), None
    step = torch.ldexp(torch.ones_like(z3.scales, dtype=torch.float64), z3.scales.int() - 133)
    step = step.repeat_interleave(32, dim=1)[:, :n]
    near = 0.5 * step + acc + torch.where(z3.codes.abs() == 127, 0.5 * step, 0.0)
    assert bool(((got - z).abs() <= near).all())
    top = torch.nn.functional.pad(z.abs(), (0, -n % 32)).view(T, -1, 32)
    slop = torch.nn.functional.pad(acc, (0, -n % 32)).view(T, -1, 32).amax(2)
    s = z3.scales.double()
    assert bool((torch.exp2(s - 127) <= top.amax(2) + slop).logical_or(s == 7).all())
    assert bool((torch.exp2(s - 126) >= top.amax(2) - slop).all())


GRADS = [(1, 1, 1), (1, 1024, 512), (3, 65, 31), (16, 128, 64), (40, 4096, 24), (77, 40, 1000), (128, 256, 128),
         (200, 520, 264), (257, 1031, 519), (512, 1024, 2048), (1000, 300, 777), (2100, 520, 392), (2050, 1800, 2100)]


@pytest.mark.parametrize("T,k,n", GRADS)
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("how", ["plain", "act16", "act8", "in16", "in8", "both8", "odd"])
def test_backward(cuda, T, k, n, dt, how):
    i = GRADS.index((T, k, n))
    g = gen(100 + i)
    pad = 1 if how == "odd" else 8 * (i % 2)
    name = ref.ACTS[1 + (i + len(how)) % 4] if how in ("act16", "act8", "both8", "odd") else "none"
    inner = ref.ACTS[1 + (i + 2 * len(how)) % 4] if how in ("in16", "in8", "both8") else "none"
    dy, w = rows(g, T, n, dt, pad, 0.1, shift=pad), rows(g, n, k, dt, pad, k ** -0.5)
    x, z = rows(g, T, k, dt, pad), rows(g, T, n, dt, pad)
    add = rows(g, T, k, dt, pad, 0.1) if i % 2 else None
    xv, zv, xa, za = x.double(), z.double(), x, z
    if how in ("act8", "both8"):
        za = ckpt8.Ckpt8(*ref.pack(z), dt)
        zv = ref.unpack(*za[:2])
    if how in ("in8", "both8", "odd"):
        xa = ckpt8.Ckpt8(*ref.pack(x), dt)
        xv = ref.unpack(*xa[:2])
    G = dy.double() * ref.slope(zv, name)
    D = G @ w.double()
    Dabs = G.abs() @ w.double().abs()
    u = ref.UNIT[dt]
    gu = (u if name != "none" else 0.0)                   # G is rounded to dt where an activation made it
    xu = (u if inner != "none" else 0.0)
    act_g = 2.0 ** -17 * dy.double().abs()               # error of act' times dy
    tiny = ref.TINY[dt]                                   # a rounding that ends among F16's subnormals
    s_in, X = ref.slope(xv, inner), ref.act(xv, inner)
    e_g = gu * G.abs() + (act_g + tiny if name != "none" else 0.0)
    e_d = e_g @ w.double().abs() + ref.add_error(n) * Dabs
    dx = D * s_in + (add.double() if add is not None else 0.0)
    slack = e_d * s_in.abs().clamp(min=1) + 2.0 ** -17 * D.abs() + 2.0 ** -24 * dx.abs()
    out, sea = out_like(T, k, dt, pad)
    got = linear.backward(dy, xa, w, act=name, z=za if name != "none" else None, in_act=inner, add=add, dx=out, dx_sum=True)
    # the sum over the tokens of dX's FP32 values: its slack without the rounding, and an addition's for each token
    sums = dx.sum(0)
    ref.check(got[3], sums, dt, (slack + ref.add_error(T) * dx.abs()).sum(0), "dx_sum", 2)
    ref.check(got[0], dx, dt, slack, "dx", 2)
    assert bool((sea[:, k:] == 7).all())
    e_x = xu * X.abs() + (2.0 ** -18 * xv.abs() + tiny if inner != "none" else 0.0)
    dw, wabs = G.t() @ X, G.abs().t() @ X.abs()
    e_w = e_g.t() @ (X.abs() + e_x) + G.abs().t() @ e_x + ref.add_error(T) * wabs
    ref.check(got[1], dw, dt, e_w, "dw", 3)
    db, e_b = G.sum(0), (ref.add_error(T) * G.abs() + (act_g if name != "none" else 0.0)).sum(0)
    ref.check(got[2], db, dt, e_b, "db")
    # FP32 gradients, added to what is there; only some of the outputs
    dw0, db0 = torch.randn(n, k, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g)
    dw32, db32 = dw0.clone(), db0.clone()
    none, a, b = linear.backward(dy, xa, w, act=name, z=za if name != "none" else None, in_act=inner, need_dx=False, dw=dw32,
                                 db=db32, accumulate=True)
    assert none is None and a is dw32 and b is db32
    ref.check(dw32, dw0.double() + dw, FP, e_w + 2.0 ** -23 * wabs, "dw in FP32", 1e9)
    ref.check(db32, db0.double() + db, FP, e_b + 2.0 ** -23 * G.abs().sum(0), "db in FP32", 1e9)
    sum0 = torch.randn(k, device="cuda", generator=g)
    sum32 = sum0.clone()
    four = linear.backward(dy, xa if inner != "none" else None, w, act=name, z=za if name != "none" else None, in_act=inner, add=add,
                           need_dw=False, need_db=False, dx_sum=sum32, grad_dtype=FP, accumulate=True)
    assert torch.equal(four[0], got[0]) and four[3] is sum32
    ref.check(sum32, sum0.double() + sums, FP, (slack + ref.add_error(T) * dx.abs()).sum(0) + 1e-6, "dx_sum in FP32", 1e9)
    only = linear.backward(dy, xa if inner != "none" else None, w, act=name, z=za if name != "none" else None, in_act=inner,
                           add=add, need_dw=False, need_db=False)
    assert torch.equal(only[0], got[0]) and only[1] is None and only[2] is None


@pytest.mark.parametrize("name", ref.ACTS)
def test_gradients_against_differences(cuda, name):
    """<dX, v>, <dW, V>, <db, b'> against central differences of the FP64 forward (step 1e-4: error below 1e-6)."""
    g, dt, T, k, n = gen(5), BF, 96, 160, 224
    x, w, b, dy = rows(g, T, k, dt), rows(g, n, k, dt, 0, k ** -0.5), rows(g, 1, n, dt)[0].contiguous(), rows(g, T, n, dt)
    _, z, _ = ref.forward(x, w, b, None, name)
    zin = z.to(dt)   # the kept pre-activation is Z rounded to 16 bits: |dG| <= |dy| max|act''| u |Z|, max|act''| < 1.6
    got = linear.backward(dy, x, w, act=name, z=zin)
    h = 1e-4
    for what, v in (("x", x), ("w", w), ("b", b)):
        d = torch.randn(v.shape, dtype=torch.float64, device="cuda", generator=g)
        side = []
        for sgn in (1, -1):
            p = {"x": x.double(), "w": w.double(), "b": b.double()}
            p[what] = p[what] + sgn * h * d
            side.append((ref.act(p["x"] @ p["w"].t() + p["b"], name) * dy.double()).sum())
        want = (side[0] - side[1]) / (2 * h)
        mine = got["xwb".index(what)].double()
        # the 2-norm of a gradient's error is at most 3 u of its norm, plus the kept Z's rounding (1.6 u |Z dy| through W or X)
        lim = (3 * mine.norm() + 1.6 * (z * dy.double()).norm() * {"x": w.double().norm(2), "w": x.double().norm(2),
                                                                   "b": torch.tensor(T ** 0.5)}[what]) * 2.0 ** -8
        kinks = (z.abs() < h * 40).sum() * 40 * 4 if name == "relu" else 0  # differences across ReLU's corner
        assert abs(want - (mine * d).sum()) <= lim * d.norm() / d.numel() ** 0.5 * 4 + kinks * h + 1e-3


@pytest.mark.parametrize("dt", [BF, HF])
def test_empty_and_zero_lengths(cuda, dt):
    g = gen(1)
    for T, k, n in ((0, 8, 8), (4, 0, 8), (4, 8, 0)):
        x, w, b = rows(g, T, k, dt), rows(g, n, k, dt), torch.randn(n, device="cuda").to(dt)
        r = rows(g, T, n, dt)
        y = linear.forward(x, w, b, residual=r, act="silu")
        assert y.shape == (T, n)
        ref.check(y, ref.act(b.double(), "silu")[None] + r.double() if k == 0 else ref.forward(x, w, b, r, "silu")[0], dt,
                  2.0 ** -17 * torch.ones(T, n, dtype=torch.float64, device="cuda"), "y")
        dy, add = rows(g, T, n, dt), rows(g, T, k, dt)
        dx, dw, db = linear.backward(dy, x, w, add=add)
        if n == 0:
            assert torch.equal(dx, add)
            ref.check(linear.backward(dy, x, w, add=add, dx_sum=True)[3], add.double().sum(0), dt,
                      1e-6 * torch.ones(k, dtype=torch.float64, device="cuda"), "dx_sum")
        if T == 0:
            assert bool((dw == 0).all()) and bool((db == 0).all())
            assert bool((linear.backward(dy, x, w, dx_sum=True)[3] == 0).all())
            dw1, db1 = torch.ones(n, k, dtype=dt, device="cuda"), torch.ones(n, dtype=dt, device="cuda")
            linear.backward(dy, x, w, dw=dw1, db=db1, accumulate=True)
            assert bool((dw1 == 1).all()) and bool((db1 == 1).all())
        if k == 0:
            ref.check(db, dy.double().sum(0), dt, 1e-5 * torch.ones(n, dtype=torch.float64, device="cuda"), "db")


def test_aliased_outputs_and_given_memory(cuda):
    g, dt, T, k, n = gen(2), BF, 150, 264, 400
    x, w, r = rows(g, T, k, dt), rows(g, n, k, dt, 0, k ** -0.5), rows(g, T, n, dt)
    want = linear.forward(x, w, residual=r, act="relu")
    mine = r.clone()
    assert linear.forward(x, w, residual=mine, act="relu", out=mine) is mine
    assert torch.equal(mine, want)
    dy, add = rows(g, T, n, dt), rows(g, T, k, dt)
    dx, _, _ = linear.backward(dy, x, w, add=add)
    mine = add.clone()
    linear.backward(dy, x, w, add=mine, dx=mine, need_dw=False, need_db=False)
    assert torch.equal(mine, dx)
    # a workspace of the caller's own, for rows that need copying
    xo = rows(g, T, 129, dt, 2)
    wo = rows(g, n, 129, dt, 2)
    y = linear.forward(xo, wo)
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    assert torch.equal(linear.forward(xo, wo, work=work), y)
    with pytest.raises(_lib.ChplError) as err:
        linear.forward(xo, wo, work=work[:512])
    assert err.value.code == _lib.CHPL_ERR_WORKSPACE


@pytest.mark.parametrize("T", [1, 40, 700])
def test_infinities_and_nan_stay_in_their_rows(cuda, T):
    """A token with a NaN or an infinity spoils its own row only; one in a checkpoint, its own group."""
    g, dt, k, n = gen(3), BF, 200, 300
    x, w = rows(g, T + 2, k, dt), rows(g, n, k, dt, 0, k ** -0.5)
    clean, z_clean = linear.forward(x, w, act="gelu", save="z8")
    x[0, 3], x[-1, 7] = float("nan"), float("inf")
    y, z = linear.forward(x, w, act="gelu", save="z8")
    assert torch.equal(y[1:-1], clean[1:-1]) and torch.equal(z.codes[1:-1], z_clean.codes[1:-1])
    assert bool(torch.isnan(y[0]).all()) and not bool(torch.isfinite(y[-1].float()).any() and (w[:, 7] != 0).all())
    assert bool((z.scales[0] == 255).all()) and bool((z.codes[0] == 0).all())
    assert bool(torch.isnan(ckpt8.unpack(z)[0]).all())
    # huge but finite pre-activations: act and act' stay finite
    big = torch.tensor([[3e38, -3e38, 1e20, -1e20, 100.0, -100.0, 0.0, -0.0]], device="cuda").to(dt)
    one = torch.ones(1, 8, dtype=dt, device="cuda")
    for name in ref.ACTS:
        _, _, db = linear.backward(one, one, torch.zeros(8, 8, dtype=dt, device="cuda"), act=name, z=big)
        ref.check(db, ref.slope(big.double().clamp(-200, 200), name)[0], dt, 2.0 ** -17 * torch.ones(8, dtype=torch.float64, device="cuda"), name)
        eye = torch.eye(8, dtype=dt, device="cuda")
        y = linear.forward(big, eye, act=name)
        assert bool(torch.isfinite(y.float()).all())


def test_results_repeat_bit_for_bit(cuda):
    g, dt = gen(4), BF
    for T, k, n in ((1, 4096, 512), (48, 2048, 1000), (600, 1000, 520)):
        x, w, dy = rows(g, T, k, dt), rows(g, n, k, dt, 0, k ** -0.5), rows(g, T, n, dt)
        z = rows(g, T, n, dt)
        one = [linear.forward(x, w, act="gelu"), *linear.backward(dy, x, w, act="gelu", z=z)]
        for _ in range(3):
            two = [linear.forward(x, w, act="gelu"), *linear.backward(dy, x, w, act="gelu", z=z)]
            assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_streams_and_graphs(cuda):
    """On a stream of its own, behind work queued there, and replayed from a CUDA graph on new inputs."""
    g, dt, T, k, n = gen(6), HF, 33, 1001, 600
    x, w, dy = rows(g, T, k, dt), rows(g, n, k, dt, 0, k ** -0.5), rows(g, T, n, dt)
    want = [linear.forward(x, w, act="relu"), *linear.backward(dy, x, w)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        later = torch.zeros_like(x.contiguous())
        filler = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            filler = filler @ filler * 1e-3
        later.copy_(x)
        got = [linear.forward(later, w, act="relu"), *linear.backward(dy, later, w)]
    other = [linear.forward(x, w, act="relu", stream=s), *linear.backward(dy, x, w, stream=s)]
    s.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, other))
    buf = torch.zeros_like(x.contiguous())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [linear.forward(buf, w, act="relu"), *linear.backward(dy, buf, w)]
    buf.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_offsets_past_32_bits(cuda):
    """An output of more than 2^31 elements: rows at its start, middle and end."""
    dt, T, k, n = BF, 70000, 32, 32768
    g = gen(7)
    x, w = rows(g, T, k, dt), rows(g, n, k, dt, 0, k ** -0.5)
    y, z = linear.forward(x, w, act="relu", save="z8")
    back = ckpt8.unpack(z)
    for t in (0, T // 2, T - 1):
        want, zz, size = ref.forward(x[t:t + 1], w, None, None, "relu")
        ref.check(y[t:t + 1], want, dt, 1.2 * ref.add_error(k) * size, f"row {t}")
        codes, scales = z.codes[t:t + 1], z.scales[t:t + 1]
        assert torch.equal(back[t:t + 1].double(), ref.unpack(codes, scales))
    del y, z
    dx, dw, db = linear.backward(back, x, w)
    for t in (0, T - 1):
        D = back[t:t + 1].double() @ w.double()
        ref.check(dx[t:t + 1], D, dt, ref.add_error(n) * (back[t:t + 1].double().abs() @ w.double().abs()), f"dx row {t}")
    col = back[:, -40:].double()
    ref.check(dw[-40:], col.t() @ x.double(), dt, ref.add_error(T) * (col.abs().t() @ x.double().abs()), "dw")
    ref.check(db[-40:], col.sum(0), dt, ref.add_error(T) * col.abs().sum(0), "db")


def test_refusals(cuda):
    g = gen(8)
    x, w = rows(g, 4, 16, BF), rows(g, 8, 16, BF)
    dy = rows(g, 4, 8, BF)
    bad = [lambda: linear.forward(x.float(), w), lambda: linear.forward(x, w.half()), lambda: linear.forward(x, w[:, :8]),
           lambda: linear.forward(x, w, act="swish"), lambda: linear.forward(x, w, save="z16"),
           lambda: linear.forward(x.cpu(), w), lambda: linear.forward(x, w, torch.zeros(7, dtype=BF, device="cuda")),
           lambda: linear.forward(x, w, residual=x), lambda: linear.forward(x.t().contiguous().t(), w),
           lambda: linear.forward(x, w, out=torch.empty(4, 9, dtype=BF, device="cuda")),
           lambda: linear.forward(x[:1].expand(4, 16), w),
           lambda: linear.backward(dy, x, w, act="gelu"), lambda: linear.backward(dy, None, w),
           lambda: linear.backward(dy, x[:3], w), lambda: linear.backward(dy, x, w, grad_dtype=HF),
           lambda: linear.backward(dy, x, w, accumulate=True), lambda: linear.backward(dy, x, w, need_dx=False, dx_sum=True),
           lambda: linear.backward(dy, x, w, dx_sum=torch.zeros(15, dtype=BF, device="cuda")), lambda: linear.backward(dy, x, w[:, :8]),
           lambda: linear.backward(dy, x, w, act="gelu", z=x),
           lambda: linear.backward(dy, ckpt8.Ckpt8(x.to(torch.int8), x.to(torch.uint8), BF), w)]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.ChplError) as err:
            f()
        assert err.value.code == _lib.CHPL_ERR_INVALID, i
    assert linear.backward(dy, None, w, need_dw=False)[0].shape == (4, 16)


@pytest.mark.parametrize("T,k,n", [(777, 1024, 1024), (400, 2048, 1040), (1024, 1023, 2100)])
@pytest.mark.parametrize("dt", [BF, HF])
def test_relu_codes_settle_at_the_slope(cuda, T, k, n, dt):
    """Whether a code is 0, and with it ReLU's slope at the checkpoint, follows the exact Z and not the tiling: of some
    thousand quotients within 1e-3 of 1/2, those further than 1e-6 from it (FP32's rounding of partial sums of eight,
    2^-24 of a few steps) have the code that Z has."""
    g = gen(31)
    x, w = rows(g, T, k, dt), rows(g, n, k, dt, 0, k ** -0.5)
    z = x.double() @ w.double().t()
    b = torch.zeros(n, dtype=dt, device="cuda")
    codes, scales = ref.pack(z)
    step = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 133).repeat_interleave(32, 1)[:, :n]
    q = z / step
    near = (q.abs() - 0.5).abs()
    assert bool((near < 1e-3).any())                      # there are some to settle
    _, c = linear.forward(x, w, b, act="relu", save="z8")
    want = q.abs() > 0.5
    sure = near > 1e-6                                     # beyond FP64's own doubt and the exact sum's FP32 eights
    same = c.scales.repeat_interleave(32, 1)[:, :n] == scales.repeat_interleave(32, 1)[:, :n]
    assert torch.equal(((c.codes != 0) == want) | ~sure | ~same, torch.ones_like(want))
