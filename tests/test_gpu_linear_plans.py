"""Every kernel, tile and split of the linear layers' products on the GPU, with and without what an epilogue reads and
adds, against the FP64 definitions; FP32 gradients to more than 16 bits."""
import pytest
import torch

import linear_plans as lp
import linear_ref as ref
from chpl_b200 import ckpt8, linear

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def mk(g, *shape, dt=FP, scale=1.0):
    return torch.empty(*shape, dtype=dt, device="cuda").normal_(0.0, scale, generator=g)


def check_codes(c, z, acc):
    """Codes within half a step of Z (a whole one where the code is clamped) and scales of its groups' magnitudes, up to
    the error `acc` of an FP32 Z."""
    n = z.shape[1]
    step = torch.ldexp(torch.ones_like(c.scales, dtype=torch.float64), c.scales.int() - 133)
    step = step.repeat_interleave(32, dim=1)[:, :n]
    near = 0.5 * step + acc + torch.where(c.codes.abs() == 127, 0.5 * step, 0.0)
    assert bool(((ref.unpack(c.codes, c.scales) - z).abs() <= near).all())
    pad = lambda v: torch.nn.functional.pad(v, (0, -n % 32)).view(len(z), -1, 32).amax(2)
    top, slop, s = pad(z.abs()), pad(acc), c.scales.double()
    assert bool((torch.exp2(s - 127) <= top + slop).logical_or(s == 7).all())
    assert bool((torch.exp2(s - 126) >= top - slop).all())


def check_fp32(got, want, size, terms, what, dt):
    """A 2-norm bound of FP32 accumulation: the tensor cores add 16 products at a time into FP32 by cutting, an error of
    at most 2^-23 of a partial sum each, whose 2-norm over an output is at most that of `size` (the 2-norm that sums of
    random signs have).  The same result rounded to the operands' 16 bits has to fail it."""
    lim = 2.0 ** -23 * ((terms / 16 + 3) * size.norm() + 2 * want.norm())
    assert (got.double() - want).norm() <= lim, f"{what}: {(got.double() - want).norm()} over {lim}"
    if (want.to(dt).double() - want).norm() > 0:  # one token's db is in 16 bits as it stands
        assert (got.to(dt).double() - want).norm() > lim, f"{what}: the bound {lim} lets {dt} pass"


def test_this_gpu_takes_the_plans_that_the_sizes_were_chosen_for(cuda):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    found = {p for s in lp.SIZES + lp.LARGE for p in lp.plans(*s)}
    assert sms == 148 and len(found) >= 170, (sms, len(found))


@pytest.mark.parametrize("T,k,n", lp.SIZES + lp.LARGE)
@pytest.mark.parametrize("dt", [BF, HF])
def test_forward(cuda, T, k, n, dt):
    i = (lp.SIZES + lp.LARGE).index((T, k, n))
    g = gen(i)
    x, w, b = mk(g, T, k, dt=dt), mk(g, n, k, dt=dt, scale=k ** -0.5), mk(g, n, dt=dt) if i % 3 else None
    z = x.double() @ w.double().t()
    acc = ref.add_error(k) * (x.double().abs() @ w.double().abs().t())
    if b is not None:
        z, acc = z + b.double(), acc + ref.add_error(k) * b.double().abs()
    r = mk(g, T, n, dt=dt)
    for name in ("relu", ("none", "gelu", "gelu_tanh", "silu")[i % 4]):
        act = ref.act(z, name)
        for res in (None, r):
            y, want = linear.forward(x, w, b, residual=res, act=name), act if res is None else act + res.double()
            ref.check(y, want, dt, 1.2 * acc + ref.ACT_ERROR * z.abs() + 2.0 ** -24 * want.abs(), f"y {name}")
            y8, z8 = linear.forward(x, w, b, residual=res, act=name, save="z8")
            assert torch.equal(y8, y)
            check_codes(z8, z, acc)
        y16, z16 = linear.forward(x, w, b, residual=r.clone(), act=name, save="z")
        assert torch.equal(y16, y)
        ref.check(z16, z, dt, acc, "z")
    mine = r.clone()  # Y in place of R
    assert torch.equal(linear.forward(x, w, b, residual=mine, act=name, out=mine), y)


@pytest.mark.parametrize("T,k,n", lp.SIZES + lp.LARGE)
@pytest.mark.parametrize("dt", [BF, HF])
def test_backward_from_a_checkpoint(cuda, T, k, n, dt):
    """dX with its slope and Xv from an 8-bit or 16-bit pre-activation, an addend (in place too) and the sum over the
    tokens; dW of the recomputed Xv."""
    i = (lp.SIZES + lp.LARGE).index((T, k, n))
    g, u, name = gen(1000 + i), ref.UNIT[dt], ref.ACTS[1 + i % 4]
    dy, w, add = mk(g, T, n, dt=dt, scale=0.1), mk(g, n, k, dt=dt, scale=k ** -0.5), mk(g, T, k, dt=dt, scale=0.1)
    x16 = mk(g, T, k, dt=dt)
    x8 = ckpt8.Ckpt8(*ref.pack(x16), dt)
    D, Dabs = dy.double() @ w.double(), dy.double().abs() @ w.double().abs()
    for x, xv in ((x8, ref.unpack(*x8[:2])), (x16, x16.double())):
        s, X = ref.slope(xv, name), ref.act(xv, name)
        plain = D * s
        slack = ref.add_error(n) * Dabs * s.abs().clamp(min=1) + 2.0 ** -17 * D.abs()
        dx, dw, db, total = linear.backward(dy, x, w, in_act=name, add=add, dx_sum=True)
        want = plain + add.double()
        here = slack + 2.0 ** -24 * want.abs()
        ref.check(dx, want, dt, here, "dx")
        ref.check(total, want.sum(0), dt, (here + ref.add_error(T) * want.abs()).sum(0), "dx_sum", 2)
        ref.check(db, dy.double().sum(0), dt, ref.add_error(T) * dy.double().abs().sum(0), "db")
        e_x = u * X.abs() + 2.0 ** -18 * xv.abs() + ref.TINY[dt]   # Xv is rounded to dt
        e_w = dy.double().abs().t() @ e_x + ref.add_error(T) * (dy.double().abs().t() @ X.abs())
        ref.check(dw, dy.double().t() @ X, dt, e_w, "dw", 2)
        mine = add.clone()
        assert linear.backward(dy, x, w, in_act=name, add=mine, dx=mine, need_dw=False, need_db=False)[0] is mine
        assert torch.equal(mine, dx)
        bare = linear.backward(dy, x, w, in_act=name, need_dw=False, need_db=False)[0]
        ref.check(bare, plain, dt, slack + 2.0 ** -24 * plain.abs(), "dx without an addend")


@pytest.mark.parametrize("T,k,n", lp.SIZES + lp.LARGE)
@pytest.mark.parametrize("dt", [BF, HF])
def test_gradients_in_fp32_and_accumulated(cuda, T, k, n, dt):
    """dW, db and dX's sum in FP32, new and added to what is held; dW added to in 16 bits; dX that reads nothing."""
    i = (lp.SIZES + lp.LARGE).index((T, k, n))
    g = gen(2000 + i)
    dy, w, x = mk(g, T, n, dt=dt, scale=0.1), mk(g, n, k, dt=dt, scale=k ** -0.5), mk(g, T, k, dt=dt)
    D, Dabs = dy.double() @ w.double(), dy.double().abs() @ w.double().abs()
    W, Wabs = dy.double().t() @ x.double(), dy.double().abs().t() @ x.double().abs()
    Wsize = (dy.double().square().t() @ x.double().square()).sqrt()
    rows, columns = D.square().sum(0).sqrt(), dy.double().square().sum(0).sqrt()
    sums, db = D.sum(0), dy.double().sum(0)
    dx, *first = linear.backward(dy, x, w, grad_dtype=FP, dx_sum=True)
    ref.check(dx, D, dt, ref.add_error(n) * Dabs, "dx")
    assert torch.equal(linear.backward(dy, x, w, need_dw=False, need_db=False)[0], dx)
    assert all(v.dtype == FP for v in first)
    start = [mk(g, n, k, scale=0.1 * T ** 0.5), mk(g, n, scale=0.1 * T ** 0.5), mk(g, k, scale=float(rows.mean()))]
    held = [v.clone() for v in start]
    linear.backward(dy, x, w, dw=held[0], db=held[1], dx_sum=held[2], grad_dtype=FP, accumulate=True)
    for got, base in ((first, [0.0, 0.0, 0.0]), (held, start)):
        want = [v + (o.double() if isinstance(o, torch.Tensor) else o) for v, o in zip((W, db, sums), base)]
        check_fp32(got[0], want[0], Wsize, T, "dw", dt)
        # sums over the tokens: an error of 2^-24 of a partial sum for each token, of random signs
        check_fp32(got[1], want[1], columns, 16 * T ** 0.5, "db", dt)
        check_fp32(got[2], want[2], rows, n + 16 * T ** 0.5, "dx_sum", dt)
        for v, o, slack, what in zip(got, want, (ref.add_error(T) * Wabs, ref.add_error(T) * dy.double().abs().sum(0),
                                                 (ref.add_error(n) * Dabs + ref.add_error(T) * D.abs()).sum(0)), ("dw", "db", "dx_sum")):
            worst = ((v.double() - o).abs() - slack - 2.0 ** -23 * o.abs() - ref.TINY[FP]).max()
            assert worst <= 0, f"{what}: {worst} over its bound"
    start16 = start[0].to(dt)
    held16 = start16.clone()
    linear.backward(dy, x, w, need_dx=False, need_db=False, dw=held16, accumulate=True)
    want = W + start16.double()
    ref.check(held16, want, dt, ref.add_error(T) * Wabs + 2.0 ** -24 * want.abs(), "dw added in 16 bits")
    new16 = linear.backward(dy, x, w, need_dx=False, need_db=False)[1]
    ref.check(new16, W, dt, ref.add_error(T) * Wabs, "dw in 16 bits")


PAIRS = [(4100, 16384, 4200), (2300, 16383, 4200), (3000, 8200, 4200)]


@pytest.mark.parametrize("T,k,n", PAIRS)
@pytest.mark.parametrize("dt", [BF, HF])
def test_relu_codes_of_pairs_settle_at_the_exact_code(cuda, T, k, n, dt):
    """Products on pairs of CTAs: with ReLU a quotient near 1/2 has the code that the exact Z has, unless it is nearer
    than what settling can tell: its FP32 sums of eight products round by 2^-24 of a partial sum for each term, of random
    signs, a standard deviation of at most 1.3 2^-24 sqrt(sum x^2 w^2); six of them are held off.  Without ReLU the longest
    contraction's own error (some 10^-4 of a step) decides over a few of them.  A warp's 16 rows of 32 features hold
    0.02 quotients within the settled width, eight or more never."""
    assert lp.plan(0, n, T, k)[0] == 1
    g = gen(41)
    x, w = mk(g, T, k, dt=dt), mk(g, n, k, dt=dt, scale=k ** -0.5)
    z = x.double() @ w.double().t()
    size = (x.double().square() @ w.double().square().t()).sqrt()
    codes, scales = ref.pack(z)
    step = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 133).repeat_interleave(32, 1)[:, :n]
    q = z.abs() / step
    sure = (q - 0.5).abs() > 8 * 2.0 ** -24 * size / step

    def wrong(c):
        same = (c.scales == scales).repeat_interleave(32, 1)[:, :n]
        return int((((c.codes != 0) != (q > 0.5)) & sure & same).sum())

    for res in (None, mk(g, T, n, dt=dt)):
        assert wrong(linear.forward(x, w, residual=res, act="relu", save="z8")[1]) == 0
    if k == 16384:
        assert wrong(linear.forward(x, w, act="silu", save="z8")[1]) > 0


@pytest.mark.parametrize("T,k,n", [(1, 512, 1000), (40, 1024, 300), (333, 256, 1100), (2300, 320, 4200)])
@pytest.mark.parametrize("dt", [BF, HF])
def test_relu_codes_of_data_made_of_ties(cuda, T, k, n, dt):
    """Whole numbers whose sums are exact, one feature of each group far above the rest: most quotients are 1/2 or 3/2 to
    the last bit, more than a warp's list holds, and every code is the rule's."""
    g = gen(7)
    x = torch.randint(-1, 2, (T, k), device="cuda", generator=g).to(dt)
    w = torch.zeros(n, k, dtype=dt, device="cuda")
    w[torch.arange(n, device="cuda"), torch.randint(0, k - 1, (n,), device="cuda", generator=g)] = 1  # z in -1, 0, 1
    x[:, -1] = 1
    w[::32, :] = 0
    w[::32, -1] = 128                                                                                   # step 2
    z = x.double() @ w.double().t()
    codes, scales = ref.pack(z)
    for b in (None, torch.ones(n, dtype=dt, device="cuda")):
        want = (codes, scales) if b is None else ref.pack(z + 1)
        one = linear.forward(x, w, b, act="relu", save="z8")[1]
        assert torch.equal(one.scales, want[1]) and torch.equal(one.codes, want[0])
        two = linear.forward(x, w, b, act="relu", save="z8")[1]
        assert torch.equal(one.codes, two.codes)


def test_relu_codes_of_more_rows_than_the_lists_are_made_for(cuda):
    """A product in several launches: Y, the addend and the codes of all of them, rows apart."""
    T, k, n, dt = 24000, 16384, 4096, BF
    g = gen(43)
    x, w, b = mk(g, T, k, dt=dt), mk(g, n, k, dt=dt, scale=k ** -0.5), mk(g, n, dt=dt)
    r = mk(g, T, n + 8, dt=dt)[:, :n]
    held = ckpt8.Ckpt8(torch.empty(T, n + 32, dtype=torch.int8, device="cuda")[:, :n],
                       torch.empty(T, n // 32 + 1, dtype=torch.uint8, device="cuda")[:, : n // 32], dt)
    y, z8 = linear.forward(x, w, b, residual=r, act="relu", save="z8", z=held)
    assert z8 is held
    wrong = 0
    for t0 in range(0, T, 4000):
        rows = slice(t0, t0 + 4000)
        z = x[rows].double() @ w.double().t() + b.double()
        want = ref.act(z, "relu") + r[rows].double()
        size = (x[rows].double().square() @ w.double().square().t()).sqrt()
        # random operands: cut sums are off by 1e-5 of their size in the standard deviation, ten of them allowed
        ref.check(y[rows], want, dt, 1e-4 * size + 2.0 ** -24 * want.abs(), "y")
        codes, scales = ref.pack(z)
        step = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 133).repeat_interleave(32, 1)
        q = z.abs() / step
        sure = (q - 0.5).abs() > 8 * 2.0 ** -24 * size / step
        same = (held.scales[rows] == scales).repeat_interleave(32, 1)
        assert float(same.double().mean()) > 0.999
        wrong += int((((held.codes[rows] != 0) != (q > 0.5)) & sure & same).sum())
    assert wrong == 0
