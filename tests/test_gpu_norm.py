"""Norms and residual joins on the GPU against their FP64 restatement: every kind, the widths at which threads, warps, groups of
warps and clusters begin and end, rows apart and unaligned, what lies beside the rows, and the calls that the documents allow."""
import pytest
import torch

import linear_ref as lin
import norm_ref as ref
from chpl_b200 import _lib, check_device, norm

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
# one lane, one eight, a half warp's and a warp's features and one more, several warps, a CTA's most, clusters, the widest
WIDTHS = [1, 7, 8, 9, 255, 256, 257, 512, 513, 1031, 2048, 4097, 5120, 8192, 9217, 16384]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows(g, T, n, dt, pad=0, scale=1.0):
    """T x n, rows n + pad apart, NaN between them."""
    full = torch.full((T, n + pad), float("nan"), dtype=dt, device="cuda")
    full[:, :n] = torch.empty(T, n, device="cuda").normal_(0.0, scale, generator=g).to(dt)
    return full[:, :n]


def vec(g, n, dt, mean=0.0):
    return torch.empty(n, device="cuda").normal_(mean, 0.3, generator=g).to(dt)


def a_norm(g, n, dt, kind, bias=None):
    if kind == "none":
        return None
    return norm.Norm(vec(g, n, dt, 1.0), vec(g, n, dt) if (kind == "layer" if bias is None else bias) else None, kind, 1e-5)


def same(got, want, dt, what, factor=ref.ERROR):
    """Within the bound of want's size elementwise, and for 16-bit results in the 2-norm, where a sum's own error is far below
    their one rounding.  Not so for FP32 results, sums over T tokens: every term has some four roundings of its own and
    enters T / 2 partial sums of its size times sqrt(T / 2) in the mean, so the sum is off by about sqrt(4 T + T / 2 * T / 2 / T)
    2^-25 terms, and its size is about sqrt(T) terms: a unit and a half of it, more than the unit that check() leaves."""
    if dt is FP:
        assert bool(((got.double() - want[0]).abs() <= lin.UNIT[FP] * want[0].abs() + factor * want[1]).all()), what
    else:
        lin.check(got, want[0], dt, factor * want[1], what)


def opened(T, n, dt, pad):
    """(memory for T x n, what surrounds it)"""
    full = torch.full((T + 2, n + pad), 7.0, dtype=dt, device="cuda")
    return full[1:T + 1, :n], full


def untouched(full, T, n):
    assert bool((full[0] == 7).all()) and bool((full[T + 1:] == 7).all()) and bool((full[:, n:] == 7).all())


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("T,pad,dt,kind", [(1, 0, BF, "rms"), (5, 1, HF, "layer"), (301, 3, BF, "layer"), (150, 8, HF, "rms"), (700, 0, BF, "rms")])
def test_forward_and_backward(cuda, T, n, pad, dt, kind):
    g = gen(T + n)
    x, dh, add, v = rows(g, T, n, dt, pad), rows(g, T, n, dt, pad, 0.1), rows(g, T, n, dt, pad, 0.1), a_norm(g, n, dt, kind)
    if T > 4:
        x[3] = 0  # a padding token
    out, around = opened(T, n, dt, pad)
    h, st = norm.forward(x, v, save=True, out=out)
    assert h is out
    w = ref.wide(v)
    want = ref.apply(x.double(), w)
    same(h, want, dt, "h")
    untouched(around, T, n)
    exact = ref.stats(x.double(), w)
    assert bool(((st.double() - exact).abs() <= ref.ERROR * torch.stack([x.double().abs().mean(1), exact[:, 1] * (1 + x.double().abs().mean(1) * exact[:, 1])], 1)).all())
    for skip in (None, add):
        out, around = opened(T, n, dt, pad)
        dx, dw, db = norm.backward(dh, x, st, v, add=skip, dx=out)
        (rx, rxs), rw, rb = ref.pull(dh.double(), x.double(), st, w)
        if skip is not None:
            rx, rxs = rx + skip.double(), rxs + skip.double().abs()
        same(dx, (rx, rxs), dt, "dx")
        untouched(around, T, n)
        same(dw, rw, dt, "dw", ref.sum_error(T))
        assert (db is None) == (v.bias is None)
        if db is not None:
            same(db, rb, dt, "db", ref.sum_error(T))
    # FP32 gradients, added to
    into = torch.full((n,), 2.0, device="cuda"), torch.full((n,), 3.0, device="cuda") if v.bias is not None else None
    _, dw, db = norm.backward(dh, x, st, v, need_dx=False, dweight=into[0], dbias=into[1], accumulate=True)
    same(dw, (rw[0] + 2, rw[1] + 2), FP, "dw added to", ref.sum_error(T))
    if db is not None:
        same(db, (rb[0] + 3, rb[1] + 3), FP, "db added to", ref.sum_error(T))
    check_device()


@pytest.mark.parametrize("post", ["none", "rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "vector", "matrix"])
@pytest.mark.parametrize("pre", ["none", "rms", "layer"])
@pytest.mark.parametrize("T,n,pad,dt,bias", [(1, 264, 0, BF, None), (37, 1031, 1, HF, True), (400, 768, 0, BF, False), (160, 5121, 5, HF, None), (20, 16384, 0, BF, None)])
def test_join_and_its_gradients(cuda, post, gate, pre, T, n, pad, dt, bias):
    """bias: of all norms, of none, or of layer norms."""
    g = gen(T + n + len(post + gate + pre))
    x, y, dr = rows(g, T, n, dt, pad), rows(g, T, n, dt, pad), rows(g, T, n, dt, pad, 0.1)
    post, pre = a_norm(g, n, dt, post, bias), a_norm(g, n, dt, pre, bias)
    gate = {"none": lambda: None, "vector": lambda: vec(g, n, dt), "matrix": lambda: rows(g, T, n, dt, pad)}[gate]()
    dh = rows(g, T, n, dt, pad, 0.1) if pre else None
    how = dict(post=post, gate=gate, scale=0.5, residual_scale=0.75, pre=pre)
    wide = dict(post=ref.wide(post), gate=None if gate is None else gate.double(), scale=0.5, residual_scale=0.75, pre=ref.wide(pre))
    out, around = opened(T, n, dt, pad)
    out_h, around_h = opened(T, n, dt, pad)
    *got, (post_stats, pre_stats) = norm.join(x, y, save=True, out=out, out_h=out_h, **how)
    want = ref.join(x.double(), y.double(), **wide)
    same(got[0], want["r"], dt, "r")
    untouched(around, T, n)
    assert (post_stats is None) == (post is None) and (pre_stats is None) == (pre is None)
    if pre:
        same(got[1], want["h"], dt, "h")
        untouched(around_h, T, n)
    r = got[0]
    for first in (dr, None) if pre else (dr,):
        grads = norm.join_backward(first, dh, r, y, post_stats, pre_stats, **how)
        want = ref.join_backward(None if first is None else first.double(), None if dh is None else dh.double(), r.double(), y.double(), post_stats, pre_stats, **wide)
        assert {name for name, v in grads._asdict().items() if v is not None} == set(want)
        for name, v in want.items():
            same(getattr(grads, name), v, dt, name, ref.ERROR if v[0].dim() == 2 else ref.sum_error(T))
    check_device()


def test_what_is_left_out_changes_nothing(cuda):
    """need_*=False: the other outputs are bit for bit those of the whole call, and runs repeat bit for bit."""
    g = gen(3)
    T, n, dt = 333, 1030, BF
    x, y, dr, dh, gate = (rows(g, T, n, dt) for _ in range(5))
    post, pre = a_norm(g, n, dt, "layer"), a_norm(g, n, dt, "rms")
    how = dict(post=post, gate=gate, scale=0.5, pre=pre)
    r, h, st = norm.join(x, y, save=True, **how)
    assert torch.equal(r, norm.join(x, y, **how)[0]) and torch.equal(h, norm.join(x, y, **how)[1])
    whole = norm.join_backward(dr, dh, r, y, *st, **how)
    for off in ("need_dx", "need_dy", "need_dgate", "need_dparams"):
        part = norm.join_backward(dr, dh, r, y, *st, **how, **{off: False})
        for name, a, b in zip(whole._fields, whole, part):
            gone = {"need_dx": name == "dx", "need_dy": name == "dy", "need_dgate": name == "dgate", "need_dparams": name.startswith("dp")}[off]
            assert b is None if gone or a is None else torch.equal(a, b), (off, name)
    f32 = norm.join_backward(dr, dh, r, y, *st, **how, grad_dtype=FP)
    assert f32.dpost_weight.dtype == FP and torch.equal(f32.dpost_weight.to(dt), whole.dpost_weight) and f32.dx.dtype == dt


@pytest.mark.parametrize("pad", [0, 1])
def test_in_place(cuda, pad):
    """r over x or y, h over x, dx over dr or dh: bit for bit the calls with memory of their own."""
    g = gen(5)
    T, n, dt = 500, 770, HF
    v = a_norm(g, n, dt, "layer")
    x, y, dr, dh = (rows(g, T, n, dt, pad) for _ in range(4))
    h, st = norm.forward(x, v, save=True)
    z = x.as_strided(x.shape, x.stride()).clone(memory_format=torch.preserve_format) if pad == 0 else rows(g, T, n, dt, pad)
    z.copy_(x)
    assert torch.equal(norm.forward(z, v, out=z), h)
    want = norm.backward(dh, x, st, v, add=dr)
    for over in (dr, dh):
        z = rows(g, T, n, dt, pad)
        z.copy_(over)
        args = (z, x, st, v) if over is dh else (dh, x, st, v)
        got = norm.backward(*args, add=z if over is dr else dr, dx=z)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    r, h = norm.join(x, y, post=v, pre=v)
    for over in (x, y):
        z = rows(g, T, n, dt, pad)
        z.copy_(over)
        got = norm.join(z if over is x else x, z if over is y else y, post=v, pre=v, out=z)
        assert torch.equal(got[0], r) and torch.equal(got[1], h)


def test_rows_of_large_mean_infinities_and_nan(cuda):
    """A mean far above the deviation keeps its variance; a row with an infinity or a NaN spoils itself and no other; eps 0 and a
    zero row follow the formula (0 times infinity)."""
    g = gen(7)
    T, n = 6, 1000
    v = norm.Norm(torch.ones(n, device="cuda", dtype=HF), torch.zeros(n, device="cuda", dtype=HF), "layer", 0.0)
    x = rows(g, T, n, HF) + 1000
    h, st = norm.forward(x, v, save=True)
    same(h, ref.apply(x.double(), ref.wide(v)), HF, "large mean")
    y = rows(g, T, n, HF)
    want = norm.forward(y, v)
    for bad in (float("inf"), float("-inf"), float("nan")):
        z = y.clone()
        z[2, 900] = bad
        got = norm.forward(z, v)
        keep = [0, 1, 3, 4, 5]
        assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[2]).all())
    z = y.clone()
    z[4] = 0
    got = norm.forward(z, norm.Norm(v.weight, None, "rms", 0.0))
    assert bool(torch.isnan(got[4]).all()) and bool(torch.isfinite(got[[0, 1, 2, 3, 5]]).all())


def test_no_tokens_no_features(cuda):
    w = torch.ones(40, device="cuda", dtype=BF)
    v = norm.Norm(w, w, "layer")
    e = torch.empty(0, 40, device="cuda", dtype=BF)
    h, st = norm.forward(e, v, save=True)
    assert h.shape == (0, 40) and st.shape == (0, 2)
    dx, dw, db = norm.backward(e, e, st, v)
    assert dx.shape == (0, 40) and bool((dw == 0).all()) and bool((db == 0).all())
    keep = torch.full((40,), 5.0, device="cuda")
    _, dw, db = norm.backward(e, e, st, v, dweight=keep, dbias=keep.clone(), accumulate=True)
    assert dw is keep and bool((dw == 5).all()) and bool((db == 5).all())
    for gate in (w, e):
        out = norm.join_backward(e, e, e, e, st, st, post=v, gate=gate, pre=v)
        assert out.dgate.shape == gate.shape and all(bool((t == 0).all()) for t in out[3:])
    z = torch.empty(3, 0, device="cuda", dtype=BF)
    u = norm.Norm(torch.empty(0, device="cuda", dtype=BF))
    h, st = norm.forward(z, u, save=True)
    assert h.shape == (3, 0) and norm.backward(z, z, st, u)[1].shape == (0,)


def test_streams_devices_and_graphs(cuda):
    """Another stream than the current one; two graphs captured from calls that share nothing but the module, replayed in turn
    on new inputs."""
    g = gen(11)
    T, n, dt = 300, 9000, BF
    v = a_norm(g, n, dt, "rms")
    x, y = rows(g, T, n, dt), rows(g, T, n, dt)
    want = norm.join(x, y, post=v, pre=v, save=True)
    grads = norm.join_backward(y, x, want[0], y, *want[2], post=v, pre=v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = norm.join(x, y, post=v, pre=v, save=True, stream=side)
    more = norm.join_backward(y, x, got[0], y, *got[2], post=v, pre=v, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(more, grads))
    a, b = x.clone(), y.clone()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            o = norm.join(a, b, post=v, pre=v, save=True)
            outs.append((o, norm.join_backward(b, a, o[0], b, *o[2], post=v, pre=v)))
    for seed in (1, 2):
        x2, y2 = rows(gen(seed), T, n, dt), rows(gen(seed + 10), T, n, dt)
        a.copy_(x2)
        b.copy_(y2)
        for graph in graphs:
            graph.replay()
        want = norm.join(x2, y2, post=v, pre=v, save=True)
        grads = norm.join_backward(y2, x2, want[0], y2, *want[2], post=v, pre=v)
        for o, m in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
            assert all(p is q is None or torch.equal(p, q) for p, q in zip(m, grads))
    check_device()


def test_gradients_follow_differences(cuda):
    """<dx, e> against the difference of <dh, h> along e: (L(x + e) - L(x - e)) / 2 differs from it by h's third derivative along
    e, which a step of 1/16 of a deviation-one row makes at most 2^-12 |dh| |e| a feature, and by the roundings of h, 2^-11 of
    it each, of random signs: four standard deviations of their sum over the features are allowed."""
    g = gen(13)
    T, n, dt = 64, 2048, HF
    for kind in ("rms", "layer"):
        v = a_norm(g, n, dt, kind)
        x, dh, e = rows(g, T, n, dt), rows(g, T, n, dt), (rows(g, T, n, dt) / 16)
        h, st = norm.forward(x, v, save=True)
        dx, dw, _ = norm.backward(dh, x, st, v, grad_dtype=FP)
        up, down = (x + e), (x - e)
        step = (up.double() - down.double()) / 2  # what the rounded arguments differ by
        diff = (dh.double() * (norm.forward(up, v).double() - norm.forward(down, v).double())).sum(1) / 2
        along = (dx.double() * step).sum(1)
        slack = 4 * 2.0 ** -11 * (dh.double() * h.double()).norm(dim=1) + 2.0 ** -12 * (dh.double().norm(dim=1) * step.norm(dim=1)) + 2.0 ** -11 * (dx.double() * step).norm(dim=1) * 4
        assert bool(((diff - along).abs() <= slack).all()), kind
        # the weight enters linearly
        e = vec(g, n, dt)
        up = norm.Norm(v.weight + e, v.bias, kind, v.eps)
        step = up.weight.double() - v.weight.double()
        diff = (dh.double() * (norm.forward(x, up).double() - h.double())).sum()
        slack = 4 * 2.0 ** -11 * 2 * (dh.double() * h.double()).norm() + 2.0 ** -17 * (dw.double() * step).abs().sum()
        assert abs(diff - (dw.double() * step).sum()) <= slack


def test_refusals(cuda):
    T, n = 4, 64
    x = torch.randn(T, n, device="cuda", dtype=BF)
    w = torch.ones(n, device="cuda", dtype=BF)
    v = norm.Norm(w)
    h, st = norm.forward(x, v, save=True)
    bad = [lambda: norm.forward(x.float(), norm.Norm(w.float())), lambda: norm.forward(x.t(), v), lambda: norm.forward(x[0], v), lambda: norm.forward(x.cpu(), v),
           lambda: norm.forward(x, norm.Norm(w[:63])), lambda: norm.forward(x, norm.Norm(w.float())), lambda: norm.forward(x, norm.Norm(w, w[:3])),
           lambda: norm.forward(x, norm.Norm(w, kind="batch")), lambda: norm.forward(x, norm.Norm(w, eps=-1.0)), lambda: norm.forward(x, norm.Norm(w, eps=float("nan"))),
           lambda: norm.forward(x, None), lambda: norm.forward(x, v, out=x[:3]), lambda: norm.forward(x.expand(T, n)[:1].expand(T, n), v),
           lambda: norm.backward(x, x, st[:3], v), lambda: norm.backward(x, x[:3], st, v), lambda: norm.backward(x, x, st.double(), v), lambda: norm.backward(x, x, st.t().contiguous().t(), v),
           lambda: norm.backward(x, x, st, v, grad_dtype=HF), lambda: norm.backward(x, x, st, v, accumulate=True), lambda: norm.backward(x, x, st, v, add=x[:2]),
           lambda: norm.join(x, x[:3]), lambda: norm.join(x, x, gate=w[:5]), lambda: norm.join(x, x, gate=x[:2]), lambda: norm.join(x, x, gate=x[None]),
           lambda: norm.join(x, x, scale=float("inf")), lambda: norm.join(x, x.half()), lambda: norm.join(x, x, post=norm.Norm(w.cpu())),
           lambda: norm.join_backward(None, None, x, x, st, st, pre=v), lambda: norm.join_backward(x, x, x, x, st, st), lambda: norm.join_backward(x, None, x, x, st, st, pre=v),
           lambda: norm.join_backward(x, None, None, None, st, None, post=v), lambda: norm.join_backward(x, None, None, x, None, None, post=v),
           lambda: norm.join_backward(x, None, None, None, None, None, gate=w)]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.ChplError) as err:
            f()
        assert err.value.code == _lib.CHPL_ERR_INVALID, (i, err.value)
    wide = torch.zeros(2, 16385, device="cuda", dtype=BF)
    with pytest.raises(_lib.ChplError) as err:
        norm.forward(wide, norm.Norm(wide[0]))
    assert err.value.code == _lib.CHPL_ERR_UNSUPPORTED
    with pytest.raises(_lib.ChplError) as err:
        norm.backward(x, x, st, v, work=torch.empty(16, dtype=torch.uint8, device="cuda"))
    assert err.value.code == _lib.CHPL_ERR_WORKSPACE
    torch.cuda.synchronize()
