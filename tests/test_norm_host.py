"""CPU checks of the norms: what the C entry points refuse before any launch, the formulas of the reference against differences,
and the functions' place in torch's autograd, with the passes replaced by plain torch (the kernels need a GPU)."""
import ctypes

import pytest
import torch

import norm_ref as ref
from chpl_b200 import _lib, norm

INVALID, UNSUPPORTED, WORKSPACE = _lib.CHPL_ERR_INVALID, _lib.CHPL_ERR_UNSUPPORTED, _lib.CHPL_ERR_WORKSPACE
P = [4096 * (i + 1) for i in range(32)]  # addresses that are never looked at


def a_norm(kind=_lib.CHPL_NORM_LAYER, **kw):
    return _lib.Norm(**{**dict(kind=kind, eps=1e-6, weight=P[20], bias=P[21]), **kw})


def fwd(**kw):
    a = dict(type=_lib.CHPL_TYPE_BF16, join=1, tokens=4, n=16, scale=1.0, residual_scale=1.0, x=P[0], ldx=16, y=P[1], ldy=16, gate=P[2], ldgate=16,
             post=a_norm(), pre=a_norm(), r=P[3], ldr=16, h=P[4], ldh=16, post_stats=P[5], pre_stats=P[6])
    return _lib.NormFwd(**{**a, **kw})


def bwd(**kw):
    a = dict(type=_lib.CHPL_TYPE_BF16, join=1, grad_type=_lib.CHPL_TYPE_BF16, tokens=4, n=16, scale=1.0, residual_scale=1.0, dr=P[0], lddr=16, dh=P[1], lddh=16,
             r=P[2], ldr=16, y=P[3], ldy=16, gate=P[4], ldgate=16, post=a_norm(), pre=a_norm(), post_stats=P[5], pre_stats=P[6], dx=P[7], lddx=16, dy=P[8],
             lddy=16, dgate=P[9], lddgate=16, dpost_weight=P[10], dpost_bias=P[11], dpre_weight=P[12], dpre_bias=P[13])
    return _lib.NormBwd(**{**a, **kw})


NONE = _lib.Norm()
FORWARD = [dict(type=2), dict(type=7), dict(tokens=-1), dict(n=-1), dict(x=None), dict(y=None), dict(r=None), dict(h=None), dict(ldx=15), dict(ldy=15),
           dict(ldr=15), dict(ldh=15), dict(ldgate=15), dict(x=P[0] + 1), dict(gate=P[2] + 1), dict(post=a_norm(kind=3)), dict(pre=a_norm(kind=-1)),
           dict(post=a_norm(weight=None)), dict(pre=a_norm(weight=P[20] + 1)), dict(pre=a_norm(bias=P[21] + 1)), dict(pre=a_norm(eps=-1e-6)),
           dict(pre=a_norm(eps=float("nan"))), dict(post=a_norm(eps=float("inf"))), dict(scale=float("nan")), dict(residual_scale=float("inf")),
           dict(post_stats=P[5] + 4), dict(pre_stats=P[6] + 4), dict(r=P[0], ldr=24), dict(r=P[1], ldr=24), dict(h=P[1], ldh=24), dict(h=P[3]),
           dict(join=0), dict(join=0, post=NONE, pre=NONE), dict(join=0, post=NONE, h=P[0], ldh=24)]
BACKWARD = [dict(type=2), dict(grad_type=_lib.CHPL_TYPE_F16), dict(tokens=-1), dict(n=-3), dict(dr=P[0] + 1), dict(lddr=15), dict(dh=None), dict(lddh=15),
            dict(r=None), dict(ldr=15), dict(y=None), dict(ldy=15), dict(gate=P[4] + 1), dict(ldgate=15), dict(post_stats=None), dict(pre_stats=None),
            dict(pre_stats=P[6] + 4), dict(dx=P[7] + 1), dict(lddx=15), dict(lddy=15), dict(dy=P[8] + 1), dict(lddgate=15), dict(dpost_weight=P[10] + 1),
            dict(dpre_bias=P[13] + 1), dict(dx=P[0], lddx=24), dict(dx=P[1], lddx=24), dict(pre=NONE), dict(post=NONE), dict(gate=None),
            dict(post=a_norm(weight=None)), dict(pre=a_norm(weight=None)), dict(join=0), dict(join=0, post=NONE, dpost_weight=None, dpost_bias=None),
            dict(join=0, post=NONE, dpost_weight=None, dpost_bias=None, dgate=None), dict(pre=NONE, dr=None, dpre_weight=None, dpre_bias=None),
            dict(scale=float("inf")), dict(post=a_norm(kind=9)), dict(grad_type=_lib.CHPL_TYPE_F32, dpost_bias=P[11] + 2)]


@pytest.mark.parametrize("kw", FORWARD, ids=str)
def test_forward_refuses(kw):
    a = fwd(**kw)
    assert _lib.load().chpl_norm_forward(None, ctypes.byref(a)) == INVALID


@pytest.mark.parametrize("kw", BACKWARD, ids=str)
def test_backward_refuses(kw):
    a = bwd(**kw)
    assert _lib.load().chpl_norm_backward(None, ctypes.byref(a), P[30], 1 << 40) == INVALID


def test_other_refusals():
    L = _lib.load()
    for a, call in ((fwd(n=16385, ldx=20000, ldy=20000, ldr=20000, ldh=20000, ldgate=20000), lambda a: L.chpl_norm_forward(None, ctypes.byref(a))),
                    (bwd(n=16385), lambda a: L.chpl_norm_backward(None, ctypes.byref(a), None, 0)), (fwd(tokens=(1 << 30) + 1), lambda a: L.chpl_norm_forward(None, ctypes.byref(a))),
                    (fwd(ldx=(1 << 32) + 1), lambda a: L.chpl_norm_forward(None, ctypes.byref(a)))):
        assert call(a) == UNSUPPORTED
    assert L.chpl_norm_forward(None, None) == INVALID and L.chpl_norm_backward(None, None, None, 0) == INVALID
    size = ctypes.c_size_t()
    assert L.chpl_norm_backward_worksize(ctypes.byref(bwd()), None) == INVALID
    assert L.chpl_norm_backward_worksize(ctypes.byref(bwd()), ctypes.byref(size)) == 0 and size.value >= 4 * 16 * 4
    assert L.chpl_norm_backward(None, ctypes.byref(bwd()), P[30], size.value - 1) == WORKSPACE
    assert L.chpl_norm_backward(None, ctypes.byref(bwd()), None, size.value) == WORKSPACE
    assert L.chpl_norm_backward(None, ctypes.byref(bwd()), P[30] + 8, size.value) == INVALID
    # nothing to sum up: no workspace; nothing to do: nothing is looked at
    none = dict(dpost_weight=None, dpost_bias=None, dpre_weight=None, dpre_bias=None)
    assert L.chpl_norm_backward_worksize(ctypes.byref(bwd(**none)), ctypes.byref(size)) == 0 and size.value == 0
    assert L.chpl_norm_forward(None, ctypes.byref(fwd(tokens=0, x=None, y=None, r=None, h=None))) == 0
    assert L.chpl_norm_forward(None, ctypes.byref(fwd(n=0, x=None, y=None, r=None, h=None))) == 0


def test_workspace_covers_every_shape():
    """The workspace holds the sums of every unit that a launch may have: growing in the tokens up to one to an SM, and enough
    for one part of each sum."""
    L = _lib.load()
    size = ctypes.c_size_t()
    for n in (1, 500, 513, 4096, 5120, 9000, 16384):
        last = 0
        for tokens in (1, 2, 147, 148, 149, 1000, 100000, 1 << 30):
            a = bwd(tokens=tokens, n=n, **{k: n for k in ("lddr", "lddh", "ldr", "ldy", "ldgate", "lddx", "lddy", "lddgate")})
            assert L.chpl_norm_backward_worksize(ctypes.byref(a), ctypes.byref(size)) == 0
            assert 4 * 4 * n <= size.value <= 4 * 4 * (n + 3) * 148 + 256
            last = max(last, size.value)
        assert last == size.value or n < 16384


# ------------------------------------------------------------------------------- the reference's formulas
def test_reference_gradients_follow_differences():
    g = torch.Generator().manual_seed(1)

    def mk(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    T, n = 3, 11
    for kind in ("rms", "layer"):
        for gate in (None, mk(n), mk(T, n)):
            post, pre = (ref.N(mk(n), mk(n), kind, 1e-3) for _ in range(2))
            leaves = dict(x=mk(T, n), y=mk(T, n), pw=post.weight, pb=post.bias, qw=pre.weight, qb=pre.bias)
            if gate is not None:
                leaves["gate"] = gate
            dr, dh = mk(T, n), mk(T, n)

            def loss(x, y, pw, pb, qw, qb, gate=None):
                out = ref.join(x, y, ref.N(pw, pb, kind, 1e-3), gate, 0.5, 0.75, ref.N(qw, qb, kind, 1e-3))
                return (dr * out["r"][0]).sum() + (dh * out["h"][0]).sum()

            r = ref.join(leaves["x"], leaves["y"], post, gate, 0.5, 0.75, pre)["r"][0]
            got = ref.join_backward(dr, dh, r, leaves["y"], ref.stats(leaves["y"], post), ref.stats(r, pre), post, gate, 0.5, 0.75, pre)
            names = dict(x="dx", y="dy", pw="dpost_weight", pb="dpost_bias", qw="dpre_weight", qb="dpre_bias", gate="dgate")
            for name, leaf in leaves.items():
                e = mk(*leaf.shape)
                step = 1e-5
                diff = (loss(**{**leaves, name: leaf + step * e}) - loss(**{**leaves, name: leaf - step * e})) / (2 * step)
                # the third derivative's share is some 1e-10, that of the roundings 1e-16 |loss| / step
                assert abs(diff - (got[names[name]][0] * e).sum()) <= 1e-7 * (1 + abs(diff)), (kind, name)


# --------------------------------------------------------------------------------------------- autograd
class Passes:
    """norm.forward, backward, join and join_backward in plain FP64 torch."""

    def __init__(self):
        self.calls = []

    def forward(self, x, v, *, save=False):
        assert x.dim() == 2
        self.calls.append(("forward", save))
        h = ref.apply(x, ref.N(*v))[0]
        return (h, ref.stats(x, v)) if save else h

    def backward(self, dh, x, st, v, *, need_dx=True, need_dparams=True):
        self.calls.append(("backward", need_dx, need_dparams))
        (dx, _), (dw, _), db = ref.pull(dh, x, st, ref.N(*v))
        return dx if need_dx else None, dw if need_dparams else None, db[0] if db and need_dparams else None

    def join(self, x, y, *, post=None, gate=None, scale=1.0, residual_scale=1.0, pre=None, save=False):
        assert x.dim() == 2 == y.dim()
        self.calls.append(("join", save))
        out = {k: v[0] for k, v in ref.join(x, y, post, gate, scale, residual_scale, pre).items()}
        got = (out["r"],) if pre is None else (out["r"], out["h"])
        if save:
            return *got, (ref.stats(y, post) if post else None, ref.stats(out["r"], pre) if pre else None)
        return got[0] if pre is None else got

    def join_backward(self, dr, dh, r, y, post_stats, pre_stats, *, post=None, gate=None, scale=1.0, residual_scale=1.0, pre=None, need_dx=True,
                      need_dy=True, need_dgate=True, need_dparams=True):
        self.calls.append(("join_backward", dr is None, dh is None, need_dx, need_dy, need_dgate, need_dparams))
        y = torch.zeros_like(dr if dr is not None else dh) if y is None else y
        out = {k: v[0] for k, v in ref.join_backward(dr, dh, r, y, post_stats, pre_stats, post, gate, scale, residual_scale, pre).items()}
        need = dict(dx=need_dx, dy=need_dy, dgate=need_dgate)
        return norm.Joined(*(out.get(f) if need.get(f, need_dparams) else None for f in norm.Joined._fields))


@pytest.fixture
def passes(monkeypatch):
    p = Passes()
    for name in ("forward", "backward", "join", "join_backward"):
        monkeypatch.setattr(norm, name, getattr(p, name))
    return p


def leaves(lead=(4,), n=5, frozen=(), matrix=True):
    g = torch.Generator().manual_seed(2)
    t = dict(x=torch.randn(*lead, n, generator=g), y=torch.randn(*lead, n, generator=g), gate=torch.randn(*(lead if matrix else ()), n, generator=g))
    t.update({k: torch.randn(n, generator=g) for k in ("pw", "pb", "qw", "qb")})
    return {k: v.double().requires_grad_(k not in frozen) for k, v in t.items()}


def plain_norm(v, w, b, kind, eps):
    m = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return (v - m) / ((v - m).square().mean(-1, keepdim=True) + eps).sqrt() * w + b


def plain_join(t):
    r = 0.75 * t["x"] + 0.5 * t["gate"] * plain_norm(t["y"], t["pw"], t["pb"], "layer", 1e-3)
    return r, plain_norm(r, t["qw"], t["qb"], "rms", 1e-3)


def own_join(t):
    return norm.joined(t["x"], t["y"], post=norm.Norm(t["pw"], t["pb"], "layer", 1e-3), gate=t["gate"], scale=0.5, residual_scale=0.75,
                       pre=norm.Norm(t["qw"], t["qb"], "rms", 1e-3))


@pytest.mark.parametrize("lead,matrix", [((4,), True), ((4,), False), ((), False), ((2, 3), True), ((1, 1, 4), False), ((0, 3), True)])
def test_joined(passes, lead, matrix):
    t = leaves(lead, matrix=matrix)
    want, got = plain_join(t), own_join(t)
    dr, dh = torch.randn(want[0].shape, dtype=torch.float64), torch.randn(want[0].shape, dtype=torch.float64)
    assert all(a.shape == b.shape and torch.allclose(a, b) for a, b in zip(got, want))
    for a, b in zip(torch.autograd.grad(got, list(t.values()), (dr, dh)), torch.autograd.grad(want, list(t.values()), (dr, dh))):
        assert a.shape == b.shape and torch.allclose(a, b)


def test_only_one_of_the_outputs_is_used(passes):
    for i in (0, 1):
        t = leaves()
        d = torch.randn(4, 5, dtype=torch.float64)
        want = torch.autograd.grad(plain_join(t)[i], list(t.values()), d, allow_unused=True)
        got = torch.autograd.grad(own_join(t)[i], list(t.values()), d, allow_unused=True)
        assert all(a is b is None or torch.allclose(a, b) for a, b in zip(got, want))
        assert passes.calls[-1][1:3] == (i == 1, i == 0)


def test_normalized(passes):
    for lead in ((4,), (), (2, 3), (0,)):
        for kind in ("rms", "layer"):
            t = leaves(lead)
            want, got = plain_norm(t["x"], t["pw"], t["pb"], kind, 1e-3), norm.normalized(t["x"], norm.Norm(t["pw"], t["pb"], kind, 1e-3))
            d = torch.randn(want.shape, dtype=torch.float64)
            assert torch.allclose(want, got) and want.shape == got.shape
            some = [t["x"], t["pw"], t["pb"]]
            assert all(torch.allclose(a, b) for a, b in zip(torch.autograd.grad(got, some, d), torch.autograd.grad(want, some, d)))


def test_frozen_inputs_cost_nothing(passes):
    for frozen in (("x",), ("y",), ("gate",), ("pw", "pb", "qw", "qb"), ("x", "y", "gate")):
        t = leaves(frozen=frozen)
        some = [v for v in t.values() if v.requires_grad]
        d = torch.randn(4, 5, dtype=torch.float64)
        want, got = torch.autograd.grad(plain_join(t), some, (d, d)), torch.autograd.grad(own_join(t), some, (d, d))
        assert all(torch.allclose(a, b) for a, b in zip(got, want))
        assert passes.calls[-1][3:] == ("x" not in frozen, "y" not in frozen, "gate" not in frozen, "pw" not in frozen)
    with torch.no_grad():
        own_join(leaves())
    assert passes.calls[-1] == ("join", False)
    t = leaves(frozen=("x", "y", "gate", "pw", "pb", "qw", "qb"))
    own_join(t)
    norm.normalized(t["x"], norm.Norm(t["pw"]))
    assert passes.calls[-2:] == [("join", False), ("forward", False)]


def test_a_second_differentiation_raises(passes):
    t = leaves()
    for f, inputs in ((lambda: own_join(t)[1], t["x"]), (lambda: norm.normalized(t["x"], norm.Norm(t["pw"])), t["x"])):
        dx, = torch.autograd.grad((f() * 2).sum(), inputs, create_graph=True)
        with pytest.raises(_lib.ChplError, match="differentiated again"):
            dx.square().sum().backward()


def test_shapes_that_do_not_fit(passes):
    x = torch.zeros(2, 3, 5)
    for kw in (dict(y=torch.zeros(2, 3, 4)), dict(y=torch.zeros(6, 5)), dict(y=x, gate=torch.zeros(2, 1, 5)), dict(y=x, gate=torch.zeros(6, 5))):
        with pytest.raises(_lib.ChplError):
            norm.joined(x, kw["y"], gate=kw.get("gate"))
