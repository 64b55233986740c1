"""What norms and joins are launched as: rows of a batch run one after another only where more at once would not fit."""
import ctypes

import pytest

from chpl_b200 import _lib

P = [4096 * (i + 1) for i in range(32)]  # addresses that are never looked at
NONE = _lib.Norm()


def norm_(kind=_lib.CHPL_NORM_LAYER):
    return _lib.Norm(kind=kind, eps=1e-6, weight=P[20], bias=P[21])


def forward(tokens, n, join, pad):
    ld = {k: n + pad for k in ("ldx", "ldy", "ldr", "ldh")}
    return _lib.NormFwd(type=0, join=join, tokens=tokens, n=n, scale=1.0, residual_scale=1.0, x=P[0], y=P[1], gate=P[2] if join else None, post=norm_() if join else NONE,
                        pre=norm_(), r=P[3], h=P[4], **ld)


def backward(tokens, n, join, pad):
    ld = {k: n + pad for k in ("lddr", "lddh", "ldr", "ldy", "lddx", "lddy")}
    sums = dict(dgate=P[9], dpost_weight=P[10], dpost_bias=P[11], dy=P[8]) if join else {}
    return _lib.NormBwd(type=0, join=join, grad_type=0, tokens=tokens, n=n, scale=1.0, residual_scale=1.0, dr=P[0], dh=P[1], r=P[2], y=P[3], gate=P[4] if join else None,
                        post=norm_() if join else NONE, pre=norm_(), post_stats=P[5], pre_stats=P[6], dx=P[7], dpre_weight=P[12], dpre_bias=P[13], **sums, **ld)


def plan(a):
    p = (ctypes.c_int64 * 3)()
    call = _lib.load().chpl_diag_norm_forward_plan if isinstance(a, _lib.NormFwd) else _lib.load().chpl_diag_norm_backward_plan
    assert call(ctypes.byref(a), p) == 0
    return tuple(p)


@pytest.mark.parametrize("of", [forward, backward], ids=["forward", "backward"])
@pytest.mark.parametrize("join", [0, 1])
@pytest.mark.parametrize("pad", [0, 1])
def test_rows_wait_only_for_room(of, join, pad):
    clusters = set()
    for n in (1, 500, 513, 1024, 2048, 4096, 5120, 6144, 8192, 9216, 10000, 12288, 16384):
        cluster, rows, units = plan(of(1 << 20, n, join, pad))  # as many at once as there may be
        clusters.add(cluster)
        for tokens in (1, 24, 33, 34, 60, 74, 75, 100, 147, 148, 149, 222, 223, 296, 297, 444, 700, 5000):
            c, r, u = plan(of(tokens, n, join, pad))
            assert c == cluster and 1 <= r <= rows and 1 <= u <= units
            assert -(-tokens // (r * u)) <= -(-tokens // (rows * units)), (n, tokens)
            assert r * (u - 1) < tokens  # no unit without a row
    assert clusters >= {1, 2}


@pytest.mark.parametrize("of", [forward, backward], ids=["forward", "backward"])
def test_every_width_has_a_shape(of):
    """A cluster exchanges the sums of four rows at most, and a row's warps fit into its CTAs."""
    for n in range(1, 16385, 5):
        for join in (0, 1):
            cluster, rows, units = plan(of(1 << 20, n, join, n % 3))
            assert cluster in (1, 2, 4) and (cluster == 1 or rows <= 4) and rows * -(-n // (512 * cluster)) <= (32 if of is forward else 16)
            assert units == {1: 148, 2: 74, 4: 33}[cluster]


def test_refusals():
    p = (ctypes.c_int64 * 3)()
    L = _lib.load()
    for a, call in ((forward, L.chpl_diag_norm_forward_plan), (backward, L.chpl_diag_norm_backward_plan)):
        assert call(None, p) == _lib.CHPL_ERR_INVALID and call(ctypes.byref(a(3, 64, 1, 0)), None) == _lib.CHPL_ERR_INVALID
        assert call(ctypes.byref(a(0, 64, 1, 0)), p) == _lib.CHPL_ERR_INVALID and call(ctypes.byref(a(3, 0, 1, 0)), p) == _lib.CHPL_ERR_INVALID
        assert call(ctypes.byref(a(3, 64, 1, -1)), p) == _lib.CHPL_ERR_INVALID
