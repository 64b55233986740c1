"""CPU checks of the 4-bit module: what the C entry points refuse before any launch, sizes, and that the tests' sizes reach every
kernel, tile and split on 148 SMs."""
import ctypes
import math
import random

import pytest

import mx4_ref as ref
from chpl_b200 import _lib

INVALID, UNSUPPORTED, WORKSPACE = _lib.CHPL_ERR_INVALID, _lib.CHPL_ERR_UNSUPPORTED, _lib.CHPL_ERR_WORKSPACE
P = [4096 * (i + 1) for i in range(16)]  # addresses that are never looked at


def fwd(**kw):
    a = dict(type=_lib.CHPL_TYPE_BF16, act=0, tokens=40, n=64, k=96, x=P[0], ldx=96, w4=_lib.Mx4(P[1], P[2], 48), bias=P[3], residual=P[4], ldr=64, y=P[5],
             ldy=64)
    return _lib.Mx4Fwd(**{**a, **kw})


BAD = [dict(type=2), dict(type=-1), dict(act=5), dict(act=-1), dict(tokens=-1), dict(n=-1), dict(k=-1), dict(x=None), dict(x=P[0] + 1), dict(ldx=95),
       dict(w4=_lib.Mx4(None, P[2], 48)), dict(w4=_lib.Mx4(P[1], None, 48)), dict(w4=_lib.Mx4(P[1] + 8, P[2], 48)), dict(w4=_lib.Mx4(P[1], P[2] + 8, 48)),
       dict(w4=_lib.Mx4(P[1], P[2], 32)), dict(w4=_lib.Mx4(P[1], P[2], 56)), dict(x4=_lib.Mx4(P[6], P[7], 47)), dict(x4=_lib.Mx4(P[6], None, 48)),
       dict(x4=_lib.Mx4(P[6] + 1, P[7], 48)), dict(bias=P[3] + 1), dict(residual=P[4] + 1), dict(ldr=63), dict(y=None), dict(y=P[5] + 1), dict(ldy=63),
       dict(y=P[4], ldy=72)]


@pytest.mark.parametrize("kw", BAD, ids=range(len(BAD)))
def test_linear_refuses(kw):
    assert _lib.load().chpl_mx4_linear(None, ctypes.byref(fwd(**kw)), P[10], 1 << 40) == INVALID


def test_workspace_and_sizes():
    L = _lib.load()
    size, bytes_ = ctypes.c_size_t(), ctypes.c_int64()

    def need(**kw):
        assert L.chpl_mx4_linear_worksize(ctypes.byref(fwd(**kw)), ctypes.byref(size)) == 0
        return size.value

    # codes of whole groups and scales of whole pieces and blocks of rows; none where X is coded already, or by the product
    assert need() == 40 * 48 // 256 * 256 + 256 + 1024 and need(tokens=8) == 0 and need(x4=_lib.Mx4(P[6], P[7], 48)) == 0
    assert need(tokens=0) == need(n=0) == need(k=0) == 0
    assert need(tokens=300, k=257, w4=_lib.Mx4(P[1], P[2], 144), ldx=257) == -(-300 * 144 // 256) * 256 + 3 * 2048
    assert L.chpl_mx4_linear(None, ctypes.byref(fwd()), P[10], need() - 1) == WORKSPACE
    assert L.chpl_mx4_linear(None, ctypes.byref(fwd()), None, need()) == WORKSPACE
    assert L.chpl_mx4_linear(None, ctypes.byref(fwd()), P[10] + 16, need()) == INVALID
    assert L.chpl_mx4_linear(None, None, None, 0) == INVALID and L.chpl_mx4_linear_worksize(ctypes.byref(fwd()), None) == INVALID
    assert L.chpl_mx4_linear(None, ctypes.byref(fwd(tokens=0, x=None, y=None)), None, 0) == 0
    assert L.chpl_mx4_linear(None, ctypes.byref(fwd(k=(1 << 30) + 1)), None, 0) == UNSUPPORTED
    for rows, cols, want in ((1, 1, 1024), (128, 256, 1024), (129, 256, 2048), (128, 257, 2048), (0, 5, 0), (5, 0, 0)):
        assert L.chpl_mx4_scale_bytes(rows, cols, ctypes.byref(bytes_)) == 0 and bytes_.value == want
    assert L.chpl_mx4_scale_bytes(-1, 1, ctypes.byref(bytes_)) == INVALID and L.chpl_mx4_scale_bytes(1, 1, None) == INVALID


@pytest.mark.parametrize("call", ["chpl_mx4_pack", "chpl_mx4_unpack"])
def test_pack_and_unpack_refuse(call):
    L = _lib.load()

    def run(type=0, rows=4, cols=96, x=P[0], ldx=96, c=_lib.Mx4(P[1], P[2], 48)):
        c = None if c is None else ctypes.byref(c)
        args = (type, rows, cols, x, ldx, c) if call == "chpl_mx4_pack" else (type, rows, cols, c, x, ldx)
        return getattr(L, call)(None, *args)

    for kw in (dict(type=3), dict(rows=-1), dict(cols=-1), dict(x=None), dict(x=P[0] + 1), dict(ldx=95), dict(c=None), dict(c=_lib.Mx4(None, P[2], 48)),
               dict(c=_lib.Mx4(P[1], None, 48)), dict(c=_lib.Mx4(P[1], P[2], 47)), dict(c=_lib.Mx4(P[1], P[2], 56)), dict(c=_lib.Mx4(P[1] + 4, P[2], 48)),
               dict(c=_lib.Mx4(P[1], P[2] + 4, 48)), dict(type=2, x=P[0] + 2)):
        assert run(**kw) == INVALID, kw
    assert run(rows=(1 << 30) + 1) == UNSUPPORTED
    assert run(rows=0, x=None) == 0 and run(cols=0, x=None) == 0


def test_sizes_reach_every_plan():
    have = {ref.plan(*s) for s in ref.SIZES}
    assert len(have) == len(ref.SIZES)
    rng = random.Random(9)

    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    met = {ref.plan(size(1, 8192), size(32, 16384), size(32, 16384)) for _ in range(50000)}
    assert met <= have, met - have
