"""CPU checks of what the linear-layer entry points refuse where a size is zero: whatever a kernel would read is checked
before any launch, also where another operand's emptiness leaves less to compute."""
import ctypes
import itertools

import pytest

from chpl_b200 import _lib

INVALID = _lib.CHPL_ERR_INVALID


def bwd(**kw):
    a = _lib.LinearBwd(type=_lib.CHPL_TYPE_BF16, grad_type=_lib.CHPL_TYPE_BF16, tokens=4, n=8, k=16, dy=4096, lddy=8, w=8192,
                       ldw=16, x=16384, ldx=16, dx=32768, lddx=16, dw=65536, lddw=16, db=131072)
    for name, v in kw.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize("dw", [None, 65536])
@pytest.mark.parametrize("in_act", [_lib.CHPL_ACT_RELU, _lib.CHPL_ACT_GELU, _lib.CHPL_ACT_SILU])
def test_pre_activation_of_dx_is_checked_without_outputs_of_the_layer(dw, in_act):
    """n = 0: dX = in_act'(X) * 0 still reads X, whether or not a dW (of no rows) is asked for."""
    L = _lib.load()
    for kw in (dict(x=None), dict(ldx=15), dict(x=None, x8=_lib.Ckpt8(4096, None, 16, 1)), dict(x=None, x8=_lib.Ckpt8(4096, 4096, 15, 1))):
        a = bwd(n=0, lddy=8, in_act=in_act, dw=dw, **kw)
        assert L.chpl_linear_backward(None, ctypes.byref(a), None, 0) == INVALID, kw


def test_every_operand_that_is_read_is_checked():
    """All choices of outputs, activations and zero sizes: a call that reads an operand refuses its absence."""
    L = _lib.load()
    acts = (_lib.CHPL_ACT_NONE, _lib.CHPL_ACT_GELU)
    for tokens, n, k, act, in_act, dx, dw, db in itertools.product((0, 4), (0, 8), (0, 16), acts, acts, (0, 1), (0, 1), (0, 1)):
        kw = dict(tokens=tokens, n=n, k=k, act=act, in_act=in_act, z=262144, ldz=8, dx=32768 if dx else None,
                  dw=65536 if dw else None, db=131072 if db else None)
        some = tokens > 0 and n > 0
        reads = {"dy": some and bool(db or (k > 0 and (dx or dw))),
                 "z": some and act != _lib.CHPL_ACT_NONE and bool(db or (k > 0 and (dx or dw))),
                 "w": some and k > 0 and bool(dx),
                 "x": tokens > 0 and k > 0 and bool((dw and n > 0) or (dx and in_act != _lib.CHPL_ACT_NONE))}
        for name, read in reads.items():
            if read:
                a = bwd(**{**kw, name: None})
                assert L.chpl_linear_backward(None, ctypes.byref(a), None, 0) == INVALID, (kw, name)
