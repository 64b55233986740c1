"""CPU checks of the linear-layer entry points: what they refuse and how much workspace they ask for, before any CUDA
call, and the gradients of the tests' FP64 definitions against differences."""
import ctypes

import pytest
import torch

import linear_ref as ref
from chpl_b200 import _lib


def fwd(**kw):
    a = _lib.LinearFwd(type=_lib.CHPL_TYPE_BF16, act=_lib.CHPL_ACT_GELU, tokens=4, n=8, k=16, x=4096, ldx=16, w=8192, ldw=16,
                       y=16384, ldy=8)
    for name, v in kw.items():
        setattr(a, name, v)
    return a


def bwd(**kw):
    a = _lib.LinearBwd(type=_lib.CHPL_TYPE_F16, grad_type=_lib.CHPL_TYPE_F16, tokens=4, n=8, k=16, dy=4096, lddy=8, w=8192,
                       ldw=16, x=16384, ldx=16, dx=32768, lddx=16, dw=65536, lddw=16, db=131072)
    for name, v in kw.items():
        setattr(a, name, v)
    return a


def size(entry, a):
    L, need = _lib.load(), ctypes.c_size_t(12345)
    rc = getattr(L, entry + "_worksize")(ctypes.byref(a), ctypes.byref(need))
    return rc, need.value


INVALID, UNSUPPORTED, WORKSPACE = _lib.CHPL_ERR_INVALID, _lib.CHPL_ERR_UNSUPPORTED, _lib.CHPL_ERR_WORKSPACE


@pytest.mark.parametrize("kw,code", [
    (dict(type=2), INVALID), (dict(type=-1), INVALID), (dict(act=5), INVALID), (dict(tokens=-1), INVALID), (dict(n=-8), INVALID),
    (dict(k=(1 << 30) + 1), UNSUPPORTED), (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(y=None), INVALID),
    (dict(x=4097), INVALID), (dict(ldx=15), INVALID), (dict(ldw=8), INVALID), (dict(ldy=7), INVALID), (dict(ldy=1 << 33), UNSUPPORTED),
    (dict(bias=8193), INVALID), (dict(residual=4096, ldr=4), INVALID), (dict(residual=16384, ldr=16), INVALID), (dict(z=16384, ldz=2), INVALID),
    (dict(z8=_lib.Ckpt8(4096, None, 8, 1)), INVALID), (dict(z8=_lib.Ckpt8(4096, 4096, 8, 0)), INVALID), (dict(ldx=17), WORKSPACE)])
def test_forward_refuses(kw, code):
    L = _lib.load()
    assert L.chpl_linear_forward(None, ctypes.byref(fwd(**kw)), None, 0) == code
    assert L.chpl_last_error_string().startswith(b"linear_forward")


@pytest.mark.parametrize("kw,code", [
    (dict(type=2), INVALID), (dict(act=9), INVALID), (dict(in_act=-1), INVALID), (dict(grad_type=0), INVALID), (dict(tokens=-1), INVALID),
    (dict(dy=None), INVALID), (dict(lddy=7), INVALID), (dict(w=None), INVALID), (dict(x=None), INVALID), (dict(lddx=8), INVALID),
    (dict(lddw=8), INVALID), (dict(db=131073), INVALID), (dict(act=_lib.CHPL_ACT_SILU), INVALID), (dict(add=4096, ldadd=8), INVALID),
    (dict(add=32768, ldadd=24), INVALID), (dict(grad_type=2, dw=65538), INVALID), (dict(x8=_lib.Ckpt8(4096, 4096, 8, 1)), INVALID),
    (dict(dw=None, in_act=2, x=None), INVALID), (dict(tokens=4000), WORKSPACE)])
def test_backward_refuses(kw, code):
    L = _lib.load()
    assert L.chpl_linear_backward(None, ctypes.byref(bwd(**kw)), None, 0) == code
    assert L.chpl_last_error_string().startswith(b"linear_backward")


def test_c_program_calls_the_worksize_functions(tmp_path):
    """A C program fills the argument structures by name and links against libchpl.so."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "lin.c"
    src.write_text(r"""
#include "chpl.h"
int main(void) {
    chpl_linear_fwd f = {0};
    chpl_linear_bwd g = {0};
    chpl_ckpt8 c = {0, 0, 32, 1};
    size_t need = 1;
    f.type = CHPL_TYPE_BF16; f.act = CHPL_ACT_GELU; f.tokens = 8; f.n = 64; f.k = 32; f.ldx = 32; f.ldw = 32; f.ldy = 64;
    if (chpl_linear_forward_worksize(&f, &need) != CHPL_OK || need != 0) return 2;
    f.ldx = 33;
    if (chpl_linear_forward_worksize(&f, &need) != CHPL_OK || need < 8 * 32 * 2) return 3;
    g.type = CHPL_TYPE_F16; g.grad_type = CHPL_TYPE_F32; g.in_act = CHPL_ACT_SILU; g.tokens = 8; g.n = 64; g.k = 32;
    if (chpl_linear_backward_worksize(&g, &need) != CHPL_OK || need != 0) return 4;
    if (chpl_linear_backward(0, &g, 0, 0) != CHPL_OK) return 5;   /* no output wanted */
    if (chpl_ckpt8_pack(0, CHPL_TYPE_F32, -1, 32, 0, 32, &c) != CHPL_ERR_INVALID) return 6;
    return 0;
}
""")
    exe, libdir = tmp_path / "lin", os.path.dirname(_lib.LIB_PATH)
    cc = subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(exe), "-L",
                         libdir, "-lchpl", f"-Wl,-rpath,{libdir}"], capture_output=True, text=True)
    assert cc.returncode == 0, cc.stderr
    assert subprocess.run([str(exe)], timeout=60).returncode == 0


def test_null_arguments():
    L, need = _lib.load(), ctypes.c_size_t()
    assert L.chpl_linear_forward(None, None, None, 0) == INVALID
    assert L.chpl_linear_backward(None, None, None, 0) == INVALID
    assert L.chpl_linear_forward_worksize(ctypes.byref(fwd()), None) == INVALID
    assert L.chpl_linear_backward_worksize(None, ctypes.byref(need)) == INVALID
    assert L.chpl_linear_backward(None, ctypes.byref(bwd(dx=None, dw=None, db=None)), None, 0) == _lib.CHPL_OK
    assert L.chpl_linear_forward(None, ctypes.byref(fwd(tokens=0, x=None, y=None)), None, 0) == _lib.CHPL_OK
    c = _lib.Ckpt8(4096, 4096, 64, 2)
    assert L.chpl_ckpt8_pack(None, 3, 4, 64, 4096, 64, ctypes.byref(c)) == INVALID
    assert L.chpl_ckpt8_pack(None, 2, 4, 64, 4098, 64, ctypes.byref(c)) == INVALID
    assert L.chpl_ckpt8_pack(None, 2, 4, 65, 4096, 65, ctypes.byref(c)) == INVALID
    assert L.chpl_ckpt8_unpack(None, 2, 4, 64, None, 4096, 64) == INVALID
    assert L.chpl_ckpt8_unpack(None, 2, -4, 64, ctypes.byref(c), 4096, 64) == INVALID
    assert L.chpl_ckpt8_pack(None, 2, 0, 64, None, 64, ctypes.byref(c)) == _lib.CHPL_OK


def test_worksize():
    assert size("chpl_linear_forward", fwd()) == (0, 0)                       # every row aligned: nothing
    rc, need = size("chpl_linear_forward", fwd(ldx=17))                       # X is copied: 4 rows of 16
    assert rc == 0 and 4 * 16 * 2 <= need <= 4 * 16 * 2 + 256
    assert size("chpl_linear_forward", fwd(tokens=1, ldx=17)) == (0, 0)       # a single row has no distance
    rc, need = size("chpl_linear_forward", fwd(w=8194, k=15))
    assert rc == 0 and need >= 8 * 16 * 2
    small = size("chpl_linear_backward", bwd(db=None))
    assert small == (0, 0)
    rc, need = size("chpl_linear_backward", bwd(db=None, act=_lib.CHPL_ACT_SILU, z=4096, ldz=8))
    assert rc == 0 and need >= 4 * 8 * 2
    rc, need = size("chpl_linear_backward", bwd(db=None, x8=_lib.Ckpt8(4096, 4096, 16, 1)))
    assert rc == 0 and need >= 4 * 16 * 2
    assert size("chpl_linear_forward", fwd(tokens=-1))[0] == INVALID


@pytest.mark.parametrize("name", ref.ACTS)
def test_slopes_against_differences(name):
    """act' of the tests' definitions against central differences, h = 1e-5: truncation below 1e-9, rounding 1e-10."""
    z = torch.linspace(-7, 7, 1003, dtype=torch.float64)
    d = (ref.act(z + 1e-5, name) - ref.act(z - 1e-5, name)) / 2e-5
    keep = z.abs() > 1e-4
    assert torch.allclose(ref.slope(z, name)[keep], d[keep], rtol=0, atol=1e-8)


def test_checkpoint_rule_on_known_values():
    x = torch.zeros(1, 40, dtype=torch.float64)
    x[0, :4] = torch.tensor([1.0, -0.5, 1.99, 1.0 / 128])
    x[0, 32] = 100.0
    codes, scales = ref.pack(x)
    assert scales.tolist() == [[127, 133]] and codes[0, :4].tolist() == [64, -32, 127, 0] and codes[0, 32] == 100
    assert ref.unpack(codes, scales)[0, 0] == 1.0 and ref.unpack(codes, scales)[0, 32] == 100.0


def test_python_entry_points_refuse_without_a_gpu():
    """The torch binding loads without a GPU and refuses what is not on one, as ChplError with the C ABI's code."""
    from chpl_b200 import ckpt8, ffn, linear
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    bad = [lambda: linear.forward(x, w), lambda: linear.forward(x, w, act="swish"), lambda: linear.forward(x, w, save="16"),
           lambda: linear.forward(None, w), lambda: linear.forward(x[0], w), lambda: linear.backward(x, x, w),
           lambda: linear.backward(x, x, w, grad_dtype=torch.float64), lambda: linear.backward(x, x, w, accumulate=True),
           lambda: ckpt8.pack(x), lambda: ckpt8.unpack(ckpt8.empty(4, 16, torch.bfloat16, "cpu")),
           lambda: ffn.forward(x, w, None, w, None), lambda: _lib.torch_ops().linear_forward(x, w)]
    for i, f in enumerate(bad):
        with pytest.raises(_lib.ChplError) as err:
            f()
        assert err.value.code == INVALID, i
