"""Linear layers of a model on libchpl's tensor-core products.

``forward``:  Y = act(X W^T + b) + R, with the pre-activation kept in 16 bits or as an 8-bit checkpoint.
``backward``: dX, dW and db of such a layer, from 16-bit tensors or from checkpoints.

X is tokens x k, W is n x k, Y is tokens x n: CUDA tensors of BF16 or F16 whose rows are contiguous; rows may lie
any distance apart (include/chpl.h has the rules, and which copies unaligned rows cost).  Calls are asynchronous on torch's
current stream, or on `stream`, on which the inputs have to be ready; outputs that are not given and the workspace are
allocated from that stream's memory.  Errors raise ChplError.  Everything runs in libchpl.so on the GPU; there is no
host implementation here.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ckpt8 import GROUP, Ckpt8, current_handle, elsewhere, empty, invalid, matrix, on_stream, pointers

ACTS = {"none": _lib.CHPL_ACT_NONE, "relu": _lib.CHPL_ACT_RELU, "gelu": _lib.CHPL_ACT_GELU,
        "gelu_tanh": _lib.CHPL_ACT_GELU_TANH, "silu": _lib.CHPL_ACT_SILU}
_TYPES = {torch.bfloat16: _lib.CHPL_TYPE_BF16, torch.float16: _lib.CHPL_TYPE_F16}
_NO_CKPT = (0, 0, 0, 0)


def _lead(where: str, name: str, t) -> tuple[int, int, int, int, int]:
    """(type, rows, columns, row distance, device) of the matrix that sets a call's type and device."""
    try:
        code, (rows, cols), (ld, unit), device = _TYPES[t.dtype], t.shape, t.stride(), t.get_device()
        if unit == 1 and ld >= cols and device >= 0:
            return code, rows, cols, ld, device
    except (AttributeError, KeyError, TypeError, ValueError):
        pass
    ld = matrix(where, name, t, None, None, None)
    if t.dtype not in _TYPES:
        raise invalid(where, f"{name} is {t.dtype}: bfloat16 or float16 is wanted")
    return _TYPES[t.dtype], *t.shape, ld, t.get_device()


def _act(where: str, name: str) -> int:
    code = ACTS.get(name)
    if code is None:
        raise invalid(where, f"activation {name!r} is none of {', '.join(ACTS)}")
    return code


def _vector(where: str, name: str, t, n: int, dtype, device: int) -> int:
    if not isinstance(t, torch.Tensor) or t.shape != (n,) or t.stride() != (1,) and n > 1:
        raise invalid(where, f"{name} is not a contiguous vector of {n}")
    if t.dtype is not dtype or t.get_device() != device:
        raise invalid(where, f"{name} is {t.dtype} on {t.device}, not {dtype} on cuda:{device}")
    return t.data_ptr()


def _workspace(worksize, entry: str, args: bytes, device):
    need = ctypes.c_size_t()
    _lib.check(worksize(args, need), entry)
    return torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None


def forward(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
            act: str = "none", save: str = "none", out: torch.Tensor | None = None, z=None, work=None, stream=None):
    """Y = act(x w^T + bias) + residual.

    save="z" returns (Y, Z) with the pre-activation Z in x's type, save="z8" (Y, checkpoint of Z).  out and z may
    give the memory for Y and for what is saved; out may be residual itself.  work: a uint8 CUDA tensor to use as
    workspace instead of allocating one.
    """
    where = "linear.forward"
    code, tokens, k, ldx, dev = _lead(where, "x", x)
    act_code, dt = _act(where, act), x.dtype
    if elsewhere(dev, stream):
        with on_stream(x.device, stream):
            return forward(x, w, bias, residual=residual, act=act, save=save, out=out, z=z, work=work)
    n = w.shape[0]
    ldw = matrix(where, "w", w, dt, dev, (n, k))
    bp = _vector(where, "bias", bias, n, dt, dev) if bias is not None else 0
    rp, ldr = (residual.data_ptr(), matrix(where, "residual", residual, dt, dev, (tokens, n))) if residual is not None else (0, 0)
    if out is None:
        out, ldy = x.new_empty(tokens, n), n
    else:
        ldy = matrix(where, "out", out, dt, dev, (tokens, n))
    zp, ldz, z8 = 0, 0, _NO_CKPT
    if save == "z":
        z = x.new_empty(tokens, n) if z is None else z
        zp, ldz = z.data_ptr(), matrix(where, "z", z, dt, dev, (tokens, n))
    elif save == "z8":
        if z is None:
            z = empty(tokens, n, dt, x.device)
            z8 = (z.codes.data_ptr(), z.scales.data_ptr(), n, -(-n // GROUP))
        else:
            z8 = pointers(where, "z", z, dev, (tokens, n))
    elif save != "none":
        raise invalid(where, f"save {save!r} is none of none, z, z8")
    a = _lib.LINEAR_FWD.pack(code, act_code, tokens, n, k, x.data_ptr(), ldx, w.data_ptr(), ldw, bp, rp, ldr,
                             out.data_ptr(), ldy, zp, ldz, *z8)
    L = _lib.load()
    # rows that TMA can read (a base and a row distance of whole 16 bytes) need no workspace
    if work is None and ((ldx | ldw) & 7 or (x.data_ptr() | w.data_ptr()) & 15):
        work = _workspace(L.chpl_linear_forward_worksize, "chpl_linear_forward_worksize", a, x.device)
    ptr, size = (work.data_ptr(), work.numel() * work.element_size()) if work is not None else (None, 0)
    _lib.check(L.chpl_linear_forward(current_handle(dev), a, ptr, size), "chpl_linear_forward")
    return out if save == "none" else (out, z)


def backward(dy: torch.Tensor, x, w: torch.Tensor, *, act: str = "none", z=None, in_act: str = "none",
             add: torch.Tensor | None = None, need_dx: bool = True, need_dw: bool = True, need_db: bool = True,
             dx: torch.Tensor | None = None, dw: torch.Tensor | None = None, db: torch.Tensor | None = None,
             grad_dtype: torch.dtype | None = None, accumulate: bool = False, work=None, stream=None):
    """(dX, dW, db) of Y = act(X w^T + b) + R from dY; dR is dY itself.

    x is X, or with in_act the pre-activation that X = in_act(x) came from (dX is then x's gradient); z is the
    layer's own pre-activation, wanted where act is not none.  Either may be a tensor of dY's type or a Ckpt8.
    add is added to dX (the gradient that a skip connection brings); dx may be add itself.  need_*=False leaves an output
    out (None).  dW and db are of grad_dtype: dY's type, or torch.float32; accumulate adds them to the dw and db given.
    """
    where = "linear.backward"
    code, tokens, n, lddy, dev = _lead(where, "dy", dy)
    act_code, in_code, dt = _act(where, act), _act(where, in_act), dy.dtype
    if elsewhere(dev, stream):
        with on_stream(dy.device, stream):
            return backward(dy, x, w, act=act, z=z, in_act=in_act, add=add, need_dx=need_dx, need_dw=need_dw, need_db=need_db,
                            dx=dx, dw=dw, db=db, grad_dtype=grad_dtype, accumulate=accumulate, work=work)
    k = w.shape[-1]
    ldw = matrix(where, "w", w, dt, dev, (n, k))
    gt = grad_dtype or (dw.dtype if dw is not None else db.dtype if db is not None else dt)
    if gt != dt and gt != torch.float32:
        raise invalid(where, f"gradients in {gt}: {dt} or float32 is wanted")
    if accumulate and ((need_dw and dw is None) or (need_db and db is None)):
        raise invalid(where, "accumulate wants dw and db to add to")

    def saved(name, v, width):
        if v is None:
            return (0, 0, *_NO_CKPT)
        if isinstance(v, Ckpt8):
            return (0, 0, *pointers(where, name, v, dev, (tokens, width)))
        return (v.data_ptr(), matrix(where, name, v, dt, dev, (tokens, width)), *_NO_CKPT)

    xs = saved("x", x, k)
    zs = saved("z", z, n) if act != "none" else (0, 0, *_NO_CKPT)
    ap, ldadd = (add.data_ptr(), matrix(where, "add", add, dt, dev, (tokens, k))) if add is not None else (0, 0)
    lddx = lddw = 0
    if not need_dx:
        dx = None
    elif dx is None:
        dx, lddx = dy.new_empty(tokens, k), k
    else:
        lddx = matrix(where, "dx", dx, dt, dev, (tokens, k))
    if not need_dw:
        dw = None
    elif dw is None:
        dw, lddw = dy.new_empty(n, k, dtype=gt), k
    else:
        lddw = matrix(where, "dw", dw, gt, dev, (n, k))
    if not need_db:
        db = None
    elif db is None:
        db = dy.new_empty(n, dtype=gt)
    else:
        _vector(where, "db", db, n, gt, dev)
    xp, wp, bp = (v.data_ptr() if v is not None else 0 for v in (dx, dw, db))
    a = _lib.LINEAR_BWD.pack(code, act_code, in_code, _lib.CHPL_TYPE_F32 if gt == torch.float32 else code, bool(accumulate),
                             tokens, n, k, dy.data_ptr(), lddy, w.data_ptr(), ldw, *xs, *zs, ap, ldadd, xp, lddx, wp, lddw, bp)
    L = _lib.load()
    if work is None:
        work = _workspace(L.chpl_linear_backward_worksize, "chpl_linear_backward_worksize", a, dy.device)
    ptr, size = (work.data_ptr(), work.numel() * work.element_size()) if work is not None else (None, 0)
    _lib.check(L.chpl_linear_backward(current_handle(dev), a, ptr, size), "chpl_linear_backward")
    return dx, dw, db
