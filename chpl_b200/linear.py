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
from .ckpt8 import Ckpt8, empty, invalid, matrix, on_stream, struct_of

ACTS = {"none": _lib.CHPL_ACT_NONE, "relu": _lib.CHPL_ACT_RELU, "gelu": _lib.CHPL_ACT_GELU,
        "gelu_tanh": _lib.CHPL_ACT_GELU_TANH, "silu": _lib.CHPL_ACT_SILU}
_TYPES = {torch.bfloat16: _lib.CHPL_TYPE_BF16, torch.float16: _lib.CHPL_TYPE_F16}
_NONE = _lib.Ckpt8()


def _type(where: str, t) -> int:
    code = _TYPES.get(getattr(t, "dtype", None))
    if code is None:
        raise invalid(where, f"{getattr(t, 'dtype', type(t).__name__)}: bfloat16 or float16 is wanted")
    return code


def _act(where: str, name: str) -> int:
    code = ACTS.get(name)
    if code is None:
        raise invalid(where, f"activation {name!r} is none of {', '.join(ACTS)}")
    return code


def _vector(where: str, name: str, t, n: int, dtype, device) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise invalid(where, f"{name} is not a contiguous vector of {n}")
    if t.dtype != dtype or t.device != device:
        raise invalid(where, f"{name} is {t.dtype} on {t.device}, not {dtype} on {device}")


def _run(entry: str, args, device, on, work) -> None:
    L = _lib.load()
    need = ctypes.c_size_t()
    _lib.check(getattr(L, entry + "_worksize")(args, need), entry + "_worksize")
    if work is None:
        work = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
    ptr, size = (work.data_ptr(), work.numel() * work.element_size()) if work is not None else (None, 0)
    _lib.check(getattr(L, entry)(on.handle, args, ptr, size), entry)


def forward(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
            act: str = "none", save: str = "none", out: torch.Tensor | None = None, z=None, work=None, stream=None):
    """Y = act(x w^T + bias) + residual.

    save="z" returns (Y, Z) with the pre-activation Z in x's type, save="z8" (Y, checkpoint of Z).  out and z may
    give the memory for Y and for what is saved; out may be residual itself.  work: a uint8 CUDA tensor to use as
    workspace instead of allocating one.
    """
    where = "linear.forward"
    code, act_code = _type(where, x), _act(where, act)
    dt, dev = x.dtype, x.device
    ldx = matrix(where, "x", x)
    ldw = matrix(where, "w", w, dt, None, dev)
    tokens, k = x.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise invalid(where, f"x has {k} features and w {w.shape[1]}")
    if save not in ("none", "z", "z8"):
        raise invalid(where, f"save {save!r} is none of none, z, z8")
    if bias is not None:
        _vector(where, "bias", bias, n, dt, dev)
    ldr = matrix(where, "residual", residual, dt, (tokens, n), dev) if residual is not None else 0
    with on_stream(dev, stream) as on:
        if out is None:
            out = torch.empty(tokens, n, dtype=dt, device=dev)
        ldy = matrix(where, "out", out, dt, (tokens, n), dev)
        ldz, z8 = 0, _NONE
        if save == "z":
            z = torch.empty(tokens, n, dtype=dt, device=dev) if z is None else z
            ldz = matrix(where, "z", z, dt, (tokens, n), dev)
        elif save == "z8":
            z = empty(tokens, n, dt, dev) if z is None else z
            z8 = struct_of(where, "z", z, (tokens, n), dev)
        a = _lib.LinearFwd(code, act_code, tokens, n, k, x.data_ptr(), ldx, w.data_ptr(), ldw,
                           bias.data_ptr() if bias is not None else None,
                           residual.data_ptr() if residual is not None else None, ldr, out.data_ptr(), ldy,
                           z.data_ptr() if save == "z" else None, ldz, z8)
        _run("chpl_linear_forward", a, dev, on, work)
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
    code, act_code, in_code = _type(where, dy), _act(where, act), _act(where, in_act)
    dt, dev = dy.dtype, dy.device
    lddy = matrix(where, "dy", dy)
    ldw = matrix(where, "w", w, dt, None, dev)
    tokens, n = dy.shape
    k = w.shape[1]
    if w.shape[0] != n:
        raise invalid(where, f"dy has {n} features and w {w.shape[0]} rows")
    gt = grad_dtype or (dw.dtype if dw is not None else db.dtype if db is not None else dt)
    if gt != dt and gt != torch.float32:
        raise invalid(where, f"gradients in {gt}: {dt} or float32 is wanted")
    if accumulate and ((need_dw and dw is None) or (need_db and db is None)):
        raise invalid(where, "accumulate wants dw and db to add to")

    def saved(name, v, width):
        if v is None:
            return None, 0, _NONE
        if isinstance(v, Ckpt8):
            return None, 0, struct_of(where, name, v, (tokens, width), dev)
        return v.data_ptr(), matrix(where, name, v, dt, (tokens, width), dev), _NONE

    xp, ldx, x8 = saved("x", x, k)
    zp, ldz, z8 = saved("z", z, n) if act != "none" else (None, 0, _NONE)
    ldadd = matrix(where, "add", add, dt, (tokens, k), dev) if add is not None else 0
    with on_stream(dev, stream) as on:
        lddx = lddw = 0
        if need_dx:
            dx = torch.empty(tokens, k, dtype=dt, device=dev) if dx is None else dx
            lddx = matrix(where, "dx", dx, dt, (tokens, k), dev)
        if need_dw:
            dw = torch.empty(n, k, dtype=gt, device=dev) if dw is None else dw
            lddw = matrix(where, "dw", dw, gt, (n, k), dev)
        if need_db:
            db = torch.empty(n, dtype=gt, device=dev) if db is None else db
            _vector(where, "db", db, n, gt, dev)
        a = _lib.LinearBwd(code, act_code, in_code, _lib.CHPL_TYPE_F32 if gt == torch.float32 else code, int(accumulate),
                           tokens, n, k, dy.data_ptr(), lddy, w.data_ptr(), ldw, xp, ldx, x8, zp, ldz, z8,
                           add.data_ptr() if add is not None else None, ldadd, dx.data_ptr() if need_dx else None,
                           lddx, dw.data_ptr() if need_dw else None, lddw, db.data_ptr() if need_db else None)
        _run("chpl_linear_backward", a, dev, on, work)
    return dx if need_dx else None, dw if need_dw else None, db if need_db else None
