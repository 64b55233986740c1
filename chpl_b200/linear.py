"""Linear layers of a model on libchpl's tensor-core products.

``forward``:  Y = act(X W^T + b) + R, with the pre-activation kept in 16 bits or as an 8-bit checkpoint.
``backward``: dX, dW and db of such a layer, from 16-bit tensors or from checkpoints.

X is tokens x k, W is n x k, Y is tokens x n: CUDA tensors of BF16 or F16 whose rows are contiguous; rows may lie
any distance apart (include/chpl.h has the rules, and which copies unaligned rows cost).  Calls are asynchronous on torch's
current stream, or on `stream`, on which the inputs have to be ready; outputs that are not given and the workspace are
allocated from that stream's memory.  Errors raise ChplError; a wait inside a kernel that runs out is reported by
chpl_b200.check_device(), which waits for the GPU (these calls do not).  Everything runs in libchpl.so on the GPU; there is no
host implementation here.

Autograd does not see these functions: what they return carries no graph and no tangents, whatever the inputs require.
A program calls ``backward`` for the gradients, or uses ``ffn.block``.
"""
from __future__ import annotations

import torch

from . import _lib
from .ckpt8 import Ckpt8, on

_ops = _lib.torch_ops()
ACTS = {"none": _lib.CHPL_ACT_NONE, "relu": _lib.CHPL_ACT_RELU, "gelu": _lib.CHPL_ACT_GELU,
        "gelu_tanh": _lib.CHPL_ACT_GELU_TANH, "silu": _lib.CHPL_ACT_SILU}
_SAVE = {"none": 0, "z": 1, "z8": 2}


def _choice(where: str, what: str, table: dict, name) -> int:
    code = table.get(name)
    if code is None:
        raise _lib.ChplError(_lib.CHPL_ERR_INVALID, where, f"{what} {name!r} is none of {', '.join(table)}")
    return code


def forward(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
            act: str = "none", save: str = "none", out: torch.Tensor | None = None, z=None, work=None, stream=None):
    """Y = act(x w^T + bias) + residual.

    save="z" returns (Y, Z) with the pre-activation Z in x's type, save="z8" (Y, checkpoint of Z).  out and z may
    give the memory for Y and for what is saved; out may be residual itself.  work: a uint8 CUDA tensor to use as
    workspace instead of allocating one.
    """
    if stream is not None:
        with on(stream, x.device):
            return forward(x, w, bias, residual=residual, act=act, save=save, out=out, z=z, work=work)
    code, how = _choice("linear.forward", "activation", ACTS, act), _choice("linear.forward", "save", _SAVE, save)
    if how == 2:
        codes, scales = (None, None) if z is None else (z.codes, z.scales)
        y, codes, scales = _ops.linear_forward(x, w, bias, residual, code, how, out, None, codes, scales, work)
        return y, Ckpt8(codes, scales, x.dtype) if z is None else z if z.dtype is x.dtype else z._replace(dtype=x.dtype)
    return _ops.linear_forward(x, w, bias, residual, code, how, out, z, None, None, work)


def backward(dy: torch.Tensor, x, w: torch.Tensor, *, act: str = "none", z=None, in_act: str = "none",
             add: torch.Tensor | None = None, need_dx: bool = True, need_dw: bool = True, need_db: bool = True,
             dx: torch.Tensor | None = None, dw: torch.Tensor | None = None, db: torch.Tensor | None = None,
             dx_sum=False, grad_dtype: torch.dtype | None = None, accumulate: bool = False, work=None, stream=None):
    """(dX, dW, db) of Y = act(X w^T + b) + R from dY; dR is dY itself.

    x is X, or with in_act the pre-activation that X = in_act(x) came from (dX is then x's gradient); z is the
    layer's own pre-activation, wanted where act is not none.  Either may be a tensor of dY's type or a Ckpt8.
    add is added to dX (the gradient that a skip connection brings); dx may be add itself.  need_*=False leaves an output
    out (None).  dx_sum=True returns a fourth, the sum of dX over the tokens (with in_act, the db of the layer that made
    x); a tensor gives the memory for it.  dW, db and that sum are of grad_dtype: dY's type, or torch.float32; accumulate
    adds them to the dw, db and dx_sum given.
    """
    if stream is not None:
        with on(stream, dy.device):
            return backward(dy, x, w, act=act, z=z, in_act=in_act, add=add, need_dx=need_dx, need_dw=need_dw, need_db=need_db,
                            dx=dx, dw=dw, db=db, dx_sum=dx_sum, grad_dtype=grad_dtype, accumulate=accumulate, work=work)
    where = "linear.backward"
    code, in_code = _choice(where, "activation", ACTS, act), _choice(where, "activation", ACTS, in_act)
    xc = xs = zc = zs = None
    if isinstance(x, Ckpt8):
        xc, xs, x = x.codes, x.scales, None
    if isinstance(z, Ckpt8):
        zc, zs, z = z.codes, z.scales, None
    gt = grad_dtype or (dw.dtype if dw is not None else db.dtype if db is not None else dy.dtype)
    if gt is not dy.dtype and gt is not torch.float32:
        raise _lib.ChplError(_lib.CHPL_ERR_INVALID, where, f"gradients in {gt}: {dy.dtype} or float32 is wanted")
    total = dx_sum if isinstance(dx_sum, torch.Tensor) else None
    if accumulate and ((need_dw and dw is None) or (need_db and db is None) or (dx_sum is True)):
        raise _lib.ChplError(_lib.CHPL_ERR_INVALID, where, "accumulate wants dw, db and dx_sum to add to")
    want_sum = dx_sum is True or total is not None
    out = _ops.linear_backward(dy, w, x, xc, xs, z, zc, zs, add, code, in_code, gt is torch.float32, accumulate, need_dx, need_dw,
                               need_db, want_sum, dx, dw, db, total, work)
    return out if want_sum else out[:3]
