"""Linear layers served from 4-bit weights: microscaled 4-bit floating point (OCP MXFP4) and products on the 4-bit tensor cores.

    w4 = mx4.pack(w)                                   # once; 0.53 bytes a weight
    y = mx4.linear(x, w4, bias, residual=r, act="gelu")

A matrix in this format holds E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, and one power-of-two
step for each 32 consecutive features of a row; include/chpl.h has the exact rule and where codes and scales lie.  ``linear``
codes x the same way on its way into the product, whose sums are FP32.  ``ffn.forward`` takes such weights too.  Calls follow
linear's rules: torch's current stream or `stream`, outputs allocated from it, ChplError; a wait inside a kernel that runs
out is reported by chpl_b200.check_device().  Autograd does not see these functions.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .ckpt8 import on
from .linear import ACTS, _choice

_ops = _lib.torch_ops()
GROUP = 32


class Mx4(NamedTuple):
    """codes: uint8 rows x 16 ceil(cols / 32) (rows may lie apart, on 16-byte boundaries); scales: uint8, in the tensor cores'
    order; cols: features of a row; dtype: the type of what was coded."""
    codes: torch.Tensor
    scales: torch.Tensor
    cols: int
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.codes.shape[0], self.cols))

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def pack(x: torch.Tensor, out: Mx4 | None = None, stream=None) -> Mx4:
    """x (rows x cols, BF16, F16 or FP32) in 4 bits, on torch's current stream or on `stream`.  out gives the memory; what is
    returned is in it and of x's type, out itself where that is its type already."""
    if stream is not None:
        with on(stream, x.device):
            return pack(x, out)
    if out is not None:
        if out.shape != x.shape:
            raise _lib.ChplError(_lib.CHPL_ERR_INVALID, "mx4.pack", f"out is {tuple(out.shape)}, x {tuple(x.shape)}")
        _ops.mx4_pack(x, out.codes, out.scales)
        return out if out.dtype is x.dtype else out._replace(dtype=x.dtype)
    return Mx4(*_ops.mx4_pack(x, None, None), x.shape[1], x.dtype)


def unpack(c: Mx4, dtype: torch.dtype | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The values that codes and scales stand for, in `dtype` (default: the type of what was coded)."""
    if stream is not None:
        with on(stream, c.codes.device):
            return unpack(c, dtype, out)
    return _ops.mx4_unpack(c.codes, c.scales, c.cols, out.dtype if out is not None else dtype or c.dtype, out)


def linear(x, w: Mx4, bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None, act: str = "none",
           out: torch.Tensor | None = None, work=None, stream=None) -> torch.Tensor:
    """act(Q(x) w^T + bias) + residual, of x's type.  x: tokens x k in BF16 or F16, coded by this call, or an Mx4 of such a
    tensor.  out may give the memory for the result and may be residual itself; work: a uint8 CUDA tensor to use as
    workspace instead of allocating one."""
    if not isinstance(w, Mx4):
        raise _lib.ChplError(_lib.CHPL_ERR_INVALID, "mx4.linear", "w is not an Mx4")
    if stream is not None:
        with on(stream, w.codes.device):
            return linear(x, w, bias, residual=residual, act=act, out=out, work=work)
    code = _choice("mx4.linear", "activation", ACTS, act)
    if isinstance(x, Mx4):
        return _ops.mx4_linear(None, x.codes, x.scales, x.cols, x.dtype, w.codes, w.scales, w.cols, bias, residual, code, out, work)
    return _ops.mx4_linear(x, None, None, None, None, w.codes, w.scales, w.cols, bias, residual, code, out, work)
