"""8-bit activation checkpoints: what a training step holds between its forward and its backward pass.

A checkpoint codes a matrix (rows x cols, BF16, F16 or FP32) in 8 bits per element plus one byte per 32: the
consecutive features 32g..32g+31 of a row share a power-of-two step, and each is stored as a signed code of 7 bits
(the OCP Microscaling MXINT8 elements and scales; include/chpl.h has the exact rule).  ``linear.forward`` writes
one from its epilogue, ``linear.backward`` reads it in its products; ``pack`` and ``unpack`` convert whole tensors.
Everything runs in libchpl.so on the GPU; there is no host implementation here.  Autograd does not see these functions:
a gradient does not pass a checkpoint.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

_ops = _lib.torch_ops()
GROUP = 32


class Ckpt8(NamedTuple):
    """codes: int8 rows x cols (rows may lie apart: new ones start every 16 bytes); scales: uint8 rows x ceil(cols / 32);
    dtype: the type of what was coded."""
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def empty(rows: int, cols: int, dtype: torch.dtype, device) -> Ckpt8:
    """Memory for the checkpoint of a rows x cols matrix."""
    return Ckpt8(torch.empty(rows, -(-cols // 16) * 16, dtype=torch.int8, device=device)[:, :cols],
                 torch.empty(rows, -(-cols // GROUP), dtype=torch.uint8, device=device), dtype)


def on(stream, device: torch.device):
    """The context in which `stream` (a torch stream, or a raw handle) is torch's current one, so that outputs and
    workspaces come from that stream's memory."""
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream)


def pack(x: torch.Tensor, out: Ckpt8 | None = None, stream=None) -> Ckpt8:
    """The checkpoint of x (rows x cols), on torch's current stream or on `stream`."""
    if stream is not None:
        with on(stream, x.device):
            return pack(x, out)
    if out is not None:
        _ops.ckpt8_pack(x, out.codes, out.scales)
        return out
    return Ckpt8(*_ops.ckpt8_pack(x, None, None), x.dtype)


def unpack(c: Ckpt8, dtype: torch.dtype | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The values that a checkpoint stands for, in `dtype` (default: the type of what was coded)."""
    if stream is not None:
        with on(stream, c.codes.device):
            return unpack(c, dtype, out)
    return _ops.ckpt8_unpack(c.codes, c.scales, out.dtype if out is not None else dtype or c.dtype, out)
