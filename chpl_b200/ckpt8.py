"""8-bit activation checkpoints: what a training step holds between its forward and its backward pass.

A checkpoint codes a matrix (rows x cols, BF16, F16 or FP32) in 8 bits per element plus one byte per 32: the
consecutive features 32g..32g+31 of a row share a power-of-two step, and each is stored as a signed code of 7 bits
(the OCP Microscaling MXINT8 elements and scales; include/chpl.h has the exact rule).  ``linear.forward`` writes
one from its epilogue, ``linear.backward`` reads it in its products; ``pack`` and ``unpack`` convert whole tensors.
Everything runs in libchpl.so on the GPU; there is no host implementation here.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

GROUP = 32
_TYPES = {torch.bfloat16: _lib.CHPL_TYPE_BF16, torch.float16: _lib.CHPL_TYPE_F16, torch.float32: _lib.CHPL_TYPE_F32}


class Ckpt8(NamedTuple):
    """codes: int8 rows x cols; scales: uint8 rows x ceil(cols / 32); dtype: the type of what was coded."""
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def invalid(where: str, msg: str) -> _lib.ChplError:
    return _lib.ChplError(_lib.CHPL_ERR_INVALID, where, msg)


def matrix(where: str, name: str, t, dtype, device: int, shape) -> int:
    """The distance between the rows of a CUDA matrix with unit column stride, of this type, device and shape; any may
    be None.  Raises ChplError for another."""
    try:
        if t.shape == shape and t.dtype is dtype and t.get_device() == device:  # what nearly every call passes
            ld, unit = t.stride()
            if unit == 1 and ld >= shape[1]:
                return ld
    except (AttributeError, TypeError, ValueError):
        pass
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise invalid(where, f"{name} is not a matrix")
    if not t.is_cuda or (device is not None and t.get_device() != device):
        raise invalid(where, f"{name} is on {t.device}, not on {'a GPU' if device is None else f'cuda:{device}'}")
    if dtype is not None and t.dtype != dtype:
        raise invalid(where, f"{name} is {t.dtype}, not {dtype}")
    if shape is not None and t.shape != shape:
        raise invalid(where, f"{name} is {tuple(t.shape)}, not {tuple(shape)}")
    rows, cols = t.shape
    ld, unit = t.stride()
    if unit != 1 and cols > 1:
        raise invalid(where, f"{name} has column stride {unit}: rows must be contiguous")
    if rows > 1 and ld < cols:  # an expanded or overlapping view
        raise invalid(where, f"{name} has row stride {ld} below its {cols} columns")
    return ld if rows > 1 else cols


def pointers(where: str, name: str, c: Ckpt8, device, shape) -> tuple[int, int, int, int]:
    """(codes, scales, ldc, lds) of a checkpoint, as chpl_ckpt8 has them."""
    ldc = matrix(where, name + ".codes", c.codes, torch.int8, device, shape)
    rows, cols = c.codes.shape
    lds = matrix(where, name + ".scales", c.scales, torch.uint8, c.codes.get_device(), (rows, -(-cols // GROUP)))
    return c.codes.data_ptr(), c.scales.data_ptr(), ldc, lds


def empty(rows: int, cols: int, dtype: torch.dtype, device) -> Ckpt8:
    return Ckpt8(torch.empty(rows, cols, dtype=torch.int8, device=device),
                 torch.empty(rows, -(-cols // GROUP), dtype=torch.uint8, device=device), dtype)


def elsewhere(device: int, stream) -> bool:
    """Whether a call has to change torch's current device or stream first."""
    return stream is not None or device != _current_device()


class on_stream:
    """Makes `device` and `stream` (a torch stream, a raw handle, or None for that device's current one) torch's
    current ones, so that outputs and workspaces come from that stream's memory."""

    def __init__(self, device: torch.device, stream):
        self._stack = [torch.cuda.device(device)]
        if stream is not None:
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream, device=device)
            self._stack.append(torch.cuda.stream(stream))

    def __enter__(self):
        for c in self._stack:
            c.__enter__()

    def __exit__(self, *exc):
        for c in reversed(self._stack):
            c.__exit__(*exc)


# torch's current device, and the handle of a device's current stream, without the checks and objects that the public
# calls put around them (2.5 us a call, a quarter of a one-token product's)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
current_handle = getattr(torch._C, "_cuda_getCurrentRawStream", lambda i: torch.cuda.current_stream(i).cuda_stream)


def pack(x: torch.Tensor, out: Ckpt8 | None = None, stream=None) -> Ckpt8:
    """The checkpoint of x (rows x cols), on torch's current stream or on `stream`."""
    where = "ckpt8.pack"
    ldx = matrix(where, "x", x, None, None, None)
    code = _TYPES.get(x.dtype)
    if code is None:
        raise invalid(where, f"x is {x.dtype}: bfloat16, float16 or float32 is wanted")
    dev = x.get_device()
    if elsewhere(dev, stream):
        with on_stream(x.device, stream):
            return pack(x, out)
    rows, cols = x.shape
    if out is None:
        out = empty(rows, cols, x.dtype, x.device)
        c = (out.codes.data_ptr(), out.scales.data_ptr(), cols, -(-cols // GROUP))
    else:
        c = pointers(where, "out", out, dev, x.shape)
    _lib.check(_lib.load().chpl_ckpt8_pack(current_handle(dev), code, rows, cols, x.data_ptr(), ldx,
                                           _lib.CKPT8.pack(*c)), "chpl_ckpt8_pack")
    return out


def unpack(c: Ckpt8, dtype: torch.dtype | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The values that a checkpoint stands for, in `dtype` (default: the type of what was coded)."""
    where = "ckpt8.unpack"
    s = pointers(where, "c", c, None, None)
    dtype = out.dtype if out is not None else dtype or c.dtype
    code = _TYPES.get(dtype)
    if code is None:
        raise invalid(where, f"{dtype}: bfloat16, float16 or float32 is wanted")
    dev = c.codes.get_device()
    if elsewhere(dev, stream):
        with on_stream(c.codes.device, stream):
            return unpack(c, dtype, out)
    rows, cols = c.codes.shape
    if out is None:
        out, ldx = torch.empty(rows, cols, dtype=dtype, device=c.codes.device), cols
    else:
        ldx = matrix(where, "out", out, dtype, dev, c.codes.shape)
    _lib.check(_lib.load().chpl_ckpt8_unpack(current_handle(dev), code, rows, cols, _lib.CKPT8.pack(*s),
                                             out.data_ptr(), ldx), "chpl_ckpt8_unpack")
    return out
