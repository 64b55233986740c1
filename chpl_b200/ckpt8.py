"""8-bit activation checkpoints: what a training step holds between its forward and its backward pass.

A checkpoint codes a matrix (rows x cols, BF16, F16 or FP32) in 8 bits per element plus one byte per 32: the
consecutive features 32g..32g+31 of a row share a power-of-two step, and each is stored as a signed code of 7 bits
(the OCP Microscaling MXINT8 elements and scales; include/chpl.h has the exact rule).  ``linear.forward`` writes
one from its epilogue, ``linear.backward`` reads it in its products; ``pack`` and ``unpack`` convert whole tensors.
Everything runs in libchpl.so on the GPU; there is no host implementation here.
"""
from __future__ import annotations

import ctypes
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


def matrix(where: str, name: str, t, dtype=None, shape=None, device=None) -> int:
    """Checks a CUDA matrix with unit column stride; returns the distance between its rows."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise invalid(where, f"{name} is not a matrix")
    if not t.is_cuda or (device is not None and t.device != device):
        raise invalid(where, f"{name} is on {t.device}, not on {device or 'a GPU'}")
    if dtype is not None and t.dtype != dtype:
        raise invalid(where, f"{name} is {t.dtype}, not {dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise invalid(where, f"{name} is {tuple(t.shape)}, not {tuple(shape)}")
    rows, cols = t.shape
    ld, unit = t.stride()
    if unit != 1 and cols > 1:
        raise invalid(where, f"{name} has column stride {unit}: rows must be contiguous")
    if rows > 1 and ld < cols:  # an expanded or overlapping view
        raise invalid(where, f"{name} has row stride {ld} below its {cols} columns")
    return ld if rows > 1 else cols


def struct_of(where: str, name: str, c: Ckpt8, shape=None, device=None) -> _lib.Ckpt8:
    ldc = matrix(where, f"{name}.codes", c.codes, torch.int8, shape, device)
    rows, cols = c.codes.shape
    lds = matrix(where, f"{name}.scales", c.scales, torch.uint8, (rows, -(-cols // GROUP)), c.codes.device)
    return _lib.Ckpt8(c.codes.data_ptr(), c.scales.data_ptr(), ldc, lds)


def empty(rows: int, cols: int, dtype: torch.dtype, device) -> Ckpt8:
    return Ckpt8(torch.empty(rows, cols, dtype=torch.int8, device=device),
                 torch.empty(rows, -(-cols // GROUP), dtype=torch.uint8, device=device), dtype)


class on_stream:
    """The device of `device` and, where one is given, `stream`: outputs and workspaces come from that stream's
    memory.  `self.handle` is the stream's handle."""

    def __init__(self, device: torch.device, stream):
        self.handle = None
        self._stack = []
        if device.index != torch.cuda.current_device():
            self._stack.append(torch.cuda.device(device))
        if stream is not None:
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream, device=device)
            self._stack.append(torch.cuda.stream(stream))
        self._device = device

    def __enter__(self):
        for c in self._stack:
            c.__enter__()
        self.handle = torch.cuda.current_stream(self._device).cuda_stream
        return self

    def __exit__(self, *exc):
        for c in reversed(self._stack):
            c.__exit__(*exc)


def pack(x: torch.Tensor, out: Ckpt8 | None = None, stream=None) -> Ckpt8:
    """The checkpoint of x (rows x cols), on torch's current stream or on `stream`."""
    where = "ckpt8.pack"
    ldx = matrix(where, "x", x)
    if x.dtype not in _TYPES:
        raise invalid(where, f"x is {x.dtype}: bfloat16, float16 or float32 is wanted")
    rows, cols = x.shape
    with on_stream(x.device, stream) as on:
        if out is None:
            out = empty(rows, cols, x.dtype, x.device)
        c = struct_of(where, "out", out, x.shape, x.device)
        _lib.check(_lib.load().chpl_ckpt8_pack(on.handle, _TYPES[x.dtype], rows, cols, x.data_ptr(), ldx,
                                               ctypes.byref(c)), "chpl_ckpt8_pack")
    return out


def unpack(c: Ckpt8, dtype: torch.dtype | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The values that a checkpoint stands for, in `dtype` (default: the type of what was coded)."""
    where = "ckpt8.unpack"
    s = struct_of(where, "c", c)
    dtype = out.dtype if out is not None else dtype or c.dtype
    if dtype not in _TYPES:
        raise invalid(where, f"{dtype}: bfloat16, float16 or float32 is wanted")
    rows, cols = c.codes.shape
    with on_stream(c.codes.device, stream) as on:
        if out is None:
            out = torch.empty(rows, cols, dtype=dtype, device=c.codes.device)
        ldx = matrix(where, "out", out, dtype, c.codes.shape, c.codes.device)
        _lib.check(_lib.load().chpl_ckpt8_unpack(on.handle, _TYPES[dtype], rows, cols, ctypes.byref(s),
                                                 out.data_ptr(), ldx), "chpl_ckpt8_unpack")
    return out
