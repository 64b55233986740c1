"""chpl_b200 -- a B200-native (sm_100a) HPL engine with the drop-in surface of
Koyingtw/CHPL: the Ozaki-II emulated trailing update (GEMMul8 interface), the
FP64 panel/pivoting path and the chpl_single / chpl_p2 solvers; and, beside them
on tensor-core kernels of their own, a model's linear layers with their gradients
and 8-bit activation checkpoints (linear, ckpt8, ffn).

All compute runs in the in-tree CUDA library libchpl.so (C ABI: include/chpl.h);
importing a submodule that needs it raises if the library is missing.
"""
from ._lib import ChplError, check_device, load  # noqa: F401

__all__ = ["ChplError", "check_device", "load", "oz2", "hpl", "linear", "ckpt8", "ffn"]
__version__ = "0.1"
