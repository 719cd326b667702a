"""The native call path (qlin/_native.so, csrc/qlin_torch.cpp), bound to the loaded library.

Its functions take the calls that need no copy, no conversion and no change of device, and return None for every
other one, which the Python functions of the same names then handle.  There is no fallback for a module that is
missing: it is built with the library.
"""
import ctypes

import torch  # noqa: F401  (the module links against its libraries)

from ._lib import check, lib

try:
    from . import _native as native
except ImportError as e:
    raise ImportError(f"qlin/_native.so: {e}; build it with `python mac-kernels-public_b200/build.py`") from e

native.bind(check, *(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in (
    "qlin_fp8_linear", "qlin_fp8_linear_workspace", "qlin_fp8_linear_grad_input",
    "qlin_fp8_linear_grad_input_workspace", "qlin_rotary_table", "qlin_qk_norm_rotary", "qlin_qk_norm_rotary_backward",
    "qlin_qk_norm_rotary_backward_workspace")))
