"""The native call path (qlin/_native.so, csrc/qlin_torch.cpp), bound to the loaded library.

Its functions take the calls that need no copy, no conversion and no change of device, and return None for every
other one, which the Python functions of the same names then handle.  Where the module is missing, or was built for
another torch or Python, they handle every call: the same kernels, with more host time for each call, and one
warning at the first.
"""
import ctypes
import sysconfig
import warnings

import torch

from ._lib import check, lib

_BOUND = ("qlin_fp8_linear", "qlin_fp8_linear_workspace", "qlin_fp8_linear_grad_input",
          "qlin_fp8_linear_grad_input_workspace", "qlin_rotary_table", "qlin_qk_norm_rotary",
          "qlin_qk_norm_rotary_backward", "qlin_qk_norm_rotary_backward_workspace")


class _Missing:
    """In the place of the module: takes no call."""

    def __init__(self, why):
        self.why = why

    def _none(self, *_args):
        if self.why is not None:
            why, self.why = self.why, None
            warnings.warn(f"qlin/_native.so: {why}; these operators' calls take more host time until it is built again "
                          "with `python mac-kernels-public_b200/build.py`", RuntimeWarning, stacklevel=3)

    fp8_linear = fp8_linear_grad_input = rotary_table = qk_norm_rotary = qk_norm_rotary_backward = _none


def _load():
    try:
        from . import _native
    except ImportError as e:
        return _Missing(str(e))
    here = f"torch {torch.__version__}, {sysconfig.get_config_var('SOABI')}"
    if getattr(_native, "built_for", None) != here:
        return _Missing(f"built for {getattr(_native, 'built_for', 'an unknown torch')}, this is {here}")
    _native.bind(check, *(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _BOUND))
    return _native


native = _load()
