"""Kernels that are launched dependent on the work before them are resident while that work still writes their inputs.
The read-only load path is defined only for memory that stays unchanged while a kernel lives, so no source that such a
kernel is made of may use it, or let the compiler choose it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mac-kernels-public_b200", "csrc")


def _code(name):
    """The file without its comments."""
    src = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", src, flags=re.S)


def _with_includes(name, seen):
    if name not in seen and os.path.exists(os.path.join(CSRC, name)):
        seen.add(name)
        for inc in re.findall(r'#include "([^"/]+)"', _code(name)):
            _with_includes(inc, seen)
    return seen


def test_dependent_kernels_use_no_read_only_loads():
    units = [f for f in os.listdir(CSRC) if f.endswith(".cu")]
    dependent = [u for u in units if any("griddep_wait();" in _code(f) for f in _with_includes(u, set()) - {"qlin_ptx.cuh"})]
    assert {"qlin_fp8.cu", "qlin_rotary.cu"} <= set(dependent)
    found = []
    for unit in dependent:
        for f in sorted(_with_includes(unit, set())):
            for word in ("__ldg", "ld.global.nc", "__restrict__"):
                if word in _code(f):
                    found.append((f, word))
    assert not found, found
