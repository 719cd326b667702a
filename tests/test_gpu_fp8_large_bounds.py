"""The larger forms of the block-scaled linear once more on the bounds-checked build, as test_gpu_attention_input_bounds.py
runs the smaller ones."""
import os
import subprocess
import sys

import pytest

from test_gpu_attention_input_bounds import CHECKED, HERE, _Clean


@pytest.mark.gpu
def test_no_out_of_bounds_access():
    assert os.path.exists(CHECKED), "build it with: python mac-kernels-public_b200/build.py --checks"
    r = subprocess.run([sys.executable, os.path.abspath(__file__)], env=dict(os.environ, QLIN_LIB=CHECKED),
                       capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and "all clean" in r.stdout, r.stdout[-4000:] + r.stderr[-2000:]


def _child():
    code = pytest.main(["-q", "-x", "-m", "gpu", "-p", "no:cacheprovider", os.path.join(HERE, "test_gpu_fp8_large.py")],
                       plugins=[_Clean()])
    from qlin import _lib
    assert os.path.samefile(_lib.LIB_PATH, CHECKED), _lib.LIB_PATH
    if code == 0:
        print("all clean")
    return int(code)


if __name__ == "__main__":
    sys.path.insert(0, HERE)
    sys.exit(_child())
