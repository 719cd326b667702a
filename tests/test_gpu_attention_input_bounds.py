"""The tests of the block-scaled 8-bit linear, the rotary tables and the head norm once more on the bounds-checked
build (libqlin_checked.so): after every one of them no check of a global access or a shared-memory index has failed.
The tests run in a child process that loads the checked library through QLIN_LIB."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CHECKED = os.path.join(os.path.dirname(HERE), "mac-kernels-public_b200", "qlin", "libqlin_checked.so")


@pytest.mark.gpu
def test_no_out_of_bounds_access():
    assert os.path.exists(CHECKED), "build it with: python mac-kernels-public_b200/build.py --checks"
    r = subprocess.run([sys.executable, os.path.abspath(__file__)], env=dict(os.environ, QLIN_LIB=CHECKED),
                       capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and "all clean" in r.stdout, r.stdout[-4000:] + r.stderr[-2000:]


class _Clean:
    @pytest.hookimpl(wrapper=True)
    def pytest_runtest_call(self, item):
        result = yield
        import qlin
        record = qlin.bounds_check()
        assert record is None, record
        return result


def _child():
    code = pytest.main(["-q", "-x", "-m", "gpu", "-p", "no:cacheprovider", os.path.join(HERE, "test_gpu_fp8.py"),
                        os.path.join(HERE, "test_gpu_rotary.py")], plugins=[_Clean()])
    from qlin import _lib
    assert os.path.samefile(_lib.LIB_PATH, CHECKED), _lib.LIB_PATH
    if code == 0:
        print("all clean")
    return int(code)


if __name__ == "__main__":
    sys.exit(_child())
