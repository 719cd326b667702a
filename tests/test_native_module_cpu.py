"""The package where the native call path's module is missing, was built for something else, or cannot be built."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "mac-kernels-public_b200")


@pytest.fixture
def package(tmp_path):
    """A copy of the Python package beside the library itself, without the module."""
    shutil.copytree(os.path.join(PKG, "qlin"), tmp_path / "qlin", ignore=shutil.ignore_patterns("*.so", "__pycache__"))
    return tmp_path


def _run(package, code):
    env = dict(os.environ, PYTHONPATH=str(package), QLIN_LIB=os.path.join(PKG, "qlin", "libqlin.so"))
    r = subprocess.run([sys.executable, "-c", code], env=env, cwd=package, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    return r.stdout


CALLS = """
import warnings, torch, qlin
assert qlin.__file__.startswith({where!r}), qlin.__file__
try:
    qlin.int8_linear(torch.zeros(2, 16), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4))
except NotImplementedError:
    print("int8 answers")
w = torch.zeros(64, 128).to(torch.float8_e4m3fn)
with warnings.catch_warnings(record=True) as told:
    warnings.simplefilter("always")
    for _ in range(2):
        for call in (lambda: qlin.fp8_linear(torch.zeros(2, 128), w, torch.ones(1, 1)),
                     lambda: qlin.rotary_table(torch.zeros(3, 1), [8])):
            try:
                call()
            except NotImplementedError:
                print("answers")
told = [str(t.message) for t in told if "_native" in str(t.message)]
assert len(told) == 1, told
print(told[0])
"""


def test_package_without_the_module(package):
    out = _run(package, CALLS.format(where=str(package)))
    assert "int8 answers" in out and out.count("answers") == 5 and "build.py" in out


def test_library_builds_without_torch(tmp_path, monkeypatch, capsys):
    """The C library needs no torch: the module is left out with a note where there is none."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("qlin_build", os.path.join(PKG, "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    real = importlib.util.find_spec
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else real(name, *a))
    monkeypatch.setattr(build, "OUT_NATIVE", str(tmp_path / "_native.so"))
    monkeypatch.setattr(build, "compile_one", lambda *a, **k: (build.OUT, ""))  # the objects are not what is tested
    assert build.build() == build.OUT
    assert not os.path.exists(build.OUT_NATIVE) and "torch" in capsys.readouterr().err


@pytest.mark.parametrize("line", ["", "built_for = 'torch 1.0.0, cpython-39-x86_64-linux-gnu'"])
def test_module_built_for_another_torch_is_not_used(package, line):
    """Structures of another torch's tensors would be read: the module is left alone."""
    calls = "".join(f"\ndef {f}(*a):\n    raise SystemError('called')\n" for f in ("bind", "fp8_linear", "rotary_table"))
    (package / "qlin" / "_native.py").write_text(line + "\n" + calls)
    out = _run(package, CALLS.format(where=str(package)))
    assert "int8 answers" in out and out.count("answers") == 5 and "this is torch" in out


def test_module_that_is_built_is_used():
    from qlin import _fast
    assert _fast.native.__name__ == "qlin._native", _fast.native.why
