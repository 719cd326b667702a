"""Builds libqlin.so (sm_100a) in-tree: mac-kernels-public_b200/qlin/libqlin.so.

    python mac-kernels-public_b200/build.py [--jobs N] [--verbose] [--checks]

--checks builds the same library with -DQLIN_CHECKS (bounds checks on every plain global access
and computed shared-memory index, recorded and read back with qlin_bounds_check) as
qlin/libqlin_checked.so, from objects in _build/checks/; select it with QLIN_LIB.

qlin/_native.so, the call path of the small operators from torch tensors to the C ABI, is compiled from
csrc/qlin_torch.cpp against the installed torch (no device code; it does not link libqlin.so).  Without torch it is
left out.

Each csrc/*.cu is compiled with nvcc for `-gencode arch=compute_100a,code=sm_100a` into
_build/, then linked into one shared library with the CUDA runtime linked statically, so the
library does not depend on which libcudart the host process (PyTorch) loaded.
"""
import argparse
import concurrent.futures as cf
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "qlin", "libqlin.so")
OUT_CHECKED = os.path.join(HERE, "qlin", "libqlin_checked.so")
OUT_NATIVE = os.path.join(HERE, "qlin", "_native.so")
BUILD = os.path.join(HERE, "_build")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-Xptxas", "-v" if os.environ.get("QLIN_PTXAS_V") else "-O3"]


def nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def compile_one(src, verbose=False, checks=False):
    obj = os.path.join(BUILD, "checks" if checks else "", os.path.basename(src) + ".o")
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "qlin.h")]
    if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(d) for d in deps):
        return obj, ""
    cmd = [nvcc(), *ARCH, *FLAGS, *(["-DQLIN_CHECKS"] if checks else []), "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj, (r.stdout + r.stderr) if verbose else ""


def build_native():
    """qlin/_native.so: a CPython extension on torch's tensors.  Left out where there is no torch: the C library
    needs none."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        print("torch is not installed: qlin/_native.so is not built", file=sys.stderr)
        return None
    src = os.path.join(CSRC, "qlin_torch.cpp")
    torch_dir = list(spec.submodule_search_locations)[0]
    deps = [src, os.path.join(HERE, "..", "include", "qlin.h"), os.path.join(torch_dir, "version.py")]
    with open(os.path.join(torch_dir, "version.py")) as f:
        version = re.search(r"^__version__ = ['\"](.+)['\"]", f.read(), re.M).group(1)
    built_for = f"torch {version}, {sysconfig.get_config_var('SOABI')}"
    stamp = os.path.join(BUILD, "native_built_for")
    if os.path.exists(OUT_NATIVE) and os.path.getmtime(OUT_NATIVE) >= max(os.path.getmtime(d) for d in deps) and \
            os.path.exists(stamp) and open(stamp).read() == built_for:
        return OUT_NATIVE
    inc, libs = os.path.join(torch_dir, "include"), os.path.join(torch_dir, "lib")
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I" + inc,
           "-I" + os.path.join(inc, "torch", "csrc", "api", "include"), "-I" + cuda,
           "-I" + sysconfig.get_paths()["include"], f'-DQLIN_BUILT_FOR="{built_for}"', src, "-o", OUT_NATIVE, "-L" + libs, "-ltorch_python", "-ltorch_cpu",
           "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src}:\n{r.stdout}\n{r.stderr}")
    os.makedirs(BUILD, exist_ok=True)
    with open(stamp, "w") as f:
        f.write(built_for)
    return OUT_NATIVE


def build(jobs=None, verbose=False, checks=False):
    out = OUT_CHECKED if checks else OUT
    os.makedirs(os.path.join(BUILD, "checks") if checks else BUILD, exist_ok=True)
    srcs = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))
    with cf.ThreadPoolExecutor(max_workers=jobs or min(8, os.cpu_count() or 1)) as ex:
        results = list(ex.map(lambda s: compile_one(s, verbose, checks), srcs))
    objs = [o for o, _ in results]
    if verbose:
        for _, log in results:
            if log:
                print(log)
    newest = max(os.path.getmtime(o) for o in objs)
    if not os.path.exists(out) or os.path.getmtime(out) < newest:
        cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", out, *objs, "-lpthread", "-ldl", "-lrt"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    build_native()
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=None)
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--checks", action="store_true")
    a = ap.parse_args()
    try:
        print(build(a.jobs, a.verbose, a.checks))
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
