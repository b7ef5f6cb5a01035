"""Build the in-tree C-ABI library ``hsd_b200/libhsd_b200.so`` for sm_100a.

    python -m hsd_b200.build [--verbose]

Compiles every ``hsd_b200/csrc/*.cu`` with nvcc
(``-gencode arch=compute_100a,code=sm_100a -lineinfo -O3``) and links them
into one shared library with the CUDA runtime linked statically, so the
library loads next to PyTorch's own runtime without version coupling.  Then
compiles ``csrc/ops.cpp``, the Python binding of the entry points whose calls
have to be cheap on the host (``hsd_b200/_ops.so``; it links PyTorch and the
library).  The build is incremental: nothing is recompiled when the outputs
are newer than every source and header, and the binding was built for the
PyTorch and the interpreter that run this.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig

from ._native import ops_target

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(PKG, "libhsd_b200.so")
OPS = os.path.join(PKG, "_ops.so")
OPS_STAMP = os.path.join(PKG, "_build", "ops_built_for.txt")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path():
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(cand):
        raise RuntimeError("nvcc not found; the hsd_b200 library needs CUDA 12.8+")
    return cand


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps():
    return sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        glob.glob(os.path.join(INCLUDE, "*.h"))


def _newer(out, deps):
    if not os.path.exists(out):
        return False
    t = os.path.getmtime(out)
    return all(os.path.getmtime(p) <= t for p in deps)


def up_to_date():
    return _newer(LIB, _deps()) and _ops_up_to_date()


def _ops_up_to_date():
    """The binding is newer than its sources and built for this PyTorch and
    interpreter (a stamp beside the object files says for which)."""
    if not _newer(OPS, _ops_deps()) or not os.path.exists(OPS_STAMP):
        return False
    with open(OPS_STAMP) as f:
        return f.read() == ops_target()


def _ops_deps():
    return [os.path.join(CSRC, "ops.cpp")] + glob.glob(os.path.join(INCLUDE, "*.h"))


def _ops_command(out):
    """The host compiler's command for the Python binding; its symbols of the
    library resolve in ``libhsd_b200.so`` beside it, PyTorch's in the libraries
    that ``import torch`` has loaded."""
    import torch
    cxx = os.environ.get("CXX") or shutil.which("g++")
    if not cxx:
        raise RuntimeError("g++ not found; the Python binding needs a host compiler")
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc_path())), "include")
    home = os.path.dirname(torch.__file__)
    inc = [INCLUDE, cuda, sysconfig.get_paths()["include"], os.path.join(home, "include"),
           os.path.join(home, "include", "torch", "csrc", "api", "include")]
    lib = os.path.join(home, "lib")
    return [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            f'-DHSD_BUILT_FOR="{ops_target()}"',
            os.path.join(CSRC, "ops.cpp"), "-o", out] + ["-I" + d for d in inc] + \
        ["-L" + PKG, "-l:libhsd_b200.so", "-Wl,-rpath,$ORIGIN", "-L" + lib, "-ltorch_python",
         "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda"]


def build(verbose=False, force=False, jobs=None):
    if force or not _newer(LIB, _deps()):
        _build_library(verbose)
    if force or not _ops_up_to_date():
        tmp = OPS + ".tmp"
        r = subprocess.run(_ops_command(tmp), stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                           text=True)
        if verbose or r.returncode:
            sys.stderr.write(r.stdout)
        if r.returncode:
            raise RuntimeError("the Python binding (csrc/ops.cpp) failed to build")
        os.replace(tmp, OPS)
        os.makedirs(os.path.dirname(OPS_STAMP), exist_ok=True)
        with open(OPS_STAMP, "w") as f:
            f.write(ops_target())
    return LIB


def _build_library(verbose):
    nvcc = nvcc_path()
    objdir = os.path.join(PKG, "_build")
    os.makedirs(objdir, exist_ok=True)
    flags = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
                    "-I", INCLUDE, "-I", CSRC, "--expt-relaxed-constexpr"]
    if verbose:
        flags += ["-Xptxas", "-v"]
    objs = []
    procs = []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        objs.append(obj)
        cmd = [nvcc, "-c", src, "-o", obj] + flags
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE,
                                            stderr=subprocess.STDOUT, text=True)))
    failed = False
    for cmd, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode:
            sys.stderr.write(out)
        if p.returncode:
            failed = True
            sys.stderr.write("FAILED: " + " ".join(cmd) + "\n")
    if failed:
        raise RuntimeError("nvcc failed building hsd_b200")
    tmp = LIB + ".tmp"
    link = [nvcc, "-shared", "-o", tmp] + objs + ARCH + ["-cudart", "static"]
    r = subprocess.run(link, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode:
        sys.stderr.write(r.stdout)
        raise RuntimeError("nvcc link failed building hsd_b200")
    os.replace(tmp, LIB)


if __name__ == "__main__":
    build(verbose="--verbose" in sys.argv, force="--force" in sys.argv)
    print(LIB)
