"""Builds kore_b200/libkore_cuda.so (the C-ABI library) with nvcc for sm_100a.

Usage: ``python -m kore_b200.build [--force] [--verbose] [--trace]``; also
kore_b200/_tensors.*.so, with which the Python operators describe torch tensors
(without it they do so themselves). The library is built in-tree so that it travels with the repository to the GPU
machine. ``--trace`` builds kore_b200/libkore_cuda_trace.so instead: the same
library compiled with KORE_TRACE, whose decode and merge CTAs record
%globaltimer stamps (read by ``python -m kore_b200.trace_decode``).
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB = os.path.join(PKG, "libkore_cuda.so")
# the Python module that describes torch tensors for the library, named for the Python that it is compiled for
TENSORS = os.path.join(PKG, "_tensors" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
TRACE_LIB = os.path.join(PKG, "libkore_cuda_trace.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC,-O2",
              "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _stale(lib: str = LIB) -> bool:
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False, trace: bool = False, out: str | None = None,
          defines: tuple[str, ...] = ()) -> str:
    """Compiles every .cu under csrc/ into one shared library; returns its path.
    `out` and `defines` (NAME=VALUE, e.g. KORE_ROWS_WARPS=12) build a variant
    with other compile-time shapes elsewhere (loaded through $KORE_CUDA_LIB)."""
    lib = out or (TRACE_LIB if trace else LIB)
    if not force and not out and not _stale(lib):
        return lib
    objdir = os.path.join(os.path.dirname(lib), "_build_" + os.path.basename(lib)) if out else \
        os.path.join(PKG, "_build_trace" if trace else "_build")
    os.makedirs(objdir, exist_ok=True)
    objs = []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-3] + ".o")
        cmd = [nvcc(), *ARCH, *NVCC_FLAGS, *(["-DKORE_TRACE"] if trace else []), *("-D" + d for d in defines),
               "-I", INCLUDE, "-c", src, "-o", obj]
        if verbose:
            cmd += ["-Xptxas", "-v"]
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        objs.append(obj)
    tmp = lib + ".tmp"
    subprocess.run([nvcc(), *ARCH, "-shared", "-o", tmp, *objs, "-lcudart_static", "-lrt", "-ldl", "-lpthread"],
                   check=True)
    os.replace(tmp, lib)
    return lib


def _tensors_stale(deps: list[str], version: str) -> bool:
    if not os.path.exists(TENSORS) or any(os.path.getmtime(d) > os.path.getmtime(TENSORS) for d in deps):
        return True
    # another torch may be older than the module: the module holds the version it was compiled against
    with open(TENSORS, "rb") as f:
        return version.encode() + b"\0" not in f.read()


def build_tensors(force: bool = False) -> str | None:
    """Compiles csrc/tensors.cpp against the torch and for the Python that are installed; returns the module's path. None,
    and no module, where it cannot be: without torch there are no tensors to describe, and without a C++ compiler or
    Python's headers kore_b200/paged.py describes them itself, in some microseconds more a call."""
    try:
        import torch
    except (ImportError, OSError):
        return None
    untagged = os.path.join(PKG, "_tensors.so")   # (every Python would import one of this name)
    if untagged != TENSORS and os.path.exists(untagged):
        os.remove(untagged)
    src = os.path.join(CSRC, "tensors.cpp")
    version = torch.__version__.split("+")[0]
    if not force and not _tensors_stale([src, os.path.join(INCLUDE, "kore_cuda.h"), torch.__file__], version):
        return TENSORS
    home = os.path.dirname(torch.__file__)
    cxx = os.environ.get("CXX") or shutil.which("g++") or "c++"
    tmp = TENSORS + ".tmp"
    try:
        subprocess.run([cxx, "-O2", "-std=c++17", "-fPIC", "-shared",
                        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
                        "-I", INCLUDE, "-I", sysconfig.get_paths()["include"], "-isystem", os.path.join(home, "include"),
                        "-isystem", os.path.join(home, "include", "torch", "csrc", "api", "include"),
                        src, "-o", tmp, "-L", os.path.join(home, "lib"), "-lc10", "-ltorch_cpu", "-ltorch_python"], check=True)
    except (OSError, subprocess.CalledProcessError) as e:
        for f in (tmp, TENSORS):   # (what is there is not of these sources)
            if os.path.exists(f):
                os.remove(f)
        print(f"{os.path.basename(TENSORS)} is not built, tensors are described in Python: {e}", file=sys.stderr)
        return None
    os.replace(tmp, TENSORS)
    return TENSORS


if __name__ == "__main__":
    import argparse
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--trace", action="store_true")
    ap.add_argument("--out", default=None, help="build a variant library at this path")
    ap.add_argument("-D", dest="defines", action="append", default=[], help="NAME=VALUE for a variant build")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose, trace=a.trace, out=a.out, defines=tuple(a.defines)))
    if not a.trace and not a.out:
        print(build_tensors(force=a.force))
