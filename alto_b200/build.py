"""Builds ``libaltob200.so`` (the C-ABI CUDA library) in-tree with nvcc for sm_100a, and ``_autograd.so`` (autograd functions
around some of its entry points, compiled against the installed torch) with the C++ compiler.

Run as ``python -m alto_b200.build``.  The shared objects land next to this file so that
``alto_b200._lib`` finds them without any installation step.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libaltob200.so"
AUTOGRAD_PATH = PKG_DIR / "_autograd.so"
HEADER = PKG_DIR.parent / "include" / "altob200.h"
SOURCES = ["quant.cu", "macro_scale.cu", "rht_dense.cu", "rows.cu", "swiglu.cu", "norm.cu", "route.cu", "dge.cu", "deosc.cu",
           "gemm_sm100.cu", "linear.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--shared", "--cudart", "static",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or add it to PATH")
    return cand


def needs_build() -> bool:
    if not LIB_PATH.exists():
        return True
    t = LIB_PATH.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + [HEADER]
    return any(p.stat().st_mtime > t for p in deps)


def build_autograd(force: bool = False) -> Path:
    """Compile ``csrc/autograd.cpp`` against the torch that this interpreter imports; returns the module's path."""
    src = CSRC / "autograd.cpp"
    if not force and AUTOGRAD_PATH.exists() and AUTOGRAD_PATH.stat().st_mtime >= max(src.stat().st_mtime, HEADER.stat().st_mtime):
        return AUTOGRAD_PATH
    import torch
    at = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    includes = [HEADER.parent, at / "include", at / "include" / "torch" / "csrc" / "api" / "include", sysconfig.get_paths()["include"],
                cuda / "include"]
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(a for i in includes for a in ("-I", str(i))),
           "-o", str(AUTOGRAD_PATH), str(src), "-L", str(at / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("the C++ compiler failed building _autograd.so")
    return AUTOGRAD_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every CUDA source into one shared library, and the autograd functions; returns the library's path."""
    build_autograd(force)
    if not force and not needs_build():
        return LIB_PATH
    srcs = [str(CSRC / s) for s in SOURCES if (CSRC / s).exists()]
    cmd = [_nvcc(), *NVCC_FLAGS, "-I", str(HEADER.parent), "-o", str(LIB_PATH), *srcs]
    if verbose:
        cmd.insert(1, "-Xptxas")
        cmd.insert(2, "-v")
        print(" ".join(cmd))
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building libaltob200.so")
    if verbose:
        print(res.stderr)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
