"""Build libbonsai_khq_b200.so in-tree with nvcc for sm_100a, and with g++ the CPython extension through which ``paged.py`` calls it.

Run as ``python -m bonsai_mojo_1bit_optimization_t4_cuda_b200.build``.  nvcc cross-compiles, so
no GPU is needed to build.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_NAME = "libbonsai_khq_b200.so"
LIB_PATH = PKG_DIR / LIB_NAME
HOST_PATH = PKG_DIR / "_khq_paged_host.so"
HOST_SOURCE = CSRC / "khq_paged_host.cpp"
SOURCES = ["khq_compress.cu", "khq_decode.cu", "khq_engine.cu", "khq_prefill.cu", "khq_prefill_tc5.cu", "khq_prestep.cu", "khq_calib.cu", "khq_paged.cu",
           "khq_paged_attn.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-shared", "-Xcompiler", "-fPIC",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: set NVCC or put it on PATH")


def needs_build() -> bool:
    if not LIB_PATH.exists():
        return True
    t = LIB_PATH.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + [PKG_DIR.parent / "include" / "khq_b200.h"]
    return any(p.stat().st_mtime > t for p in deps if p.exists())


def needs_host_build() -> bool:
    deps = [HOST_SOURCE, PKG_DIR.parent / "include" / "khq_b200.h"]
    return not HOST_PATH.exists() or any(p.stat().st_mtime > HOST_PATH.stat().st_mtime for p in deps)


def build_host(force: bool = False) -> Path:
    """The extension: torch's and Python's headers, no CUDA code."""
    if not force and not needs_host_build():
        return HOST_PATH
    import sysconfig

    import torch

    torch_dir = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent / "include"
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", str(PKG_DIR.parent / "include"), "-I", str(torch_dir / "include"), "-I", str(torch_dir / "include" / "torch" / "csrc" / "api" / "include"),
           "-I", sysconfig.get_paths()["include"], "-I", str(cuda), str(HOST_SOURCE), "-o", str(HOST_PATH), "-L", str(torch_dir / "lib"),
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed building " + HOST_PATH.name)
    return HOST_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every CUDA source into one shared library next to this file, and the extension."""
    build_host(force)
    if not force and not needs_build():
        return LIB_PATH
    cmd = [_nvcc(), *NVCC_FLAGS, "-I", str(PKG_DIR.parent / "include")]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    cmd += ["-o", str(LIB_PATH)] + [str(CSRC / s) for s in SOURCES]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("nvcc failed building " + LIB_NAME)
    if verbose:
        sys.stderr.write(res.stderr)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
