"""Build libbonsai_khq_b200.so in-tree with nvcc for sm_100a, and with g++ the CPython extension through which ``paged.py`` calls it.

The library needs neither torch nor Python; the extension is built for the torch and the Python that are there, which its file name says,
and where it cannot be built only ``paged.py`` is without it.

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


def host_path() -> Path:
    """The extension's file for the torch and the Python that are there (ImportError: no torch)."""
    from importlib import metadata
    import sysconfig

    try:
        torch_version = metadata.version("torch")
    except metadata.PackageNotFoundError as e:
        raise ImportError("torch is not installed") from e
    return PKG_DIR / f"_khq_paged_host-torch{torch_version}{sysconfig.get_config_var('EXT_SUFFIX')}"


def needs_host_build() -> bool:
    path, deps = host_path(), [HOST_SOURCE, PKG_DIR.parent / "include" / "khq_b200.h"]
    return not path.exists() or any(p.stat().st_mtime > path.stat().st_mtime for p in deps)


def build_host(force: bool = False) -> Path:
    """The extension: torch's and Python's headers, no CUDA code."""
    path = host_path()
    if not force and not needs_host_build():
        return path
    import sysconfig

    import torch

    torch_dir = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent / "include"
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", str(PKG_DIR.parent / "include"), "-I", str(torch_dir / "include"), "-I", str(torch_dir / "include" / "torch" / "csrc" / "api" / "include"),
           "-I", sysconfig.get_paths()["include"], "-I", str(cuda), str(HOST_SOURCE), "-o", str(path), "-L", str(torch_dir / "lib"),
           "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed building " + path.name)
    return path


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every CUDA source into one shared library next to this file, then the extension.  Where that one cannot be built the reason is
    printed; ``build_host`` raises."""
    if force or needs_build():
        _build_library(verbose)
    try:
        build_host(force)
    except (ImportError, OSError, RuntimeError) as e:
        sys.stderr.write(f"the paged operators' extension was not built ({type(e).__name__}: {e}); everything else works without it\n")
    return LIB_PATH


def _build_library(verbose: bool) -> None:
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


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
