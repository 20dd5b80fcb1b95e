"""Build libmi_paged.so (sm_100a) in-tree: ``python -m mini_infra_b200.build``.

One nvcc invocation over the unity translation unit ``csrc/libmi_paged.cu``; the shared object
lands in ``mini_infra_b200/_lib/`` so that it travels with the source tree.  Beside it ``_mi_calls.so``, a
CPython extension over that library (``csrc/torch_calls.cpp``, g++ against PyTorch's headers): the ordinary
calls of the 4-bit operators without the cost of ctypes.
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG.parent / "csrc"
LIB_DIR = PKG / "_lib"
LIB_PATH = LIB_DIR / "libmi_paged.so"
CALLS_PATH = LIB_DIR / "_mi_calls.so"
CALLS_SOURCE = CSRC / "torch_calls.cpp"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
]


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted((PKG.parent.parent / "include").glob("*.h"))


def needs_build() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    return any(p.stat().st_mtime > built for p in sources() if p.exists())


def build_calls(force: bool = False, verbose: bool = False) -> Path:
    """The CPython extension; needs libmi_paged.so."""
    inputs = [CALLS_SOURCE, *(PKG.parent.parent / "include").glob("*.h")]
    if not force and CALLS_PATH.exists() and CALLS_PATH.stat().st_mtime >= max(p.stat().st_mtime for p in inputs):
        return CALLS_PATH
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    tmp = CALLS_PATH.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{root}/include", f"-I{root}/include/torch/csrc/api/include", f"-I{sysconfig.get_paths()['include']}",
           f"-I{cuda}/include", f"-I{PKG.parent.parent / 'include'}", "-o", str(tmp), str(CALLS_SOURCE),
           f"-L{root}/lib", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", f"-L{LIB_DIR}", "-lmi_paged",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    tmp.replace(CALLS_PATH)
    return CALLS_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not needs_build():
        build_calls(verbose=verbose)
        return LIB_PATH
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    nvcc = os.environ.get("NVCC", "nvcc")
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc, *NVCC_FLAGS, "-o", str(tmp), str(CSRC / "libmi_paged.cu")]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    tmp.replace(LIB_PATH)
    build_calls(force, verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
