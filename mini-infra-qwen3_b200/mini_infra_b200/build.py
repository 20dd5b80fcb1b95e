"""Build libmi_paged.so (sm_100a) in-tree: ``python -m mini_infra_b200.build``.

One nvcc invocation over the unity translation unit ``csrc/libmi_paged.cu``; the shared object
lands in ``mini_infra_b200/_lib/`` so that it travels with the source tree.  Beside it ``_mi_calls.*.so``, a
CPython extension over that library (``csrc/torch_calls.cpp``, g++ against PyTorch's headers): the ordinary
calls of the 4-bit operators without the cost of ctypes.  It belongs to one Python and one PyTorch, which its name
says; where it cannot be built, those calls go through ctypes like the others.
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG.parent / "csrc"
LIB_DIR = PKG / "_lib"
LIB_PATH = LIB_DIR / "libmi_paged.so"
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


def calls_path() -> Path:
    """The CPython extension of this Python and this PyTorch (whose C++ interface changes between versions)."""
    import torch

    return LIB_DIR / f"_mi_calls.{sysconfig.get_config_var('SOABI')}.torch-{torch.__version__}.so"


def build_calls(force: bool = False, verbose: bool = False) -> Path:
    """The CPython extension; needs libmi_paged.so, PyTorch's and Python's headers and g++."""
    path = calls_path()
    inputs = [CALLS_SOURCE, *(PKG.parent.parent / "include").glob("*.h")]
    if not force and path.exists() and path.stat().st_mtime >= max(p.stat().st_mtime for p in inputs):
        return path
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))
    tmp = path.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{root}/include", f"-I{root}/include/torch/csrc/api/include", f"-I{sysconfig.get_paths()['include']}",
           f"-I{cuda}/include", f"-I{PKG.parent.parent / 'include'}", "-o", str(tmp), str(CALLS_SOURCE),
           f"-L{root}/lib", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python", f"-L{LIB_DIR}", "-lmi_paged",
           "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    tmp.replace(path)
    return path


def _try_build_calls(force: bool, verbose: bool) -> None:
    try:
        build_calls(force, verbose)
    except (ImportError, OSError, subprocess.CalledProcessError) as e:
        warnings.warn(f"the CPython extension was not built ({e}); the 4-bit operators go through ctypes", RuntimeWarning,
                      stacklevel=3)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not needs_build():
        _try_build_calls(False, verbose)
        return LIB_PATH
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    nvcc = os.environ.get("NVCC", "nvcc")
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc, *NVCC_FLAGS, "-o", str(tmp), str(CSRC / "libmi_paged.cu")]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    tmp.replace(LIB_PATH)
    _try_build_calls(force, verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
