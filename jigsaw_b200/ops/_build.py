"""Build the sm_100a kernel library in-tree with nvcc.

The library is a plain C-ABI shared object (``libjb_kernels.so``) next to this file, loaded
with :mod:`ctypes`.  It is compiled for ``sm_100a`` only; nvcc cross-compiles on a machine
without a GPU.  Beside it stands a torch binding (``_jb_torch.so``, host code only, compiled with the
C++ compiler against torch's headers) that drives the 8-bit kernels without Python between the launches.
"""

from __future__ import annotations

import hashlib
import importlib.machinery
import importlib.util
import os
import shutil
import subprocess
import sysconfig
from pathlib import Path
from typing import Any

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
LIB_PATH = HERE / "libjb_kernels.so"
_STAMP = HERE / "libjb_kernels.stamp"
BINDING_PATH = HERE / "_jb_torch.so"
_BINDING_STAMP = HERE / "_jb_torch.stamp"
_BINDING_SOURCES = ("torch_binding.cpp", "scaled_abi.h")

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "--use_fast_math",
    "-shared",
    "-Xcompiler",
    "-fPIC",
]


def _nvcc() -> str | None:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand if cand and os.path.exists(cand) else None


def source_hash() -> str:
    """Hash of every file under ``csrc`` (rebuild trigger)."""
    h = hashlib.sha256()
    for p in sorted(CSRC.glob("*")):
        if p.suffix in (".cu", ".cuh", ".h"):
            h.update(p.name.encode())
            h.update(p.read_bytes())
    h.update(" ".join(NVCC_FLAGS).encode())
    return h.hexdigest()


def is_fresh() -> bool:
    return LIB_PATH.exists() and _STAMP.exists() and _STAMP.read_text().strip() == source_hash()


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile ``csrc/jb_kernels.cu`` into ``libjb_kernels.so`` if the sources changed."""
    if not force and is_fresh():
        return LIB_PATH
    nvcc = _nvcc()
    if nvcc is None:
        raise RuntimeError("nvcc not found; cannot build jigsaw_b200 kernels")
    tmp = LIB_PATH.with_suffix(".so.tmp%d" % os.getpid())
    cmd = [nvcc, *NVCC_FLAGS, "-o", str(tmp), str(CSRC / "jb_kernels.cu")]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + proc.stdout + proc.stderr)
    if verbose:
        print(proc.stderr)
    os.replace(tmp, LIB_PATH)
    _STAMP.write_text(source_hash())
    return LIB_PATH


# ----------------------------------------------------------------------------- torch binding
def _cuda_home() -> Path:
    nvcc = _nvcc()
    return Path(nvcc).resolve().parent.parent if nvcc else Path("/usr/local/cuda")


def binding_hash() -> str:
    import torch

    h = hashlib.sha256()
    for name in _BINDING_SOURCES:
        h.update((CSRC / name).read_bytes())
    h.update(f"{torch.__version__} {sysconfig.get_python_version()}".encode())
    return h.hexdigest()


def binding_is_fresh() -> bool:
    return BINDING_PATH.exists() and _BINDING_STAMP.exists() and _BINDING_STAMP.read_text().strip() == binding_hash()


def build_binding(force: bool = False) -> Path:
    """Compile ``csrc/torch_binding.cpp`` into ``_jb_torch.so`` if it or torch changed."""
    if not force and binding_is_fresh():
        return BINDING_PATH
    import torch

    cxx = os.environ.get("CXX") or shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        raise RuntimeError("no C++ compiler found; cannot build the torch binding of jigsaw_b200")
    root = Path(torch.__file__).parent
    tmp = BINDING_PATH.with_suffix(".so.tmp%d" % os.getpid())
    cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{root / 'include'}", f"-I{root / 'include/torch/csrc/api/include'}", f"-I{_cuda_home() / 'include'}",
           f"-I{sysconfig.get_paths()['include']}", str(CSRC / "torch_binding.cpp"), "-o", str(tmp), f"-L{root / 'lib'}",
           "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10", "-lc10_cuda"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("the C++ compiler failed on the torch binding:\n" + proc.stdout + proc.stderr)
    os.replace(tmp, BINDING_PATH)
    _BINDING_STAMP.write_text(binding_hash())
    return BINDING_PATH


def load_binding() -> Any:
    """The extension module (``JIGSAW_B200_BINDING``, or the in-tree one, built first if its source is newer)."""
    path = os.environ.get("JIGSAW_B200_BINDING") or str(build_binding())
    loader = importlib.machinery.ExtensionFileLoader("_jb_torch", path)
    spec = importlib.util.spec_from_file_location("_jb_torch", path, loader=loader)
    module = importlib.util.module_from_spec(spec)
    loader.exec_module(module)
    return module


if __name__ == "__main__":
    import sys

    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_binding(force="--force" in sys.argv))
