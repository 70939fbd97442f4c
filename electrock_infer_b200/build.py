"""Builds libb200moe.so (the C-ABI library, declared in include/b200moe.h) with nvcc for sm_100a, and
_binding.so (csrc/torch_binding.cpp, the decode-step ops for torch tensors) with the host compiler.

Run as ``python -m electrock_infer_b200.build``.  The shared objects are written next to this
file so that they are found by :mod:`electrock_infer_b200._lib` and travel with the source tree.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libb200moe.so"
INCLUDE_DIR = PKG_DIR.parent / "include"
BINDING_PATH = PKG_DIR / "_binding.so"
BINDING_SOURCE = CSRC / "torch_binding.cpp"
BINDING_STAMP = PKG_DIR / "_binding.built_for"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
]


def find_nvcc() -> str:
    nvcc = os.environ.get("NVCC") or shutil.which("nvcc")
    if nvcc is None and Path("/usr/local/cuda/bin/nvcc").exists():
        nvcc = "/usr/local/cuda/bin/nvcc"
    if nvcc is None:
        raise RuntimeError("nvcc not found: set NVCC or put the CUDA toolkit on PATH")
    return nvcc


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def is_stale() -> bool:
    if not LIB_PATH.exists():
        return True
    built = LIB_PATH.stat().st_mtime
    deps = list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cuh")) + list(INCLUDE_DIR.glob("*.h"))
    return any(p.stat().st_mtime > built for p in deps)


def binding_target() -> str:
    """The torch, C++ ABI and interpreter that a binding is compiled against; one that was compiled against
    others may load and misread tensors."""
    import sysconfig

    import torch
    return f"torch {torch.__version__}, C++11 ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, {sysconfig.get_config_var('SOABI')}"


def binding_is_stale() -> bool:
    if not BINDING_PATH.exists() or not BINDING_STAMP.exists() or BINDING_STAMP.read_text() != binding_target():
        return True
    built = BINDING_PATH.stat().st_mtime
    return any(p.stat().st_mtime > built for p in [BINDING_SOURCE, *INCLUDE_DIR.glob("*.h")])


def build_binding(force: bool = False) -> Path:
    """Compiles the binding against the torch of this interpreter; needs libb200moe.so in place."""
    if not force and not binding_is_stale():
        return BINDING_PATH
    import sysconfig

    import torch
    home = Path(torch.__file__).resolve().parent
    cuda = Path(find_nvcc()).resolve().parent.parent
    includes = [sysconfig.get_paths()["include"], home / "include", home / "include/torch/csrc/api/include",
                cuda / "include"]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DB200MOE_BUILT_FOR="{binding_target()}"',
           "-o", str(BINDING_PATH), str(BINDING_SOURCE), *(f"-I{d}" for d in includes),
           f"-L{PKG_DIR}", f"-l:{LIB_PATH.name}", f"-L{home / 'lib'}",
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    BINDING_STAMP.write_text(binding_target())
    return BINDING_PATH


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles every kernel into one shared library, and the binding; returns the library's path."""
    if not force and not is_stale():
        build_binding()
        return LIB_PATH
    cmd = [find_nvcc(), *NVCC_FLAGS]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    cmd += ["-o", str(LIB_PATH), *map(str, sources())]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed ({proc.returncode}):\n{proc.stdout}\n{proc.stderr}")
    if verbose:
        print(proc.stderr)
    build_binding(force)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
