"""In-tree build of libfastnn_b200.so (nvcc, sm_100a only) and of its torch binding.

``python -m fastnn_b200.build`` compiles the CUDA sources under ``csrc/`` into
``fastnn_b200/libfastnn_b200.so``.  nvcc cross-compiles, so no GPU is needed to build.  Then
``csrc/binding.cpp`` becomes ``fastnn_b200/_binding.so``, which holds no device code: torch tensors in,
calls of the library's C ABI out, linked against the library beside it.
"""
from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libfastnn_b200.so")
BINDING = os.path.join(HERE, "_binding.so")
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "-shared",
]


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps():
    return _sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        glob.glob(os.path.join(HERE, "..", "include", "*.h")) + [__file__]


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(d) > t for d in _deps())


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not needs_build():
        build_binding()
        return LIB
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    # built beside the target and renamed into place, so a reader never sees a half-written library
    tmp = LIB + ".tmp"
    cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-o", tmp] + _sources()
    subprocess.check_call(cmd)
    os.replace(tmp, LIB)
    build_binding(force)
    return LIB


def build_binding(force: bool = False) -> str:
    """The torch binding, built with the interpreter's torch; needs the library to link against."""
    src = os.path.join(CSRC, "binding.cpp")
    deps = [src, os.path.join(HERE, "..", "include", "fastnn_b200_kernels.h"), __file__]
    if not force and os.path.exists(BINDING) and all(os.path.getmtime(BINDING) > os.path.getmtime(d) for d in deps):
        return BINDING
    import sysconfig

    import torch
    from torch.utils import cpp_extension
    tmp = BINDING + ".tmp"
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           "-DTORCH_EXTENSION_NAME=_binding", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for d in cpp_extension.include_paths() + [sysconfig.get_paths()["include"], "/usr/local/cuda/include"]:
        cmd += ["-isystem", d]
    # the library beside it by name; torch's own libraries are in the process before this one is imported
    cmd += [src, "-o", tmp, "-L" + HERE, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"]
    cmd += ["-L" + d for d in cpp_extension.library_paths()]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    subprocess.check_call(cmd)
    os.replace(tmp, BINDING)
    return BINDING


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
