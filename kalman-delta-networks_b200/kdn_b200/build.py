"""Build ``lib/libkdn_b200.so`` from ``csrc/*.cu`` for sm_100a with nvcc.

Each translation unit is compiled in parallel to ``_build/*.o`` and linked
into one shared library exporting the C ABI declared in ``include/kdn_b200.h``.
Beside it g++ builds ``lib/_kdn_torch.<torch>.<python>.so`` from ``csrc/host``:
the C++ host path of the serving operators (``_native.host``), one per torch and
interpreter.  Rebuilds only when a source or header is newer than the libraries.

    python -m kdn_b200.build [--force]
"""
from __future__ import annotations

import concurrent.futures
import glob
import os
import shutil
import subprocess
import sys
import warnings

from ._native import HOST_LIB

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIB_DIR, "libkdn_b200.so")
HOST_SRC = os.path.join(CSRC, "host", "kdn_torch.cpp")
BUILD_DIR = os.path.join(HERE, "_build")
INCLUDE = os.path.abspath(os.path.join(HERE, "..", "..", "include"))

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC"] + ARCH


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put the CUDA toolkit on PATH")


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps():
    return _sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h")) + [__file__]


def _newer(lib: str, deps) -> bool:
    return os.path.exists(lib) and all(os.path.getmtime(d) <= os.path.getmtime(lib) for d in deps)


def up_to_date() -> bool:
    return _newer(LIB, _deps())


def host_up_to_date() -> bool:
    return _newer(HOST_LIB, [HOST_SRC, __file__] + glob.glob(os.path.join(INCLUDE, "*.h")))


def build_host(verbose: bool = False) -> str:
    """The C++ host path, against the running torch."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    cmd = ["g++", "-O2", "-fPIC", "-shared", "-std=c++17", "-DTORCH_EXTENSION_NAME=_kdn_torch",
           "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for path in include:
        cmd += ["-isystem", path]
    cmd += [HOST_SRC, "-o", HOST_LIB + ".tmp"]
    cmd += [f"-L{path}" for path in cpp_extension.library_paths()]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {os.path.basename(HOST_SRC)}:\n{res.stderr}")
    os.replace(HOST_LIB + ".tmp", HOST_LIB)
    return HOST_LIB


def build(force: bool = False, verbose: bool = False) -> str:
    """Build what is out of date; returns the C library's path.  Without the C++ host path's compiler or headers the
    kernels are built all the same, with a warning."""
    os.makedirs(BUILD_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    with concurrent.futures.ThreadPoolExecutor(max_workers=1) as pool:  # beside the kernels
        host = None if not force and host_up_to_date() else pool.submit(build_host, verbose)
        if force or not up_to_date():
            _build_kernels(verbose)
        if host is not None:
            try:
                host.result()
            except Exception as e:  # no compiler, no Python headers: the operators work without it
                if os.path.exists(HOST_LIB):
                    os.remove(HOST_LIB)  # of an older source
                warnings.warn(f"kdn_b200: the C++ host path is not built ({e}); the Python path serves")
    return LIB


def _build_kernels(verbose: bool) -> None:
    nvcc = _nvcc()

    def compile_one(src: str) -> str:
        obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-3] + ".o")
        cmd = [nvcc, *NVCC_FLAGS, "-I", INCLUDE, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{res.stderr}")
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        objs = list(pool.map(compile_one, _sources()))
    tmp = LIB + ".tmp"
    cmd = [nvcc, *ARCH, "-shared", "-o", tmp, *objs, "-lcudart"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, LIB)


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
