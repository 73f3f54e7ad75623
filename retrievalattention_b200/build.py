"""Build ``libri_b200.so`` in-tree with nvcc for sm_100a.

    python -m retrievalattention_b200.build [--force]

One translation unit per ``csrc/*.cu`` / ``csrc/*.cpp`` file, compiled in parallel, then
linked into ``retrievalattention_b200/lib/libri_b200.so``.  nvcc cross-compiles, so no GPU is
needed to build.  Beside it ``binding/paged.cpp``, the host side of ``paged.py`` (C++ on torch's
headers), becomes ``lib/_paged_binding.so``.
"""
from __future__ import annotations

import os
import shlex
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(os.path.dirname(PKG), "include")
LIB_DIR = os.path.join(PKG, "lib")
OBJ_DIR = os.path.join(LIB_DIR, "obj")
LIB_PATH = os.path.join(LIB_DIR, "libri_b200.so")
BINDING_SOURCE = os.path.join(PKG, "binding", "paged.cpp")
BINDING_PATH = os.path.join(LIB_DIR, "_paged_binding.so")

NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", f"-I{INCLUDE}", f"-I{CSRC}"]
NVCC_FLAGS += shlex.split(os.environ.get("RI_NVCC_EXTRA", ""))   # extra compiler flags (e.g. -Xptxas=-v)


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cpp")))


def _newest_input() -> float:
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + \
            [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    return max(os.path.getmtime(f) for f in files)


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.join(OBJ_DIR, os.path.splitext(src)[0] + ".o")
    cmd = ["nvcc", *NVCC_FLAGS, "-x", "cu", "-c", os.path.join(CSRC, src), "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{res.stdout}\n{res.stderr}")
    if verbose:
        sys.stderr.write(res.stderr)
    return obj


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile if the library is missing or older than any source.  Returns its path."""
    if not force and os.path.exists(LIB_PATH) and os.path.getmtime(LIB_PATH) >= _newest_input():
        return LIB_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    with ThreadPoolExecutor(max_workers=8) as pool:
        objs = list(pool.map(lambda s: _compile(s, verbose), _sources()))
    cmd = ["nvcc", "-shared", "-o", LIB_PATH, *objs, "-Xcompiler", "-fPIC", "-lpthread"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    return LIB_PATH


def build_binding(force: bool = False) -> str:
    """Compile the host side of ``paged.py`` if it is missing or older than what it is made from.  Returns its path."""
    newest = max(os.path.getmtime(f) for f in (BINDING_SOURCE, os.path.join(INCLUDE, "ri_b200.h")))
    if not force and os.path.exists(BINDING_PATH) and os.path.getmtime(BINDING_PATH) >= newest:
        return BINDING_PATH
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    include = [INCLUDE, os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
               sysconfig.get_paths()["include"], os.path.join(cuda, "include")]
    os.makedirs(LIB_DIR, exist_ok=True)
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-I{d}" for d in include), BINDING_SOURCE, "-o", BINDING_PATH, "-L" + os.path.join(root, "lib"),
           "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {BINDING_SOURCE}:\n{res.stdout}\n{res.stderr}")
    return BINDING_PATH


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
    print(build_binding(force="--force" in sys.argv))
