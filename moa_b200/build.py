"""Builds libmoa_b200.so (the C-ABI library) in-tree with nvcc for sm_100a, and _paged_host.so beside it.

    python moa_b200/build.py [--force] [--verbose]

The library is a plain shared object (no Python, no torch in its interface); the Python
package loads it with ctypes.  nvcc cross-compiles, so no GPU is needed to build.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmoa_b200.so")
SOURCES = ["errors.cu", "decode.cu", "cache.cu", "prefill.cu", "peer.cu", "paged.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
#: the host's share of the paged calls, compiled against the installed torch (moa_b200/paged.py does without it, slower)
HOST = os.path.join(HERE, "_paged_host.so")
HOST_SOURCE = os.path.join(CSRC, "paged_host.cpp")


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put it on PATH")


def _stale() -> bool:
    if not os.path.exists(LIB) or not os.path.exists(HOST):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(HOST))
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, "..", "include", "moa_b200.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu under csrc/ into libmoa_b200.so; returns the library path."""
    if not force and not _stale():
        return LIB
    objs = []
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    for src in SOURCES:
        obj = os.path.join(HERE, "build", src.replace(".cu", ".o"))
        cmd = [_nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "--use_fast_math", "-Xcompiler", "-fPIC",
               "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        objs.append(obj)
    cmd = [_nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    build_host(verbose)
    return LIB


def build_host(verbose: bool = False) -> str:
    """Compile csrc/paged_host.cpp with the host compiler against the installed torch."""
    import sysconfig

    import torch

    base = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           *("-I" + d for d in (os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"),
                                os.path.join(cuda, "include"), sysconfig.get_paths()["include"])),
           HOST_SOURCE, "-o", HOST, "-L" + os.path.join(base, "lib"), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    return HOST


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
