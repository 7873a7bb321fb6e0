"""Builds libmoa_b200.so (the C-ABI library) in-tree with nvcc for sm_100a, and _paged_host.*.so beside it.

    python moa_b200/build.py [--force] [--verbose]

The library is a plain shared object (no Python, no torch in its interface); the Python
package loads it with ctypes.  nvcc cross-compiles, so no GPU is needed to build.
"""
from __future__ import annotations

import argparse
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
import warnings

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmoa_b200.so")
SOURCES = ["errors.cu", "decode.cu", "cache.cu", "prefill.cu", "peer.cu", "paged.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
HOST_SOURCE = os.path.join(CSRC, "paged_host.cpp")
HEADER = os.path.join(HERE, "..", "include", "moa_b200.h")


def _torch_version() -> str:
    """Of the installed torch, without importing it; empty where there is none."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return ""
    with open(os.path.join(os.path.dirname(spec.origin), "version.py")) as f:
        found = re.search(r"^__version__ = '(.*)'", f.read(), flags=re.M)
    return found.group(1) if found else ""


#: the host's share of the paged calls, compiled against the installed torch (moa_b200/paged.py does without it, slower); it
#: reads torch's objects in place, so its name says which Python and torch it is for and no other ones load it
HOST = os.path.join(HERE, f"_paged_host.{sys.implementation.cache_tag}-torch{_torch_version()}.so")


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put it on PATH")


def _stale(made: str, sources) -> bool:
    return not os.path.exists(made) or any(os.path.getmtime(d) > os.path.getmtime(made) for d in sources)


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile every .cu under csrc/ into libmoa_b200.so, and the host part where that is possible; returns the library's
    path."""
    kernels = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if os.path.join(CSRC, f) != HOST_SOURCE]
    if force or _stale(LIB, kernels + [HEADER]):
        _build_library(verbose)
    if force or _stale(HOST, [HOST_SOURCE, HEADER]):
        if os.path.exists(HOST):
            os.remove(HOST)                       # should the new one fail, the old one's arguments may no longer fit
        try:
            build_host(verbose)
        except (OSError, subprocess.CalledProcessError) as e:
            why = f"exit status {e.returncode}" if isinstance(e, subprocess.CalledProcessError) else e
            warnings.warn(f"the host part of the paged calls was not built ({why}): each takes some ten microseconds more "
                          "from Python", RuntimeWarning, stacklevel=2)
    return LIB


def _build_library(verbose: bool) -> None:
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


def build_host(verbose: bool = False) -> str:
    """Compile csrc/paged_host.cpp with the host compiler against the installed torch."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        raise FileNotFoundError("torch is not installed")
    base = os.path.dirname(spec.origin)
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
