"""Build recipe for the C-ABI library (``libqssm.so``): one nvcc call per translation unit, sm_100a only.

Run ``python -m quick_ssm_b200.build`` (add ``--force`` to rebuild, ``-v`` for ptxas
resource usage).  The library links the CUDA runtime statically and resolves the one driver
entry point it needs at run time, so it loads on a machine without a GPU driver.
"""
from __future__ import annotations

import concurrent.futures
import os
import subprocess
import sys

_PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_PKG, "csrc")
UNITS = ["qssm.cu", "qssm_addnorm_fwd.cu", "qssm_addnorm_bwd.cu", "qssm_fp8.cu"]
HEADER = os.path.join(os.path.dirname(_PKG), "include", "qssm.h")
LIB = os.path.join(_PKG, "libqssm.so")


def _nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = os.path.join(cuda_home, "bin", "nvcc")
    return cand if os.path.exists(cand) else "nvcc"


def _sources():
    return [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh"))] + [HEADER]


def is_stale() -> bool:
    if not os.path.exists(LIB):
        return True
    built = os.path.getmtime(LIB)
    return any(os.path.getmtime(p) > built for p in _sources())


def _includes(path: str, seen: set) -> set:
    """The files a translation unit is made of, itself included."""
    if path in seen:
        return seen
    seen.add(path)
    with open(path) as f:
        for line in f:
            if line.startswith('#include "'):
                dep = os.path.normpath(os.path.join(os.path.dirname(path), line.split('"')[1]))
                if os.path.exists(dep):
                    _includes(dep, seen)
    return seen


def _compile(unit: str, force: bool, flags) -> str:
    src = os.path.join(CSRC, unit)
    obj = os.path.join(CSRC, unit[:-3] + ".o")
    if not force and os.path.exists(obj):
        built = os.path.getmtime(obj)
        if all(os.path.getmtime(p) <= built for p in _includes(src, set())):
            return obj
    part = f"{obj}.{os.getpid()}"  # moved into place whole: another build may be reading the object
    subprocess.check_call([_nvcc(), *flags, "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
                           "-Xcompiler", "-fPIC", "-c", "-o", part, src])
    os.replace(part, obj)
    return obj


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not is_stale():
        return LIB
    flags = (["-Xptxas", "-v"] if verbose else [])
    extra = os.environ.get("QSSM_NVCC_FLAGS")  # e.g. -DQSSM_RESIDENT_SWEEP for measurement builds
    if extra:
        flags = extra.split() + flags
    with concurrent.futures.ThreadPoolExecutor(len(UNITS)) as pool:
        objs = list(pool.map(lambda u: _compile(u, force or bool(extra), flags), UNITS))
    part = f"{LIB}.{os.getpid()}"
    subprocess.check_call([_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC",
                           "-o", part, *objs])
    os.replace(part, LIB)
    if extra:  # the next plain build must not link these
        for obj in objs:
            os.remove(obj)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
