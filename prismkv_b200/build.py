"""Build libprismkv_b200.so in-tree with nvcc for sm_100a.

``python -m prismkv_b200.build`` (or ``build()``) compiles the translation
units csrc/pkv_lib.cu and csrc/pkv_paged_lib.cu side by side and links
prismkv_b200/libprismkv_b200.so; a unit whose sources are older than its object
in prismkv_b200/_build is not compiled again.  The library statically links the
CUDA runtime, takes streams from the caller and exports only the C ABI declared
in include/prismkv_b200.h.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libprismkv_b200.so")

OBJ_DIR = os.path.join(HERE, "_build")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    *ARCH_FLAGS,
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr", "-c",
]
LINK_FLAGS = [*ARCH_FLAGS, "-shared", "-cudart", "static"]
UNITS = ("pkv_lib", "pkv_paged_lib")


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; the PrismKV B200 library needs the CUDA toolkit to build")


def _sources(unit: str) -> list:
    """The files a unit is built from: the paged sources, or all the others; headers are shared."""
    csrc = os.path.join(HERE, "csrc")
    deps = [os.path.join(ROOT, "include", "prismkv_b200.h")]
    for s in os.listdir(csrc):
        if s.endswith(".cu") and s.startswith("pkv_paged") == (unit == "pkv_paged_lib"):
            deps.append(os.path.join(csrc, s))
        elif s.endswith(".cuh") and (unit == "pkv_paged_lib" or not s.startswith("pkv_paged")):
            deps.append(os.path.join(csrc, s))
    return deps


def _stale(target: str, deps: list) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _object(unit: str) -> str:
    return os.path.join(OBJ_DIR, unit + ".o")


def _compile(unit: str, verbose: bool) -> None:
    obj = _object(unit)
    cmd = [_nvcc(), *NVCC_FLAGS, "-I", os.path.join(ROOT, "include"),
           os.path.join(HERE, "csrc", unit + ".cu"), "-o", obj + ".tmp"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}) on {unit}.cu:\n{res.stdout}\n{res.stderr}")
    os.replace(obj + ".tmp", obj)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and not _stale(LIB, [d for u in UNITS for d in _sources(u)]):
        return LIB
    os.makedirs(OBJ_DIR, exist_ok=True)
    todo = [u for u in UNITS if force or _stale(_object(u), _sources(u))]
    with ThreadPoolExecutor(len(UNITS)) as pool:
        list(pool.map(lambda u: _compile(u, verbose), todo))
    cmd = [_nvcc(), *LINK_FLAGS, *(_object(u) for u in UNITS), "-o", LIB + ".tmp"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed to link ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
