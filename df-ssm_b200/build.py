"""Build libdfssm.so in-tree with nvcc for sm_100a (no torch headers, static cudart), and dfssm_pycalls.so, the host
path of ops.py (Python's C API only).

    python -m dfssm_b200.build        (or python df-ssm_b200/build.py)
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIBDIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIBDIR, "libdfssm.so")
PYCALLS = os.path.join(LIBDIR, "dfssm_pycalls.so")
SOURCES = ["dfssm_capi.cu", "persistent.cu", "gated_delta.cu", "sample_filtered.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(p) > t for p in deps if os.path.exists(p))


def build_pycalls(force: bool = False, verbose: bool = False) -> str:
    source = os.path.join(CSRC, "pycalls.cpp")
    if not force and not _stale(PYCALLS, [source]):
        return PYCALLS
    os.makedirs(LIBDIR, exist_ok=True)
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-Wall", "-shared", "-fPIC", "-fvisibility=hidden",
           "-I" + sysconfig.get_paths()["include"], "-o", PYCALLS + ".tmp", source]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True, cwd=CSRC)
    os.replace(PYCALLS + ".tmp", PYCALLS)
    return PYCALLS


def build(force: bool = False, verbose: bool = False) -> str:
    build_pycalls(force, verbose)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if not f.endswith(".cpp")]
    if not force and not _stale(LIB, deps + [os.path.join(PKG, "..", "include", "dfssm.h")]):
        return LIB
    tmp = LIB + ".tmp"
    cmd = [nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-shared", "-Xcompiler", "-fPIC,-O3",
           "-cudart", "static", "-o", tmp] + [os.path.join(CSRC, s) for s in SOURCES]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd))
    subprocess.run(cmd, check=True, cwd=CSRC)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
