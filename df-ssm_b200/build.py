"""Build libdfssm.so in-tree with nvcc for sm_100a (no torch headers, static cudart), and dfssm_pycalls, the host path of
ops.py (Python's C API only), as a module of the running interpreter.

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
PYCALLS = os.path.join(LIBDIR, "dfssm_pycalls" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
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


def build_pycalls(force: bool = False, verbose: bool = False):
    """The module's path, or None where Python's headers are not installed: the C library works without it, ops.py does
    not and says so when it is called."""
    source = os.path.join(CSRC, "pycalls.cpp")
    if not force and not _stale(PYCALLS, [source]):
        return PYCALLS
    include = sysconfig.get_paths()["include"]
    if not os.path.exists(os.path.join(include, "Python.h")):
        print(f"no Python.h in {include}: built without {os.path.basename(PYCALLS)}, which dfssm_b200.ops needs", file=sys.stderr)
        return None
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-Wall", "-shared", "-fPIC", "-fvisibility=hidden",
           "-I" + include, "-o", PYCALLS + ".tmp", source]
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True, cwd=CSRC)
    os.replace(PYCALLS + ".tmp", PYCALLS)
    return PYCALLS


def build_library(force: bool = False, verbose: bool = False) -> str:
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


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(LIBDIR, exist_ok=True)
    build_library(force, verbose)
    build_pycalls(force, verbose)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
