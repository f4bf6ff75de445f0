"""Builds realm_b200/librealm_b200.so (sm_100a) in-tree with nvcc.

Usage: python realm_b200/build.py [--force]   (run by path: the package import needs the library)
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "librealm_b200.so")
SOURCES = ["gemv.cu", "attention.cu", "engine.cu", "sample.cu", "scheduler.cpp", "gguf.cpp", "rows_plan.cpp",
           "rows_append.cu", "rows_attn.cu", "rows_tile.cu", "filter.cu", "adapters.cu", "adapters_tile.cu", "verify.cu",
           "residual.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo",
         "-Xcompiler", "-fPIC"]


def _mtime(p: str) -> float:
    return os.path.getmtime(p) if os.path.exists(p) else 0.0


def _newest(path: str, seen: set) -> float:
    """The newest modification time of a source and of what it includes."""
    path = os.path.normpath(path)
    if path in seen:
        return 0.0
    seen.add(path)
    with open(path) as f:
        names = re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M)
    return max([_mtime(path)] + [_newest(os.path.join(os.path.dirname(path), n), seen) for n in names])


def _compile(src: str, force: bool) -> str:
    obj = os.path.join(BUILD, os.path.splitext(src)[0] + ".o")
    path = os.path.join(CSRC, src)
    if force or _mtime(obj) < _newest(path, set()):
        cmd = [NVCC, *FLAGS, "-c", path, "-o", obj]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def build(force: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    with cf.ThreadPoolExecutor(len(SOURCES)) as ex:
        objs = list(ex.map(lambda s: _compile(s, force), SOURCES))
    if force or _mtime(LIB) < max(_mtime(o) for o in objs):
        # the exported C ABI keeps default visibility through the header's extern "C" block
        cmd = [NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", LIB, *objs,
               "-Xcompiler", "-fPIC", "-lcudart"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv))
