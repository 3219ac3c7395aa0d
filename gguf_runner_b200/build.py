"""Builds libggr_attn.so (CUDA kernels + C ABI) in-tree for sm_100a with nvcc.

Usage: python -m gguf_runner_b200.build [--force] [-v] [--trace]
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libggr_attn.so")
# diagnostic build: the kernels additionally write phase time stamps (see `bench.py --case decode_stamps`)
TRACE_LIB_PATH = os.path.join(PKG_DIR, "libggr_attn_trace.so")
SOURCES = ["ggr_attn.cu", "paged.cu", "host_plan.cpp"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the attention library can only be built with the CUDA toolkit")


def _stale(path: str = LIB_PATH) -> bool:
    if not os.path.exists(path):
        return True
    built = os.path.getmtime(path)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps.append(os.path.join(PKG_DIR, "..", "include", "ggr_attn.h"))
    return any(os.path.getmtime(d) > built for d in deps if os.path.exists(d))


def _sources_of(path: str, seen: set) -> set:
    """`path` and the files of this project that it includes."""
    path = os.path.realpath(path)
    if path not in seen and os.path.exists(path):
        seen.add(path)
        with open(path) as f:
            for name in re.findall(r'^\s*#include "([^"]+)"', f.read(), flags=re.M):
                _sources_of(os.path.join(os.path.dirname(path), name), seen)
    return seen


def build_library(force: bool = False, verbose: bool = False, trace: bool = False) -> str:
    """Compiles the library if it is missing or older than its sources; returns its path. Each source has an object of its
    own under build/, compiled again when it or a file that it includes is newer, all at the same time.
    trace=True builds the diagnostic variant (-DGGR_TC_TRACE) next to it."""
    out = TRACE_LIB_PATH if trace else LIB_PATH
    if not force and not _stale(out):
        return out
    nvcc, objects_dir = _nvcc(), os.path.join(PKG_DIR, "build")
    os.makedirs(objects_dir, exist_ok=True)
    flags = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]
    if trace:
        flags += ["-DGGR_TC_TRACE"]
    if verbose:
        flags += ["-Xptxas", "-v"]

    def compiled(source: str) -> str:
        path = os.path.join(CSRC, source)
        obj = os.path.join(objects_dir, source + (".trace.o" if trace else ".o"))
        deps = _sources_of(path, {os.path.realpath(__file__)})
        if force or verbose or not os.path.exists(obj) or any(os.path.getmtime(d) > os.path.getmtime(obj) for d in deps):
            proc = subprocess.run([nvcc, *flags, "-c", "-o", obj + ".tmp", path], capture_output=True, text=True)
            if proc.returncode != 0:
                raise RuntimeError("nvcc failed:\n" + proc.stdout + proc.stderr)
            os.replace(obj + ".tmp", obj)
            if verbose:
                sys.stderr.write(proc.stderr)
        return obj

    with ThreadPoolExecutor(len(SOURCES)) as pool:
        objects = list(pool.map(compiled, SOURCES))
    proc = subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", out, *objects], capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + proc.stdout + proc.stderr)
    return out


if __name__ == "__main__":
    path = build_library(force="--force" in sys.argv, verbose="-v" in sys.argv, trace="--trace" in sys.argv)
    print(path)
