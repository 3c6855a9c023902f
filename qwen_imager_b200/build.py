"""Builds libqmm.so (the CUDA library behind include/qmm.h) in-tree with nvcc.

The library is compiled for sm_100a only and written to
qwen_imager_b200/_build/libqmm.so, next to the sources, so that it travels with
the repository to the machine that runs it.  The CUDA runtime is linked
statically; the driver API entry point for tensor maps is resolved at run time.
Beside it, _build/_qmm_host.so: the block operators' ordinary calls in C++ (g++).

Usage: python -m qwen_imager_b200.build [--verbose]
"""
from __future__ import annotations

import glob
import hashlib
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OUT_DIR = os.path.join(PKG, "_build")
LIB = os.path.join(OUT_DIR, "libqmm.so")
HOST_SRC = os.path.join(CSRC, "host", "block_host.cpp")
HOST = os.path.join(OUT_DIR, "_qmm_host.so")

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "-I" + os.path.join(ROOT, "include"),
]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the qmm CUDA library cannot be built")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def headers() -> list[str]:
    return (sorted(glob.glob(os.path.join(CSRC, "*.cuh"))) + sorted(glob.glob(os.path.join(CSRC, "*.h")))
            + sorted(glob.glob(os.path.join(ROOT, "include", "*.h"))))


def _older(target: str, files: list[str]) -> bool:
    if not os.path.exists(target):
        return True
    built = os.path.getmtime(target)
    return any(os.path.getmtime(f) > built for f in files)


def is_stale() -> bool:
    return _older(LIB, sources() + headers() + [__file__])


def host_key() -> str:
    """What the extension is built from and for: its sources, this file, and the torch and
    Python whose binary interfaces it uses.  Compiled into it (`key`)."""
    import torch

    h = hashlib.sha256()
    for path in (HOST_SRC, os.path.join(ROOT, "include", "qmm_block.h"), os.path.join(ROOT, "include", "qmm.h"), __file__):
        with open(path, "rb") as f:
            h.update(f.read())
    h.update(f"{torch.__version__} {sys.implementation.cache_tag}".encode())
    return h.hexdigest()


def host_is_stale() -> bool:
    """Whether the extension is missing or does not hold the present key (times of files say
    nothing about the torch that it was built for)."""
    if not os.path.exists(HOST):
        return True
    with open(HOST, "rb") as f:
        return host_key().encode() not in f.read()


def build_host(force: bool = False) -> str:
    """Compiles the Python extension of the block operators' calls (g++, against
    torch's headers; the entry points it calls are bound at run time)."""
    if not force and not host_is_stale():
        return HOST
    import torch

    os.makedirs(OUT_DIR, exist_ok=True)
    base = os.path.dirname(torch.__file__)
    inc = os.path.join(base, "include")
    cuda = os.path.dirname(os.path.dirname(nvcc_path()))
    with tempfile.TemporaryDirectory(dir=OUT_DIR) as work:  # this build's own: several processes may find the file stale at once
        made = os.path.join(work, os.path.basename(HOST))
        cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
               "-I" + os.path.join(ROOT, "include"), "-I" + inc, "-I" + os.path.join(inc, "torch", "csrc", "api", "include"),
               "-I" + os.path.join(cuda, "include"), "-I" + sysconfig.get_paths()["include"], f'-DQMM_HOST_KEY="{host_key()}"', HOST_SRC, "-o", made,
               "-L" + os.path.join(base, "lib"), "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", "-lc10_cuda"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("g++ failed on block_host.cpp")
        os.replace(made, HOST)
    return HOST


def build(verbose: bool = False, force: bool = False) -> str:
    """Compiles every csrc/*.cu into one shared library; returns its path."""
    if not force and not is_stale():
        return LIB
    os.makedirs(OUT_DIR, exist_ok=True)
    nvcc = nvcc_path()

    with tempfile.TemporaryDirectory(dir=OUT_DIR) as work:  # this build's own, as above

        def compile_one(src: str):
            obj = os.path.join(work, os.path.basename(src)[:-3] + ".o")
            cmd = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, "-c", src, "-o", obj]
            if verbose:
                cmd += ["-Xptxas", "-v"]
            return src, obj, subprocess.run(cmd, capture_output=True, text=True)

        objs = []
        with ThreadPoolExecutor(os.cpu_count() or 1) as pool:
            results = list(pool.map(compile_one, sources()))
        for src, obj, res in results:
            if verbose or res.returncode != 0:
                sys.stderr.write(res.stdout + res.stderr)
            if res.returncode != 0:
                raise RuntimeError(f"nvcc failed on {os.path.basename(src)}")
            objs.append(obj)
        made = os.path.join(work, os.path.basename(LIB))
        cmd = [nvcc, *ARCH_FLAGS, "-shared", "-o", made, *objs, "-Xcompiler", "-fPIC"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("nvcc link of libqmm.so failed")
        os.replace(made, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="--verbose" in sys.argv, force=True))
    print(build_host(force=True))
