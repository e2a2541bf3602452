"""Build ``libvesper_moe.so`` (the C-ABI library and its sm_100a kernels) in-tree.

    python -m velvetoptimizer_b200.build [--force] [--verbose]

Each ``csrc/*.cu`` is compiled by nvcc for ``sm_100a`` into ``_build/`` in parallel and
linked into ``velvetoptimizer_b200/lib/libvesper_moe.so``.  The CUDA runtime is linked
statically; kernels launch on the caller's stream.  nvcc cross-compiles, so this runs on
a machine without a GPU.
"""
from __future__ import annotations

import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
BUILD = os.path.join(REPO, "_build")
LIB_DIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIB_DIR, "libvesper_moe.so")
INCLUDE = os.path.join(REPO, "include")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3,-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-I", INCLUDE, "-I", CSRC]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: set NVCC or install the CUDA toolkit")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _deps() -> list[str]:
    return sources() + glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) \
        + glob.glob(os.path.join(INCLUDE, "*.h"))


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    return all(os.path.getmtime(p) <= t for p in _deps())


def _compile(src: str, verbose: bool, extra: list[str]) -> str:
    obj = os.path.join(BUILD, os.path.basename(src)[:-3] + ".o")
    cmd = [nvcc(), *ARCH, *FLAGS, *extra, "-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{r.stdout}\n{r.stderr}")
    if verbose and (r.stdout or r.stderr):
        print(r.stdout + r.stderr, flush=True)
    return obj


CSRC_PY = os.path.join(PKG, "csrc_py")


def build_host_module(name: str, force: bool = False, verbose: bool = False) -> str:
    """A host helper of the PyTorch layer (csrc_py/<name>.cpp, a CPython extension against
    torch's headers): g++ only, no GPU code.  Skips work when up to date."""
    src = os.path.join(CSRC_PY, f"{name}.cpp")
    out = os.path.join(LIB_DIR, f"_{name}.so")
    deps = [src] + ([os.path.join(INCLUDE, "vesper_moe.h")] if name == "dense_ops" else [])
    if (not force and os.path.exists(out)
            and all(os.path.getmtime(d) <= os.path.getmtime(out) for d in deps)):
        return out
    import sysconfig

    import torch
    tdir = os.path.dirname(torch.__file__)
    abi = int(getattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", True))
    cuda = os.path.join(os.path.dirname(os.path.dirname(nvcc())), "include")
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={abi}",
           "-I", sysconfig.get_paths()["include"], "-I", INCLUDE, "-I", cuda,
           "-I", os.path.join(tdir, "include"),
           "-I", os.path.join(tdir, "include", "torch", "csrc", "api", "include"),
           src, "-o", out + ".tmp", "-L", os.path.join(tdir, "lib"),
           "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python",
           # the libstdc++ that torch has loaded, also where $CXX would link one statically: the
           # module's streams, locales and exceptions are then torch's
           "-l:libstdc++.so.6"]
    if name == "dense_ops":  # calls the C ABI library beside it
        cmd += ["-lc10_cuda", "-ltorch_cuda", LIB, "-Wl,-rpath,$ORIGIN"]
    cmd += [f"-Wl,-rpath,{os.path.join(tdir, 'lib')}"]
    os.makedirs(LIB_DIR, exist_ok=True)
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{name} build failed:\n{r.stdout}\n{r.stderr}")
    os.replace(out + ".tmp", out)
    return out


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> str:
    """Compile and link the library (and the PyTorch layer's host helpers); returns the
    library's path.  Skips work when up to date."""
    build_host_module("param_key", force=force, verbose=verbose)
    if force or extra or not up_to_date():
        _build_library(verbose, extra)
    build_host_module("dense_ops", force=force, verbose=verbose)
    return LIB


def _build_library(verbose: bool, extra: list[str] | None) -> None:
    os.makedirs(BUILD, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose, extra or []), srcs))
    tmp = LIB + ".tmp"
    cmd = [nvcc(), *ARCH, "-shared", "-o", tmp, *objs, "-Xcompiler", "-fPIC",
           "-Xlinker", "-soname=libvesper_moe.so"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)


if __name__ == "__main__":
    force = "--force" in sys.argv
    verbose = "--verbose" in sys.argv or "-v" in sys.argv
    extra = ["-Xptxas", "-v"] if "--ptxas" in sys.argv else None
    print(build(force=force or bool(extra), verbose=verbose or bool(extra), extra=extra))
