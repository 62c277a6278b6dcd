"""Build libbfa.so (the C-ABI attention library) for sm_100a with nvcc, and
bfa_torch.so (the PyTorch side of the rotary and tree-decoding operators) with
the host compiler.

Usage: python build.py [--force] [--jobs N]

Objects are compiled in parallel under ``_build/`` next to this file and
linked into ``libbfa.so`` in this directory. The runtime is linked shared
(libcudart.so.12), so inside a PyTorch process the library uses the CUDA
runtime torch already loaded.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libbfa.so")
BINDING = os.path.join(HERE, "bfa_torch.so")
BINDING_SRC = os.path.join(CSRC, "torch_binding.cpp")
CXX = "g++"  # the compiler nvcc calls too: its libstdc++ is the shared one that torch uses
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-I", INCLUDE, "-I", CSRC]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _deps_mtime():
    paths = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    paths += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    return max(os.path.getmtime(p) for p in paths)


def compile_one(src: str, force: bool) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    if (not force and os.path.exists(obj)
            and os.path.getmtime(obj) >= max(os.path.getmtime(src), _deps_mtime())):
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def build_binding(force: bool = False, verbose: bool = True) -> str:
    """bfa_torch.so, a CPython module against this Python's torch and libbfa.so's
    C ABI (found next to it)."""
    deps = [BINDING_SRC, os.path.join(INCLUDE, "bfa.h")]
    if not force and os.path.exists(BINDING) and os.path.getmtime(BINDING) >= max(map(os.path.getmtime, deps)):
        return BINDING
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda = os.path.dirname(os.path.dirname(NVCC))
    inc = [x for d in [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include"), INCLUDE]
           for x in ("-isystem" if d != INCLUDE else "-I", d)]
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=bfa_torch",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *inc,
           BINDING_SRC, "-o", BINDING, "-L", HERE, "-lbfa", "-Wl,-rpath,$ORIGIN", "-L", lib, "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python", f"-Wl,-rpath,{lib}",
           "-L", os.path.join(cuda, "lib64"), "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{CXX} failed for {BINDING_SRC}:\n{r.stdout}\n{r.stderr}")
    if verbose:
        print("built", BINDING)
    return BINDING


def build(force: bool = False, jobs: int | None = None, verbose: bool = True) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs), os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(jobs) as ex:
        objs = list(ex.map(lambda s: compile_one(s, force), srcs))
    newest = max(os.path.getmtime(o) for o in objs)
    if force or not os.path.exists(LIB) or os.path.getmtime(LIB) < newest:
        cmd = [NVCC, *ARCH, "-shared", "-o", LIB, *objs, "-cudart", "shared",
               "-Xlinker", "-rpath,/usr/local/cuda/lib64"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        if verbose:
            print("built", LIB)
    build_binding(force, verbose)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    args = ap.parse_args()
    try:
        build(force=args.force, jobs=args.jobs)
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
