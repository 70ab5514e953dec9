"""Build libtosa_b200.so and its torch binding in-tree for sm_100a (nvcc cross-compiles without a GPU).

Usage: python -m tosa_b200.build [--force]

Each translation unit under csrc/ is compiled in parallel into _build/ and the
objects are linked into tosa_b200/libtosa_b200.so (CUDA runtime linked
statically; driver entry points are resolved at run time).
csrc/torch_binding.cpp is compiled with the host compiler against the
installed torch into tosa_b200/_torch_binding.so, which loads that library;
without torch the library is built alone.
"""

from __future__ import annotations

import glob
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
OUT = os.path.join(HERE, "libtosa_b200.so")
BINDING_SRC = os.path.join(CSRC, "torch_binding.cpp")
BINDING = os.path.join(HERE, "_torch_binding.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
CFLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden"]


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def _newest_input():
    files = [f for f in glob.glob(os.path.join(CSRC, "*")) if f != BINDING_SRC] + glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    return max(os.path.getmtime(f) for f in files)


def _start_binding(force, verbose):
    """Starts compiling the torch binding when it is out of date; returns the process or None."""
    inputs = [BINDING_SRC] + glob.glob(os.path.join(HERE, "..", "include", "*.h"))
    if not force and os.path.exists(BINDING) and os.path.getmtime(BINDING) >= max(os.path.getmtime(f) for f in inputs):
        return None
    import sysconfig

    try:
        import torch
    except ImportError:
        print("torch is not installed: built without the torch binding (tosa_b200/attention.py needs it)", file=sys.stderr)
        return None
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(NVCC))
    obj = os.path.join(BUILD, "torch_binding.cpp.o")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-c", "-o", obj, BINDING_SRC,
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-isystem", os.path.join(root, "include"),
           "-isystem", os.path.join(root, "include", "torch", "csrc", "api", "include"), "-isystem",
           os.path.join(cuda, "include"), "-isystem", sysconfig.get_paths()["include"]]
    if verbose:
        print(" ".join(cmd), flush=True)
    return subprocess.Popen(cmd), obj, os.path.join(root, "lib")


def _link_binding(started, verbose):
    process, obj, libs = started
    if process.wait() != 0:
        raise RuntimeError(f"the host compiler failed for {BINDING_SRC}")
    cmd = [os.environ.get("CXX", "g++"), "-shared", "-o", BINDING + ".tmp", obj, "-L" + HERE, "-l:libtosa_b200.so", "-L" + libs,
           "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    os.replace(BINDING + ".tmp", BINDING)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    binding = _start_binding(force, verbose)
    try:
        out = _build_library(force, verbose)
    finally:
        if binding is not None:
            binding[0].wait()
    if binding is not None:
        _link_binding(binding, verbose)
    return out


def _build_library(force: bool, verbose: bool) -> str:
    if not force and os.path.exists(OUT) and os.path.getmtime(OUT) >= _newest_input():
        return OUT
    newest_header = max(os.path.getmtime(f) for f in glob.glob(os.path.join(CSRC, "*.cuh")) +
                        glob.glob(os.path.join(CSRC, "*.hpp")) + glob.glob(os.path.join(HERE, "..", "include", "*.h")))
    procs, objs = [], []
    for src in _sources():
        obj = os.path.join(BUILD, os.path.basename(src) + ".o")
        objs.append(obj)
        if not force and os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), newest_header):
            continue
        cmd = [NVCC, *CFLAGS, "-c", "-o", obj, src]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd)))
    failed = [src for src, p in procs if p.wait() != 0]
    if failed:
        raise RuntimeError(f"nvcc failed for {failed}")
    link = [NVCC, *ARCH, "-shared", "-o", OUT + ".tmp", *objs]
    if verbose:
        print(" ".join(link), flush=True)
    subprocess.check_call(link)
    os.replace(OUT + ".tmp", OUT)
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
