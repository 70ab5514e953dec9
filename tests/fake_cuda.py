"""The library's own objects linked with a CUDA runtime of host memory (fake_cuda.cpp), so that its host code runs
without a GPU and on more devices than one. Nothing is computed."""

import ctypes
import glob
import os
import subprocess

from tosa_b200 import _lib as L
from tosa_b200 import build as B


def load(folder):
    B.build()
    objects = sorted(glob.glob(os.path.join(B.BUILD, "*.cu.o")))
    if not objects:  # a library without its objects
        B.build(force=True)
        objects = sorted(glob.glob(os.path.join(B.BUILD, "*.cu.o")))
    out = os.path.join(str(folder), "libtosa_fake.so")
    source = os.path.join(os.path.dirname(os.path.abspath(__file__)), "fake_cuda.cpp")
    include = os.path.join(os.path.dirname(os.path.dirname(B.NVCC)), "include")
    subprocess.check_call([os.environ.get("CXX", "g++"), "-O1", "-std=c++17", "-fPIC", "-shared", "-o", out, source, *objects,
                           "-I" + include, "-Wl,-Bsymbolic", "-lpthread", "-ldl"])
    lib = ctypes.CDLL(out)
    for name, res, args in L.SIGNATURES:
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


def events(lib):
    """What happened since the last look, one text an event."""
    text = ctypes.create_string_buffer(1 << 16)
    lib.fake_events(text, ctypes.c_size_t(len(text)))
    return text.value.decode().splitlines()


def context(lib, device):
    h = ctypes.c_void_p()
    assert lib.tb_context_create(device, ctypes.byref(h)) == 0, lib.tb_last_error()
    return h


class HostCache:
    """A small cache of host memory."""

    def __init__(self, lib, ctx):
        self.k, self.v = ctypes.create_string_buffer(1 << 17), ctypes.create_string_buffer(1 << 17)
        self.words = (ctypes.c_int32 * 64)()
        up = lambda b: (ctypes.addressof(b) + 255) & ~255  # noqa: E731
        w = ctypes.addressof(self.words)
        desc = L.CacheDesc(dtype=L.DT_BF16, layers=1, kv_heads=1, head_dim=64, page_size=16, num_pages=8, max_seqs=4, max_pages=4)
        buffers = L.CacheBuffers(up(self.k), up(self.v), w, w + 64, w + 128)
        self.h = ctypes.c_void_p()
        assert lib.tb_cache_create(ctx, ctypes.byref(desc), ctypes.byref(buffers), ctypes.byref(self.h)) == 0, lib.tb_last_error()
