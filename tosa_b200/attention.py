"""Attention over packed prompts and a paged key-value cache, on torch tensors.

The Python form of the header's tb_attention and tb_cache_* entry points:

    out, lse = attention(ctx, q, k, v, cu_q, cu_k, causal=True)

    cache = PagedCache.allocate(ctx, layers=2, num_pages=512, page_size=16, kv_heads=8, head_dim=128,
                                dtype=torch.bfloat16, max_seqs=64, max_pages=128)
    cache.reserve(slots, counts)                  # grow sequences, taking pages
    cache.write(layer, slots, offsets, k, v)      # keys and values of the new tokens
    out, lse = cache.attend(layer, slots, q)      # one new token a sequence
    cache.fork(parents, children); cache.free(slots); cache.compact()

Index tensors are int32 on the device. Calls are asynchronous on the current
stream, or on `stream`; what a kernel finds wrong in an index tensor is raised
by the next ctx.synchronize(). Everything that can be seen on the host (types,
shapes, strides, alignment) raises TbError at the call. There is no backward
pass: a tensor that requires a gradient is refused outside torch.no_grad().
"""

from __future__ import annotations

import ctypes
import os

import torch

from . import _lib as L

if not os.path.exists(os.path.join(L.HERE, "_torch_binding.so")):
    raise OSError("tosa_b200/_torch_binding.so is missing: build it with `python -m tosa_b200.build`")
from . import _torch_binding as _native  # noqa: E402

_native.init(L.TbError)


def _refuse(status: int, message: str):
    raise L.TbError(status, message)


def _hold(stream, *tensors):
    """Tensors that a call on another stream uses are held for it by the allocator until its work is done."""
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.is_cuda:
            t.record_stream(stream)


def _results_on(stream, call, *tensors):
    """The results of `call`, allocated with `stream` current: a block of the caller's stream may still be in use there
    by work queued before it was freed, and nothing orders that work with `stream`. The results are held for the
    caller's stream, where they are used next."""
    caller = torch.cuda.current_stream(stream.device)
    with torch.cuda.stream(stream):
        results = call(stream.cuda_stream)
    _hold(stream, *tensors, *results)
    _hold(caller, *results)
    return results


def attention(ctx, q, k, v, cu_q, cu_k, *, causal=True, scale=None, out=None, lse=None, stream=None):
    """Attention of packed sequences (tb_attention): q [total_q, q_heads, head_dim], k and v
    [total_k, kv_heads, head_dim], cu_q and cu_k int32 offsets of batch + 1. Returns (out, lse), out
    like q, lse float32 [q_heads, total_q]. `scale` defaults to 1 / sqrt(head_dim)."""
    if stream is None:
        return _native.attention(ctx, q, k, v, cu_q, cu_k, causal, scale, out, lse, None)
    return _results_on(stream, lambda s: _native.attention(ctx, q, k, v, cu_q, cu_k, causal, scale, out, lse, s),
                       q, k, v, cu_q, cu_k)


class PagedCache:
    """Keys and values of up to max_seqs sequences in pages (tb_cache). The tensors are the caller's:
    k_pages and v_pages [layers, num_pages, kv_heads, page_size, head_dim], page_table int32
    [max_seqs, max_pages], lengths int32 [max_seqs], refs int32 [num_pages]. Calls on one cache must
    not overlap on the GPU."""

    def __init__(self, ctx, k_pages, v_pages, page_table, lengths, refs):
        op = "cache"
        code = {torch.bfloat16: L.DT_BF16, torch.float16: L.DT_FP16}.get(k_pages.dtype)
        if code is None:
            _refuse(L.TB_ERR_DTYPE_MISMATCH, f"{op}: unsupported type {k_pages.dtype} (float16 or bfloat16)")
        if v_pages.dtype != k_pages.dtype:
            _refuse(L.TB_ERR_DTYPE_MISMATCH, f"{op}: k_pages are {k_pages.dtype}, v_pages {v_pages.dtype}")
        if k_pages.dim() != 5 or v_pages.shape != k_pages.shape:
            _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: k_pages and v_pages must be [layers, num_pages, kv_heads, page_size, head_dim]")
        if page_table.dim() != 2 or page_table.shape[0] != lengths.numel() or refs.numel() != k_pages.shape[1]:
            _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: page_table, lengths and refs do not fit each other or the pages")
        for name, t in (("page_table", page_table), ("lengths", lengths), ("refs", refs)):
            if t.dtype != torch.int32:
                _refuse(L.TB_ERR_DTYPE_MISMATCH, f"{op}: {name} must be int32")
        for t in (k_pages, v_pages, page_table, lengths, refs):
            if not t.is_contiguous():
                _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: buffers must be contiguous")
            if t.device != k_pages.device or not t.is_cuda:
                _refuse(L.TB_ERR_INVALID_ARGUMENT, f"{op}: buffers must be on one CUDA device")
        layers, num_pages, kv_heads, page_size, head_dim = k_pages.shape
        self.ctx = ctx
        self.k_pages, self.v_pages = k_pages, v_pages
        self.page_table, self.lengths, self.refs = page_table, lengths, refs
        d = L.CacheDesc(code, layers, kv_heads, head_dim, page_size, num_pages, page_table.shape[0], page_table.shape[1])
        b = L.CacheBuffers(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), refs.data_ptr())
        h = ctypes.c_void_p()
        self.h = None
        self._destroy_left()
        with torch.cuda.device(k_pages.device):
            L.check(L.load().tb_cache_create(ctx.h, ctypes.byref(d), ctypes.byref(b), ctypes.byref(h)))
        self.h = h

    @classmethod
    def allocate(cls, ctx, *, layers, num_pages, page_size, kv_heads, head_dim, dtype, max_seqs, max_pages):
        """An empty cache with buffers of its own on the context's device."""
        dev = torch.device("cuda", ctx.device)
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        pages = [torch.empty(shape, dtype=dtype, device=dev) for _ in range(2)]
        table = torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=dev)
        return cls(ctx, *pages, table, torch.zeros(max_seqs, dtype=torch.int32, device=dev),
                   torch.zeros(num_pages, dtype=torch.int32, device=dev))

    _left = []  # handles of caches that were closed during a capture

    def close(self):
        """Frees the workspace, after the device's work. That waiting would spoil a graph that the current stream is
        capturing, so a cache that is closed (or collected) then is destroyed with the next one made or closed."""
        if self.h:
            self._left.append(self.h)
            self.h = None
            self._destroy_left()

    @classmethod
    def _destroy_left(cls):
        if cls._left and not torch.cuda.is_current_stream_capturing():
            while cls._left:
                L.load().tb_cache_destroy(cls._left.pop())

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @staticmethod
    def _on(stream, *tensors):
        if stream is None:
            return None
        _hold(stream, *tensors)
        return stream.cuda_stream

    def reserve(self, slots, counts=None, *, stream=None):
        """Grow slots[i] by counts[i] tokens (one each by default)."""
        _native.cache_reserve(self, self.k_pages, slots, counts, self._on(stream, slots, counts))

    def write(self, layer, slots, offsets, k, v, *, stream=None):
        """Rows offsets[i]..offsets[i+1] of k and v are the last tokens of slots[i]."""
        _native.cache_write(self, self.k_pages, layer, slots, offsets, k, v, self._on(stream, slots, offsets, k, v))

    def attend(self, layer, slots, q, *, scale=None, out=None, lse=None, stream=None):
        """Attention of one new token q [n, q_heads, head_dim] a slot. Returns (out, lse), out like q,
        lse float32 [n, q_heads]."""
        if stream is None:
            return _native.cache_attend(self, self.k_pages, layer, slots, q, scale, out, lse, None)
        return _results_on(stream, lambda s: _native.cache_attend(self, self.k_pages, layer, slots, q, scale, out, lse, s),
                           slots, q)

    def fork(self, parents, children, *, stream=None):
        """children[i] becomes a copy of parents[i]; full pages are shared."""
        _native.cache_fork(self, self.k_pages, parents, children, self._on(stream, parents, children))

    def free(self, slots, *, stream=None):
        """Empty the slots."""
        _native.cache_free(self, self.k_pages, slots, self._on(stream, slots))

    def copy_pages(self, src, dst, *, stream=None):
        """Copy the contents of pages src[i] to pages dst[i]."""
        _native.cache_copy_pages(self, self.k_pages, src, dst, self._on(stream, src, dst))

    def compact(self, page_table=None, refs=None, *, stream=None):
        """Move the pages in use to the front, in place or with the new table and counts in other tensors."""
        _native.cache_compact(self, self.page_table, self.refs, page_table, refs, self._on(stream, page_table, refs))
