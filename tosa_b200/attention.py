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
shapes, strides, alignment) raises TbError at the call.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib as L

_DTYPES = {torch.bfloat16: L.DT_BF16, torch.float16: L.DT_FP16}


def _refuse(status: int, message: str):
    raise L.TbError(status, message)


def _dtype(t, op):
    code = _DTYPES.get(t)
    if code is None:
        _refuse(L.TB_ERR_DTYPE_MISMATCH, f"{op}: unsupported type {t} (float16 or bfloat16)")
    return code


def _heads(op, name, t, dtype, device, rows=None, heads=None, dim=None):
    """Checks a [rows, heads, head_dim] tensor whose heads are contiguous; returns its token and head strides."""
    if t.dtype != dtype:
        _refuse(L.TB_ERR_DTYPE_MISMATCH, f"{op}: {name} is {t.dtype}, not {dtype}")
    if t.device != device:
        _refuse(L.TB_ERR_INVALID_ARGUMENT, f"{op}: {name} is on {t.device}, not on {device}")
    if t.dim() != 3 or any(w is not None and w != g for w, g in zip((rows, heads, dim), t.shape)):
        _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: {name} has shape {tuple(t.shape)}")
    if t.stride(2) != 1:
        _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: the last dimension of {name} must be contiguous")
    # the stride of a dimension of one element says nothing
    token, head = t.stride(0), t.stride(1)
    return (token if t.shape[0] > 1 else t.shape[1] * t.shape[2]), (head if t.shape[1] > 1 else t.shape[2])


def _index(op, name, t, n, device):
    if t.dtype != torch.int32 or t.dim() != 1 or (n is not None and t.shape[0] != n) or not t.is_contiguous():
        _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: {name} must be a contiguous int32 vector" + ("" if n is None else f" of {n}"))
    if t.device != device:
        _refuse(L.TB_ERR_INVALID_ARGUMENT, f"{op}: {name} is on {t.device}, not on {device}")


def _on(stream, tensors):
    """The raw stream a call runs on. Tensors that meet another stream than the current one are held
    for it by the allocator until the call's work is done."""
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return stream.cuda_stream


def attention(ctx, q, k, v, cu_q, cu_k, *, causal=True, scale=None, out=None, lse=None, stream=None):
    """Attention of packed sequences (tb_attention): q [total_q, q_heads, head_dim], k and v
    [total_k, kv_heads, head_dim], cu_q and cu_k int32 offsets of batch + 1. Returns (out, lse), out
    like q, lse float32 [q_heads, total_q]. `scale` defaults to 1 / sqrt(head_dim)."""
    op = "attention"
    code = _dtype(q.dtype, op)
    device = q.device
    sq = _heads(op, "q", q, q.dtype, device)
    rows, heads, dim = q.shape
    sk = _heads(op, "k", k, q.dtype, device, dim=dim)
    sv = _heads(op, "v", v, q.dtype, device, k.shape[0], k.shape[1], dim)
    _index(op, "cu_q", cu_q, None, device)
    _index(op, "cu_k", cu_k, cu_q.shape[0], device)
    if cu_q.shape[0] < 1:
        _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: cu_q needs batch + 1 offsets")
    if out is None:
        out, so = torch.empty((rows, heads, dim), dtype=q.dtype, device=device), (heads * dim, dim)
    else:
        so = _heads(op, "out", out, q.dtype, device, rows, heads, dim)
    if lse is None:
        lse = torch.empty((heads, rows), dtype=torch.float32, device=device)
    elif lse.dtype != torch.float32 or tuple(lse.shape) != (heads, rows) or not lse.is_contiguous() or lse.device != device:
        _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: lse must be contiguous float32 of ({heads}, {rows})")
    d = L.AttentionDesc(code, cu_q.shape[0] - 1, heads, k.shape[1], dim, int(bool(causal)),
                        1.0 / math.sqrt(dim) if scale is None else scale, rows, k.shape[0],
                        sq, sk, sv, so)
    s = _on(stream, (q, k, v, cu_q, cu_k, out, lse))
    L.check(L.load().tb_attention(ctx.h, ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(),
                                  cu_k.data_ptr(), out.data_ptr(), lse.data_ptr(), s))
    return out, lse


class PagedCache:
    """Keys and values of up to max_seqs sequences in pages (tb_cache). The tensors are the caller's:
    k_pages and v_pages [layers, num_pages, kv_heads, page_size, head_dim], page_table int32
    [max_seqs, max_pages], lengths int32 [max_seqs], refs int32 [num_pages]. Calls on one cache must
    not overlap on the GPU."""

    def __init__(self, ctx, k_pages, v_pages, page_table, lengths, refs):
        op = "cache"
        code = _dtype(k_pages.dtype, op)
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
        self._default_scale = 1.0 / math.sqrt(head_dim)
        d = L.CacheDesc(code, layers, kv_heads, head_dim, page_size, num_pages, page_table.shape[0], page_table.shape[1])
        b = L.CacheBuffers(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), refs.data_ptr())
        h = ctypes.c_void_p()
        self.h = None
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

    def close(self):
        if self.h:
            L.load().tb_cache_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _slots(self, op, name, t, n=None):
        _index(op, name, t, n, self.k_pages.device)
        return t.data_ptr()

    def reserve(self, slots, counts=None, *, stream=None):
        """Grow slots[i] by counts[i] tokens (one each by default)."""
        p = self._slots("cache reserve", "slots", slots)
        c = None if counts is None else self._slots("cache reserve", "counts", counts, slots.shape[0])
        L.check(L.load().tb_cache_reserve(self.h, p, c, slots.shape[0], _on(stream, (slots, counts))))

    def write(self, layer, slots, offsets, k, v, *, stream=None):
        """Rows offsets[i]..offsets[i+1] of k and v are the last tokens of slots[i]."""
        op = "cache write"
        p = self._slots(op, "slots", slots)
        o = self._slots(op, "offsets", offsets, slots.shape[0] + 1)
        pages = self.k_pages
        sk = _heads(op, "k", k, pages.dtype, pages.device, None, pages.shape[2], pages.shape[4])
        sv = _heads(op, "v", v, pages.dtype, pages.device, k.shape[0], pages.shape[2], pages.shape[4])
        L.check(L.load().tb_cache_write(self.h, layer, p, o, slots.shape[0], k.shape[0], k.data_ptr(), *sk, v.data_ptr(), *sv,
                                        _on(stream, (slots, offsets, k, v))))

    def attend(self, layer, slots, q, *, scale=None, out=None, lse=None, stream=None):
        """Attention of one new token q [n, q_heads, head_dim] a slot. Returns (out, lse), out like q,
        lse float32 [n, q_heads]."""
        op = "cache attend"
        p = self._slots(op, "slots", slots)
        pages = self.k_pages
        n, heads, dim = slots.shape[0], q.shape[1] if q.dim() == 3 else 0, pages.shape[4]
        sq = _heads(op, "q", q, pages.dtype, pages.device, n, None, dim)
        if out is None:
            out, so = torch.empty((n, heads, dim), dtype=q.dtype, device=q.device), (heads * dim, dim)
        else:
            so = _heads(op, "out", out, q.dtype, q.device, n, heads, dim)
        if lse is None:
            lse = torch.empty((n, heads), dtype=torch.float32, device=q.device)
        elif lse.dtype != torch.float32 or tuple(lse.shape) != (n, heads) or not lse.is_contiguous() or lse.device != q.device:
            _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: lse must be contiguous float32 of ({n}, {heads})")
        L.check(L.load().tb_cache_attend(self.h, layer, p, n, heads, self._default_scale if scale is None else scale,
                                         q.data_ptr(), *sq, out.data_ptr(), *so, lse.data_ptr(), _on(stream, (slots, q, out, lse))))
        return out, lse

    def fork(self, parents, children, *, stream=None):
        """children[i] becomes a copy of parents[i]; full pages are shared."""
        p = self._slots("cache fork", "parents", parents)
        c = self._slots("cache fork", "children", children, parents.shape[0])
        L.check(L.load().tb_cache_fork(self.h, p, c, parents.shape[0], _on(stream, (parents, children))))

    def free(self, slots, *, stream=None):
        """Empty the slots."""
        p = self._slots("cache free", "slots", slots)
        L.check(L.load().tb_cache_free(self.h, p, slots.shape[0], _on(stream, (slots,))))

    def copy_pages(self, src, dst, *, stream=None):
        """Copy the contents of pages src[i] to pages dst[i]."""
        p = self._slots("cache copy_pages", "src", src)
        o = self._slots("cache copy_pages", "dst", dst, src.shape[0])
        L.check(L.load().tb_cache_copy_pages(self.h, p, o, src.shape[0], _on(stream, (src, dst))))

    def compact(self, page_table=None, refs=None, *, stream=None):
        """Move the pages in use to the front, in place or with the new table and counts in other tensors."""
        for name, t, own in (("page_table", page_table, self.page_table), ("refs", refs, self.refs)):
            if t is not None and (t.dtype != torch.int32 or t.shape != own.shape or not t.is_contiguous() or t.device != own.device):
                _refuse(L.TB_ERR_SHAPE_MISMATCH, f"cache compact: {name} must be like the cache's own")
        L.check(L.load().tb_cache_compact(self.h, None if page_table is None else page_table.data_ptr(),
                                          None if refs is None else refs.data_ptr(), _on(stream, (page_table, refs))))
