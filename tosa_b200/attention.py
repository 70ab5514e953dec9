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


import torch

from . import _lib as L

_DTYPES = {torch.bfloat16: L.DT_BF16, torch.float16: L.DT_FP16}
_INT32 = torch.int32
_F32 = torch.float32


def _refuse(status: int, message: str):
    raise L.TbError(status, message)


def _dtype(t, op):
    code = _DTYPES.get(t)
    if code is None:
        _refuse(L.TB_ERR_DTYPE_MISMATCH, f"{op}: unsupported type {t} (float16 or bfloat16)")
    return code


# Small calls take a few microseconds on the GPU, so the checks that every call makes are written to be
# quick: one look at each tensor, and the reason of a refusal is worked out only when there is one.

def _heads(op, name, t, dtype, device, rows=None, heads=None, dim=None):
    """Checks a [rows, heads, head_dim] tensor on device number `device` whose heads are contiguous (None: any
    number); returns its token and head strides."""
    try:
        n, h, d = t.shape
        token, head, last = t.stride()
    except ValueError:
        n = None
    if (n is None or t.dtype is not dtype or t.get_device() != device or last != 1 or (rows is not None and n != rows)
            or (heads is not None and h != heads) or (dim is not None and d != dim)):
        if t.dtype is not dtype:
            _refuse(L.TB_ERR_DTYPE_MISMATCH, f"{op}: {name} is {t.dtype}, not {dtype}")
        if t.get_device() != device:
            _refuse(L.TB_ERR_INVALID_ARGUMENT, f"{op}: {name} is on {t.device}, not on device {device}")
        if t.dim() == 3 and t.stride(2) != 1:
            _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: the last dimension of {name} must be contiguous")
        _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: {name} has shape {tuple(t.shape)}")
    # the stride of a dimension of one element says nothing
    return (token if n > 1 else h * d), (head if h > 1 else d)


def _index(op, name, t, n, device):
    """Checks a contiguous int32 vector of n (None: any number) on the device; returns its length."""
    if t.dtype is not _INT32 or t.dim() != 1 or (n is not None and t.numel() != n) or not t.is_contiguous():
        _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: {name} must be a contiguous int32 vector" + ("" if n is None else f" of {n}"))
    if t.get_device() != device:
        _refuse(L.TB_ERR_INVALID_ARGUMENT, f"{op}: {name} is on {t.device}, not on device {device}")
    return t.numel()


def _sums(op, lse, rows, columns, device):
    if lse.dtype is not _F32 or tuple(lse.shape) != (rows, columns) or not lse.is_contiguous() or lse.get_device() != device:
        _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: lse must be contiguous float32 of ({rows}, {columns})")


# The current stream's handle; torch.cuda.current_stream() makes a stream object first, a few microseconds.
_current = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _on(stream, device, *tensors):
    """The raw stream a call runs on. Tensors that meet another stream than the current one are held
    for it by the allocator until the call's work is done."""
    if stream is None:
        return _current(device)
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return stream.cuda_stream


def attention(ctx, q, k, v, cu_q, cu_k, *, causal=True, scale=None, out=None, lse=None, stream=None):
    """Attention of packed sequences (tb_attention): q [total_q, q_heads, head_dim], k and v
    [total_k, kv_heads, head_dim], cu_q and cu_k int32 offsets of batch + 1. Returns (out, lse), out
    like q, lse float32 [q_heads, total_q]. `scale` defaults to 1 / sqrt(head_dim)."""
    op = "attention"
    dtype = q.dtype
    code = _dtype(dtype, op)
    device = q.get_device()
    q_token, q_head = _heads(op, "q", q, dtype, device)
    rows, heads, dim = q.shape
    k_token, k_head = _heads(op, "k", k, dtype, device, None, None, dim)
    keys, kv_heads, _ = k.shape
    v_token, v_head = _heads(op, "v", v, dtype, device, keys, kv_heads, dim)
    offsets = _index(op, "cu_q", cu_q, None, device)
    _index(op, "cu_k", cu_k, offsets, device)
    if offsets < 1:
        _refuse(L.TB_ERR_SHAPE_MISMATCH, f"{op}: cu_q needs batch + 1 offsets")
    if out is None:
        out, o_token, o_head = torch.empty((rows, heads, dim), dtype=dtype, device=q.device), heads * dim, dim
    else:
        o_token, o_head = _heads(op, "out", out, dtype, device, rows, heads, dim)
    if lse is None:
        lse = torch.empty((heads, rows), dtype=_F32, device=q.device)
    else:
        _sums(op, lse, heads, rows, device)
    d = L.AttentionDesc(code, offsets - 1, heads, kv_heads, dim, 1 if causal else 0, dim ** -0.5 if scale is None else scale,
                        rows, keys, q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head)
    L.check(L.load().tb_attention(ctx.h, d, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(),
                          out.data_ptr(), lse.data_ptr(), _on(stream, device, q, k, v, cu_q, cu_k, out, lse)))
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
        self._device = k_pages.get_device()
        self._lib = L.load()
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
        return _index(op, name, t, n, self._device)

    def reserve(self, slots, counts=None, *, stream=None):
        """Grow slots[i] by counts[i] tokens (one each by default)."""
        n = self._slots("cache reserve", "slots", slots)
        if counts is not None:
            self._slots("cache reserve", "counts", counts, n)
        L.check(self._lib.tb_cache_reserve(self.h, slots.data_ptr(), None if counts is None else counts.data_ptr(), n,
                                           _on(stream, self._device, slots, counts)))

    def write(self, layer, slots, offsets, k, v, *, stream=None):
        """Rows offsets[i]..offsets[i+1] of k and v are the last tokens of slots[i]."""
        op, device = "cache write", self._device
        n = self._slots(op, "slots", slots)
        self._slots(op, "offsets", offsets, n + 1)
        _, _, heads, _, dim = self.k_pages.shape
        dtype = self.k_pages.dtype
        k_token, k_head = _heads(op, "k", k, dtype, device, None, heads, dim)
        rows = k.shape[0]
        v_token, v_head = _heads(op, "v", v, dtype, device, rows, heads, dim)
        L.check(self._lib.tb_cache_write(self.h, layer, slots.data_ptr(), offsets.data_ptr(), n, rows, k.data_ptr(),
                                         k_token, k_head, v.data_ptr(), v_token, v_head,
                                         _on(stream, device, slots, offsets, k, v)))

    def attend(self, layer, slots, q, *, scale=None, out=None, lse=None, stream=None):
        """Attention of one new token q [n, q_heads, head_dim] a slot. Returns (out, lse), out like q,
        lse float32 [n, q_heads]."""
        op, device = "cache attend", self._device
        n = self._slots(op, "slots", slots)
        dtype, dim = self.k_pages.dtype, self.k_pages.shape[4]
        q_seq, q_head = _heads(op, "q", q, dtype, device, n, None, dim)
        heads = q.shape[1]
        if out is None:
            out, o_seq, o_head = torch.empty((n, heads, dim), dtype=dtype, device=q.device), heads * dim, dim
        else:
            o_seq, o_head = _heads(op, "out", out, dtype, device, n, heads, dim)
        if lse is None:
            lse = torch.empty((n, heads), dtype=_F32, device=q.device)
        else:
            _sums(op, lse, n, heads, device)
        L.check(self._lib.tb_cache_attend(self.h, layer, slots.data_ptr(), n, heads, dim ** -0.5 if scale is None else scale,
                                          q.data_ptr(), q_seq, q_head, out.data_ptr(), o_seq, o_head, lse.data_ptr(),
                                          _on(stream, device, slots, q, out, lse)))
        return out, lse

    def fork(self, parents, children, *, stream=None):
        """children[i] becomes a copy of parents[i]; full pages are shared."""
        n = self._slots("cache fork", "parents", parents)
        self._slots("cache fork", "children", children, n)
        L.check(self._lib.tb_cache_fork(self.h, parents.data_ptr(), children.data_ptr(), n,
                                        _on(stream, self._device, parents, children)))

    def free(self, slots, *, stream=None):
        """Empty the slots."""
        n = self._slots("cache free", "slots", slots)
        L.check(self._lib.tb_cache_free(self.h, slots.data_ptr(), n, _on(stream, self._device, slots)))

    def copy_pages(self, src, dst, *, stream=None):
        """Copy the contents of pages src[i] to pages dst[i]."""
        n = self._slots("cache copy_pages", "src", src)
        self._slots("cache copy_pages", "dst", dst, n)
        L.check(self._lib.tb_cache_copy_pages(self.h, src.data_ptr(), dst.data_ptr(), n, _on(stream, self._device, src, dst)))

    def compact(self, page_table=None, refs=None, *, stream=None):
        """Move the pages in use to the front, in place or with the new table and counts in other tensors."""
        for name, t, own in (("page_table", page_table, self.page_table), ("refs", refs, self.refs)):
            if t is not None and (t.dtype is not _INT32 or t.shape != own.shape or not t.is_contiguous() or t.get_device() != self._device):
                _refuse(L.TB_ERR_SHAPE_MISMATCH, f"cache compact: {name} must be like the cache's own")
        L.check(self._lib.tb_cache_compact(self.h, None if page_table is None else page_table.data_ptr(),
                                           None if refs is None else refs.data_ptr(),
                                           _on(stream, self._device, page_table, refs)))
