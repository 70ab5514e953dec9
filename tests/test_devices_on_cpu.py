"""Which device the library's host code waits for, allocates and launches on, without a GPU (fake_cuda.py)."""

import ctypes

import pytest

from tests import fake_cuda as F
from tosa_b200 import _lib as L


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return F.load(tmp_path_factory.mktemp("fake"))


@pytest.fixture
def contexts(lib):
    both = [F.context(lib, d) for d in (0, 1)]
    yield both
    for h in both:
        lib.tb_context_destroy(h)


def test_a_cache_waits_for_its_own_device(lib, contexts):
    """Its workspace may go to another cache of its context, so it is its context's device that has to be through,
    whichever is current; and the current one stays current."""
    lib.fake_set_device(0)
    cache = F.HostCache(lib, contexts[0])
    lib.fake_set_device(1)
    F.events(lib)
    lib.tb_cache_destroy(cache.h)
    assert F.events(lib) == ["synchronize 0", "free on 0"]
    assert lib.fake_device() == 1


def test_a_cache_may_outlive_its_context(lib):
    ctx = F.context(lib, 0)
    lib.fake_set_device(0)
    cache = F.HostCache(lib, ctx)
    lib.tb_context_destroy(ctx)
    lib.fake_set_device(1)
    F.events(lib)
    lib.tb_cache_destroy(cache.h)
    assert F.events(lib) == ["synchronize 0", "free on 0"]


def test_a_workspace_whose_calls_may_still_run_is_not_freed(lib, contexts):
    """A device cannot be waited for while one of its streams is captured."""
    lib.fake_set_device(0)
    cache = F.HostCache(lib, contexts[0])
    F.events(lib)
    lib.fake_sync_result(900)
    lib.tb_cache_destroy(cache.h)
    lib.fake_sync_result(0)
    assert F.events(lib) == ["synchronize 0"]


def test_calls_launch_on_the_contexts_device_only(lib, contexts):
    lib.fake_set_device(0)
    cache = F.HostCache(lib, contexts[0])
    up = (ctypes.addressof(cache.k) + 255) & ~255
    desc = L.AttentionDesc(dtype=L.DT_BF16, batch=1, q_heads=2, kv_heads=1, head_dim=64, causal=1, scale=0.125, total_q=4, total_k=4,
                           q_token_stride=128, q_head_stride=64, k_token_stride=64, k_head_stride=64, v_token_stride=64,
                           v_head_stride=64, out_token_stride=128, out_head_stride=64)
    calls = [
        lambda: lib.tb_attention(contexts[0], ctypes.byref(desc), up, up, up, up, up, up, None, None),
        lambda: lib.tb_cache_reserve(cache.h, up, None, 1, None),
        lambda: lib.tb_cache_write(cache.h, 0, up, up, 1, 1, up, 64, 64, up, 64, 64, None),
        lambda: lib.tb_cache_attend(cache.h, 0, up, 1, 1, 0.125, up, 64, 64, up, 64, 64, None, None),
        lambda: lib.tb_cache_fork(cache.h, up, up, 1, None),
        lambda: lib.tb_cache_free(cache.h, up, 1, None),
        lambda: lib.tb_cache_copy_pages(cache.h, up, up, 1, None),
        lambda: lib.tb_cache_compact(cache.h, None, None, None),
    ]
    F.events(lib)
    for i, call in enumerate(calls):
        lib.fake_set_device(1)
        assert call() == L.TB_ERR_INVALID_ARGUMENT, i
        assert F.events(lib) == [], i
        lib.fake_set_device(0)
        assert call() == 0, (i, lib.tb_last_error())
        assert set(F.events(lib)) == {"launch on 0"}, i
    lib.tb_cache_destroy(cache.h)


def test_sizes_whose_indexes_pass_32_bits_are_refused(lib, contexts):
    """A token's key of 2^31 vectors of 16 bytes, and a write of more slots than the search of their offsets can count."""
    lib.fake_set_device(0)
    cache = F.HostCache(lib, contexts[0])
    w = ctypes.addressof(cache.words)
    desc = L.CacheDesc(dtype=L.DT_BF16, layers=1, kv_heads=1 << 27, head_dim=128, page_size=8, num_pages=1, max_seqs=1, max_pages=1)
    up = (ctypes.addressof(cache.k) + 255) & ~255
    buffers, h = L.CacheBuffers(up, up, w, w, w), ctypes.c_void_p()
    assert lib.tb_cache_create(contexts[0], ctypes.byref(desc), ctypes.byref(buffers), ctypes.byref(h)) == L.TB_ERR_NOT_ACCELERATED
    assert not h.value
    F.events(lib)
    assert lib.tb_cache_write(cache.h, 0, up, up, 2**31 - 1, 1, up, 64, 64, up, 64, 64, None) == L.TB_ERR_NOT_ACCELERATED
    assert F.events(lib) == []
    lib.tb_cache_destroy(cache.h)


def test_every_device_gets_the_shared_memory_that_a_kernel_needs(lib, contexts):
    """The limit of a function's dynamic shared memory is each device's own: one process may have contexts on several."""
    for device, ctx in enumerate(contexts):
        lib.fake_set_device(device)
        cache = F.HostCache(lib, ctx)
        up = (ctypes.addressof(cache.k) + 255) & ~255
        heads = L.AttentionDesc(dtype=L.DT_FP16, batch=1, q_heads=2, kv_heads=1, head_dim=128, causal=1, scale=0.125, total_q=4,
                                total_k=4, q_token_stride=256, q_head_stride=128, k_token_stride=128, k_head_stride=128,
                                v_token_stride=128, v_head_stride=128, out_token_stride=256, out_head_stride=128)
        product = L.MatmulDesc(n=1, h=64, c=64, w=64, a_dtype=L.DT_BF16, b_dtype=L.DT_BF16, out_dtype=L.DT_FP32)
        F.events(lib)
        assert lib.tb_attention(ctx, ctypes.byref(heads), up, up, up, up, up, up, None, None) == 0, (device, lib.tb_last_error())
        assert lib.tb_cache_attend(cache.h, 0, up, 1, 2, 0.125, up, 128, 64, up, 128, 64, None, None) == 0, (device, lib.tb_last_error())
        assert lib.tb_matmul_t(ctx, product, 1, None, up, up, up, None) == 0, (device, lib.tb_last_error())
        assert set(F.events(lib)) == {f"launch on {device}"}
        lib.tb_cache_destroy(cache.h)
