"""Which device the library's host code waits for, allocates and launches on, without a GPU (fake_cuda.py)."""

import pytest

from tests import fake_cuda as F


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
