"""What the torch form of attention and the cache refuses before anything reaches the library, without a GPU."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from tosa_b200 import _lib as L  # noqa: E402
from tosa_b200.attention import PagedCache, attention  # noqa: E402


class Handle:
    """A context with a handle that nothing may look behind."""

    def __init__(self, device=0):
        self.h, self.device = ctypes.c_void_p(1 << 12), device


def _call(ctx=None, **kw):
    # (a head_dim that the library refuses first thing, should the call get there)
    t = dict(q=torch.zeros(4, 2, 24).half(), k=torch.zeros(6, 1, 24).half(), v=torch.zeros(6, 1, 24).half(),
             cu_q=torch.tensor([0, 4], dtype=torch.int32), cu_k=torch.tensor([0, 6], dtype=torch.int32))
    t.update(kw)
    with pytest.raises(L.TbError) as e:
        attention(ctx or Handle(), **t)
    return e.value


def test_tensors_that_are_not_on_a_gpu():
    e = _call()
    assert e.kind == "InvalidArgument" and "cpu" in str(e)


@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_a_gradient_that_would_be_lost(name):
    """There is no backward pass: results would come without a gradient, silently."""
    rows = 6 if name in "kv" else 4
    t = {name: torch.zeros(rows, 1 if name in "kv" else 2, 24).half().requires_grad_()}
    e = _call(**t)
    assert e.kind == "InvalidArgument" and "gradient" in str(e) and f": {name} " in str(e)
    with torch.no_grad():
        assert "gradient" not in str(_call(**t))


@pytest.mark.parametrize("op", ["reserve", "write", "attend", "fork", "free", "copy_pages"])
def test_a_cache_whose_context_is_closed(op):
    """The library's cache points into its context. (What stands for one here is zeros, and the calls have nothing to do.)"""
    zeros = ctypes.create_string_buffer(1 << 12)
    c = PagedCache.__new__(PagedCache)
    c.h, c.ctx = ctypes.c_void_p(ctypes.addressof(zeros)), Handle()
    c.ctx.h = None
    c.k_pages = torch.zeros(1, 4, 1, 8, 64).half()
    none, x = torch.zeros(0, dtype=torch.int32), torch.zeros(0, 1, 64).half()
    args = dict(write=(0, none, torch.zeros(1, dtype=torch.int32), x, x), attend=(0, none, x), fork=(none, none), copy_pages=(none, none))
    try:
        with pytest.raises(L.TbError) as e:
            getattr(c, op)(*args.get(op, (none,)))
        assert e.value.kind == "InvalidArgument" and "closed" in str(e.value)
    finally:
        c.h = None
