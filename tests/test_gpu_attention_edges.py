"""Attention and the paged cache where calls meet values that are not finite, other streams, captures and very
large pages."""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tosa_b200 import _lib as L  # noqa: E402
from tosa_b200.attention import PagedCache, attention  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return _ints(at)


def _filled(ctx, lens, heads, d, dtype=torch.bfloat16, page=16, seed=0):
    """A cache that holds the given lengths, its keys and values, and one query row a slot and four to a key head."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = sum(-(-n // page) for n in lens)
    c = PagedCache.allocate(ctx, layers=1, num_pages=pages + 1, page_size=page, kv_heads=heads, head_dim=d, dtype=dtype,
                            max_seqs=len(lens), max_pages=max(-(-n // page) for n in lens) + 1)
    k, v = (torch.randn(sum(lens), heads, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(len(lens), 4 * heads, d, generator=g, device="cuda").to(dtype)
    slots = _ints(range(len(lens)))
    c.reserve(slots, _ints(lens))
    c.write(0, slots, _offsets(lens), k, v)
    return c, slots, q, k, v


# A unit that one CTA finishes, and one that several share.
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", ["q", "every key", "one key"])
@pytest.mark.parametrize("lens", [[40, 50, 30], [5000, 9000, 7000]], ids=["whole", "split"])
def test_scores_of_nan_make_the_rows_sum_nan(ctx, lens, where, d):
    """exp(NaN) is NaN and so is the logarithm of a sum with it; -inf is the sum of a row without keys. Other rows keep theirs."""
    c, slots, q, k, v = _filled(ctx, lens, 2, d)
    want, wlse = c.attend(0, slots, q)
    if where == "q":
        q[1, :4, 3] = math.nan  # the first key head's rows of slot 1
    else:
        rows = slice(lens[0], lens[0] + lens[1]) if where == "every key" else lens[0] + lens[1] // 2
        k[rows, 0, 3] = math.nan
        c.write(0, slots, _offsets(lens), k, v)
    out, lse = c.attend(0, slots, q)
    ctx.synchronize()
    assert torch.isnan(out[1, :4]).all() and torch.isnan(lse[1, :4]).all()
    assert torch.equal(out[1, 4:], want[1, 4:]) and torch.equal(lse[1, 4:], wlse[1, 4:])
    assert torch.equal(out[[0, 2]], want[[0, 2]]) and torch.equal(lse[[0, 2]], wlse[[0, 2]])


def _busy(tensor):
    """Work on the current stream that lasts some milliseconds and then writes all of `tensor`."""
    x = torch.ones(1 << 28, device="cuda")
    for _ in range(20):
        x.add_(1.0)
    tensor.fill_(7.0)


@pytest.mark.parametrize("op", ["prompt", "token"])
def test_results_on_another_stream_are_not_memory_in_use(ctx, op):
    """A block that was freed while work queued on the caller's stream still writes it is no place for results that
    another stream writes at once."""
    if op == "prompt":
        q, k, v = (torch.randn(2048, h, 128, device="cuda").bfloat16() for h in (8, 2, 2))
        cu = _offsets([2048])
        call = lambda **kw: attention(ctx, q, k, v, cu, cu, **kw)  # noqa: E731
    else:
        c, slots, q, k, v = _filled(ctx, [200 + i for i in range(256)], 2, 128)
        call = lambda **kw: c.attend(0, slots, q, **kw)  # noqa: E731
    want, wlse = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for one in (want, wlse):
        last = torch.empty_like(one)
        place = last.data_ptr()
        _busy(last)
        del last
        out, lse = call(stream=side)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, wlse)
        assert place not in (out.data_ptr(), lse.data_ptr())


def test_results_given_by_the_caller_are_used_on_another_stream(ctx):
    q, k, v = (torch.randn(300, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
    cu = _offsets([300])
    want, wlse = attention(ctx, q, k, v, cu, cu)
    out, lse = torch.zeros_like(want), torch.zeros_like(wlse)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = attention(ctx, q, k, v, cu, cu, out=out, lse=lse, stream=side)
    side.synchronize()
    assert got[0] is out and got[1] is lse and torch.equal(out, want) and torch.equal(lse, wlse)


@pytest.mark.parametrize("collected", [True, False])
def test_a_cache_that_ends_during_a_capture_leaves_the_graph_whole(ctx, collected):
    caches = [PagedCache.allocate(ctx, layers=1, num_pages=4, page_size=16, kv_heads=1, head_dim=64, dtype=torch.bfloat16,
                                  max_seqs=2, max_pages=2) for _ in range(2)]
    q, k, v = (torch.randn(50, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
    cu = _offsets([50])
    want, wlse = attention(ctx, q, k, v, cu, cu)
    out, lse = torch.zeros_like(want), torch.zeros_like(wlse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention(ctx, q, k, v, cu, cu, out=out, lse=lse)
        if collected:
            del caches[0]
        else:
            caches[0].close()
            assert caches[0].h is None
    assert len(PagedCache._left) == 1
    graph.replay()
    ctx.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    caches[-1].close()  # and with it the other one
    assert not PagedCache._left


def test_tensors_on_another_device_than_the_contexts(ctx):
    class Elsewhere:
        h, device = ctx.h, ctx.device + 1

    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(L.TbError) as e:
        attention(Elsewhere(), q, q, q, _offsets([4]), _offsets([4]))
    assert e.value.kind == "InvalidArgument"


def test_pages_of_more_than_32_bits_of_vectors(ctx):
    """Pages of 2^27 tokens of 128, 2^31 vectors of 16 bytes each: a write to the second head of one, a copy of a whole
    one. Keys and values are the same memory here, with the same contents, so that 64 GB are enough."""
    tokens = 1 << 27
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip("needs 70 GB of free memory")
    memory = torch.empty(2 * tokens * 128, dtype=torch.bfloat16, device="cuda")
    table, lengths, refs = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), _ints([tokens]), _ints([1])
    pages = memory.view(1, 1, 2, tokens, 128)
    c = PagedCache(ctx, pages, pages, table, lengths, refs)
    pages[0, 0, :, -6:] = 0
    x = torch.randn(5, 2, 128, device="cuda").bfloat16()
    c.write(0, _ints([0]), _ints([0, 5]), x, x)
    ctx.synchronize()
    assert torch.equal(pages[0, 0, :, -5:], x.transpose(0, 1)) and (pages[0, 0, :, -6] == 0).all()
    c.close()
    pages = memory.view(1, 2, 1, tokens, 128)
    c = PagedCache(ctx, pages, pages, table, lengths, _ints([1, 0]))
    places = [0, 1, 12345677, tokens // 2, tokens - 2, tokens - 1]
    x = torch.randn(len(places), 128, device="cuda").bfloat16()
    for i, at in enumerate(places):
        pages[0, 0, 0, at] = x[i]
    c.copy_pages(_ints([0]), _ints([1]))
    ctx.synchronize()
    assert all(torch.equal(pages[0, 1, 0, at], x[i]) for i, at in enumerate(places))
    c.close()
    del pages, memory, c
    torch.cuda.empty_cache()


@pytest.mark.parametrize("heads,d", [(2, 128), (1, 64)])
def test_attend_under_a_bound_of_zero_is_right_or_says_that_a_wait_ran_out(heads, d):
    """Its waits are for copies of some microseconds, which the first look at a barrier may outlast: a wait that gives up
    cannot be brought about at will. Where one does, the kernel goes through its units without data, its loads land and
    the next synchronize reports it. The call after that is right either way."""
    lib, ctx = L.load(), L.Context(0)
    c, slots, q, k, v = _filled(ctx, [5000, 70, 9000], heads, d)
    want, wlse = c.attend(0, slots, q)
    ctx.synchronize()
    for _ in range(20):
        L.check(lib.tb_context_set_wait_timeout_ms(ctx.h, 0.0))
        out, lse = c.attend(0, slots, q)
        try:
            ctx.synchronize()
        except L.TbError as e:
            assert e.kind == "Timeout"
        else:
            assert torch.equal(out, want) and torch.equal(lse, wlse)
        L.check(lib.tb_context_set_wait_timeout_ms(ctx.h, 2000.0))
        out, lse = c.attend(0, slots, q)
        ctx.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, wlse)
    c.close()
    ctx.close()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,at", [(40, 3), (40, 39), (5000, 0), (5000, 31), (5000, 64), (5000, 4999)])
def test_infinite_scores_of_one_new_token_and_of_a_prompts_row(ctx, n, at, d):
    """Every score -inf: 0 divided by 0, and the logarithm of 0. One of +inf, anywhere: infinity by infinity. In one CTA and
    in several, in the first 32 keys and after them."""
    lens = [n, n, 50]
    c, slots, q, k, v = _filled(ctx, lens, 1, d)
    q[:2], k[:2 * n] = q[:2].abs(), k[:2 * n].abs()
    want, wlse = c.attend(0, slots, q)
    k[:n, :, 5] = -math.inf
    k[n + at, :, 5] = math.inf
    c.write(0, slots, _offsets(lens), k, v)
    out, lse = c.attend(0, slots, q)
    rows, rlse = attention(ctx, q, k, v, _offsets([1, 1, 1]), _offsets(lens))
    ctx.synchronize()
    for o, s in ((out, lse), (rows, rlse.T)):
        assert torch.isnan(o[0]).all() and (s[0] == -math.inf).all()
        assert torch.isnan(o[1]).all() and torch.isnan(s[1]).all()
        assert torch.isfinite(o[2]).all() and torch.isfinite(s[2]).all()
    assert torch.equal(out[2], want[2]) and torch.equal(lse[2], wlse[2])
