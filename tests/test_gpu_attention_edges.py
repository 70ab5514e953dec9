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
