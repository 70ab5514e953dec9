"""The paged key-value cache: its bookkeeping against a page-by-page model, the contents that its operators
write and move, and the attention of one new token against the definition in 64 bits."""

import ctypes
import math
import random

import numpy as np
import pytest

from tests import attention_oracle as A

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tosa_b200 import _lib as L  # noqa: E402
from tosa_b200.attention import PagedCache, attention  # noqa: E402

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(lens):
    return _ints(np.concatenate([[0], np.cumsum(lens)]).tolist())


def _cache(ctx, dtype="bf16", layers=1, pages=32, page=16, heads=2, d=64, seqs=8, max_pages=8):
    c = PagedCache.allocate(ctx, layers=layers, num_pages=pages, page_size=page, kv_heads=heads, head_dim=d,
                            dtype=DT[dtype], max_seqs=seqs, max_pages=max_pages)
    c.k_pages.fill_(math.nan)  # pages that nothing was written to
    c.v_pages.fill_(math.nan)
    return c


def _state(c):
    return c.page_table.tolist(), c.lengths.tolist(), c.refs.tolist()


def _same(c, m):
    assert c.lengths.tolist() == m.lengths
    assert c.page_table.tolist() == m.rows()
    assert c.refs.tolist() == m.refs


# ---------------------------------------------------------------------------
# One new token
# ---------------------------------------------------------------------------

def _filled(ctx, seed, dtype, lens, hk, d, page, shuffle=True, spare=3):
    """A cache whose slots hold the given lengths in pages in no order; what no token fills is NaN."""
    r = random.Random(seed)
    need = [-(-n // page) for n in lens]
    order = list(range(sum(need) + spare))
    if shuffle:
        r.shuffle(order)
    c = _cache(ctx, dtype, 1, len(order), page, hk, d, len(lens), max(need + [1]))
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.randn(sum(lens), hk, d, generator=g, device="cuda").to(DT[dtype])
    v = torch.randn(sum(lens), hk, d, generator=g, device="cuda").to(DT[dtype])
    table, refs, at = [], [0] * len(order), 0
    for n in need:
        row = order[at:at + n]
        at += n
        for p in row:
            refs[p] = 1
        table.append(row + [-1] * (c.page_table.shape[1] - n))
    c.page_table.copy_(_ints(table))
    c.refs.copy_(_ints(refs))
    c.lengths.copy_(_ints(lens))
    c.write(0, _ints(list(range(len(lens)))), _offsets(lens), k, v)
    return c, k, v


def _check(dtype, q, k, v, lens, slots, scale, out, lse):
    q, k, v, out, lse = (t.detach().double().cpu().numpy() for t in (q, k, v, out, lse))
    start = np.concatenate([[0], np.cumsum(lens)])
    group = q.shape[1] // k.shape[1]
    for i, s in enumerate(slots):
        for h in range(k.shape[1]):
            hs = slice(h * group, (h + 1) * group)
            want, wlse, mean, size, tail = A.attend(q[i, hs], k[start[s]:start[s + 1], h], v[start[s]:start[s + 1], h],
                                                    np.full(group, lens[s]), scale)
            tol, ltol = A.tolerance(dtype, want, mean, size, tail)
            bad = ~(np.abs(out[i, hs] - want) <= tol)
            assert not bad.any(), (i, s, lens[s], h, np.argwhere(bad)[:4], np.abs(out[i, hs] - want).max())
            none = np.isneginf(wlse)
            assert np.array_equal(np.isneginf(lse[i, hs]), none), (i, s, h)
            assert (np.abs(lse[i, hs][~none] - wlse[~none]) <= ltol[~none]).all(), (i, s, h)


ATTEND = [
    # lengths, query heads, key heads, head_dim, page
    ([1], 1, 1, 16, 8),
    ([0, 1, 2], 2, 1, 64, 16),
    ([15, 16, 17, 0, 31, 33], 8, 2, 128, 16),
    ([63, 64, 65, 127, 128, 129], 4, 4, 128, 16),
    ([100, 7, 300], 6, 2, 96, 24),
    ([257, 511, 40], 7, 1, 80, 64),
    ([999], 16, 1, 64, 8),
    ([513, 3], 32, 1, 112, 32),
    ([700, 70], 24, 1, 128, 128),
    ([90, 600], 48, 2, 32, 256),
    ([40] * 70, 4, 2, 48, 16),
    ([5000, 1, 0, 77], 4, 1, 128, 16),
    ([12007], 8, 8, 64, 64),
    ([20011, 19], 8, 2, 128, 72),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{len(c[0])}x{max(c[0])}-h{c[1]}-{c[2]}-d{c[3]}-p{c[4]}")
def test_attend_matches_the_definition(ctx, dtype, case):
    lens, hq, hk, d, page = case
    c, k, v = _filled(ctx, sum(lens) + hq, dtype, lens, hk, d, page)
    slots = list(range(len(lens)))[::-1]
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(len(lens), hq, d, generator=g, device="cuda").to(DT[dtype])
    out, lse = c.attend(0, _ints(slots), q)
    again, lse2 = c.attend(0, _ints(slots), q)
    ctx.synchronize()
    _check(dtype, q, k, v, lens, slots, np.float32(1 / math.sqrt(d)), out, lse)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_attend_rising_scores(ctx):
    lens = [1500]
    c, k, v = _filled(ctx, 2, "bf16", lens, 1, 64, 16)
    k[:, 0, 0] = torch.linspace(-15, 15, 1500, device="cuda").bfloat16()
    c.write(0, _ints([0]), _offsets(lens), k, v)
    q = torch.randn(1, 3, 64, device="cuda").bfloat16()
    q[..., 0] = torch.tensor([8.0, -8.0, 0.5])
    out, lse = c.attend(0, _ints([0]), q, scale=1.0)
    ctx.synchronize()
    _check("bf16", q, k, v, lens, [0], 1.0, out, lse)


def test_attend_equals_the_prompts_last_row(ctx):
    """Both operators within their tolerance of each other, over the same keys."""
    lens = [37, 400, 128]
    c, k, v = _filled(ctx, 3, "bf16", lens, 2, 128, 16)
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    out, lse = c.attend(0, _ints([0, 1, 2]), q)
    want, wlse = attention(ctx, q, k, v, _offsets([1, 1, 1]), _offsets(lens))
    ctx.synchronize()
    _check("bf16", q, k, v, lens, [0, 1, 2], np.float32(1 / math.sqrt(128)), out, lse)
    _check("bf16", q, k, v, lens, [0, 1, 2], np.float32(1 / math.sqrt(128)), want, wlse.T)


def test_attend_layouts_streams_and_graphs(ctx):
    lens = [50, 333]
    c, k, v = _filled(ctx, 4, "f16", lens, 2, 64, 16)
    slots = _ints([1, 0])
    qkv = torch.randn(2, 8 + 4, 64, device="cuda").half()
    q = qkv[:, :8]
    want, wlse = c.attend(0, slots, q.contiguous())
    wide = torch.full((2, 16, 72), 7.0, dtype=torch.float16, device="cuda")
    got, lse = c.attend(0, slots, q, out=wide[:, ::2, :64])
    torch.cuda.synchronize()
    assert torch.equal(want, got) and torch.equal(lse, wlse) and (wide[:, 1::2] == 7).all() and (wide[..., 64:] == 7).all()
    side = torch.cuda.Stream()
    got, _ = c.attend(0, slots, q, stream=side)
    side.synchronize()
    assert torch.equal(want, got)
    out, lse = torch.zeros_like(want), torch.zeros_like(wlse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(0, slots, q, out=out, lse=lse)
    c.lengths.copy_(_ints([17, 300]))  # the lengths are read when the graph runs
    graph.replay()
    ctx.synchronize()
    k2 = torch.cat([k[:17], k[50:350]])
    v2 = torch.cat([v[:17], v[50:350]])
    _check("f16", q, k2, v2, [17, 300], [1, 0], np.float32(0.125), out, lse)


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_attend_values_that_are_not_finite(ctx, value):
    lens = [100, 100]
    c, k, v = _filled(ctx, 5, "bf16", lens, 1, 64, 16)
    q = torch.randn(2, 2, 64, device="cuda").bfloat16()
    want, wlse = c.attend(0, _ints([0, 1]), q)
    v[130, 0, 9] = value
    c.write(0, _ints([0, 1]), _offsets(lens), k, v)
    got, lse = c.attend(0, _ints([0, 1]), q)
    ctx.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(lse, wlse)
    assert not torch.isfinite(got[1, :, 9]).any()
    keep = [x for x in range(64) if x != 9]
    assert torch.equal(got[1][:, keep], want[1][:, keep])


def test_attend_bad_indices_are_reported(ctx):
    lens = [30, 40, 50]
    c, k, v = _filled(ctx, 6, "bf16", lens, 1, 64, 16)
    q = torch.randn(3, 2, 64, device="cuda").bfloat16()
    keep = c.page_table.clone(), c.lengths.clone()

    def refused(slots, *right):
        """The call is refused; the rows of `right` are right all the same."""
        out, lse = c.attend(0, _ints(slots), q)
        with pytest.raises(L.TbError) as e:
            ctx.synchronize()
        assert e.value.kind == "InvalidArgument"
        right = list(right)
        _check("bf16", q[right], k, v, lens, [slots[r] for r in right], np.float32(0.125), out[right], lse[right])
        c.page_table.copy_(keep[0])
        c.lengths.copy_(keep[1])

    refused([0, 3, 2], 0, 2)
    refused([-1, 1, 2], 1, 2)
    c.page_table[1, 1] = 1000000
    refused([0, 1, 2], 0, 2)
    c.page_table[1, 2] = -7
    refused([0, 1, 2], 0, 2)
    c.lengths[2] = 1 << 30
    refused([0, 1, 2], 0, 1)
    c.lengths[0] = -1
    refused([0, 1, 2], 1, 2)
    out, lse = c.attend(0, _ints([0, 1, 2]), q)
    ctx.synchronize()
    _check("bf16", q, k, v, lens, [0, 1, 2], np.float32(0.125), out, lse)


def test_a_cache_beyond_32_bit_offsets(ctx):
    """2.4e9 elements a tensor: write, attend, fork, copy and compact at its far end."""
    page, heads, d, pages, layers = 16, 8, 128, 1600, 92
    c = PagedCache.allocate(ctx, layers=layers, num_pages=pages, page_size=page, kv_heads=heads, head_dim=d,
                            dtype=torch.bfloat16, max_seqs=4, max_pages=16)
    assert c.k_pages.numel() > 1 << 31
    n = 200
    table = torch.full((4, 16), -1, dtype=torch.int32)
    table[1, :13] = torch.arange(pages - 13, pages, dtype=torch.int32)
    c.page_table.copy_(table)
    c.lengths.copy_(_ints([0, n, 0, 0]))
    c.refs[pages - 13:] = 1
    k, v = (torch.randn(n, heads, d, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(1, 16, d, device="cuda").bfloat16()
    scale = np.float32(1 / math.sqrt(d))
    for layer in (layers - 1, 0):
        c.write(layer, _ints([1]), _offsets([n]), k, v)
    out, lse = c.attend(layers - 1, _ints([1]), q)
    ctx.synchronize()
    _check("bf16", q, k, v, [n], [0], scale, out, lse)
    c.fork(_ints([1]), _ints([3]))
    c.free(_ints([1]))
    c.compact()
    got, glse = c.attend(layers - 1, _ints([3]), q)
    first, _ = c.attend(0, _ints([3]), q)
    ctx.synchronize()
    assert torch.equal(got, out) and torch.equal(glse, lse) and torch.equal(first, out)
    assert c.page_table[3, :13].max() < 13
    c.copy_pages(_ints([int(c.page_table[3, 2])]), _ints([pages - 1]))
    ctx.synchronize()
    assert torch.equal(c.v_pages[layers - 1, pages - 1], c.v_pages[layers - 1, c.page_table[3, 2].long()])


# ---------------------------------------------------------------------------
# Bookkeeping
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("seed,pages,page,seqs", [(0, 40, 8, 9), (1, 300, 16, 40), (2, 64, 24, 16), (3, 9000, 16, 70)])
def test_bookkeeping_follows_the_model(ctx, seed, pages, page, seqs):
    """A few hundred random operations, every state compared, every refusal too; contents follow the pages."""
    r = random.Random(seed)
    max_pages = 12
    c = _cache(ctx, "f16", 2, pages, page, 1, 16, seqs, max_pages)
    m = A.Cache(pages, page, seqs, max_pages)
    data = [[] for _ in range(seqs)]  # token numbers of each slot
    count = 0
    for step in range(150):
        op = r.choice(["reserve", "reserve", "fork", "free", "compact"])
        n = r.randint(1, seqs)
        slots = r.sample(range(seqs), n)
        refused = False
        if op == "reserve":
            counts = [min(r.choice([0, 1, 1, r.randrange(40)]), max_pages * page - m.lengths[s]) for s in slots]
            ones = r.random() < 0.3 and all(m.lengths[s] < max_pages * page for s in slots)
            counts = [1] * n if ones else counts
            refused = not m.reserve(slots, counts)
            c.reserve(_ints(slots), None if ones else _ints(counts))
            if not refused and sum(counts):
                new = list(range(count, count + sum(counts)))
                count = (count + len(new)) % 1000
                at = 0
                for s, k in zip(slots, counts):
                    data[s] = data[s] + new[at:at + k]
                    at += k
                x = torch.tensor(new, device="cuda").half()[:, None, None].expand(-1, 1, 16).contiguous()
                for layer in range(2):
                    c.write(layer, _ints(slots), _offsets(counts), x + layer, -x)
        elif op == "fork":
            k = r.randint(0, n // 2)
            parents, children = [r.choice(slots[k:]) for _ in range(k)], slots[:k]
            copies = m.fork(parents, children)
            refused = copies is None
            c.fork(_ints(parents), _ints(children))
            if not refused:
                for p, s in zip(parents, children):
                    data[s] = list(data[p])
        elif op == "free":
            m.free(slots)
            c.free(_ints(slots))
            for s in slots:
                data[s] = []
        elif r.random() < 0.5:
            c.compact()
            m.compact()
        else:
            table, refs = torch.empty_like(c.page_table), torch.empty_like(c.refs)
            before = _state(c)
            c.compact(table, refs)
            ctx.synchronize()
            assert _state(c) == before
            m.compact()
            c.page_table.copy_(table)
            c.refs.copy_(refs)
        if refused:
            with pytest.raises(L.TbError) as e:
                ctx.synchronize()
            assert e.value.kind == "OutOfPages"
        else:
            ctx.synchronize()
        _same(c, m)
        if step % 10 == 9:
            kp, vp = c.k_pages.float().cpu().numpy(), c.v_pages.float().cpu().numpy()
            for s in range(seqs):
                for layer in range(2):
                    rows = kp[layer, m.table[s], 0].reshape(-1, 16)[:m.lengths[s]]
                    vals = vp[layer, m.table[s], 0].reshape(-1, 16)[:m.lengths[s]]
                    want = np.float16(np.array(data[s], dtype=np.float16)[:, None] + np.float16(layer)) if data[s] else np.zeros((0, 1))
                    assert (rows == want).all() and (vals == -np.array(data[s], dtype=np.float32)[:, None]).all(), (step, s)
    assert int(c.refs.sum()) == sum(m.refs)


def test_fork_copies_only_the_tokens(ctx):
    c, k, v = _filled(ctx, 7, "bf16", [21, 0, 0], 2, 64, 16, shuffle=False, spare=4)
    c.fork(_ints([0, 0]), _ints([2, 1]))
    ctx.synchronize()
    assert c.page_table.tolist() == [[0, 1], [0, 3], [0, 2]] and c.refs.tolist() == [3, 1, 1, 1, 0, 0]
    assert torch.equal(c.k_pages[0, 2, :, :5], c.k_pages[0, 1, :, :5]) and torch.equal(c.v_pages[0, 3, :, :5], c.v_pages[0, 1, :, :5])
    assert torch.isnan(c.k_pages[0, 2, :, 5:]).all() and torch.isnan(c.v_pages[0, 3, :, 5:]).all()


def test_fork_reuses_what_its_children_held(ctx):
    """No free page is left, but the child's former page is enough."""
    c = _cache(ctx, pages=3, page=8, seqs=2, max_pages=3)
    c.reserve(_ints([0, 1]), _ints([10, 7]))
    c.fork(_ints([0]), _ints([1]))
    ctx.synchronize()
    assert _state(c) == ([[0, 1, -1], [0, 2, -1]], [10, 10], [2, 1, 1])


def test_parts_of_a_wide_projection_are_written(ctx):
    c = _cache(ctx, "bf16", 3, 8, 8, 2, 80, 3, 4)
    c.reserve(_ints([2, 0]), _ints([11, 9]))
    wide = torch.randn(20, 9, 88, device="cuda").bfloat16()
    k, v = wide[:, 1:5:2, :80], wide[:, 5:7, :80]
    c.write(1, _ints([2, 0]), _ints([0, 11, 20]), k, v)
    ctx.synchronize()
    for slot, rows in ((2, slice(0, 11)), (0, slice(11, 20))):
        pages = c.page_table[slot, :2].long()
        got = c.k_pages[1, pages].transpose(1, 2).reshape(16, 2, 80)[:rows.stop - rows.start]
        val = c.v_pages[1, pages].transpose(1, 2).reshape(16, 2, 80)[:rows.stop - rows.start]
        assert torch.equal(got, k[rows]) and torch.equal(val, v[rows])
    assert torch.isnan(c.k_pages[[0, 2]]).all() and torch.isnan(c.v_pages[[0, 2]]).all()


@pytest.mark.parametrize("name,args", [
    ("reserve", ([0, 0],)), ("reserve", ([0, 8],)), ("reserve", ([-1],)),
    ("reserve", ([0, 1], [3, -1])), ("reserve", ([0, 1], [3, 1000])), ("reserve", ([0], [2000000000])),
    ("free", ([1, 1],)), ("free", ([9],)), ("fork", ([0, 0], [2, 2])), ("fork", ([0, 1], [1, 2])), ("fork", ([0], [0])),
    ("fork", ([8], [1])), ("fork", ([0], [-3])),
])
def test_a_refused_call_changes_nothing(ctx, name, args):
    c = _cache(ctx)
    c.reserve(_ints([0, 1]), _ints([20, 16]))
    ctx.synchronize()
    before = _state(c)
    getattr(c, name)(*[_ints(a) for a in args])
    with pytest.raises(L.TbError) as e:
        ctx.synchronize()
    assert e.value.kind == "InvalidArgument" and _state(c) == before
    c.fork(_ints([0]), _ints([5]))  # and the slots are not left marked
    c.free(_ints([0, 1, 5]))
    ctx.synchronize()
    assert sum(c.refs.tolist()) == 0


@pytest.mark.parametrize("slots,offsets", [([0, 9], [0, 2, 4]), ([0, -1], [0, 2, 4]), ([0, 1], [1, 2, 4]), ([0, 1], [0, 2, 3]),
                                           ([0, 3], [0, 2, 4]), ([0, 1], [0, 40, 4])])
def test_writes_to_the_wrong_place_are_reported(ctx, slots, offsets):
    c = _cache(ctx)
    c.reserve(_ints([0, 1]), _ints([20, 16]))
    x = torch.zeros(4, 2, 64, device="cuda").bfloat16()
    c.write(0, _ints(slots), _ints(offsets), x, x)
    with pytest.raises(L.TbError) as e:
        ctx.synchronize()
    assert e.value.kind == "InvalidArgument"
    own = set(c.page_table[:2].reshape(-1).tolist()) - {-1}
    assert all(torch.isnan(c.k_pages[:, p]).all() for p in range(32) if p not in own)


def test_copied_pages(ctx):
    c = _cache(ctx, layers=3)
    c.k_pages.normal_()
    c.v_pages.normal_()
    k, v = c.k_pages.clone(), c.v_pages.clone()
    c.copy_pages(_ints([3, 7, 3]), _ints([1, 0, 31]))
    ctx.synchronize()
    for s, d in ((3, 1), (7, 0), (3, 31)):
        k[:, d], v[:, d] = k[:, s], v[:, s]
    assert torch.equal(c.k_pages, k) and torch.equal(c.v_pages, v)
    c.copy_pages(_ints([3, 32, 5]), _ints([2, 4, -1]))  # the good pair is copied
    with pytest.raises(L.TbError) as e:
        ctx.synchronize()
    assert e.value.kind == "InvalidArgument"
    k[:, 2], v[:, 2] = k[:, 3], v[:, 3]
    assert torch.equal(c.k_pages, k) and torch.equal(c.v_pages, v)


def test_nothing_to_do(ctx):
    c = _cache(ctx)
    none = _ints([])
    x = torch.empty(0, 2, 64, device="cuda").bfloat16()
    c.reserve(none)
    c.free(none)
    c.fork(none, none)
    c.copy_pages(none, none)
    c.write(0, none, _ints([0]), x, x)
    c.write(0, _ints([1]), _ints([0, 0]), x, x)
    out, lse = c.attend(0, none, x)
    c.compact()
    c.free(_ints([3]))
    c.fork(_ints([1]), _ints([2]))
    ctx.synchronize()
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2) and sum(c.refs.tolist()) == 0


def test_a_step_in_a_graph(ctx):
    """reserve, write and attend of one token a slot, captured once and replayed."""
    lens = [30, 47]
    c, k, v = _filled(ctx, 8, "bf16", lens, 2, 64, 16, spare=6)
    grown = torch.full((2, 6), -1, dtype=torch.int32, device="cuda")
    grown[:, :c.page_table.shape[1]] = c.page_table
    c = PagedCache(ctx, c.k_pages, c.v_pages, grown, c.lengths, c.refs)
    slots, one = _ints([0, 1]), _ints([0, 1, 2])
    q, nk, nv = (torch.randn(2, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
    out, lse = torch.empty_like(q), torch.empty(2, 4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        c.reserve(slots)
        c.write(0, slots, one, nk, nv)
        c.attend(0, slots, q, out=out, lse=lse)
    ks, vs = [[k[:30]], [k[30:]]], [[v[:30]], [v[30:]]]
    for step in range(4):
        for t in (q, nk, nv):
            t.normal_()
        graph.replay()
        ctx.synchronize()
        for i in range(2):
            ks[i].append(nk[i:i + 1].clone())
            vs[i].append(nv[i:i + 1].clone())
        lens = [n + 1 for n in lens]
        _check("bf16", q, torch.cat(ks[0] + ks[1]), torch.cat(vs[0] + vs[1]), lens, [0, 1], np.float32(0.125), out, lse)
    assert c.lengths.tolist() == [34, 51]


# ---------------------------------------------------------------------------
# Refusals on the host
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("change,kind", [
    (dict(dtype=L.DT_FP32), "DTypeMismatch"), (dict(layers=0), "ShapeMismatch"), (dict(kv_heads=-1), "ShapeMismatch"),
    (dict(num_pages=0), "ShapeMismatch"), (dict(max_seqs=0), "ShapeMismatch"), (dict(max_pages=0), "ShapeMismatch"),
    (dict(head_dim=144), "NotAccelerated"), (dict(head_dim=40), "NotAccelerated"), (dict(page_size=12), "NotAccelerated"),
    (dict(page_size=0), "NotAccelerated"), (dict(num_pages=(1 << 20) + 1), "NotAccelerated"),
    (dict(max_pages=(1 << 20) + 1), "NotAccelerated"), (dict(page_size=1 << 30), "NotAccelerated"),
])
def test_cache_refusals(ctx, change, kind):
    t = torch.zeros(65536, dtype=torch.bfloat16, device="cuda")
    i = _ints([0] * 64)
    d = dict(dtype=L.DT_BF16, layers=1, kv_heads=1, head_dim=64, page_size=8, num_pages=4, max_seqs=2, max_pages=2)
    d.update(change)
    b = L.CacheBuffers(t.data_ptr(), t.data_ptr(), i.data_ptr(), i.data_ptr(), i.data_ptr())
    h = ctypes.c_void_p()
    with pytest.raises(L.TbError) as e:
        L.check(L.load().tb_cache_create(ctx.h, ctypes.byref(L.CacheDesc(**d)), ctypes.byref(b), ctypes.byref(h)))
    assert e.value.kind == kind and not h.value


def test_call_refusals(ctx):
    c = _cache(ctx)
    one, q, x = _ints([0]), torch.zeros(1, 4, 64, device="cuda").bfloat16(), torch.zeros(1, 2, 64, device="cuda").bfloat16()

    def kind(f, *a, **kw):
        with pytest.raises(L.TbError) as e:
            f(*a, **kw)
        return e.value.kind

    assert kind(c.attend, 1, one, q) == "ShapeMismatch" and kind(c.attend, -1, one, q) == "ShapeMismatch"
    assert kind(c.attend, 0, one, q[:, :3]) == "ShapeMismatch"
    assert kind(c.attend, 0, one, q.half()) == "DTypeMismatch"
    assert kind(c.attend, 0, one, q, scale=0.0) == "InvalidArgument"
    assert kind(c.attend, 0, one.long(), q) == "ShapeMismatch"
    assert kind(c.attend, 0, one.cpu(), q) == "InvalidArgument"
    assert kind(c.attend, 0, _ints([0, 1]), q) == "ShapeMismatch"
    assert kind(c.attend, 0, one, q, out=torch.zeros(1, 4, 64, device="cuda")) == "DTypeMismatch"
    assert kind(c.attend, 0, one, q, lse=torch.zeros(4, 1, device="cuda")) == "ShapeMismatch"
    odd = torch.zeros(1 * 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")[1:257].view(1, 4, 64)
    assert kind(c.attend, 0, one, odd) == "InvalidArgument"
    assert kind(c.write, 3, one, _ints([0, 1]), x, x) == "ShapeMismatch"
    assert kind(c.write, 0, one, _ints([0]), x, x) == "ShapeMismatch"
    assert kind(c.write, 0, one, _ints([0, 1]), x[:, :1], x) == "ShapeMismatch"
    assert kind(c.write, 0, _ints([]), _ints([0]), x, x) == "ShapeMismatch"
    assert kind(c.reserve, _ints(list(range(9)))) == "ShapeMismatch"
    assert kind(c.reserve, one, _ints([1, 2])) == "ShapeMismatch"
    assert kind(c.fork, one, _ints([1, 2])) == "ShapeMismatch"
    assert kind(c.compact, torch.empty_like(c.page_table)) == "InvalidArgument"
    assert kind(c.compact, torch.empty_like(c.refs), torch.empty_like(c.refs)) == "ShapeMismatch"
    lib = L.load()
    assert lib.tb_cache_reserve(None, L.ptr(one), None, 1, None) == L.TB_ERR_INVALID_ARGUMENT
    assert lib.tb_cache_free(c.h, None, 1, None) == L.TB_ERR_INVALID_ARGUMENT
    assert lib.tb_cache_free(c.h, L.ptr(one), -1, None) == L.TB_ERR_SHAPE_MISMATCH
    assert lib.tb_cache_compact(None, None, None, None) == L.TB_ERR_INVALID_ARGUMENT
    ctx.synchronize()


def test_attend_many_rows(ctx):
    """More rows than one look at their lengths takes (128), slots in any order and more than once."""
    r = np.random.default_rng(20)
    lens = [int(x) for x in r.choice([0, 1, 15, 16, 17, 64, 65, 200], 90)]
    c, k, v = _filled(ctx, 21, "f16", lens, 1, 64, 16)
    slots = [int(x) for x in r.integers(0, 90, 700)]
    q = torch.randn(700, 3, 64, device="cuda").half()
    out, lse = c.attend(0, _ints(slots), q)
    ctx.synchronize()
    _check("f16", q, k, v, lens, slots, np.float32(0.125), out, lse)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hk,d,page", [(16, 1, 64, 8), (32, 2, 32, 24), (5, 1, 16, 64), (10, 1, 48, 128)])
def test_attend_narrow_heads_many_tiles(ctx, dtype, hq, hk, d, page):
    """Several tiles a CTA, an even and an odd number of them, that end anywhere in the last one or two."""
    r = np.random.default_rng(hq + d)
    lens = [int(x) for x in r.choice([64, 65, 127, 128, 129, 190, 191, 192, 193, 255, 257, 640, 1111, 2049], 40)]
    c, k, v = _filled(ctx, 31, dtype, lens, hk, d, page)
    slots = [int(x) for x in r.integers(0, 40, 200)]
    q = torch.randn(200, hq, d, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(DT[dtype])
    out, lse = c.attend(0, _ints(slots), q)
    ctx.synchronize()
    _check(dtype, q, k, v, lens, slots, np.float32(1 / math.sqrt(d)), out, lse)


def test_bookkeeping_of_more_slots_than_threads(ctx):
    """1500 slots in one call, more pages than one pass over the counts takes (4096)."""
    c = _cache(ctx, "bf16", 1, 9000, 8, 1, 16, 3000, 6)
    m = A.Cache(9000, 8, 3000, 6)
    r = np.random.default_rng(22)
    slots = [int(x) for x in r.permutation(3000)[:1500]]
    counts = [int(x) for x in r.integers(0, 40, 1500)]
    assert m.reserve(slots, counts)
    c.reserve(_ints(slots), _ints(counts))
    ctx.synchronize()
    _same(c, m)
    children = [s for s in range(3000) if s not in set(slots)]
    parents = [slots[int(x)] for x in r.integers(0, 1500, len(children))]
    assert m.fork(parents, children) is not None
    c.fork(_ints(parents), _ints(children))
    ctx.synchronize()
    _same(c, m)
    m.free(slots)
    c.free(_ints(slots))
    m.compact()
    c.compact()
    ctx.synchronize()
    _same(c, m)
