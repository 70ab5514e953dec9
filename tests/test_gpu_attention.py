"""Attention over packed prompts against the definition in 64 bits: types, head layouts, lengths from
none to a few thousand, strides, masks that leave rows empty, what masked places hold, refusals."""

import ctypes
import math

import numpy as np
import pytest

from tests import attention_oracle as A

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tosa_b200 import _lib as L  # noqa: E402
from tosa_b200.attention import attention  # noqa: E402

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ctx():
    c = L.Context(0)
    yield c
    c.close()


def _offsets(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _inputs(seed, dtype, lq, lk, hq, hk, d, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda n, h: torch.randn(n, h, d, generator=g, device="cuda").mul_(std).to(DT[dtype])  # noqa: E731
    return mk(sum(lq), hq), mk(sum(lk), hk), torch.randn(sum(lk), hk, d, generator=g, device="cuda").to(DT[dtype])


def _check(dtype, q, k, v, lq, lk, causal, scale, out, lse, rows=None):
    """Every row (or the given rows of each sequence) of every head."""
    q, k, v, out, lse = (t.detach().double().cpu().numpy() for t in (q, k, v, out, lse))
    group = q.shape[1] // k.shape[1]
    a = b = 0
    for nq, nk in zip(lq, lk):
        at = np.arange(nq) if rows is None else np.array(sorted({r for r in rows if r < nq}), dtype=np.int64)
        limits = at + nk - nq + 1 if causal else np.full(len(at), nk)
        for h in range(q.shape[1]):
            kk, vv = k[b:b + nk, h // group], v[b:b + nk, h // group]
            want, wlse, mean, size, tail = A.attend(q[a + at, h], kk, vv, limits, scale)
            tol, ltol = A.tolerance(dtype, want, mean, size, tail)
            got, glse = out[a + at, h], lse[h, a + at]
            bad = ~(np.abs(got - want) <= tol)
            assert not bad.any(), (nq, nk, h, np.argwhere(bad)[:4], np.abs(got - want).max())
            none = np.isneginf(wlse)
            assert np.array_equal(np.isneginf(glse), none), (nq, nk, h)
            off = np.abs(glse[~none] - wlse[~none])
            assert (off <= ltol[~none]).all(), (nq, nk, h, off.max())
        a, b = a + nq, b + nk


CASES = [
    # lq, lk, query heads, key heads, head_dim, causal
    ([1], [1], 1, 1, 16, True),
    ([1], [1], 4, 1, 128, False),
    ([1, 1, 1], [5, 129, 300], 8, 2, 64, True),
    ([127], [127], 2, 2, 128, True),
    ([128], [128], 2, 1, 128, True),
    ([129], [129], 3, 1, 128, True),
    ([129], [257], 2, 1, 96, True),
    ([300], [300], 6, 2, 80, False),
    ([64, 65, 1, 200, 3], [64, 65, 1, 200, 3], 4, 4, 64, True),
    ([256, 255], [256, 255], 2, 2, 128, True),
    ([0, 7, 0, 33], [12, 7, 0, 50], 4, 2, 48, True),      # a sequence without rows
    ([9, 5, 140], [0, 5, 0], 4, 2, 64, False),            # a sequence without keys: out 0, lse -inf
    ([150, 20], [40, 3], 4, 2, 128, True),                # more rows than keys: the first rows see nothing
    ([130, 270], [1, 129], 2, 1, 32, True),
    ([513], [900], 7, 1, 112, True),
    ([257], [640], 5, 5, 128, True),
    ([31] * 40, [31] * 40, 2, 1, 64, True),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{max(c[1])}-h{c[2]}-{c[3]}-d{c[4]}-{int(c[5])}")
def test_matches_the_definition(ctx, dtype, case):
    lq, lk, hq, hk, d, causal = case
    q, k, v = _inputs(sum(lq) + d, dtype, lq, lk, hq, hk, d)
    scale = 1 / math.sqrt(d)
    out, lse = attention(ctx, q, k, v, _offsets(lq), _offsets(lk), causal=causal)
    ctx.synchronize()
    _check(dtype, q, k, v, lq, lk, causal, np.float32(scale), out, lse)


@pytest.mark.parametrize("dtype,causal", [("bf16", True), ("f16", False)])
def test_long(ctx, dtype, causal):
    lq, lk = [2049, 300], [4100, 2600]
    q, k, v = _inputs(5, dtype, lq, lk, 4, 2, 128)
    out, lse = attention(ctx, q, k, v, _offsets(lq), _offsets(lk), causal=causal)
    ctx.synchronize()
    _check(dtype, q, k, v, lq, lk, causal, np.float32(1 / math.sqrt(128)), out, lse,
           rows=list(range(0, 2049, 37)) + [127, 128, 255, 256, 2047, 2048])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_rise_and_fall(ctx, dtype, rising):
    """Scores over a range of 240, rising along the keys (the running maximum moves in every block) or falling."""
    n, d = 700, 64
    q, k, v = _inputs(11, dtype, [n], [n], 2, 1, d)
    ramp = torch.linspace(-15, 15, n, device="cuda") * (1 if rising else -1)
    k[:, 0, 0] = ramp.to(k.dtype)
    q[:, :, 0] = 8.0
    out, lse = attention(ctx, q, k, v, _offsets([n]), _offsets([n]), causal=False, scale=1.0)
    ctx.synchronize()
    _check(dtype, q, k, v, [n], [n], False, 1.0, out, lse, rows=range(0, n, 9))


def test_layouts(ctx):
    """Parts of one projection's rows, head-major tensors, strided rows and outputs give the packed call's bits."""
    lq, hq, hk, d = [70, 133], 4, 2, 64
    n = sum(lq)
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(n, hq + 2 * hk, d, generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    cu = _offsets(lq)
    want, wlse = attention(ctx, q.contiguous(), k.contiguous(), v.contiguous(), cu, cu)
    got, lse = attention(ctx, q, k, v, cu, cu)
    head_major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    got2, _ = attention(ctx, *head_major, cu, cu)
    wide = torch.full((n, 2 * hq, d + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    view = wide[:, ::2, :d]
    got3, _ = attention(ctx, q, k, v, cu, cu, out=view)
    ctx.synchronize()
    assert torch.equal(want, got) and torch.equal(wlse, lse) and torch.equal(want, got2)
    assert got3 is view and torch.equal(want, view)
    assert (wide[:, 1::2] == 7).all() and (wide[:, ::2, d:] == 7).all()


def test_rows_of_one_head_or_token_may_have_any_stride(ctx):
    q, k, v = _inputs(4, "f16", [33], [33], 1, 1, 32)
    odd = [torch.as_strided(t, t.shape, (32, 5, 1)) for t in (q, k, v)]
    cu = _offsets([33])
    want, _ = attention(ctx, q, k, v, cu, cu)
    got, _ = attention(ctx, *odd, cu, cu)
    one = torch.as_strided(q, (1, 1, 32), (3, 1, 1))
    cu1 = _offsets([1])
    last, _ = attention(ctx, one, k[:1], v[:1], cu1, cu1)
    ctx.synchronize()
    assert torch.equal(want, got) and torch.equal(last[0], v[0])


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_what_is_masked_has_no_part(ctx, dtype, value):
    """NaN and infinities in other sequences' keys and in keys after a row leave the row as it was."""
    lq, lk = [50, 141, 20], [50, 141, 20]
    q, k, v = _inputs(8, dtype, lq, lk, 4, 2, 64)
    cu = _offsets(lq)
    want, wlse = attention(ctx, q, k, v, cu, cu)
    k2, v2 = k.clone(), v.clone()
    k2[:50], v2[:50] = value, value          # the first sequence
    k2[191:], v2[191:] = value, value        # the last one
    k2[150:191], v2[150:191] = value, value  # rows 0..99 of the middle one do not see these
    got, lse = attention(ctx, q, k2, v2, cu, cu)
    ctx.synchronize()
    assert torch.equal(got[50:150], want[50:150])
    assert torch.equal(lse[:, 50:150], wlse[:, 50:150])
    assert not torch.isfinite(got[150:191].float()).any()


@pytest.mark.parametrize("where", [0, 63, 64, 100, 127, 128, 190])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(ctx, where):
    n = 200
    q, k, v = _inputs(9, "bf16", [n], [n], 2, 1, 128)
    cu = _offsets([n])
    want, wlse = attention(ctx, q, k, v, cu, cu)
    v2 = v.clone()
    v2[where, 0, 5], v2[where, 0, 77], v2[where, 0, 120] = math.inf, -math.inf, math.nan
    got, lse = attention(ctx, q, k, v2, cu, cu)
    ctx.synchronize()
    keep = [c for c in range(128) if c not in (5, 77, 120)]
    assert torch.equal(got[:where], want[:where]) and torch.equal(got[..., keep], want[..., keep])
    assert torch.equal(lse, wlse)
    assert (got[where:, :, 5] == math.inf).all() and (got[where:, :, 77] == -math.inf).all()
    assert torch.isnan(got[where:, :, 120]).all()


def test_infinite_scores(ctx):
    """A row whose scores are all -inf is a division of 0 by 0; a score of +inf makes the row NaN. Other rows keep theirs."""
    q, k, v = _inputs(10, "bf16", [6], [6], 1, 1, 16)
    q[2], k[:, :, 0] = 0.0, 1.0
    q[2, 0, 0] = -math.inf
    q[4] = 0.0
    q[4, 0, 0] = math.inf
    cu = _offsets([6])
    out, lse = attention(ctx, q, k, v, cu, cu, causal=False)
    ctx.synchronize()
    assert torch.isnan(out[2]).all() and lse[0, 2] == -math.inf
    assert torch.isnan(out[4]).all() and not torch.isfinite(lse[0, 4])
    keep = [0, 1, 3, 5]
    _check("bf16", q[keep], k, v, [4], [6], False, 0.25, out[keep], lse[:, keep])


def test_the_same_call_twice_gives_the_same_bits(ctx):
    lq = [700, 33, 5]
    q, k, v = _inputs(12, "bf16", lq, lq, 8, 2, 128)
    cu = _offsets(lq)
    a = attention(ctx, q, k, v, cu, cu)
    b = attention(ctx, q, k, v, cu, cu)
    ctx.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_rows_and_no_sequences(ctx):
    e = torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    out, lse = attention(ctx, e, e, e, _offsets([0]), _offsets([0]))
    assert out.shape == (0, 2, 64) and lse.shape == (2, 0)
    attention(ctx, e, e, e, _offsets([]), _offsets([]))
    q = torch.randn(3, 2, 64, device="cuda").half()
    out, lse = attention(ctx, q, e, e, _offsets([3]), _offsets([0]))
    ctx.synchronize()
    assert (out == 0).all() and (lse == -math.inf).all()


def test_another_stream_and_a_captured_graph(ctx):
    q, k, v = _inputs(13, "bf16", [200], [200], 4, 4, 64)
    cu = _offsets([200])
    want, wlse = attention(ctx, q, k, v, cu, cu)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got, lse = attention(ctx, q, k, v, cu, cu, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, wlse)
    out, lse = torch.zeros_like(want), torch.zeros_like(wlse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attention(ctx, q, k, v, cu, cu, out=out, lse=lse)
    q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    want, wlse = attention(ctx, q, k, v, cu, cu)
    ctx.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, wlse)


@pytest.mark.parametrize("cu_q,cu_k", [([0, 10, 31], [0, 10, 30]), ([0, 20, 10], [0, 20, 30]), ([-1, 10, 30], [0, 10, 30]),
                                       ([0, 10, 30], [0, 10, 2000000000]), ([0, 10, 30], [0, -5, 30])])
def test_offsets_out_of_range_are_reported(ctx, cu_q, cu_k):
    q, k, v = _inputs(14, "bf16", [30], [30], 2, 2, 64)
    out = torch.zeros_like(q)
    attention(ctx, q, k, v, torch.tensor(cu_q, dtype=torch.int32, device="cuda"),
              torch.tensor(cu_k, dtype=torch.int32, device="cuda"), out=out)
    with pytest.raises(L.TbError) as e:
        ctx.synchronize()
    assert e.value.kind == "InvalidArgument"
    cu = _offsets([30])
    got, lse = attention(ctx, q, k, v, cu, cu)
    ctx.synchronize()
    _check("bf16", q, k, v, [30], [30], True, np.float32(0.125), got, lse)


def _desc(**kw):
    d = dict(dtype=L.DT_BF16, batch=1, q_heads=2, kv_heads=1, head_dim=64, causal=1, scale=0.125, total_q=4, total_k=4,
             q_token_stride=128, q_head_stride=64, k_token_stride=64, k_head_stride=64, v_token_stride=64, v_head_stride=64,
             out_token_stride=128, out_head_stride=64)
    d.update(kw)
    return L.AttentionDesc(**d)


@pytest.mark.parametrize("change,kind", [
    (dict(dtype=L.DT_FP32), "DTypeMismatch"), (dict(q_heads=3, kv_heads=2), "ShapeMismatch"), (dict(kv_heads=0), "ShapeMismatch"),
    (dict(head_dim=136), "NotAccelerated"), (dict(head_dim=24), "NotAccelerated"), (dict(head_dim=0), "NotAccelerated"),
    (dict(scale=0.0), "InvalidArgument"), (dict(scale=-1.0), "InvalidArgument"), (dict(scale=math.nan), "InvalidArgument"),
    (dict(scale=math.inf), "InvalidArgument"), (dict(batch=-1), "ShapeMismatch"), (dict(total_q=-1), "ShapeMismatch"),
    (dict(total_k=1 << 31), "NotAccelerated"), (dict(q_token_stride=130), "InvalidArgument"),
    (dict(v_token_stride=-64), "ShapeMismatch"), (dict(k_head_stride=4), "InvalidArgument"),
])
def test_refusals(ctx, change, kind):
    t = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    cu = _offsets([4])
    lse = torch.zeros(8, device="cuda")
    args = [L.ptr(t), L.ptr(t), L.ptr(t), L.ptr(cu), L.ptr(cu), L.ptr(t), L.ptr(lse), L.stream_ptr()]
    with pytest.raises(L.TbError) as e:
        L.check(L.load().tb_attention(ctx.h, ctypes.byref(_desc(**change)), *args))
    assert e.value.kind == kind
    ctx.synchronize()


@pytest.mark.parametrize("missing", range(6))
def test_null_pointers_are_refused(ctx, missing):
    t = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    cu = _offsets([4])
    args = [L.ptr(t), L.ptr(t), L.ptr(t), L.ptr(cu), L.ptr(cu), L.ptr(t), None, L.stream_ptr()]
    args[missing] = None
    with pytest.raises(L.TbError) as e:
        L.check(L.load().tb_attention(ctx.h, ctypes.byref(_desc()), *args))
    assert e.value.kind == "InvalidArgument"


def test_unaligned_tensors_are_refused(ctx):
    t = torch.zeros(8192, dtype=torch.bfloat16, device="cuda")
    q = t[1:1 + 4 * 2 * 64].view(4, 2, 64)
    k = t[:256].view(4, 1, 64)
    cu = _offsets([4])
    with pytest.raises(L.TbError) as e:
        attention(ctx, q, k, k, cu, cu)
    assert e.value.kind == "InvalidArgument"


def test_lse_may_be_null(ctx):
    q, k, v = _inputs(15, "bf16", [40], [40], 2, 1, 64)
    cu = _offsets([40])
    want, _ = attention(ctx, q, k, v, cu, cu)
    out = torch.zeros_like(q)
    d = _desc(total_q=40, total_k=40)
    L.check(L.load().tb_attention(ctx.h, ctypes.byref(d), L.ptr(q), L.ptr(k), L.ptr(v), L.ptr(cu), L.ptr(cu), L.ptr(out),
                                  None, L.stream_ptr()))
    ctx.synchronize()
    assert torch.equal(out, want)


def test_a_wait_that_runs_out_is_reported_and_the_context_stays_usable():
    """With a bound of zero a wait that lasts gives up (here the result warps' wait for a row of 12,000 keys): the
    kernel unwinds by design (its copies and MMAs drain, tensor memory is freed) and the next synchronize reports it."""
    lib = L.load()
    ctx = L.Context(0)
    n = 12000
    q, k, v = _inputs(16, "bf16", [n], [n], 4, 2, 128)
    cu = _offsets([n])
    L.check(lib.tb_context_set_wait_timeout_ms(ctx.h, ctypes.c_double(0.0)))
    attention(ctx, q, k, v, cu, cu)
    with pytest.raises(L.TbError) as e:
        ctx.synchronize()
    assert e.value.kind == "Timeout"
    L.check(lib.tb_context_set_wait_timeout_ms(ctx.h, ctypes.c_double(2000.0)))
    out, lse = attention(ctx, q, k, v, cu, cu)
    ctx.synchronize()
    _check("bf16", q, k, v, [n], [n], True, np.float32(1 / math.sqrt(128)), out, lse, rows=range(0, n, 997))
    ctx.close()


def test_many_sequences(ctx):
    """More sequences than one look at their lengths takes (32), of lengths in no order, some empty."""
    r = np.random.default_rng(17)
    lq = [int(x) for x in r.choice([0, 1, 3, 17, 40, 129, 200], 150)]
    lk = [n + int(x) for n, x in zip(lq, r.choice([0, 0, 5, 130], 150))]
    q, k, v = _inputs(18, "f16", lq, lk, 6, 2, 64)
    out, lse = attention(ctx, q, k, v, _offsets(lq), _offsets(lk))
    ctx.synchronize()
    _check("f16", q, k, v, lq, lk, True, np.float32(0.125), out, lse, rows=[0, 1, 2, 16, 39, 127, 128, 199])


def test_two_streams_at_once(ctx):
    """Independent calls that overlap on the GPU: nothing is shared between them."""
    q, k, v = _inputs(19, "bf16", [700], [700], 8, 2, 128)
    cu = _offsets([700])
    want, wlse = attention(ctx, q, k, v, cu, cu)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[attention(ctx, q, k, v, cu, cu, stream=s) for _ in range(8)] for s in streams]
    torch.cuda.synchronize()
    for pair in sum(got, []):
        assert torch.equal(pair[0], want) and torch.equal(pair[1], wlse)


@pytest.mark.parametrize("hq,hk", [(2, 1), (8, 2), (8, 1), (16, 1), (32, 1), (64, 1), (6, 1), (10, 2)])
def test_heads_that_share_a_tile(ctx, hq, hk):
    """Groups of a power of two share a tile's rows (up to 32 heads), others do not: tokens around a tile's and a warp's end."""
    group = hq // hk
    tokens = max(1, 128 // group)
    lq = [1, tokens - 1, tokens, tokens + 1, 2 * tokens + 3, 0, 7]
    lq = [max(n, 0) for n in lq]
    lk = [n + 3 for n in lq]
    q, k, v = _inputs(23 + hq, "bf16", lq, lk, hq, hk, 64)
    out, lse = attention(ctx, q, k, v, _offsets(lq), _offsets(lk))
    ctx.synchronize()
    _check("bf16", q, k, v, lq, lk, True, np.float32(0.125), out, lse)
