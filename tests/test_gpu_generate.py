"""The serving example (prompts, forked beams, single tokens, pages freed and moved) against the same
model in 64 bits with full recomputation.

Each layer rounds to bf16 after its four products, its attention and its two additions: 8 roundings of
relative size 2^-8 at most (and the attention's weights once more), so two layers stay within 18 * 2^-8 of
the norm, taken as if every rounding error added up."""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tosa_b200 import _lib as L  # noqa: E402
from tosa_b200 import generate as G  # noqa: E402

BOUND = 18 * 2.0 ** -8


def _reference(model, x):
    """Rows of one sequence through the layers in 64 bits; returns every row."""
    x = x.double()
    n, group = x.shape[0], model.heads // model.kv_heads
    hidden = torch.ones(n, n, device=x.device).triu(1).bool()
    for b in model.blocks:
        qkv = (x @ b.qkv.double().T).view(n, -1, model.head_dim)
        q, k, v = qkv.split((model.heads, model.kv_heads, model.kv_heads), dim=1)
        k, v = (t.repeat_interleave(group, 1) for t in (k, v))
        scores = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(model.head_dim)
        p = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).reshape(n, -1) @ b.out.double().T
        x = x + torch.relu(x @ b.up.double().T) @ b.down.double().T
    return x


def _near(got, want):
    return float((got.double() - want).norm() / want.norm()) <= BOUND


@pytest.mark.parametrize("beams,lengths", [(3, (37, 5, 130)), (1, (16, 1)), (2, (64, 31, 200, 2))])
def test_example_matches_full_recomputation(beams, lengths):
    ctx = L.Context(0)
    model, (x, rows, parents, offsets), steps, cache = G.run(ctx, lengths=lengths, tokens=6, beams=beams, seed=beams)
    for i in range(len(lengths)):
        part = slice(offsets[i], offsets[i + 1])
        assert _near(rows[part], _reference(model, x[part])), i
    history = {}  # the rows that each slot has seen
    for slots, y, out in steps:
        for j, slot in enumerate(slots):
            p = parents[slot - len(lengths)]
            seen = history.setdefault(slot, [x[offsets[p]:offsets[p + 1]]])
            seen.append(y[j:j + 1])
            assert _near(out[j], _reference(model, torch.cat(seen))[-1]), (slot, j)
    live = sorted(p for p in cache.page_table.flatten().tolist() if p >= 0)
    assert set(live) == {p for p, n in enumerate(cache.refs.tolist()) if n}
    cache.close()
    ctx.close()


def test_command_runs(capsys):
    G.main(["--tokens", "4", "--layers", "1"])
    assert "pages in use" in capsys.readouterr().out
