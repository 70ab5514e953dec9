"""A transformer block that serves prompts and single tokens: the example of how the library's
contractions, its attention over prompts and its paged cache work together.

    python -m tosa_b200.generate [--layers 2] [--tokens 12] [--beams 3]

Random weights and prompts, a linear read-out instead of a vocabulary: what it shows is the calls. The
projections are MATMUL_T (bf16 operands, FP32 result), prompts of different lengths go through the layers as
packed rows, their keys and values into the cache's pages, and then one row a sequence and step; the
sequences are forked into beams (full pages shared), beams that end are freed, and the pages in use moved
together. Additions, the activation and casts between the calls are torch's.
"""

from __future__ import annotations

import argparse

import torch

from . import _lib as L
from .attention import PagedCache, attention


class Block:
    """Weights of one layer: [out, in] matrices in bf16."""

    def __init__(self, generator, hidden, heads, kv_heads, head_dim, inner):
        def weight(rows, columns):
            w = torch.randn(rows, columns, generator=generator, device="cuda") * columns ** -0.5
            return w.to(torch.bfloat16)
        self.qkv = weight((heads + 2 * kv_heads) * head_dim, hidden)
        self.out = weight(hidden, heads * head_dim)
        self.up = weight(inner, hidden)
        self.down = weight(hidden, inner)


class Model:
    def __init__(self, ctx, *, layers=2, hidden=256, heads=8, kv_heads=2, head_dim=64, inner=512, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.heads, self.kv_heads, self.head_dim, self.hidden = ctx, heads, kv_heads, head_dim, hidden
        self.blocks = [Block(g, hidden, heads, kv_heads, head_dim, inner) for _ in range(layers)]

    def matmul(self, x, w):
        """x [rows, in] times w [out, in] transposed: bf16 operands, the FP32 result rounded to bf16."""
        out = torch.empty(x.shape[0], w.shape[0], dtype=torch.float32, device=x.device)
        d = L.MatmulDesc(n=1, h=x.shape[0], c=x.shape[1], w=w.shape[0], a_dtype=L.DT_BF16, b_dtype=L.DT_BF16, out_dtype=L.DT_FP32)
        L.check(L.load().tb_matmul_t(self.ctx.h, d, 1, None, L.ptr(x), L.ptr(w), L.ptr(out), L.stream_ptr()))
        return out.to(torch.bfloat16)

    def _layers(self, x, attend):
        """x [rows, hidden] through the layers; attend(layer, q, k, v) gives the attention of the rows."""
        for i, b in enumerate(self.blocks):
            qkv = self.matmul(x, b.qkv).view(x.shape[0], -1, self.head_dim)
            q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
            x = x + self.matmul(attend(i, q, k, v).view(x.shape[0], -1), b.out)
            x = x + self.matmul(torch.relu(self.matmul(x, b.up)), b.down)
        return x

    def prompt(self, cache, slots, offsets, lengths, x):
        """Rows of several prompts one behind the other, written to their slots; returns every row."""
        cache.reserve(slots, lengths)

        def attend(i, q, k, v):
            cache.write(i, slots, offsets, k, v)
            return attention(self.ctx, q, k, v, offsets, offsets, causal=True)[0]
        return self._layers(x, attend)

    def step(self, cache, slots, one_each, x):
        """One new row a slot; one_each is 0, 1, .. len(slots)."""
        cache.reserve(slots)

        def attend(i, q, k, v):
            cache.write(i, slots, one_each, k, v)
            return cache.attend(i, slots, q)[0]
        return self._layers(x, attend)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def run(ctx, *, layers=2, lengths=(37, 5, 130), tokens=12, beams=3, seed=0):
    """Prompts, then `tokens` steps of `beams` forks of each. Returns the model, the prompts' rows, and for
    each step its slots, its input rows and its result rows; and the cache."""
    model = Model(ctx, layers=layers, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    n = len(lengths)
    seqs = n * (1 + beams)
    longest = max(lengths) + tokens
    cache = PagedCache.allocate(ctx, layers=layers, num_pages=seqs * (-(-longest // 16)) + 4, page_size=16, kv_heads=model.kv_heads,
                                head_dim=model.head_dim, dtype=torch.bfloat16, max_seqs=seqs, max_pages=-(-longest // 16))
    offsets = [0]
    for x in lengths:
        offsets.append(offsets[-1] + x)
    x = torch.randn(offsets[-1], model.hidden, generator=g, device="cuda").to(torch.bfloat16)
    rows = model.prompt(cache, _ints(range(n)), _ints(offsets), _ints(lengths), x)
    # beams: slots n .. of prompt 0, 1, ..; the prompts' own slots end here
    parents = [i for i in range(n) for _ in range(beams)]
    slots = list(range(n, seqs))
    cache.fork(_ints(parents), _ints(slots))
    cache.free(_ints(range(n)))
    # each beam begins from its prompt's last row, a little apart
    y = rows[_ints([offsets[p + 1] - 1 for p in parents]).long()]
    y = (y + 0.1 * torch.randn(y.shape, generator=g, device="cuda")).to(torch.bfloat16)
    steps = []
    for t in range(tokens):
        if t == tokens // 2 and beams > 1:  # the last beam of each prompt ends; its pages go back and the rest move together
            cache.free(_ints(slots[beams - 1::beams]))
            y = y[_ints([i for i in range(len(slots)) if i % beams != beams - 1]).long()]
            slots = [s for i, s in enumerate(slots) if i % beams != beams - 1]
            cache.compact()
        out = model.step(cache, _ints(slots), _ints(range(len(slots) + 1)), y)
        steps.append((list(slots), y, out))
        y = torch.nn.functional.normalize(out.float(), dim=1).mul(model.hidden ** 0.5).to(torch.bfloat16)
    ctx.synchronize()
    return model, (x, rows, parents, offsets), steps, cache


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--tokens", type=int, default=12)
    ap.add_argument("--beams", type=int, default=3)
    a = ap.parse_args(argv)
    ctx = L.Context(0)
    before = ctx.launches
    _, (x, _, _, _), steps, cache = run(ctx, layers=a.layers, tokens=a.tokens, beams=a.beams)
    used = int((cache.refs > 0).sum())
    print(f"{x.shape[0]} prompt rows, {len(steps)} steps of {len(steps[0][0])} to {len(steps[-1][0])} beams, "
          f"{used} of {cache.refs.numel()} pages in use, {ctx.launches - before} kernels")
    cache.close()
    ctx.close()


if __name__ == "__main__":
    main()
