"""Attention and the paged cache in 64 bits, from their definitions, for the tests: numpy on the host,
one sequence and head at a time. The tolerances are derived here too."""

import math

import numpy as np

UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half the spacing of the type at 1


def attend(q, k, v, limits, scale):
    """q [r, d], k and v [n, d] float64; row i sees the keys before limits[i]. Returns out, lse, and what
    the tolerances need: the weighted mean of |v|, the largest sum |q||k| scale, and max|v| n / sum w."""
    r, d = q.shape
    out, lse = np.zeros((r, d)), np.full(r, -math.inf)
    mean, size, tail = np.zeros((r, d)), np.zeros(r), np.zeros(r)
    for i in range(r):
        n = min(max(int(limits[i]), 0), k.shape[0])
        if n == 0:
            continue
        s = scale * (k[:n] @ q[i])
        top = s.max()
        w = np.exp(s - (0.0 if np.isneginf(top) else top))
        total = w.sum()
        with np.errstate(invalid="ignore", divide="ignore"):
            out[i] = (w @ v[:n]) / total
            lse[i] = top + math.log(total) if total > 0 else (math.nan if math.isnan(total) else -math.inf)
            mean[i] = (w @ np.abs(v[:n])) / total
            size[i] = scale * (np.abs(k[:n]) @ np.abs(q[i])).max()
            tail[i] = n * np.abs(v[:n]).max() / total
    return out, lse, mean, size, tail


def tolerance(dtype, out, mean, size, tail):
    """Bounds on the errors of out and lse. The result is rounded once to the type (u |out|) and so is each
    weight (u times the weighted mean of |v|; weights below f16's smallest normal number, 2^-14 of the
    largest, lose up to 2^-25 each). A score is a sum of up to 128 products in 32 bits, each addition
    rounding to 2^-24: its error is at most 2^-17 sum |q||k| scale, and twice that, with two more bits for
    the exponential and the sums, is the relative error of a weight."""
    u = UNIT[dtype]
    score = 2.0 ** -16 * (1 + size)
    return (u * np.abs(out) + (u + score)[..., None] * mean + 2.0 ** -24 * tail[..., None],
            score + 2.0 ** -22 * 8 * size)


class Cache:
    """The page bookkeeping, one page at a time."""

    def __init__(self, pages, page, seqs, max_pages):
        self.page, self.max_pages = page, max_pages
        self.refs = [0] * pages
        self.table = [[] for _ in range(seqs)]
        self.lengths = [0] * seqs

    def _take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, slots, counts):
        need = sum(-(-(self.lengths[s] + c) // self.page) - len(self.table[s]) for s, c in zip(slots, counts))
        if need > self.refs.count(0):
            return False
        for s, c in zip(slots, counts):
            self.lengths[s] += c
            while len(self.table[s]) < -(-self.lengths[s] // self.page):
                self.table[s].append(self._take())
        return True

    def free(self, slots):
        for s in slots:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.table[s], self.lengths[s] = [], 0

    def fork(self, parents, children):
        """Returns the copies (source, destination, tokens), or None when pages are short."""
        before = list(self.refs), [list(t) for t in self.table], list(self.lengths)
        self.free(children)
        for p, c in zip(parents, children):
            self.table[c] = self.table[p][:self.lengths[p] // self.page]
            self.lengths[c] = self.lengths[p]
            for x in self.table[c]:
                self.refs[x] += 1
        copies = []
        for p, c in zip(parents, children):
            if self.lengths[p] % self.page:
                if 0 not in self.refs:
                    self.refs, self.table, self.lengths = before
                    return None
                to = self._take()
                copies.append((self.table[p][self.lengths[p] // self.page], to, self.lengths[p] % self.page))
                self.table[c].append(to)
        return copies

    def compact(self):
        """Returns the moves (source, destination)."""
        moves = []
        live = sum(1 for n in self.refs if n)
        for src in [p for p in range(live, len(self.refs)) if self.refs[p]]:
            to = self.refs.index(0)
            moves.append((src, to))
            self.refs[to], self.refs[src] = self.refs[src], 0
        to = dict(moves)
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return moves

    def rows(self):
        return [row + [-1] * (self.max_pages - len(row)) for row in self.table]
