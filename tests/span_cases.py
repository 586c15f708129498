"""Cases and the 64-bit oracle of the attention over parts of a row's pages
(window and sinks) and over shared pages.

A case's pools hold NaN wherever no query of the case may look, and the table
entries of pages without a visible token are -1, so a kernel that lets a
hidden token in, or reads a page it need not, shows it.

Tolerance.  A kernel's probabilities are rounded to BF16 (off by at most 2^-8
of each) before the FP32 product with V, and the output is rounded to BF16
(2^-8 of it).  With w the exact softmax weights, out = sum w v and
A = sum w |v|: rounded probabilities change the sum by at most 2^-8 A and the
normaliser, if it sums the rounded ones, by at most 2^-8 of it (2^-8 |out|);
the output's rounding adds 2^-8 |out|.  The FP32 scores (64 products of
magnitude s: below 64 * 2^-24 * sum|q k| scale, with sum|q k| scale < 30 here)
and exponentials (2^-22) are off by less than 2^-13 relative in all:
    tol = 2^-8 (A + 2 |out|) + 2^-13 A.
"""
from __future__ import annotations

import numpy as np

import workloads as W

PAGE, DIM, GROUP = W.PAGE, W.HEAD_DIM, W.GROUP


def visible(pos: int, window: int, sinks: int) -> np.ndarray:
    """Positions that a query at `pos` sees."""
    j = np.arange(pos + 1)
    return j[(j > pos - window) | (j < sinks)]


def attend(q, k, v, scale):
    """q [4, 64] against k, v [n, 64] in float64: (out [4, 64], A [4, 64])."""
    s = (q @ k.T) * scale
    w = np.exp(s - s.max(axis=1, keepdims=True))
    w /= w.sum(axis=1, keepdims=True)
    return w @ v, w @ np.abs(v)


class SpanCase:
    """Sequences of given lengths on scattered pages.  `queries`: per sequence
    the positions of its queries (decode: the last one).  `see`: per sequence,
    position -> visible positions."""

    def __init__(self, seed, lens, kv_heads=8, num_layers=1, layer=0, window=None, sinks=0,
                 q_counts=None, groups=None, scale=0.125, slack=3):
        # groups: [(rows, shared pages), ...] over the rows in order
        self.rng = rng = np.random.default_rng(seed)
        self.lens = lens = np.asarray(lens, dtype=np.int32)
        self.kv_heads, self.layer, self.scale = kv_heads, layer, scale
        self.window, self.sinks = window, sinks
        B = len(lens)
        need = -(-np.maximum(lens, 0) // PAGE)
        shared = np.zeros(B, dtype=np.int64)
        self.prefix_tables = None
        group_of = np.full(B, -1)
        n_shared = 0
        if groups is not None:
            rows = np.cumsum([0] + [n for n, _ in groups])
            self.group_rows = rows.astype(np.int32)
            self.prefix_pages = np.array([p for _, p in groups], dtype=np.int32)
            n_shared = int(self.prefix_pages.sum())
            for g in range(len(groups)):
                group_of[rows[g]:rows[g + 1]] = g
                shared[rows[g]:rows[g + 1]] = groups[g][1]
            self.prefix_tables = np.full((max(len(groups), 1), max([p for _, p in groups] + [1]) + 1), -1,
                                         dtype=np.int32)
        own = np.maximum(need - shared, 0)
        self.num_pages = int(own.sum()) + n_shared + slack
        perm = rng.permutation(self.num_pages).astype(np.int32)
        stride = max(int(need.max()) if B else 1, 1)
        full = np.full((B, stride), -1, dtype=np.int64)  # every page a row's positions are on
        used = 0
        if groups is not None:
            for g, (_, n) in enumerate(groups):
                self.prefix_tables[g, :n] = perm[used:used + n]
                used += n
        for b in range(B):
            n = min(int(shared[b]), int(need[b]))
            if group_of[b] >= 0:
                full[b, :n] = self.prefix_tables[group_of[b], :n]
            full[b, n:need[b]] = perm[used:used + own[b]]
            used += int(own[b])
        q_counts = np.ones(B, dtype=np.int64) * (lens > 0) if q_counts is None else np.asarray(q_counts)
        self.q_counts = q_counts
        shape = (num_layers, self.num_pages, PAGE, kv_heads * DIM)
        nan = np.uint16(0x7FC0)
        self.k_pool = np.full(shape, nan, dtype=np.uint16)
        self.v_pool = np.full(shape, nan, dtype=np.uint16)
        self.tables = np.full((B, stride), -1, dtype=np.int32)
        self.seen = []  # per sequence: [(visible positions) per query]
        for b in range(B):
            per_query = []
            for i in range(int(q_counts[b])):
                pos = int(lens[b]) - int(q_counts[b]) + i
                per_query.append(visible(pos, window if window else pos + 1, sinks))
            self.seen.append(per_query)
            if not per_query:
                continue
            at = np.unique(np.concatenate(per_query))
            pages = np.unique(at // PAGE)
            mine = pages[pages >= shared[b]]
            self.tables[b, mine] = full[b, mine]
            phys = full[b, at // PAGE]
            empty = np.isnan(W.bf16_to_f32(self.k_pool[layer, phys, at % PAGE, 0]))
            self.k_pool[layer, phys[empty], at[empty] % PAGE] = W.normal_bf16(rng, (int(empty.sum()), kv_heads * DIM))
            self.v_pool[layer, phys[empty], at[empty] % PAGE] = W.normal_bf16(rng, (int(empty.sum()), kv_heads * DIM))
        self.full = full
        self.decode = bool(np.all(q_counts == (lens > 0)))
        tokens = B if self.decode else int(q_counts.sum())
        self.q = W.normal_bf16(rng, (tokens, kv_heads * GROUP * DIM))
        self.cu_q = np.concatenate([[0], np.cumsum(q_counts)]).astype(np.int32)
        self.q_pos0 = (lens - q_counts).astype(np.int32)

    def oracle(self):
        """(out, tol), float64 [tokens, q width]; rows without queries are zeros with tolerance 0."""
        out = np.zeros(self.q.shape)
        tol = np.zeros(self.q.shape)
        q = W.bf16_to_f32(self.q).astype(np.float64).reshape(len(self.q), self.kv_heads, GROUP, DIM)
        for b, per_query in enumerate(self.seen):
            for i, at in enumerate(per_query):
                row = b if self.decode else int(self.cu_q[b]) + i
                phys = self.full[b, at // PAGE]
                k = W.bf16_to_f32(self.k_pool[self.layer, phys, at % PAGE]).astype(np.float64)
                v = W.bf16_to_f32(self.v_pool[self.layer, phys, at % PAGE]).astype(np.float64)
                for g in range(self.kv_heads):
                    c = slice(g * DIM, (g + 1) * DIM)
                    o, a = attend(q[row, g], k[:, c], v[:, c], self.scale)
                    cols = slice(g * GROUP * DIM, (g + 1) * GROUP * DIM)
                    out[row, cols] = o.reshape(-1)
                    tol[row, cols] = (2.0 ** -8 * (a + 2 * np.abs(o)) + 2.0 ** -13 * a).reshape(-1)
        return out, tol


def check(got_bits, case, what=""):
    out, tol = case.oracle()
    got = W.bf16_to_f32(got_bits).astype(np.float64)
    assert np.isfinite(got).all(), f"{what}: non-finite output"
    bad = np.abs(got - out) > tol
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} values off, the worst by "
                           f"{float((np.abs(got - out) - tol).max()):.3g} over its tolerance")
