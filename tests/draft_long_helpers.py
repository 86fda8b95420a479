"""Drafted tokens behind long caches, made so that every page shows in the outputs, with bounds that say so.

Averages of thousands of Gaussian values are near zero, and a tolerance in units of the values says little of them.  Here

 * `flat` batches have queries of zero and whole numbers as values, most of them a sign of their page's own: every weight is exactly
   one, sums below 2^24 are exact in float32 in whatever order they are taken, and what is left is the division's and the output's
   rounding.  A lost key shows;
 * `aimed` batches have queries that lie along the directions of a few pages' keys (another few for every row and head), so that a row's
   weight lies on these pages, its maximum moves as they come, and pieces of unlike maxima are added up.  A lost page shows."""
import numpy as np
import torch

from draft_helpers import PAGE, TreeBatch


class FlatBatch(TreeBatch):
    def __init__(self, seed, *args, **kw):
        super().__init__(seed, *args, **kw)
        rng = np.random.default_rng(seed + 1)
        self.q[:] = 0.0
        sign = rng.integers(0, 2, (self.n_pages, self.n_kv, 1, self.hd)) * 2 - 1
        self.v = (6 * sign + rng.integers(-2, 3, self.v.shape)).astype(np.float32)       # (exact in bfloat16)
        self.round_to(torch.bfloat16)

    def bound(self, dtype, ref):
        """1 / count and the product with it, 2^-24 each; half a step of the output."""
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
        return (half + 4 * 2.0 ** -24) * np.abs(ref.out)


class AimedBatch(TreeBatch):
    PAGES = 3                                            # that a row looks at

    def __init__(self, seed, *args, **kw):
        super().__init__(seed, *args, **kw)
        rng = np.random.default_rng(seed + 1)
        along = rng.integers(0, 2, (self.n_pages, self.n_kv, self.hd)) * 2 - 1
        self.k = (along[:, :, None] + 0.3 * self.k).astype(np.float32)
        sign = rng.integers(0, 2, (self.n_pages, self.n_kv, 1, self.hd)) * 2 - 1
        self.v = (sign + 0.25 * self.v).astype(np.float32)
        q = np.zeros((len(self.pos), self.n_q, self.hd))
        self.aims = set()                                # (sequence, place in its table)
        row = 0
        for s, n in enumerate(self.new):
            places = [i for i, p in enumerate(self.table[s]) if 0 <= p < self.n_pages and i * PAGE < self.old[s]]
            for i in range(n):
                for h in range(self.n_q):
                    for x in range(self.PAGES if places else 0):
                        at = places[(row + x * (len(places) // self.PAGES)) % len(places)]
                        self.aims.add((s, at))
                        # scores of 10 where the other pages' are of one unit around zero
                        q[int(self.start[s]) + i, h] += 10 * self.hd ** -0.5 * along[self.table[s, at], h * self.n_kv // self.n_q]
                    row += 1
        self.q = q.reshape(len(self.pos), -1).astype(np.float32)
        self.round_to(torch.bfloat16)

    def bound(self, dtype, ref):
        """A weight is off by what its score's rounding makes of it (D + 3 roundings of 2^-24 of the largest sum of magnitudes), the
        exponential (2^-13 at most) and, in bfloat16, half a step, 2^-8; weights that are off by w of themselves move their mean by
        no more than w of p |v - mean| (and w of that again).  Sums of n numbers in float32, whatever their order: n 2^-23 of their
        magnitudes.  Half a step of the output."""
        half, weight = (2.0 ** -8, 2.0 ** -8 + 2.0 ** -13) if dtype == torch.bfloat16 else (0.0, 2.0 ** -20)
        weight = weight + 2 * ref.score
        return (half * np.abs(ref.out) + weight * (1 + 2 * weight) * ref.spread +
                (float(self.length.max()) + 16) * 2.0 ** -23 * 2 * (ref.mean + np.abs(ref.out)))


class Reference:
    """In 64 bits: outputs [tokens, n_q, hd]; per element a bound of p |v - mean| and p |v|; per row and head a bound of what rounding the
    score does to a weight.  without: (sequence, place in its table) of pages, (sequence, position) of keys that are left out."""

    def __init__(self, b, without_pages=(), without_keys=()):
        T, G, D = len(b.pos), b.n_q // b.n_kv, b.hd
        self.out, self.spread, self.mean = (np.zeros((T, b.n_q, D)) for _ in range(3))
        self.score = np.zeros((T, b.n_q, 1))
        q = b.q.astype(np.float64).reshape(T, b.n_q, D)
        for s, (base, n) in enumerate(zip(b.old, b.new)):
            if n == 0:
                continue
            position = np.arange(int(b.length[s]))
            position = position[position // PAGE < b.table.shape[1]]
            page = b.table[s, position // PAGE]
            there = (page >= 0) & (page < b.n_pages)
            for at in (i for x, i in without_pages if x == s):
                there &= position // PAGE != at
            for at in (i for x, i in without_keys if x == s):
                there &= position != at
            sees = np.zeros((n, len(position)), bool)
            for i, have in enumerate(b.sets[s]):
                lo = max(0, b.pos[int(b.start[s]) + i] - b.window + 1) if b.window else 0
                sees[i] = (position >= lo) & (position < base)
                at = [base + j for j in have if base + j < len(position)]
                sees[i, at] = True
            sees &= there
            rows = slice(int(b.start[s]), int(b.start[s]) + n)
            if not there.any():
                continue
            page, row = np.where(there, page, page[there][0]), np.where(there, position % PAGE, (position % PAGE)[there][0])
            for g in range(b.n_kv):
                K, V = (x[page, g, row].astype(np.float64) for x in (b.k, b.v))
                for h in range(g * G, (g + 1) * G):
                    x = np.where(sees, q[rows, h] @ K.T * b.scale, -np.inf)
                    top = x.max(1, keepdims=True)
                    p = np.where(sees, np.exp(x - np.where(np.isfinite(top), top, 0.0)), 0.0)
                    total = np.maximum(p.sum(1, keepdims=True), 1e-300)
                    o = p @ V / total                    # (whole numbers under equal weights: the sum is exact)
                    self.out[rows, h], self.mean[rows, h] = o, p @ np.abs(V) / total
                    self.spread[rows, h] = np.sqrt(np.maximum(p @ V ** 2 / total - o ** 2, 0.0))      # (no less than p |v - o|: Jensen)
                    self.score[rows, h, 0] = (np.abs(K) @ np.abs(q[rows, h]).T).max(0) * abs(b.scale) * (D + 3) * 2.0 ** -24


CASES = {
    "one of 3,000, few rows": ([3000], [7], 8, 2),
    "one of 3,000, many rows": ([3000], [40], 8, 2),
    "one of 12,000, few rows": ([12000, 400], [3, 2], 2, 1),
    "one of 12,000, many rows": ([12000, 400], [70, 2], 2, 1),
    "ragged": ([5000, 64, 1, 700, 2900, 0, 1300], [9, 33, 1, 64, 17, 5, 2], 8, 2),
    "masked pages, few rows": ([3000 - 7 * i for i in range(24)], [4] * 24, 8, 2),
    "masked pages, many rows": ([3000 - 7 * i for i in range(24)], [40] * 24, 8, 2),
}


def make(cls, case, hd):
    """A batch of one of the cases.  Masked pages: a page outside the pool in every sequence, so that whole stretches of pages take the
    masked way; what nobody sees is not finite."""
    old, new, n_q, n_kv = CASES[case]
    b = cls(hd + sum(new), old, new, n_q, n_kv, hd)
    if case.startswith("masked"):
        for s in range(len(old)):
            b.table[s, 5 + s] = -1 if s % 2 else b.n_pages + s
        held = b.table[(b.table >= 0) & (b.table < b.n_pages)]
        for p in sorted(set(range(b.n_pages)) - set(held.tolist())):
            b.k[p], b.v[p] = np.nan, np.inf
        for s, n in enumerate(b.length.tolist()):
            if n % PAGE:
                page, row = b.place(s, n)
                b.k[page, :, row:], b.v[page, :, row:] = np.inf, np.nan
    return b
