"""Drafted tokens for the tests: trees, paged caches with every kind of page order, and 64-bit references."""
import numpy as np
import torch

PAGE = 64


def random_tree(rng, n, branch=3):
    """Parents of n nodes (the first: -1), each in front of its children."""
    return [-1] + [int(rng.integers(max(0, i - branch), i)) for i in range(1, n)]


def depths(parents):
    out = []
    for p in parents:
        out.append(0 if p < 0 else out[p] + 1)
    return out


def sees(parents):
    """Per node the set of nodes it sees: its ancestors and itself."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else set()) | {i})
    return out


def mask_words(sets, words):
    """int64 rows: bit j of word w = node 64 w + j."""
    m = np.zeros((len(sets), words), dtype=np.uint64)
    for i, s in enumerate(sets):
        for j in s:
            m[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return m.view(np.int64)


class TreeBatch:
    """Inputs of kernels.attention_tree on the CPU, as numpy arrays; `sets[s][i]`: what node i of sequence s sees."""

    def __init__(self, seed, old, new, n_q, n_kv, hd, window=0, words=None, width=None, spare=3, spread=1.0):
        rng = np.random.default_rng(seed)
        self.n_q, self.n_kv, self.hd, self.window, self.scale = n_q, n_kv, hd, window, hd ** -0.5
        self.old, self.new = list(old), list(new)
        held = [-(-(a + b) // PAGE) for a, b in zip(old, new)]
        n_pages = sum(held) + spare
        order = rng.permutation(n_pages)
        self.table = np.full((len(old), width or max(1, max(held))), -1, np.int32)
        at = 0
        for s, n in enumerate(held):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.trees = [random_tree(rng, n) for n in new]
        self.sets, self.pos = [], []
        for base, tree in zip(old, self.trees):
            d = depths(tree)
            self.sets.append([{j for j in have if window == 0 or d[i] - d[j] < window} for i, have in enumerate(sees(tree))])
            self.pos += [base + x for x in d]
        self.words = words or max(1, -(-max(new) // 64))
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.length = np.array([a + b for a, b in zip(old, new)], np.int32)
        T = int(self.start[-1])
        f = lambda *shape: (rng.standard_normal(shape) * spread).astype(np.float32)      # noqa: E731
        self.q, self.k, self.v = f(T, n_q * hd), f(n_pages, n_kv, PAGE, hd), f(n_pages, n_kv, PAGE, hd)
        self.n_pages = n_pages

    def place(self, s, position):
        """(page, row) of a sequence's key."""
        return int(self.table[s, position // PAGE]), position % PAGE

    def mask(self):
        rows = [mask_words(sets, self.words) for sets in self.sets if sets]
        return np.concatenate(rows) if rows else np.zeros((0, self.words), np.int64)

    def round_to(self, dtype):
        for name in ("q", "k", "v"):
            setattr(self, name, torch.from_numpy(getattr(self, name)).to(dtype).float().numpy())
        return self

    def reference(self):
        """(outputs in 64 bits [tokens, n_q * hd], per element a bound of the values it averages: (largest - smallest, mean
        of |v|), and per row and head a bound of its scores' rounding in float32)."""
        G, D = self.n_q // self.n_kv, self.hd
        out = np.zeros((int(self.start[-1]), self.n_q, D))
        span, mean, score_err = np.zeros_like(out), np.zeros_like(out), np.zeros(out.shape[:2])
        q = self.q.astype(np.float64).reshape(-1, self.n_q, D)
        for s, base in enumerate(self.old):
            for i, have in enumerate(self.sets[s]):
                t = int(self.start[s]) + i
                lo = max(0, self.pos[t] - self.window + 1) if self.window else 0
                keys = [p for p in list(range(lo, base)) + [base + j for j in sorted(have)]
                        if p < self.length[s] and p // PAGE < self.table.shape[1] and 0 <= self.table[s, p // PAGE] < self.n_pages]
                if not keys:
                    continue
                pg, row = self.table[s, np.array(keys) // PAGE], np.array(keys) % PAGE
                for h in range(self.n_q):
                    K, V = (x[pg, h // G, row].astype(np.float64) for x in (self.k, self.v))
                    with np.errstate(invalid="ignore", over="ignore"):
                        x = K @ q[t, h] * self.scale
                        p = np.exp(x - x.max())
                        p /= p.sum()
                        out[t, h] = p @ V
                        span[t, h] = V.max(0) - V.min(0)
                        mean[t, h] = p @ np.abs(V)
                        score_err[t, h] = (np.abs(K) @ np.abs(q[t, h])).max() * abs(self.scale) * (D + 3) * 2.0 ** -24
        T = out.shape[0]
        return out.reshape(T, -1), span.reshape(T, -1), mean.reshape(T, -1), np.repeat(score_err, D, 1)

    def bound(self, dtype, ref):
        """How far a kernel may be off, element by element.  bfloat16: half a step of the output (2^-8 of it); probabilities
        shortened to 8 bits, each low by a factor within 2^-7 of one, so that a mean of values moves by at most 2^-7 of their
        spread; float32 rounding of the scores (twice: in the weight and in the sum) and of the sums.  float32: the last two."""
        out, span, mean, score = ref
        n = float(self.length.max(initial=1))
        f32 = (2.0 * score + (n + 16.0) * 2.0 ** -23) * 2.0 * (mean + np.abs(out)) + 1e-30
        if dtype == torch.float32:
            return f32
        return 2.0 ** -8 * np.abs(out) + 2.0 ** -7 * span + f32


def run_tree(b, dtype, out=None, extra_q=0, extra_out=0, max_new=None, device="cuda"):
    """kernels.attention_tree on a TreeBatch; the rows of q and out lie `extra` columns further apart than they are wide."""
    from stratum_b200 import kernels as K
    dev = lambda a, dt=None: torch.from_numpy(np.ascontiguousarray(a)).to(device=device, dtype=dt)      # noqa: E731
    T, W = b.q.shape
    q = torch.zeros(T, W + extra_q, dtype=dtype, device=device)
    q[:, :W] = dev(b.q, dtype)
    if out is None:
        out = torch.full((T, W + extra_out), 7.0, dtype=dtype, device=device)
    K.attention_tree(q, dev(b.k, dtype), dev(b.v, dtype), dev(np.array(b.pos, np.int32)), dev(b.mask()), dev(b.start),
                     dev(b.length), dev(b.table), out, b.n_q, b.n_kv, b.hd, PAGE, b.window, b.scale,
                     max(b.new) if max_new is None else max_new)
    return out
