"""The target's probabilities and the walk through drafted tokens against plain implementations in 64 bits."""
import numpy as np
import pytest
import torch

from draft_helpers import random_tree

pytestmark = pytest.mark.gpu


def dev(a, dtype):
    return torch.tensor(np.asarray(a), dtype=dtype, device="cuda")


# ------------------------------------------------------------------------------------------ probabilities
def plain_probs(logits, temperature):
    out = np.zeros(logits.shape)
    for r, t in enumerate(temperature):
        x = logits[r].astype(np.float64)
        x[np.isnan(x)] = -np.inf
        m = x.max()
        if m == -np.inf:
            continue
        if not t > 0:
            out[r, int(np.argmax(x))] = 1.0
            continue
        with np.errstate(invalid="ignore"):
            e = np.where(x == m, 1.0, np.where(np.isinf(x), 0.0, np.exp((x - m) / np.float64(t))))
        out[r] = e / e.sum()
    return out


def check_probs(logits, temperature, out):
    """exp2((l - max) * (log2 e / T)): the exponent is off by three roundings of 2^-24 of itself, which is at most 160 before
    the result is zero in float32 (times ln 2: the relative error of the result), exp2f by 2 units, the sum of n values by
    its 32 + 5 + 4 + 4 levels of additions, the reciprocal and the last product by one each."""
    ref = plain_probs(logits, temperature)
    got = out.cpu().numpy().astype(np.float64)
    with np.errstate(divide="ignore"):
        exponent = np.where(ref > 0, -np.log2(np.maximum(ref, 1e-300)), 0.0) + np.log2(max(2, logits.shape[1]))
    rel = (3 * np.minimum(exponent, 200.0) * 0.7 + 4 + 64) * 2.0 ** -24
    assert (np.abs(got - ref) <= rel * ref + 2.0 ** -126 * 4).all()


@pytest.mark.parametrize("vocab", [1, 2, 31, 511, 512, 513, 4097, 16384, 16385, 32003, 128256, 262144, 262145])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_probabilities(vocab, rows):
    from stratum_b200 import kernels as K
    rng = np.random.default_rng(vocab + rows)
    logits = (rng.standard_normal((rows, vocab)) * 4).astype(np.float32)
    t = rng.uniform(0.1, 2.0, rows).astype(np.float32)
    t[rows // 2] = 0.0
    out = torch.full((rows, vocab), -1.0, device="cuda")
    K.token_probs(dev(logits, torch.float32), dev(t, torch.float32), out)
    check_probs(logits, t, out)


def test_probabilities_of_odd_rows():
    """Infinities, values that are no numbers, rows of nothing, equal largest logits, temperatures of every kind; rows apart; in place."""
    from stratum_b200 import kernels as K
    inf, nan = float("inf"), float("nan")
    rng = np.random.default_rng(0)
    base = (rng.standard_normal((12, 1003)) * 3).astype(np.float32)
    base[0, 5], base[1, :], base[2, 7:9], base[3, ::2] = nan, -inf, inf, -inf
    base[4, :], base[5, :] = nan, 2.5
    base[6, 100], base[6, 900] = 50.0, 50.0
    base[7, 3] = inf
    base[8] = -3.4e38
    base[9] = np.float32(3.4e38) * np.where(np.arange(1003) % 2, 1, -1)
    t = np.array([1, 1, 1, 0.5, 1, 2, 0, 0, 1, 1, -1, nan], np.float32)
    for extra in (0, 5):
        wide = torch.zeros(12, 1003 + extra, device="cuda")
        wide[:, :1003] = dev(base, torch.float32)
        out = torch.full((12, 1003 + extra), 9.0, device="cuda")
        K.token_probs(wide[:, :1003], dev(t, torch.float32), out[:, :1003])
        check_probs(base, t, out[:, :1003])
        assert (out[:, 1003:] == 9.0).all()
        K.token_probs(wide[:, :1003], dev(t, torch.float32), wide[:, :1003])
        assert torch.equal(wide[:, :1003], out[:, :1003])


@pytest.mark.parametrize("rows,vocab", [(600, 8192), (601, 4100), (330, 30000), (150, 65540), (100, 128256), (75, 200000)])
def test_probabilities_of_many_rows(rows, vocab):
    """Rows enough for the blocks that stay; rows apart, in place, and odd ones among them."""
    from stratum_b200 import kernels as K
    rng = np.random.default_rng(rows)
    base = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    base[3], base[5, 7:9], base[7, 11], base[9, ::2] = -np.inf, np.inf, np.nan, -np.inf
    base[11, 100], base[11, vocab - 2] = 30.0, 30.0
    t = rng.uniform(0.3, 1.5, rows).astype(np.float32)
    t[11], t[rows - 1] = 0.0, 0.0
    x = torch.zeros(rows, vocab + 4, device="cuda")
    x[:, :vocab] = dev(base, torch.float32)
    out = torch.full((rows, vocab + 8), 9.0, device="cuda")
    K.token_probs(x[:, :vocab], dev(t, torch.float32), out[:, :vocab])
    K.token_probs(x[:, :vocab], dev(t, torch.float32), x[:, :vocab])
    K.check_status()
    check_probs(base, t, out[:, :vocab])
    assert (out[:, vocab:] == 9.0).all() and (x[:, vocab:] == 0.0).all() and torch.equal(x[:, :vocab], out[:, :vocab])


def test_probabilities_do_not_depend_on_the_batch():
    """(as long as the rows are cut alike: a row's bits follow from its values and the blocks it is given)"""
    from stratum_b200 import kernels as K
    x = torch.randn(300, 128256, device="cuda")
    t = torch.ones(300, device="cuda")
    a, b = torch.empty_like(x), torch.empty(299, 128256, device="cuda")
    K.token_probs(x, t, a)
    K.token_probs(x[1:], t[1:], b)
    assert torch.equal(a[1:], b)


# ------------------------------------------------------------------------------------------ verification
def clamp(p):
    p = p.astype(np.float64)
    return np.clip(np.where(np.isnan(p), 0.0, p), 0.0, 1.0)


def plain_verify(target, draft, tokens, parents, start, u, most=1024):
    path, kept, nxt = [-1] * (start[-1]), [], []
    V = target.shape[1]
    for a, e in zip(start, start[1:]):
        n = e - a
        if n == 0:
            kept.append(0); nxt.append(-1)
            continue
        node, depth, going = 0, 0, True
        path[a] = 0
        while going:
            d, mass, going = clamp(target[a + node]), 1.0, False
            for c in range(node + 1, min(n, most)):
                x = tokens[a + c]
                if parents[a + c] != node or not 0 <= x < V:
                    continue
                if draft is None:
                    if np.float64(u[a + c]) * mass < d[x]:
                        going = True
                    else:
                        mass, d[x] = max(mass - d[x], 0.0), 0.0
                else:
                    q = clamp(draft[a + node])
                    if np.float64(u[a + c]) * mass * q[x] < d[x]:
                        going = True
                    else:
                        rest = np.maximum(d - mass * q, 0.0)
                        if rest.sum() > 0:
                            d, mass = rest, rest.sum()
                if going:
                    node, depth = c, depth + 1
                    path[a + depth] = c
                    break
        kept.append(depth)
        cum = np.cumsum(d)
        if not cum[-1] > 0:
            nxt.append(0)
            continue
        over = np.nonzero((cum > np.float64(u[a]) * cum[-1]) & (d > 0))[0]
        nxt.append(int(over[0]) if len(over) else int(np.nonzero(d > 0)[0][-1]))
    return path, kept, nxt


def run_verify(target, draft, tokens, parents, start, u, tail=0):
    from stratum_b200 import kernels as K
    T, B = target.shape[0], len(start) - 1
    path = torch.full((T,), 77, dtype=torch.int32, device="cuda")
    kept, nxt = (torch.full((B,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    K.verify_drafts(dev(target, torch.float32), None if draft is None else dev(draft, torch.float32), dev(tokens, torch.int32),
                    dev(parents, torch.int32), dev(start, torch.int32), dev(u, torch.float32), path, kept, nxt)
    return path.tolist(), kept.tolist(), nxt.tolist()


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def make(seed, new, V, drafted, branch, spread=3.0):
    rng = np.random.default_rng(seed)
    T = sum(new)
    logits = rng.standard_normal((T, V)) * spread
    target, draft = softmax(logits), softmax(logits + rng.standard_normal((T, V)))
    start = np.concatenate([[0], np.cumsum(new)]).astype(int).tolist()
    parents, tokens = [], []
    for a, n in zip(start, new):
        tree = [-1] + list(range(n - 1)) if branch == 1 else random_tree(rng, n, branch)
        parents += tree[:n]
        for p in tree[:n]:
            row = draft[a + max(p, 0)].astype(np.float64)
            tokens.append(int(rng.choice(V, p=row / row.sum())))
    u = (rng.integers(0, 2 ** 24, T) / 2.0 ** 24).astype(np.float32)
    return target, draft if drafted else None, tokens, parents, start, u


@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("branch", [1, 2, 6])
@pytest.mark.parametrize("new,V", [([1], 1), ([7], 2), ([1, 3, 0, 9, 30, 2], 517), ([5, 65, 12], 4099), ([4] * 40, 32), ([9], 128256),
                                   ([6, 2], 16385), ([0, 0, 3], 33)])
def test_verification(drafted, branch, new, V):
    for seed in range(4):
        args = make(seed + V, new, V, drafted, branch)
        assert run_verify(*args) == tuple(plain_verify(*args)), seed


def test_many_sequences():
    args = make(1, [int(n) for n in np.random.default_rng(5).integers(0, 12, 300)], 1000, True, 3)
    assert run_verify(*args) == tuple(plain_verify(*args))


def test_greedy_rows_keep_exactly_the_greedy_path():
    """One-hot targets: a draft is kept if and only if it is the target's pick."""
    for drafted in (True, False):
        target, draft, tokens, parents, start, u = make(3, [8, 20, 1], 300, drafted, 3)
        hot = np.zeros_like(target)
        hot[np.arange(len(hot)), target.argmax(1)] = 1.0
        path, kept, nxt = run_verify(hot, draft, tokens, parents, start, u)
        assert (path, kept, nxt) == tuple(plain_verify(hot, draft, tokens, parents, start, u))
        for s, (a, e) in enumerate(zip(start, start[1:])):
            node = 0
            for j in range(kept[s]):
                child = path[a + j + 1]
                assert parents[a + child] == node and tokens[a + child] == int(target[a + node].argmax())
                node = child
            assert nxt[s] == int(target[a + node].argmax())


@pytest.mark.parametrize("drafted", [True, False])
def test_odd_numbers(drafted):
    """Numbers at their ends, tokens outside the vocabulary, parents that are none, rows without weight, with NaN, above one."""
    target, draft, tokens, parents, start, u = make(9, [12, 12, 12, 6, 6], 97, drafted, 4)
    u[:12], u[12:24] = 0.0, np.float32(1.0) - np.float32(2.0 ** -24)
    tokens[3], tokens[14], tokens[30] = -1, 97, 2 ** 31 - 1
    parents[5], parents[17], parents[31] = 5, 11, -7
    target[36:42] = 0.0
    target[42:48] = np.nan
    target[42:48, 4], target[42:48, 9] = 0.25, 3.0
    if drafted:
        draft[24:30] = np.nan
        draft[42] = target[42]                       # nothing is left behind a rejection: the row stays
    args = (target, draft, tokens, parents, start, u)
    assert run_verify(*args) == tuple(plain_verify(*args))


def test_rows_of_no_sequence_are_left():
    target, draft, tokens, parents, start, u = make(4, [5, 7], 50, True, 2)
    start[-1] -= 3
    path, kept, nxt = run_verify(target, draft, tokens, parents, start, u)
    want = plain_verify(target, draft, tokens, parents, start, u)
    assert path[:9] == want[0][:9] and path[9:] == [77] * 3 and (kept, nxt) == want[1:]


def test_kept_tokens_are_distributed_as_the_target():
    """Twenty thousand walks over one small tree: the first token of each against the target's row, by a chi-square bound.
    6 ids, so 5 degrees of freedom: the statistic is above 30 in 1.5 of 100,000 samples; the numbers are fixed."""
    rng = np.random.default_rng(123)
    V, N = 6, 20000
    p, q = softmax(rng.standard_normal((1, V)) * 1.5)[0], softmax(rng.standard_normal((1, V)) * 1.5)[0]
    for drafted in (True, False):
        n = 4                                        # the first node and three tries
        target = np.tile(p, (N * n, 1)).astype(np.float32)
        tokens = np.zeros((N, n), int)
        tokens[:, 1:] = rng.choice(V, (N, 3), p=q.astype(np.float64) / q.astype(np.float64).sum())
        u = (rng.integers(0, 2 ** 24, N * n) / 2.0 ** 24).astype(np.float32)
        start = (np.arange(N + 1) * n).tolist()
        path, kept, nxt = run_verify(target, np.tile(q, (N * n, 1)).astype(np.float32) if drafted else None, tokens.reshape(-1),
                                     [-1, 0, 0, 0] * N, start, u)
        got = np.array([tokens[s, path[s * n + 1]] if kept[s] else nxt[s] for s in range(N)])
        want = p.astype(np.float64) / p.astype(np.float64).sum() * N
        count = np.bincount(got, minlength=V)
        assert ((count - want) ** 2 / want).sum() < 30.0


def test_verification_captured_and_on_two_streams():
    from stratum_b200 import kernels as K
    sets = [make(s, [9, 4, 17], 5000, True, 2) for s in range(2)]
    runs = []
    for t, d, tok, par, start, u in sets:
        held = [dev(t, torch.float32), dev(d, torch.float32), dev(tok, torch.int32), dev(par, torch.int32), dev(start, torch.int32),
                dev(u, torch.float32)]
        out = [torch.zeros(30, dtype=torch.int32, device="cuda")] + [torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2)]
        K.verify_drafts(*held, *out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.verify_drafts(*held, *out)
        runs.append((g, held, out))
    streams = [torch.cuda.Stream() for _ in runs]
    for (g, _, out), st in zip(runs, streams):
        for o in out:
            o.zero_()
    torch.cuda.synchronize()
    for (g, *_), st in zip(runs, streams):
        with torch.cuda.stream(st):
            for _ in range(10):
                g.replay()
    torch.cuda.synchronize()
    for (g, held, out), args in zip(runs, sets):
        assert tuple(o.tolist() for o in out) == tuple(plain_verify(*args))
