"""Cases for the operators of drafted decoding: attention of a tree of drafted tokens over the paged cache, the target's
probabilities, the drafts' verification against them, and what a cache does behind it (the kept tokens' rows move together,
a forked sequence's pages are copied).

Where `own` is false, `run` computes an operator in its plain form from elementary torch operations; where it is true it
makes the calls of stratum_b200.kernels.  Sizes are those of this repository's Llama shapes (32 query heads, 8 key/value heads
of 64 or 128, 16 or 32 layers, 128,256 or 32,000 ids, pages of 64 tokens).
"""
import math
import random

import torch

own = False

PAGE = 64


def listed():
    return [
        # one user, a short chat, a handful of drafted tokens: latency counts
        dict(name="attention one short", op="attention", dtype="bfloat16", seqs=1, len_lo=450, len_hi=450, new_lo=6, new_hi=6,
             n_q=32, n_kv=8, head_dim=128, window=0, sizes=1),
        # one user, a long document, a wide tree
        dict(name="attention one long", op="attention", dtype="bfloat16", seqs=1, len_lo=32700, len_hi=32700, new_lo=61,
             new_hi=61, n_q=32, n_kv=8, head_dim=128, window=0, sizes=2),
        # a ragged batch of the smaller shape, trees of all sizes down to a single token, a window
        dict(name="attention ragged", op="attention", dtype="bfloat16", seqs=24, len_lo=1, len_hi=8000, new_lo=1, new_hi=29,
             n_q=32, n_kv=8, head_dim=64, window=4096, sizes=3),
        # a full server: the largest
        dict(name="attention full batch", op="attention", dtype="bfloat16", seqs=64, len_lo=3000, len_hi=4100, new_lo=33,
             new_hi=64, n_q=32, n_kv=8, head_dim=128, window=0, sizes=4),
        # the true 32-bit path
        dict(name="attention float32", op="attention", dtype="float32", seqs=5, len_lo=300, len_hi=2500, new_lo=3, new_hi=17,
             n_q=32, n_kv=8, head_dim=64, window=0, sizes=5),
        # the target's distribution behind one user's tree
        dict(name="probabilities one tree", op="probabilities", rows=9, vocab=128256),
        # the same behind a full batch
        dict(name="probabilities full batch", op="probabilities", rows=1024, vocab=128256),
        # a draft model's chain for one user
        dict(name="verify one chain", op="verify", seqs=1, new_lo=6, new_hi=6, vocab=128256, drafted=True, branch=1, sizes=6),
        # trees of tokens looked up rather than drawn (no draft distribution), small vocabulary
        dict(name="verify looked-up trees", op="verify", seqs=37, new_lo=1, new_hi=31, vocab=32000, drafted=False, branch=4,
             sizes=7),
        # a full batch of trees drawn from a draft model, several tries per node
        dict(name="verify drawn trees", op="verify", seqs=64, new_lo=9, new_hi=16, vocab=128256, drafted=True, branch=3,
             sizes=8),
        # the kept tokens' rows move together behind a verified step of a batch, in all layers
        dict(name="keep rows", op="keep", layers=32, pages=384, seqs=32, new_lo=9, new_hi=31, n_kv=8, head_dim=128, sizes=9),
        # forks of a batch of prompts: their last pages are copied, in all layers
        dict(name="copy pages", op="copy", layers=16, pages=256, pairs=97, n_kv=8, head_dim=128),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def draw(rng):
    sizes = rng.randrange(1 << 20)
    op = rng.choice(["attention", "attention", "attention", "probabilities", "verify", "verify", "keep", "copy"])
    if op == "attention":
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        n_kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 4, 8])
        new_hi = _log(rng, 1, 64)
        seqs = _log(rng, 1, 48)
        # (a drawn case costs no more than the largest listed one: tokens in the cache, and tokens times rows)
        most = min(64, 64 * 32 * 48 // (n_kv * group * new_hi)) * 3500 if dtype == "bfloat16" else 16 * 1024
        len_hi = _log(rng, 1, max(2, min(32768, most // seqs)))
        return dict(op="attention", dtype=dtype, seqs=seqs, len_lo=rng.choice([0, max(1, len_hi // 3), len_hi]), len_hi=len_hi,
                    new_lo=rng.choice([1, new_hi]), new_hi=new_hi, n_q=n_kv * group, n_kv=n_kv,
                    head_dim=rng.choice([64, 128]), window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]), sizes=sizes)
    vocab = _log(rng, 1000, 200000)
    if op == "probabilities":
        return dict(op="probabilities", rows=_log(rng, 1, min(1024, 1024 * 128256 // vocab)), vocab=vocab)
    if op == "verify":
        seqs = _log(rng, 1, 64)
        new_hi = _log(rng, 1, max(1, min(64, 800 * 128256 // vocab // seqs)))
        return dict(op="verify", seqs=seqs, new_lo=1, new_hi=new_hi, vocab=vocab, drafted=rng.random() < 0.6,
                    branch=rng.choice([1, 2, 3, 5]), sizes=sizes)
    layers, n_kv, head_dim = _log(rng, 1, 32), rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
    if op == "keep":
        seqs = _log(rng, 1, 48)
        return dict(op="keep", layers=layers, pages=seqs * 3 + rng.randrange(50), seqs=seqs, new_lo=1, new_hi=_log(rng, 2, 64),
                    n_kv=n_kv, head_dim=head_dim, sizes=sizes)
    pairs = _log(rng, 1, 90)
    return dict(op="copy", layers=min(layers, 16), pages=2 * pairs + rng.randrange(60), pairs=pairs, n_kv=n_kv,
                head_dim=head_dim)


# ---------------------------------------------------------------- sizes and inputs
def _lengths(case):
    """(tokens in the cache in front of the drafts, drafted tokens) of every sequence."""
    rng = random.Random(case["sizes"])
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    old = [rng.randint(case.get("len_lo", 40), case.get("len_hi", 100)) for _ in range(case["seqs"])]
    new[0] = case["new_hi"]
    return old, new


def _trees(new, branch, rng):
    """Per sequence the parent of every node (the first has none, -1): at most `branch` children a node."""
    out = []
    for n in new:
        parents, room = [-1], [branch]
        for i in range(1, n):
            open_ = [j for j in range(max(0, i - 2 * branch), i) if room[j] > 0] or [j for j in range(i) if room[j] > 0]
            j = i - 1 if branch == 1 else rng.choice(open_)
            parents.append(j)
            room[j] -= 1
            room.append(branch)
        out.append(parents)
    return out


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    make = dict(attention=_prepare_attention, probabilities=_prepare_probabilities, verify=_prepare_verify,
                keep=_prepare_keep, copy=_prepare_copy)
    state = make[case["op"]](case, _generator(seed), random.Random(seed))
    state["op"] = case["op"]
    return state


def _prepare_attention(case, g, rng):
    old, new = _lengths(case)
    dt = getattr(torch, case["dtype"])
    H, G, D = case["n_q"], case["n_kv"], case["head_dim"]
    held = [(a + b + PAGE - 1) // PAGE for a, b in zip(old, new)]
    order = list(range(sum(held) + 3))
    rng.shuffle(order)                                   # pages of a sequence lie anywhere in the pool
    width = max(held)
    table, at = [], 0
    for n in held:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    pos, mask, words = [], [], (max(new) + 63) // 64
    for base, parents in zip(old, _trees(new, 4, rng)):
        depth, sees = [], []
        for i, p in enumerate(parents):
            depth.append(0 if p < 0 else depth[p] + 1)
            sees.append((0 if p < 0 else sees[p]) | (1 << i))
        W = case["window"]
        for i, m in enumerate(sees):
            if W > 0:                                    # the window counts positions among the drafted tokens too
                m = sum(1 << j for j in range(i + 1) if (m >> j) & 1 and depth[i] - depth[j] < W)
            pos.append(base + depth[i])
            mask.append([((m >> (64 * w)) & (2 ** 64 - 1)) - (((m >> (64 * w + 63)) & 1) << 64) for w in range(words)])
    T = sum(new)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    # keys with a common part, as trained heads have: the softmax leans on some keys, on others hardly at all
    keys = normal(len(order), G, PAGE, D).mul_(1.2).to(dt)
    return dict(q=normal(T, H * D).mul_(1.5).to(dt), k=keys, v=normal(len(order), G, PAGE, D).to(dt),
                pos=_ints(pos), mask=_ints(mask, torch.int64), start=_ints(_starts(new)),
                length=_ints([a + b for a, b in zip(old, new)]), table=_ints(table), out=torch.empty(T, H * D, dtype=dt, device="cuda"),
                n_q=H, n_kv=G, head_dim=D, window=case["window"], scale=1.0 / math.sqrt(D), max_new=max(new))


def _prepare_probabilities(case, g, rng):
    R, V = case["rows"], case["vocab"]
    logits = torch.randn(R, V, generator=g, device="cuda").mul_(3.0)
    warm = torch.rand(R, generator=g, device="cuda").mul_(0.8).add_(0.5)
    warm[rng.randrange(R)] = 0.0 if R > 1 else 0.7       # a greedy request among the others
    return dict(logits=logits, temperature=warm, out=torch.empty(R, V, device="cuda"))


def _prepare_verify(case, g, rng):
    _, new = _lengths(case)
    T, V = sum(new), case["vocab"]
    logits = torch.randn(T, V, generator=g, device="cuda").mul_(3.0)
    target = torch.softmax(logits, -1)
    # a draft model is the target with errors of its own; looked-up tokens are the target's likely ones, or wrong
    draft = torch.softmax(logits.add_(torch.randn(T, V, generator=g, device="cuda")), -1)
    del logits
    trees = _trees(new, case["branch"], rng)
    start = _starts(new)
    rows = _ints([s + max(p, 0) for s, parents in zip(start, trees) for p in parents], torch.int64)
    tokens = torch.multinomial(draft, 8, replacement=True, generator=g)[rows, _ints([rng.randrange(8) for _ in range(T)], torch.int64)]
    return dict(target=target, draft=draft if case["drafted"] else None, tokens=tokens.to(torch.int32),
                parents=_ints([p for parents in trees for p in parents]), start=_ints(start),
                uniform=torch.rand(T, generator=g, device="cuda"),
                path=torch.empty(T, dtype=torch.int32, device="cuda"), kept=torch.empty(len(new), dtype=torch.int32, device="cuda"),
                picked=torch.empty(len(new), dtype=torch.int32, device="cuda"), most=max(new), branch=case["branch"])


def _prepare_keep(case, g, rng):
    old, new = _lengths(case)
    held = [(a + b + PAGE - 1) // PAGE for a, b in zip(old, new)]
    order = list(range(case["pages"]))
    rng.shuffle(order)
    table, at = [], 0
    for n in held:
        table.append(order[at:at + n] + [-1] * (max(held) - n))
        at += n
    path, kept = [], []
    for n in new:                                        # the verified path: half of the drafts, wherever they lie
        some = sorted(rng.sample(range(1, n), (n - 1) // 2))
        path += [0] + some + [-1] * (n - 1 - len(some))
        kept.append(len(some))
    shape = (case["layers"], case["pages"], case["n_kv"], PAGE, case["head_dim"])
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    return dict(k=k, v=v, table=_ints(table), start=_ints(_starts(new)), length=_ints([a + b for a, b in zip(old, new)]),
                path=_ints(path), kept=_ints(kept), most=max(new))


def _prepare_copy(case, g, rng):
    some = rng.sample(range(case["pages"]), 2 * case["pairs"])
    shape = (case["layers"], case["pages"], case["n_kv"], PAGE, case["head_dim"])
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    return dict(k=k, v=v, src=some[:case["pairs"]], dst=some[case["pairs"]:])


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    make = dict(attention=_plain_attention, probabilities=_plain_probabilities, verify=_plain_verify, keep=_plain_keep,
                copy=_plain_copy)
    return make[state["op"]](state)


def _run_own(s):
    from stratum_b200 import kernels as K
    if s["op"] == "attention":
        K.attention_tree(s["q"], s["k"], s["v"], s["pos"], s["mask"], s["start"], s["length"], s["table"], s["out"], s["n_q"],
                         s["n_kv"], s["head_dim"], PAGE, s["window"], s["scale"], s["max_new"])
        return s["out"]
    if s["op"] == "probabilities":
        K.token_probs(s["logits"], s["temperature"], s["out"])
        return s["out"]
    if s["op"] == "verify":
        K.verify_drafts(s["target"], s["draft"], s["tokens"], s["parents"], s["start"], s["uniform"], s["path"], s["kept"],
                        s["picked"])
        return s["path"], s["kept"], s["picked"]
    if s["op"] == "keep":
        K.keep_rows(s["k"], s["v"], s["table"], s["start"], s["length"], s["path"], s["kept"])
    else:
        K.copy_pages(s["k"], s["v"], s["src"], s["dst"])
    return s["k"], s["v"]


def _padded(start, most):
    """(rows [sequences, most] of the packed tokens, which of them exist)."""
    at = start[:-1, None].long() + torch.arange(most, device="cuda")
    return at, at < start[1:, None]


def _plain_attention(s):
    q, table, length, start = s["q"], s["table"].long(), s["length"].long(), s["start"]
    G, D, B = s["n_kv"], s["head_dim"], s["table"].shape[0]
    group, T = s["n_q"] // G, q.shape[0]
    rows, real = _padded(start, s["max_new"])
    rows = rows.clamp(max=T - 1)
    k = s["k"][table.clamp(min=0)].float().transpose(1, 2).reshape(B, G, -1, D)          # [B, kv heads, keys, D]
    v = s["v"][table.clamp(min=0)].float().transpose(1, 2).reshape(B, G, -1, D)
    qs = q.float().view(T, G, group, D)[rows].permute(0, 2, 1, 3, 4).reshape(B, G, -1, D)   # rows: token * group + head
    key = torch.arange(k.shape[2], device="cuda")
    base = length - (start[1:] - start[:-1]).long()
    node = key[None] - base[:, None]                                                      # [B, keys]
    bits = s["mask"][rows]                                                                # [B, new, words]
    word = (node.clamp(0, 64 * bits.shape[2] - 1) >> 6)[:, None, :].expand(-1, rows.shape[1], -1)
    drafted = ((bits.gather(2, word) >> (node.clamp(min=0) & 63)[:, None, :]) & 1).bool() & (node >= 0)[:, None, :]
    cached = (node < 0)[:, None, :].expand(-1, rows.shape[1], -1)
    if s["window"] > 0:
        cached = cached & (key[None, None, :] > s["pos"][rows].long()[:, :, None] - s["window"])
    sees = (cached | drafted) & (key[None] < length[:, None])[:, None, :] & real[:, :, None]
    sees = sees[:, None, :, None, :].expand(-1, 1, -1, group, -1).reshape(B, 1, -1, key.numel())
    score = torch.matmul(qs, k.transpose(2, 3)).mul_(s["scale"]).masked_fill_(~sees, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = score.sub_(top).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(B, G, -1, group, D).permute(0, 2, 1, 3, 4).reshape(B, -1, s["n_q"] * D)
    return o[real].to(q.dtype)


def _plain_probabilities(s):
    logits, warm = s["logits"], s["temperature"][:, None]
    best = logits.argmax(-1, keepdim=True)
    e = ((logits - logits.gather(1, best)) / torch.where(warm > 0, warm, 1.0)).exp()
    p = e / e.sum(-1, keepdim=True, dtype=torch.float64).float()
    one = torch.arange(logits.shape[1], device="cuda")[None] == best
    return torch.where(warm > 0, p, one.float())


def _plain_verify(s):
    """Every node's children are tried as if the walk came to it (64 bits: a draw may lie next to a border), then the walk."""
    target, draft, tokens, parents, start = s["target"], s["draft"], s["tokens"].long(), s["parents"].long(), s["start"].long()
    T, B = tokens.numel(), start.numel() - 1
    seq = torch.searchsorted(start, torch.arange(T, device="cuda"), right=True) - 1
    first = start[seq]
    parent = torch.where(parents >= 0, parents + first, -1)                   # as rows of the batch
    # which child of its parent a node is
    same = parent[:, None] == parent[None]
    rank = (same & (torch.arange(T, device="cuda")[None] < torch.arange(T, device="cuda")[:, None])).sum(1)
    w = target.double().clamp(0.0, 1.0)
    mass = torch.ones(T, dtype=torch.float64, device="cuda")
    u = s["uniform"].double()
    chosen = torch.full((T,), -1, dtype=torch.int64, device="cuda")           # the child the walk goes on to
    for r in range(s["branch"]):
        child = torch.nonzero((rank == r) & (parent >= 0)).flatten()
        at, x = parent[child], tokens[child]
        q = draft[at].double().clamp(0.0, 1.0) if draft is not None else None
        qx = q.gather(1, x[:, None])[:, 0] if q is not None else torch.ones(child.numel(), dtype=torch.float64, device="cuda")
        wx = w[at, x]
        yes = (u[child] * mass[at] * qx < wx) & (chosen[at] < 0)
        no = ~yes & (chosen[at] < 0)
        chosen[at[yes]] = child[yes]
        at, x, wx = at[no], x[no], wx[no]
        if q is None:
            mass[at] = (mass[at] - wx).clamp(min=0.0)
            w[at, x] = 0.0
        else:
            rest = (w[at] - mass[at, None] * q[no]).clamp_(min=0.0)
            left = rest.sum(-1)
            some = left > 0
            w[at[some]] = rest[some]
            mass[at[some]] = left[some]
            del rest, q
    cur = start[:-1].clone()
    path = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    path[cur] = 0
    kept = torch.zeros(B, dtype=torch.int64, device="cuda")
    for depth in range(1, s["most"]):
        nxt = chosen[cur]
        on = nxt >= 0
        cur = torch.where(on, nxt, cur)
        path[(start[:-1] + depth)[on]] = (cur - start[:-1])[on].int()
        kept += on
    last = w[cur]
    cum = last.cumsum(-1)
    picked = torch.searchsorted(cum, (u[start[:-1]] * cum[:, -1])[:, None], right=True)[:, 0]
    most = last.shape[1] - 1 - (last > 0).flip(1).int().argmax(1)             # the last id with any weight
    return path, kept.int(), torch.minimum(picked, most).int()


def _plain_keep(s):
    table, start, length, path, kept = s["table"].long(), s["start"].long(), s["length"].long(), s["path"].long(), s["kept"].long()
    rows, _ = _padded(s["start"], s["most"])
    place = torch.arange(s["most"], device="cuda")[None]
    moves = (place >= 1) & (place <= kept[:, None])
    base = (length - (start[1:] - start[:-1]))[:, None]
    seq = torch.arange(table.shape[0], device="cuda")[:, None].expand_as(moves)[moves]
    src = (base + path[rows.clamp(max=path.numel() - 1)])[moves]
    dst = (base + place)[moves]
    for t in (s["k"], s["v"]):
        t[:, table[seq, dst // PAGE], :, dst % PAGE] = t[:, table[seq, src // PAGE], :, src % PAGE]
    return s["k"], s["v"]


def _plain_copy(s):
    src, dst = (torch.tensor(x, device="cuda") for x in (s["src"], s["dst"]))
    for t in (s["k"], s["v"]):
        t[:, dst] = t[:, src]
    return s["k"], s["v"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "attention":
        old, new = _lengths(case)
        size = 2 if case["dtype"] == "bfloat16" else 4
        seen = [min(a, case["window"]) if case["window"] else a for a in old]
        keys = sum(a + b for a, b in zip(seen, new))
        return dict(bytes=size * (keys * 2 * case["n_kv"] * case["head_dim"] + 2 * sum(new) * case["n_q"] * case["head_dim"]),
                    flops=4.0 * case["n_q"] * case["head_dim"] * sum(b * (a + 1) for a, b in zip(seen, new)))
    if case["op"] == "probabilities":
        return dict(bytes=8 * case["rows"] * case["vocab"], flops=4.0 * case["rows"] * case["vocab"])
    if case["op"] == "verify":                           # the row the last token is picked from, of every sequence
        rows = case["seqs"] * (2 if case["drafted"] else 1)
        return dict(bytes=4 * rows * case["vocab"] + 24 * sum(_lengths(case)[1]), flops=2.0 * rows * case["vocab"])
    row = 2 * 2 * case["layers"] * case["n_kv"] * case["head_dim"]           # a token's keys and values in all layers
    if case["op"] == "keep":
        return dict(bytes=2 * row * sum((n - 1) // 2 for n in _lengths(case)[1]) + 1, flops=0)
    return dict(bytes=2 * row * PAGE * case["pairs"], flops=0)


# ---------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    make = dict(attention=_exact_attention, probabilities=_exact_probabilities, verify=_exact_verify, keep=_exact_keep,
                copy=_exact_copy)
    return make[case["op"]](s)


def _exact_attention(s):
    start, length, table = s["start"].tolist(), s["length"].tolist(), s["table"].tolist()
    pos, mask = s["pos"].tolist(), s["mask"].tolist()
    G, D = s["n_kv"], s["head_dim"]
    group = s["n_q"] // G
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n_keys in enumerate(length):
        a, e = start[b], start[b + 1]
        pages = [table[b][i] for i in range((n_keys + PAGE - 1) // PAGE)]
        keys, values = (torch.cat([t[p].double() for p in pages], 1)[:, :n_keys] for t in (s["k"], s["v"]))
        base = n_keys - (e - a)
        sees = torch.zeros(e - a, n_keys, dtype=torch.bool)
        for i in range(a, e):
            lo = max(0, pos[i] - s["window"] + 1) if s["window"] > 0 else 0
            sees[i - a, min(lo, base):base] = True
            for j in range(e - a):
                sees[i - a, base + j] = bool((mask[i][j // 64] >> (j % 64)) & 1)
        sees = sees.cuda()
        for h in range(s["n_q"]):
            x = s["q"][a:e, h * D:(h + 1) * D].double() @ keys[h // group].T * s["scale"]
            p = torch.softmax(x.masked_fill(~sees, -math.inf), -1).nan_to_num(0.0)
            out[a:e, h * D:(h + 1) * D] = p @ values[h // group]
    return out


def _exact_probabilities(s):
    out = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    for r, t in enumerate(s["temperature"].tolist()):
        if t > 0:
            out[r] = torch.softmax(s["logits"][r].double() / t, -1)
        else:
            out[r, int(torch.nonzero(s["logits"][r] == s["logits"][r].max())[0])] = 1.0
    return out


def _exact_verify(s):
    start, parents, tokens, u = s["start"].tolist(), s["parents"].tolist(), s["tokens"].tolist(), s["uniform"].tolist()
    path = [-1] * len(tokens)
    kept, picked = [], []
    for a, e in zip(start, start[1:]):
        node, depth, going = 0, 0, True
        path[a] = 0
        while going:
            d, mass, going = s["target"][a + node].double().clamp(0.0, 1.0), 1.0, False
            for c in range(node + 1, e - a):
                if parents[a + c] != node:
                    continue
                x = tokens[a + c]
                if s["draft"] is None:
                    if u[a + c] * mass < float(d[x]):
                        going = True
                    else:
                        mass = max(0.0, mass - float(d[x]))
                        d[x] = 0.0
                else:
                    q = s["draft"][a + node].double().clamp(0.0, 1.0)
                    if u[a + c] * mass * float(q[x]) < float(d[x]):
                        going = True
                    else:
                        rest = torch.relu(d - mass * q)
                        if float(rest.sum()) > 0:
                            d, mass = rest, float(rest.sum())
                if going:
                    node, depth = c, depth + 1
                    path[a + depth] = c
                    break
        kept.append(depth)
        cum = torch.cumsum(d, 0)
        over = torch.nonzero(cum > u[a] * cum[-1])
        picked.append(int(over[0]) if over.numel() else int(torch.nonzero(d > 0)[-1]))
    return tuple(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (path, kept, picked))


def _exact_keep(s):
    k, v = s["k"].double(), s["v"].double()
    table, start, length, path, kept = (s[n].tolist() for n in ("table", "start", "length", "path", "kept"))
    for b, n in enumerate(kept):
        base = length[b] - (start[b + 1] - start[b])
        for j in range(1, n + 1):                        # a row's new place is never behind the row: one after the other
            src, dst = base + path[start[b] + j], base + j
            for t in (k, v):
                t[:, table[b][dst // PAGE], :, dst % PAGE] = t[:, table[b][src // PAGE], :, src % PAGE].clone()
    return k, v


def _exact_copy(s):
    k, v = s["k"].double(), s["v"].double()
    for a, b in zip(s["src"], s["dst"]):
        k[:, b], v[:, b] = k[:, a], v[:, a]
    return k, v
