"""Attention of drafted tokens over the paged cache against a plain implementation in 64 bits."""
import numpy as np
import pytest
import torch

from draft_helpers import PAGE, TreeBatch, run_tree

pytestmark = pytest.mark.gpu
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def check(b, dtype, out):
    from stratum_b200 import kernels as K
    K.check_status()
    ref = b.reference()
    W = b.n_q * b.hd
    got = out[:, :W].float().cpu().numpy().astype(np.float64)
    off, most = np.abs(got - ref[0]), b.bound(dtype, ref)
    assert np.isfinite(got).all()
    worst = int(np.argmax(off / most))
    assert (off <= most).all(), (off.flat[worst], most.flat[worst], np.unravel_index(worst, off.shape))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_q,n_kv", [(4, 4), (8, 2), (8, 1), (5, 1)])
def test_ragged_trees(dtype, hd, n_q, n_kv):
    """Caches that end at, in front of and behind a page's end, empty ones; trees of one token up to more than a page."""
    b = TreeBatch(hd + n_q, [0, 0, 1, 63, 64, 65, 200, 451], [1, 9, 5, 1, 70, 2, 17, 30], n_q, n_kv, hd).round_to(DT[dtype])
    check(b, DT[dtype], run_tree(b, DT[dtype]))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("old,new", [([0], [1]), ([5], [1]), ([700], [1]), ([3000], [7]), ([3000], [40]), ([1990, 64, 0], [130, 3, 200])])
def test_few_sequences(dtype, old, new):
    """Long caches whose pages many CTAs share, fewer pages than CTAs, trees of more than one mask word and of more rows than a CTA."""
    b = TreeBatch(sum(old), old, new, 8, 2, 64).round_to(DT[dtype])
    check(b, DT[dtype], run_tree(b, DT[dtype]))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [1, 3, 64, 100, 5000])
def test_window(dtype, window):
    b = TreeBatch(window, [0, 70, 300, 1000, 130], [3, 20, 9, 33, 1], 8, 2, 64, window=window).round_to(DT[dtype])
    check(b, DT[dtype], run_tree(b, DT[dtype]))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd,n_q,n_kv", [(16, 6, 2), (80, 6, 2), (33, 3, 3), (256, 4, 2), (200, 2, 1), (96, 40, 1)])
def test_other_head_sizes(dtype, hd, n_q, n_kv):
    b = TreeBatch(hd, [10, 130, 0], [4, 9, 2], n_q, n_kv, hd).round_to(DT[dtype])
    check(b, DT[dtype], run_tree(b, DT[dtype]))


@pytest.mark.parametrize("n_q,n_kv,new", [(3, 1, 43), (7, 1, 37), (24, 2, 11), (48, 1, 5), (128, 1, 3), (130, 1, 2)])
def test_groups_that_do_not_divide_a_tile(n_q, n_kv, new):
    b = TreeBatch(n_q, [100, 66], [new, 1], n_q, n_kv, 64).round_to(torch.bfloat16)
    check(b, torch.bfloat16, run_tree(b, torch.bfloat16))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rows_apart_and_not_aligned(dtype):
    """q and out as columns of wider rows; a distance no vector load divides takes the CUDA-core kernel."""
    b = TreeBatch(5, [100, 20], [9, 4], 8, 2, 64).round_to(DT[dtype])
    for extra in (64, 3):
        out = run_tree(b, DT[dtype], extra_q=extra, extra_out=extra)
        check(b, DT[dtype], out)
        assert (out[:, 512:] == 7.0).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("max_new", [0, 1, 16, 17, 4000])
def test_cut_does_not_follow_a_wrong_max_new(dtype, max_new):
    b = TreeBatch(6, [100, 500], [40, 4], 8, 2, 64).round_to(DT[dtype])
    check(b, DT[dtype], run_tree(b, DT[dtype], max_new=max_new))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd", [64, 128, 40])
@pytest.mark.parametrize("new", [[9, 4, 1], [45, 30, 2]])
def test_masked_keys_may_hold_anything(dtype, hd, new):
    """Rows behind a sequence's end and drafted branches that a row does not see hold NaN and infinities, in keys and values."""
    b = TreeBatch(hd + new[0], [0, 100, 190], new, 8, 2, hd).round_to(DT[dtype])
    clean = run_tree(b, DT[dtype])
    for s, n in enumerate(b.length):
        last = b.table[s, (n - 1) // PAGE]
        if n % PAGE:
            b.k[last, :, n % PAGE:] = np.nan
            b.v[last, :, n % PAGE:] = np.inf
    # the last node of the first two trees overflowed: nobody but itself (no node has it as a parent) sees it
    bad = []
    for s in (0, 1):
        node = len(b.trees[s]) - 1
        pg, row = b.place(s, b.old[s] + node)
        b.k[pg, :, row], b.v[pg, :, row, ::2] = np.nan, -np.inf
        bad.append(int(b.start[s]) + node)
    out = run_tree(b, DT[dtype])
    keep = [t for t in range(out.shape[0]) if t not in bad]
    assert torch.equal(out[keep], clean[keep])
    assert not torch.isfinite(out[bad].float()).all(1).any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("new", [4, 40])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(dtype, new):
    """An infinity in the values of a drafted token, element by element: the rows below it get it, the others do not."""
    b = TreeBatch(3, [64], [new], 8, 2, 64).round_to(DT[dtype])       # (the tree is all of its page: the first of a run too)
    clean = run_tree(b, DT[dtype]).float()
    pg, row = b.place(0, 64 + 1)
    b.v[pg, :, row, 5] = np.inf
    out = run_tree(b, DT[dtype]).float().view(-1, 8, 64)
    under = [1 in have for have in b.sets[0]]
    for t, u in enumerate(under):
        assert bool((out[t, :, 5] == float("inf")).all()) == u
    out[:, :, 5] = clean.view(-1, 8, 64)[:, :, 5]
    # (a page with such a value adds it by hand: the other elements may come out in another order of additions)
    ref = b.reference()
    most = torch.from_numpy(b.bound(DT[dtype], tuple(np.nan_to_num(x, posinf=0.0, neginf=0.0) for x in ref))).float().view(-1, 8, 64)
    diff = (out.cpu() - clean.view(-1, 8, 64).cpu()).abs()
    rest = [d for d in range(64) if d != 5]
    assert (diff[:, :, rest] <= most[:, :, rest]).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rows_that_see_nothing_and_rows_of_no_sequence(dtype):
    b = TreeBatch(8, [0, 70], [5, 6], 8, 2, 64).round_to(DT[dtype])
    b.sets[0][2] = set()
    check(b, DT[dtype], run_tree(b, DT[dtype]))
    b.start[-1] -= 2                                       # the last two rows belong to no sequence
    b.length[1] -= 2
    out = run_tree(b, DT[dtype])
    assert (out[2] == 0).all() and (out[-2:] == 7.0).all() and (out[:-2] != 7.0).any(1).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_pages_outside_the_pool_hold_keys_nobody_sees(dtype):
    b = TreeBatch(9, [400, 300], [9, 33], 8, 2, 64).round_to(DT[dtype])
    b.table[0, 2], b.table[1, 1], b.table[1, 0] = -1, b.n_pages, 2 ** 31 - 1
    check(b, DT[dtype], run_tree(b, DT[dtype]))
    b.table = np.ascontiguousarray(b.table[:, :4])         # a table that is too narrow for the lengths
    check(b, DT[dtype], run_tree(b, DT[dtype]))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_large_scores(dtype):
    """Scores of hundreds, where a running maximum is what keeps the exponentials finite."""
    b = TreeBatch(10, [500, 77], [9, 20], 8, 2, 64, spread=6.0).round_to(DT[dtype])
    check(b, DT[dtype], run_tree(b, DT[dtype]))


@pytest.mark.parametrize("dtype,new", [("bfloat16", 9), ("bfloat16", 40), ("float32", 9)])
def test_captured_and_replayed_with_other_lengths(dtype, new):
    """A captured launch serves whatever lengths its description holds at the replay, and two graphs do not meet in scratch."""
    from stratum_b200 import kernels as K
    dev = lambda a, dt=None: torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=dt)      # noqa: E731
    runs = []
    for seed in (1, 2):
        a = TreeBatch(seed, [900, 30], [new, 3], 8, 2, 64, width=20, spare=40).round_to(DT[dtype])
        b = TreeBatch(seed + 5, [64, 700], [2, new + 1], 8, 2, 64, width=20, spare=40).round_to(DT[dtype])
        T, pages = new + 3, max(a.n_pages, b.n_pages)
        pad = lambda x: np.concatenate([x, np.zeros((pages - x.shape[0],) + x.shape[1:], x.dtype)])       # noqa: E731
        make = lambda x: (dev(x.q, DT[dtype]), dev(pad(x.k), DT[dtype]), dev(pad(x.v), DT[dtype]), dev(np.array(x.pos, np.int32)),   # noqa: E731
                          dev(x.mask()), dev(x.start), dev(x.length), dev(x.table))
        held, out = make(a), torch.zeros(T, 512, dtype=DT[dtype], device="cuda")
        call = lambda: K.attention_tree(*held, out, 8, 2, 64, PAGE, 0, a.scale, new + 1)      # noqa: E731,B023
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        runs.append((g, held, out, a, b, make))
    streams = [torch.cuda.Stream() for _ in runs]
    for which in ("a", "b"):
        for g, held, out, a, b, make in runs:
            for dst, src in zip(held, make(a if which == "a" else b)):
                dst.copy_(src)
            out.zero_()
        torch.cuda.synchronize()
        for (g, *_), st in zip(runs, streams):
            with torch.cuda.stream(st):
                for _ in range(20):
                    g.replay()
        torch.cuda.synchronize()
        for g, held, out, a, b, make in runs:
            check(a if which == "a" else b, DT[dtype], out)


def test_two_streams_at_once():
    batches = [TreeBatch(i, [2000, 100], [20 + i, 5], 8, 2, 64).round_to(torch.bfloat16) for i in range(2)]
    want = [run_tree(b, torch.bfloat16) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[], []]
    for _ in range(10):
        for i, (b, st) in enumerate(zip(batches, streams)):
            with torch.cuda.stream(st):
                got[i].append(run_tree(b, torch.bfloat16))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)            # the order of additions is fixed


def test_pages_beyond_32_bits_of_bytes():
    """A page whose rows lie behind 2^31 elements of the pool."""
    n_pages, n_kv, hd = 40000, 8, 128                        # 2.6 G elements in the keys
    b = TreeBatch(11, [130], [9], 8, 8, 128).round_to(torch.bfloat16)
    from stratum_b200 import kernels as K
    dev = lambda a, dt=None: torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=dt)      # noqa: E731
    k = torch.zeros(n_pages, n_kv, PAGE, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    far = n_pages - b.n_pages
    k[far:], v[far:] = dev(b.k, torch.bfloat16), dev(b.v, torch.bfloat16)
    out = torch.empty(9, 8 * hd, dtype=torch.bfloat16, device="cuda")
    table = np.where(b.table >= 0, b.table + far, -1).astype(np.int32)
    K.attention_tree(dev(b.q, torch.bfloat16), k, v, dev(np.array(b.pos, np.int32)), dev(b.mask()), dev(b.start), dev(b.length),
                     dev(table), out, 8, 8, hd, PAGE, 0, b.scale, 9)
    check(b, torch.bfloat16, out)


@pytest.mark.parametrize("dtype,hd", [("bfloat16", 64), ("bfloat16", 128), ("bfloat16", 200), ("float32", 80), ("float32", 6)])
@pytest.mark.parametrize("new", [3, 70])
def test_pieces_of_many_stretches(dtype, hd, new):
    """One sequence that dozens of CTAs see pieces of, beside one that two see."""
    b = TreeBatch(hd, [12000, 400], [new, 2], 2, 1, hd).round_to(DT[dtype])
    check(b, DT[dtype], run_tree(b, DT[dtype]))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [4, 40])
def test_stretches_of_masked_pages(hd, new):
    """A page outside the pool in every sequence, so that whole stretches of pages take the masked way, more of them than are looked
    through at a time; the pool's other pages, and rows behind the ends, hold what is not finite."""
    b = TreeBatch(hd + new, [3000 - 7 * i for i in range(24)], [new] * 24, 8, 2, hd).round_to(torch.bfloat16)
    for s in range(24):
        b.table[s, 5 + s] = -1 if s % 2 else b.n_pages + s
    used = set(b.table[(b.table >= 0) & (b.table < b.n_pages)].tolist())
    for p in range(b.n_pages):
        if p not in used:
            b.k[p], b.v[p] = np.nan, np.inf
    for s in range(24):
        last = int(b.length[s])
        if last % PAGE:
            page, row = b.place(s, last)
            b.k[page, :, row:], b.v[page, :, row:] = np.inf, np.nan
    check(b, torch.bfloat16, run_tree(b, torch.bfloat16))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_sequences_without_drafted_tokens(dtype):
    """A padded batch: sequences without rows in front, between and behind change nothing, and a batch of nothing else writes nothing."""
    from stratum_b200 import kernels as K
    dev = lambda a, dt=None: torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=dt)      # noqa: E731
    b = TreeBatch(12, [700, 90], [9, 20], 8, 2, 64).round_to(DT[dtype])
    held = (dev(b.q, DT[dtype]), dev(b.k, DT[dtype]), dev(b.v, DT[dtype]), dev(np.array(b.pos, np.int32)), dev(b.mask()))

    def call(start, length, table):
        out = torch.full((29, 512), 7.0, dtype=DT[dtype], device="cuda")
        K.attention_tree(*held, dev(np.array(start, np.int32)), dev(np.array(length, np.int32)), dev(np.array(table, np.int32)), out, 8, 2, 64,
                         PAGE, 0, b.scale, 20)
        return out

    t, no = b.table.tolist(), [-1] * b.table.shape[1]
    out = call([0, 0, 0, 9, 9, 29, 29, 29], [0, 500, b.length[0], 0, b.length[1], 64, 0], [no, t[0], t[0], no, t[1], no, no])
    check(b, DT[dtype], out)
    assert (call([0, 0, 0, 0], [0, 700, 5], [no, t[0], t[1]]) == 7.0).all()
    assert (call([29, 29], [64], [t[0]]) == 7.0).all()
    K.check_status()
