"""Copied pages and kept rows, byte for byte."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def storage(shape, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randint(0, 255, tuple(shape[:-1]) + (shape[-1] * torch.empty(0, dtype=dtype).element_size(),), generator=g,
                      device="cuda", dtype=torch.uint8)
    return x.view(dtype)


def same(a, b):
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.bfloat16, 3), (torch.float32, 64), (torch.int8, 5), (torch.float32, 1)])
@pytest.mark.parametrize("layers,pages,heads,pairs", [(1, 4, 1, 1), (3, 40, 2, 17), (2, 2100, 1, 1000)])
def test_copy_pages(dtype, hd, layers, pages, heads, pairs):
    from stratum_b200 import kernels as K
    rng = np.random.default_rng(pairs)
    k, v = storage((layers, pages, heads, 64, hd), dtype, 1), storage((layers, pages, heads + 1, 64, hd), dtype, 2)
    some = rng.permutation(pages)[:2 * pairs].tolist()
    src, dst = some[:pairs], some[pairs:]
    want = [t.clone() for t in (k, v)]
    for w in want:
        w.view(torch.uint8)[:, dst] = w.view(torch.uint8)[:, src]
    K.copy_pages(k, v, src, dst)
    assert same(k, want[0]) and same(v, want[1])
    K.copy_pages(k, None, dst[:1], src[:1])          # keys alone; one source for several copies
    assert same(k[:, src[0]], k[:, dst[0]]) and same(v, want[1])
    if pairs > 2:
        K.copy_pages(k, v, [src[0]] * 2, dst[1:3])
        assert same(k[:, dst[1]], k[:, src[0]]) and same(v[:, dst[2]], v[:, src[0]])
    K.copy_pages(k, v, [], [])


def test_copy_pages_of_state_rows():
    """[layers, slots, anything]: a fixed-size state's rows are pages too, of any size."""
    from stratum_b200 import kernels as K
    state = torch.randn(3, 9, 7, 5, device="cuda")
    last = torch.randint(0, 1000, (2, 9, 1), dtype=torch.int32, device="cuda")
    want, want_last = state.clone(), last.clone()
    want[:, [2, 8]], want_last[:, 4] = want[:, [1, 1]], want_last[:, 0]
    K.copy_pages(state, None, [1, 1], [2, 8])
    K.copy_pages(last, None, [0], [4])
    assert torch.equal(state, want) and torch.equal(last, want_last)


def test_copy_pages_refusals():
    from stratum_b200 import kernels as K
    k = torch.zeros(2, 8, 1, 64, 4, device="cuda")
    before = k.clone()
    for src, dst in (([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [8]), ([-1], [2]), ([0, 1], [2]), ([3], [3])):
        with pytest.raises(K.KernelError):
            K.copy_pages(k, None, src, dst)
    with pytest.raises(K.KernelError):
        K.copy_pages(k, torch.zeros(2, 7, 1, 64, 4, device="cuda"), [0], [1])
    with pytest.raises(K.KernelError):
        K.copy_pages(k[:, :, :, :32], None, [0], [1])
    assert torch.equal(k, before)


def plain_keep(t, table, start, length, path, kept):
    t = t.view(torch.uint8).cpu().numpy().copy()
    for s, n in enumerate(kept):
        rows = start[s + 1] - start[s]
        base, before = length[s] - rows, 0
        for j in range(1, min(n, rows - 1) + 1):
            node = path[start[s] + j]
            if node <= before or node >= rows:
                break
            before = node
            a, b = base + node, base + j
            pages = [table[s][p // 64] if p // 64 < len(table[s]) else -1 for p in (a, b)]
            if all(0 <= p < t.shape[1] for p in pages):
                t[:, pages[1], :, b % 64] = t[:, pages[0], :, a % 64]
    return t


@pytest.mark.parametrize("dtype,hd,hv", [(torch.bfloat16, 128, 128), (torch.bfloat16, 64, 40), (torch.float32, 80, 80), (torch.float32, 300, 6),
                                         (torch.bfloat16, 3, 3)])
@pytest.mark.parametrize("layers,heads", [(1, 1), (5, 3)])
def test_keep_rows(dtype, hd, hv, layers, heads):
    from stratum_b200 import kernels as K
    rng = np.random.default_rng(hd + layers)
    new = [1, 2, 9, 40, 70, 200, 5]
    old = [0, 63, 60, 130, 64, 1, 100]
    start = np.concatenate([[0], np.cumsum(new)]).astype(int).tolist()
    length = [a + b for a, b in zip(old, new)]
    held = [-(-n // 64) for n in length]
    order = rng.permutation(sum(held) + 2).tolist()
    table, at = [], 0
    for n in held:
        table.append(order[at:at + n] + [-1] * (max(held) - n))
        at += n
    path, kept = [], []
    for n in new:
        m = int(rng.integers(0, n))
        some = sorted(rng.permutation(np.arange(1, n))[:m].tolist())
        path += [0] + some + [-1] * (n - 1 - m)
        kept.append(m)
    kept[1], path[start[1] + 1] = 1, 1               # a row that stays where it is
    kept[6] = 0
    k = storage((layers, len(order), heads, 64, hd), dtype, 3)
    v = storage((layers, len(order), heads + 1, 64, hv), dtype, 4)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")      # noqa: E731
    want = [plain_keep(t, table, start, length, path, kept) for t in (k, v)]
    K.keep_rows(k, v, i32(table), i32(start), i32(length), i32(path), i32(kept))
    for t, w in zip((k, v), want):
        assert np.array_equal(t.view(torch.uint8).cpu().numpy(), w)


def test_keep_rows_of_paths_that_are_none():
    """A path that falls, leaves the tree or is longer than it, pages outside the pool: the rows up to there move, in bounds."""
    from stratum_b200 import kernels as K
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")      # noqa: E731
    k = storage((2, 6, 2, 64, 64), torch.bfloat16, 5)
    table, start, length = [[0, 1], [2, 3], [4, 99], [5, -1]], [0, 6, 12, 18, 24], [70, 100, 66, 66]
    path = [0, 2, 4, 3, 5, -1] + [0, 2, 9, 3, 4, 5] + [0, 2, 3, 4, 5, -1] + [0, 3, 4, 5, -1, -1]
    kept = [4, 5, 4, 1000]
    want = plain_keep(k, table, start, length, path, kept)
    K.keep_rows(k, None, i32(table), i32(start), i32(length), i32(path), i32(kept))
    assert np.array_equal(k.view(torch.uint8).cpu().numpy(), want)
