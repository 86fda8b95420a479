"""Forked sequences, pages handed back, and what a step of drafted tokens refuses and describes (no GPU)."""
import random

import numpy as np
import pytest
import torch

from stratum_b200.cache import PAGE_TOKENS, CacheFull, CacheMisuse, KVSpec, PagePool, SequenceCache, StateSpec, pages_for
from stratum_b200.engine import DraftEntry
from stratum_b200.engine.step import tree_depths_and_masks


def _cache(max_tokens=64 * 8, max_seqs=4, specs=None):
    return SequenceCache(specs or [KVSpec(2, 16), KVSpec(2, 16)], max_tokens, max_seqs, torch.float32, "cpu", allocate=False)


def test_a_shared_page_is_free_when_its_last_holder_gives_it_back():
    pool = PagePool(3)
    a = pool.take(2)
    pool.share([a[0]])
    pool.give(a)
    assert pool.free_pages == 2 and pool.holders(a[0]) == 1
    pool.check()
    with pytest.raises(CacheMisuse):
        pool.share([a[1]])                     # free
    pool.give([a[0]])
    with pytest.raises(CacheMisuse):
        pool.give([a[0]])
    assert pool.free_pages == 3
    pool.check()


@pytest.mark.parametrize("length", [0, 1, 63, 64, 65, 128, 200])
def test_fork_shares_full_pages_and_copies_the_last(length):
    c = _cache()
    a = c.acquire()
    c.reserve([a], [length])
    c.advance([a], [length])
    before, epoch = c.groups[0].pool.free_pages, c.epoch
    b, d = c.fork(a, 2)
    assert c.length(b) == c.length(d) == length and c.epoch > epoch
    ta, tb, td = c.page_table_rows([a, b, d], 0)
    full = length // PAGE_TOKENS
    assert ta[:full] == tb[:full] == td[:full] and len(ta) == len(tb) == len(td) == pages_for(length)
    if length % PAGE_TOKENS:
        assert len({ta[full], tb[full], td[full]}) == 3
    assert before - c.groups[0].pool.free_pages == 2 * (length % PAGE_TOKENS > 0)
    c.check()
    for order in (a, d, b):                    # whoever goes first, the others keep their pages
        c.release(order)
        c.check()
    assert c.tokens_held() == 0


def test_fork_is_all_or_nothing():
    c = _cache(max_tokens=64 * 3, max_seqs=3)
    a = c.acquire()
    c.reserve([a], [70])
    c.advance([a], [70])
    with pytest.raises(CacheFull):
        c.fork(a, 2)                           # two more pages, one is free
    with pytest.raises(CacheFull):
        c.fork(a, 3)                           # three more slots
    with pytest.raises(CacheMisuse):
        c.fork(2)
    with pytest.raises(CacheMisuse):
        c.fork(a, -1)
    assert c.fork(a, 0) == [] and c.slots.free_slots == 2 and c.groups[0].pool.free_pages == 1
    c.check()


def test_fork_of_windowed_groups_keeps_what_was_dropped_dropped():
    c = _cache(specs=[KVSpec(2, 16), KVSpec(2, 16, window=100), StateSpec((4,))])
    a = c.acquire()
    c.reserve([a], [300])
    c.advance([a], [300])
    (b,) = c.fork(a)
    ta, tb = c.page_table_rows([a, b], 1)
    assert [p >= 0 for p in tb] == [False, False, False, True, True] and ta[3] == tb[3] and ta[4] != tb[4]
    c.check()
    c.reserve([b], [100])
    c.advance([b], [100])                      # the fork goes on alone and hands back its share
    assert c.groups[1].pool.holders(ta[3]) == 1
    c.check()
    c.release_all()
    c.check()
    assert c.tokens_held() == 0


def test_trim_hands_back_what_lies_beyond_a_sequence():
    c = _cache()
    a = c.acquire()
    c.reserve([a], [60])
    c.advance([a], [60])
    c.reserve([a], [200])                      # drafts
    assert c.tokens_held() == 5 * PAGE_TOKENS
    epoch = c.epoch
    c.advance([a], [5])
    c.trim([a])
    assert c.tokens_held() == 2 * PAGE_TOKENS and c.epoch > epoch
    epoch = c.epoch
    c.trim([a])
    assert c.epoch == epoch
    c.check()
    with pytest.raises(CacheMisuse):
        c.trim([3])


def test_random_traffic_with_forks_keeps_invariants():
    rng = random.Random(1)
    c = _cache(max_tokens=64 * 30, max_seqs=7, specs=[KVSpec(2, 16), KVSpec(1, 16, window=130)])
    live = {}
    for _ in range(3000):
        r = rng.random()
        try:
            if r < 0.15 and len(live) < 7:
                live[c.acquire()] = 0
            elif r < 0.3 and live:
                s = rng.choice(list(live))
                for b in c.fork(s, rng.randint(1, 3)):
                    live[b] = live[s]
            elif r < 0.45 and live:
                s = rng.choice(list(live))
                c.release(s)
                del live[s]
            elif live:
                s = rng.choice(list(live))
                n = rng.choice([1, 7, 64, 100])
                c.reserve([s], [n])
                keep = rng.randint(0, n)
                c.advance([s], [keep])
                c.trim([s])
                live[s] += keep
        except CacheFull:
            pass
        c.check()
        for s, n in live.items():
            assert c.length(s) == n and len(c.page_table_rows([s], 0)[0]) == pages_for(n)
    for s in list(live):
        c.release(s)
    c.check()
    assert c.tokens_held() == 0


def test_depths_and_masks():
    tree = [-1, 0, 0, 1, 3, 2]
    depth, mask = tree_depths_and_masks(tree, 0, 1)
    assert depth == [0, 1, 1, 2, 3, 2]
    assert mask[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b11011, 0b100101]
    _, mask = tree_depths_and_masks(tree, 2, 1)            # a token and the one above it
    assert mask[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1010, 0b11000, 0b100100]
    chain = DraftEntry(0, [5] * 130).tree()
    depth, mask = tree_depths_and_masks(chain, 0, 3)
    assert chain[:3] == [-1, 0, 1] and depth[129] == 129
    words = mask.view(np.uint64)
    assert words[129].tolist() == [2 ** 64 - 1, 2 ** 64 - 1, 3] and words[63].tolist() == [2 ** 64 - 1, 0, 0]


def test_which_models_take_drafts():
    """Attention over keys and values alone does; layers with a state, or with attention of other shapes, do not."""
    import dabodra_helpers
    import vitinex_helpers
    from helpers import TINY
    from stratum_b200.config import find_architecture
    from stratum_b200.engine.model import Model

    def model(cfg):
        arch = find_architecture(cfg)
        return Model(arch.describe_model(arch.config_class.from_dict(cfg)), None)
    assert all(model(TINY[name]).takes_drafts() for name in TINY)
    for helpers in (dabodra_helpers, vitinex_helpers):
        assert not any(model(cfg).takes_drafts() for cfg in helpers.CONFIGS.values())
