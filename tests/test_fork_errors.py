"""A fork whose copies cannot be launched leaves the cache as it was (no GPU: the copy is replaced)."""
import pytest
import torch

from stratum_b200.cache import KVSpec, SequenceCache, StateSpec
from stratum_b200.cache import store


@pytest.mark.parametrize("fails_at", [0, 1, 2])
@pytest.mark.parametrize("length", [64, 70])
def test_a_copy_that_fails_leaves_no_fork(monkeypatch, fails_at, length):
    """Groups of keys, of windowed keys and of states, in turn the one whose copy raises (full pages alone: only the states')."""
    c = SequenceCache([KVSpec(1, 4), KVSpec(1, 4, window=100), StateSpec((3,))], 64 * 12, 5, torch.float32, "cpu")
    a = c.acquire()
    c.reserve([a], [length])
    c.advance([a], [length])
    tables = [c.page_table_rows([a], g)[0] for g in (0, 1)]
    calls = []

    def copy(k, v, src, dst):
        calls.append(len(src))
        if len(calls) - 1 == fails_at:
            raise RuntimeError("no launch")

    monkeypatch.setattr(store.K, "copy_pages", copy)
    copies = 3 if length % 64 else 1
    epoch = c.epoch
    if fails_at < copies:
        with pytest.raises(RuntimeError, match="no launch"):
            c.fork(a, 3)
        assert c.epoch > epoch                     # tables copied meanwhile are stale
        assert c.slots.live() == [a] and c.length(a) == length
        held = len(tables[0])
        assert [g.pool.free_pages for g in c.groups[:2]] == [12 - held, 12 - held]
        assert all(g.pool.holders(p) == 1 for g, t in zip(c.groups, tables) for p in t)
        c.check()
        calls.append(0)                            # the next ones succeed
        calls.extend([0] * 3)
    forks = c.fork(a, 3)
    assert len(forks) == 3 and c.slots.free_slots == 1
    c.check()
    c.release_all()
    c.check()
    assert c.tokens_held() == 0
