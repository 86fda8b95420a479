"""Looked-up drafts that hold all of a row's weight and are refused all the same: the next token is still one that the target
can give."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

A = np.float32(0.3)
B = np.nextafter(np.float32(1.0) - A, np.float32(0.0))     # the two add up to one less 2^-24
U = np.float32(1.0) - np.float32(2.0 ** -24)               # the largest number that is drawn


def plain(row, children, u, u0):
    """(kept, next id) at one node, in 64 bits: a rejection that would leave nothing leaves the row as it was."""
    d, mass = row.astype(np.float64), 1.0
    for x in children:
        if np.float64(u) * mass < d[x]:
            return 1, None
        less = d.copy()
        less[x] = 0.0
        if less.sum() > 0:
            mass, d = max(mass - d[x], 0.0), less
    cum = np.cumsum(d)
    if not cum[-1] > 0:
        return 0, 0
    return 0, int(np.nonzero((cum > np.float64(u0) * cum[-1]) & (d > 0))[0][0])


def run(target, tokens, parents, start, u):
    from stratum_b200 import kernels as K
    up = lambda a, t: torch.tensor(np.asarray(a), dtype=t, device="cuda")               # noqa: E731
    n, B_ = len(tokens), len(start) - 1
    path = torch.empty(n, dtype=torch.int32, device="cuda")
    kept, picked = (torch.empty(B_, dtype=torch.int32, device="cuda") for _ in range(2))
    K.verify_drafts(target if torch.is_tensor(target) else up(target, torch.float32), None, up(tokens, torch.int32), up(parents, torch.int32),
                    up(start, torch.int32), up(u, torch.float32), path, kept, picked)
    return path.tolist(), kept.tolist(), picked.tolist()


@pytest.mark.parametrize("V", [40, 4099, 128256])
@pytest.mark.parametrize("children", [(7, 21), (21, 7), (7, 21, 3), (3, 7, 7, 21), (21, 3, 7, 21, 5)])
def test_the_next_token_has_weight(V, children):
    row = np.zeros(V, np.float32)
    row[7], row[21] = A, B
    n = 1 + len(children)
    for u0 in (np.float32(0.0), np.float32(0.5), U):
        want = plain(row, children, U, u0)
        assert want[0] == 0 and row[want[1]] > 0           # (the case is what it is meant to be)
        path, kept, picked = run(np.tile(row, (n, 1)), [1, *children], [-1] + [0] * len(children), [0, n], [u0] + [U] * len(children))
        assert (path, kept, picked) == ([0] + [-1] * (n - 1), [0], [want[1]])


def test_below_a_kept_draft_and_beside_other_sequences():
    """The loss belongs to the node it happened at: a kept draft's row begins anew, and a row without any weight still gives 0."""
    V = 300
    row = np.zeros(V, np.float32)
    row[7], row[21] = A, B
    zero, other = np.zeros(V, np.float32), np.zeros(V, np.float32)
    other[33] = 1.0
    # 0: both children of the node behind the kept one are refused; 1 and 2: a child is refused, the next one kept, and behind
    # that one lies a whole row or one without weight; 3: no weight at all
    target = np.stack([other, row, row, row] + [row, row, row, other] + [row, zero, zero] + [zero, zero, zero])
    tokens = [1, 33, 7, 21] + [1, 7, 21, 33] + [1, 7, 21] + [1, 7, 21]
    parents = [-1, 0, 1, 1] + [-1, 0, 0, 2] + [-1, 0, 0] + [-1, 0, 0]
    u = [0.5, 0.0, U, U] + [0.5, U, 0.0, 0.0] + [0.5, U, 0.0] + [0.5, U, U]
    path, kept, picked = run(target, tokens, parents, [0, 4, 8, 11, 14], u)
    assert kept == [1, 1, 1, 0] and picked == [21, 21, 0, 0]
    assert path == [0, 1, -1, -1, 0, 2, -1, -1, 0, 2, -1, 0, -1, -1]
