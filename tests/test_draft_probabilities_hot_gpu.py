"""The target's probabilities at temperatures without a measure: infinite ones, and ones as large as the logits' own range."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")
MOST = float(np.finfo(np.float32).max)


def plain(x, t):
    """softmax(x / t) in 64 bits; infinite logits share the row."""
    x, t = x.astype(np.float64), np.float64(t)
    x = np.where(np.isnan(x), -INF, x)
    m = x.max()
    if m == -INF:
        return np.zeros_like(x)
    if m == INF:
        e = (x == INF).astype(np.float64)
    else:
        e = np.where(x == -INF, 0.0, np.exp((np.where(x == -INF, m, x) - m) / t))
    return e / e.sum()


@pytest.mark.parametrize("vocab", [5, 1003, 32000, 128256, 262144, 262145 * 2])
@pytest.mark.parametrize("temperature", [INF, MOST, 1e38, 3e36, 1e31, 1e29, 40.0])
def test_hot_rows(vocab, temperature):
    """Relative error: the exponent's (a difference, two products, log2 e / T: 2^-24 of the exponent each, the last 2^-22 where it is
    below the smallest normal number; times ln 2), exp2f's two units, the sum's 68 levels of additions and two products."""
    from stratum_b200 import kernels as K
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((9, vocab)) * 3).astype(np.float32)
    x[1] = np.where(np.arange(vocab) % 2, MOST, -MOST)
    x[2] = (rng.uniform(-1, 1, vocab) * MOST).astype(np.float32)
    x[3, ::2], x[4, vocab // 2], x[5, 1], x[6] = -INF, INF, np.nan, -INF
    x[7, :2] = MOST, -MOST
    x[8, 0], x[8, 1], x[8, 2:4] = MOST, -INF, INF
    t = np.full(9, temperature, np.float32)
    out = torch.full((9, vocab), 7.0, device="cuda")
    K.token_probs(torch.from_numpy(x).cuda(), torch.from_numpy(t).cuda(), out)
    K.check_status()
    got = out.cpu().numpy().astype(np.float64)
    for r in range(9):
        want = plain(x[r], t[r])
        exponent = np.where(want > 0, np.log2(max(want.max(), 1e-300)) - np.log2(np.maximum(want, 1e-300)), 0.0)
        rel = 0.7 * np.minimum(exponent, 200.0) * (3 * 2.0 ** -24 + 2.0 ** -22) + (2 + 68 + 2) * 2.0 ** -24
        assert np.isfinite(got[r]).all(), r
        assert (np.abs(got[r] - want) <= rel * want + 2.0 ** -124).all(), r
