"""Attention of drafted tokens at finite scores of any size.  A score is one product of two bfloat16 numbers here (or two, of whole
numbers below 2^24): float32 holds it exactly, so that the formula's own answer is what is asked for."""
import numpy as np
import pytest
import torch

from draft_helpers import TreeBatch, run_tree

pytestmark = pytest.mark.gpu
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def outputs(b, dtype):
    from stratum_b200 import kernels as K
    out = run_tree(b, dtype).float().cpu().numpy().astype(np.float64)
    K.check_status()
    return out


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [5, 40])
@pytest.mark.parametrize("size", [1e4, 3e8, 3e9, 2e10, 1e15, 1e30, 3e36])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_score_takes_all(dtype, hd, new, size, sign):
    """Keys of 128 to 255 in one dimension: scores lie at least `size` / 255 / sqrt(hd) apart (13 halvings and more), so a row's
    output is the mean of the values of its largest ones.  bfloat16: the equal weights are rounded to 8 bits, and may be rounded
    differently, as an exponential is off by 2^-13 at most and a border may lie between two of them: (2^-8 + 2^-13) of each, which
    moves a mean by no more than that of p |v - mean|, and that is no more than p |v| + |mean|.  Half a step of the output; float32
    sums; 2^-8 of what the next ones weigh."""
    b = TreeBatch(hd + new, [3000, 70, 0], [new, 3, 2], 8, 2, hd)
    rng = np.random.default_rng(new)
    one = rng.integers(128, 256, b.k.shape[:3])
    b.k[:] = 0.0
    b.k[..., 0] = one
    b.q[:] = 0.0
    b.q.reshape(-1, 8, hd)[:, :, 0] = sign * size / 255 * rng.uniform(0.7, 1.4, (b.q.shape[0], 8))
    b.round_to(torch.bfloat16)
    ref, _, mean, _ = b.reference()
    got = outputs(b, DT[dtype])
    assert np.isfinite(got).all()
    # (the smallest gap of scores of this case, in halvings of a weight, and what 3,000 of the next ones add up to)
    gap = 0.7 * size / 255 * hd ** -0.5 * 1.44 * 0.99
    rest = min(1.0, 3000 * 2.0 ** -min(gap, 200.0))
    assert rest < 2.0 ** -3 or size < 1e5
    half, weight = (2.0 ** -8, 2.0 ** -8 + 2.0 ** -13) if dtype == "bfloat16" else (0.0, 0.0)
    most = half * np.abs(ref) + (weight + 2 * (2.0 ** -8 * rest + 64 * 2.0 ** -24)) * (mean + np.abs(ref)) + 1e-30
    assert (np.abs(got - ref) <= most).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [5, 40])
@pytest.mark.parametrize("step", [10, 50, 64, 90])
def test_a_maximum_that_moves_among_large_scores(hd, new, step):
    """Scores of some 10^7 whose later half is larger by a few units: small weights of large values, at a size where a score times
    log2 e loses the last bits of what is in front of the point.  Each weight is rounded to bfloat16 (2^-8 of it) and so is the
    output; all is positive, so the relative errors add up."""
    b = TreeBatch(new, [1024], [new], 8, 2, hd)
    b.k[:], b.q[:] = 0.0, 0.0
    q = b.q.reshape(-1, 8, hd)
    q[:, :, 0], q[:, :, 1] = 2832.0, 1.0
    b.k[..., 0] = 4096.0
    b.v = np.abs(b.v).astype(np.float32) + 0.5
    for position in range(1024 + new):
        page, row = b.place(0, position)
        b.k[page, :, row, 1] = 0.0 if position < 512 else step
        b.v[page, :, row] *= 128.0 if position < 512 else 2.0 ** -6
    b.round_to(torch.bfloat16)
    ref = b.reference()[0]
    got = outputs(b, torch.bfloat16)
    assert (np.abs(got - ref) <= ref * (3 * 2.0 ** -8 * 1.01 + 64 * 2.0 ** -23)).all()
