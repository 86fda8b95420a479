"""Attention of drafted tokens over long caches against 64 bits, with inputs whose every page (and key) shows in the outputs; that the
bounds see a lost one is tested by test_draft_long_bounds.py."""
import numpy as np
import pytest
import torch

from draft_helpers import run_tree
from draft_long_helpers import CASES, AimedBatch, FlatBatch, Reference, make

pytestmark = pytest.mark.gpu
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd", [64, 128, 80])
@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("cls", [FlatBatch, AimedBatch])
def test_long_caches(cls, case, hd, dtype):
    from stratum_b200 import kernels as K
    b = make(cls, case, hd)
    ref = Reference(b)
    out = run_tree(b, DT[dtype])
    K.check_status()
    got = out.float().cpu().numpy().astype(np.float64).reshape(ref.out.shape)
    off, most = np.abs(got - ref.out), b.bound(DT[dtype], ref)
    assert np.isfinite(got).all()
    worst = int(np.argmax(off / np.maximum(most, 1e-30)))
    assert (off <= most).all(), (off.flat[worst], most.flat[worst], np.unravel_index(worst, off.shape), int((off > most).sum()))


@pytest.mark.parametrize("window", [700, 2500])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_windows_over_long_caches(dtype, window):
    from stratum_b200 import kernels as K
    b = FlatBatch(window, [5000, 3000, 600], [9, 40, 3], 8, 2, 64, window=window)
    ref = Reference(b)
    got = run_tree(b, DT[dtype]).float().cpu().numpy().astype(np.float64).reshape(ref.out.shape)
    K.check_status()
    assert (np.abs(got - ref.out) <= b.bound(DT[dtype], ref)).all()
