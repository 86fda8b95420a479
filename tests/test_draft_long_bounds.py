"""The bounds of the long-cache tests see what they are there to see: outputs without a page, without a key, of zeros (no GPU)."""
import numpy as np
import pytest
import torch

from draft_helpers import PAGE
from draft_long_helpers import AimedBatch, FlatBatch, Reference, make

DTYPES = [torch.bfloat16, torch.float32]
SMALL = ["one of 3,000, few rows", "one of 12,000, few rows", "ragged"]


def rounded(ref, dtype):
    """The reference as a kernel without any error of its own would write it."""
    return torch.from_numpy(ref.out).to(dtype).double().numpy()


def passes(b, ref, out, dtype):
    return np.abs(out - ref.out) <= b.bound(dtype, ref)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cls", [FlatBatch, AimedBatch])
def test_the_answer_passes_and_zeros_do_not(cls, dtype):
    for case in SMALL:
        b = make(cls, case, 64)
        ref = Reference(b)
        out = rounded(ref, dtype)
        assert passes(b, ref, out, dtype).all()
        assert passes(b, ref, np.zeros_like(out), dtype).mean() < 0.05 and passes(b, ref, -out, dtype).mean() < 0.05


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", SMALL)
def test_a_lost_page_shows(case, dtype):
    """Flat batches: any page, in every row that sees it.  Aimed ones: any page that a row looks at, in that row."""
    b = make(FlatBatch, case, 64)
    ref = Reference(b)
    for s, old in enumerate(b.old):
        for at in range(0, -(-old // PAGE), 1 + old // 640):
            lost = passes(b, ref, rounded(Reference(b, without_pages=[(s, at)]), dtype), dtype)
            rows = slice(int(b.start[s]), int(b.start[s + 1]))
            assert not lost[rows].all((1, 2)).any(), (s, at)
    b = make(AimedBatch, case, 64)
    ref = Reference(b)
    for s, at in sorted(b.aims)[::11]:
        lost = passes(b, ref, rounded(Reference(b, without_pages=[(s, at)]), dtype), dtype)
        assert not lost.all(), (s, at)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_lost_key_shows(dtype):
    for case in SMALL:
        b = make(FlatBatch, case, 128)
        ref = Reference(b)
        for s, old in enumerate(b.old):
            for at in range(0, old, max(1, old // 2)):
                lost = passes(b, ref, rounded(Reference(b, without_keys=[(s, at)]), dtype), dtype)
                assert not lost.all(), (s, at)


def test_a_piece_added_up_twice_or_at_another_scale_shows():
    """What a merge may do wrong: half of a long cache's pages with twice their weight."""
    for cls in (FlatBatch, AimedBatch):
        b = make(cls, "one of 12,000, few rows", 64)
        ref = Reference(b)
        half = Reference(b, without_pages=[(0, i) for i in range(94)])
        rest = Reference(b, without_pages=[(0, i) for i in range(94, 400)])
        twice = (ref.out * 2 + rest.out) / 3 if cls is FlatBatch else (half.out + rest.out) / 2
        if cls is FlatBatch:
            assert not passes(b, ref, twice, torch.bfloat16)[:3].all((1, 2)).any()
        else:                                        # (a row looks at a page of either half, more or less alike)
            assert not passes(b, ref, half.out, torch.bfloat16)[:3].all((1, 2)).any()
            assert not passes(b, ref, rest.out, torch.bfloat16)[:3].all((1, 2)).any()
