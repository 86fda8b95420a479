"""What the kernels of drafted decoding refuse before anything runs (no GPU: a tensor on the host is the first refusal)."""
import pytest
import torch

from stratum_b200 import kernels as K


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_host_tensors_are_refused():
    q, k = torch.zeros(3, 128), torch.zeros(2, 2, 64, 64)
    calls = [
        lambda: K.attention_tree(q, k, k, i32(3), torch.zeros(3, 1, dtype=torch.int64), i32(2), i32(1), i32(1, 2), q.clone(), 2, 2, 64, 64,
                                 0, 0.125, 3),
        lambda: K.token_probs(torch.zeros(2, 5), torch.ones(2), torch.zeros(2, 5)),
        lambda: K.verify_drafts(torch.zeros(2, 5), None, i32(2), i32(2), i32(2), torch.zeros(2), i32(2), i32(1), i32(1)),
        lambda: K.keep_rows(k[None], k[None], i32(1, 2), i32(2), i32(1), i32(3), i32(1)),
        lambda: K.copy_pages(k[None], None, [0], [1]),
    ]
    for call in calls:
        with pytest.raises(K.KernelError, match="CUDA device"):
            call()


def test_half_precision_is_refused():
    with pytest.raises(K.KernelError, match="float32 or bfloat16"):
        K.attention_tree(torch.zeros(3, 128, dtype=torch.float16), None, None, None, None, None, None, None, None, 2, 2, 64, 64, 0, 1.0, 3)
