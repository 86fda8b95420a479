"""Keys and values of drafted tokens: rotated by their positions, stored at places of their own."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,hd", [(5, 48), (1, 64), (90, 64), (90, 128)])
def test_places_apart_from_positions(dtype, interleaved, T, hd):
    """The same values as tokens that are each a sequence of their own store at their positions, at the places asked for; every other
    row stays as it was."""
    from stratum_b200 import kernels as K
    rng = np.random.default_rng(T + hd)
    n_q, n_kv = 4, 2
    up = lambda x, t=torch.int32: torch.as_tensor(np.asarray(x)).to(device="cuda", dtype=t)        # noqa: E731
    qkv = up(rng.standard_normal((T, (n_q + 2 * n_kv) * hd)), dtype)
    pos = rng.integers(0, 200, T)                             # siblings share positions
    first = int(rng.integers(0, 100))
    rows = first + rng.permutation(T)
    inv = up(10000.0 ** (-np.arange(0, hd, 2) / hd), torch.float32)
    table = rng.permutation(4)[None]
    kc, vc = (torch.full((4, n_kv, 64, hd), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    q1 = qkv.clone()
    K.rope_store(q1, up(pos), up(np.zeros(T)), up(table), inv, interleaved, 1.25, kc, vc, n_q, n_kv, hd, 64, True, up(rows))
    alone = rng.permutation(4 * T).reshape(T, 4)
    ka, va = (torch.zeros(4 * T, n_kv, 64, hd, dtype=dtype, device="cuda") for _ in range(2))
    q2 = qkv.clone()
    K.rope_store(q2, up(pos), up(np.arange(T)), up(alone), inv, interleaved, 1.25, ka, va, n_q, n_kv, hd, 64, True)
    assert torch.equal(q1, q2) and not torch.equal(q1, qkv)
    for got, ref in ((kc, ka), (vc, va)):
        for t in range(T):
            assert torch.equal(got[table[0, rows[t] // 64], :, rows[t] % 64], ref[alone[t, pos[t] // 64], :, pos[t] % 64]), t
        got = got.clone()
        for r in rows:
            got[table[0, r // 64], :, r % 64] = 7.0
        assert bool((got == 7.0).all())


def test_refusals():
    from stratum_b200 import kernels as K
    qkv = torch.zeros(3, 8 * 64, device="cuda")
    z = torch.zeros(3, dtype=torch.int32, device="cuda")
    cache = torch.zeros(1, 2, 64, 64, device="cuda")
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    for wrong in (z[:2], z.long(), z.cpu()):
        with pytest.raises(K.KernelError):
            K.rope_store(qkv, z, z, table, None, False, 1.0, cache, cache.clone(), 4, 2, 64, 64, True, wrong)
