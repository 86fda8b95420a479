"""What the kernels of drafted decoding refuse of tensors on the device, each call with one thing wrong: an error that says so, and
nothing written."""
import numpy as np
import pytest
import torch

from draft_helpers import TreeBatch, run_tree

pytestmark = pytest.mark.gpu


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def refused(call, args, changes, names, outputs):
    """call(**args) runs; with each of `changes` (name, value) it is refused and `outputs` stay as they are."""
    from stratum_b200 import kernels as K
    call(**args)
    before = {n: args[n].clone() for n in outputs}
    for name, value in changes:
        assert name in names, name
        with pytest.raises(K.KernelError):
            call(**{**args, name: value})
        for n in outputs:
            assert torch.equal(args[n], before[n]), (name, n)
    K.check_status()


def test_attention_tree():
    from stratum_b200 import kernels as K
    T, n_q, n_kv, hd, pages = 5, 8, 2, 64, 6
    f = lambda *s: torch.randn(*s, device="cuda", dtype=torch.bfloat16)                 # noqa: E731
    args = dict(q=f(T, n_q * hd), k_cache=f(pages, n_kv, 64, hd), v_cache=f(pages, n_kv, 64, hd), token_pos=i32(70, 71, 72, 3, 4),
                tree_mask=torch.tensor([[1], [3], [7], [1], [3]], device="cuda"), seq_start=i32(0, 3, 5), seq_len=i32(73, 5),
                block_table=i32(0, 3, 4, -1).view(2, 2), out=f(T, n_q * hd), n_q=n_q, n_kv=n_kv, head_dim=hd, page_tokens=64, window=0,
                scale=0.125, max_new=3)
    wide = f(T, 3 * n_q * hd)
    changes = [("q", args["q"].half()), ("q", args["q"].float()), ("q", args["q"][:4]), ("q", args["q"][:, :-1]), ("q", wide[:, ::3]),
               ("q", args["q"][:1].expand(T, -1)), ("q", args["q"].cpu()), ("q", args["out"]), ("out", args["q"]),
               ("out", args["out"].float()), ("out", args["out"][:, 64:]), ("out", args["out"][:1].expand(T, -1)),
               ("k_cache", args["k_cache"].float()), ("k_cache", args["k_cache"][:, :1]), ("k_cache", args["k_cache"].transpose(0, 1)),
               ("v_cache", args["v_cache"][:5]), ("v_cache", args["v_cache"].half()), ("v_cache", args["v_cache"].cpu()),
               ("token_pos", args["token_pos"].long()), ("token_pos", args["token_pos"][:4]),
               ("tree_mask", args["tree_mask"].int()), ("tree_mask", args["tree_mask"][:4]), ("tree_mask", args["tree_mask"][:, :0]),
               ("tree_mask", args["tree_mask"][:, 0]), ("seq_start", args["seq_start"][:2]), ("seq_start", args["seq_start"].long()),
               ("seq_len", args["seq_len"].long()), ("seq_len", args["seq_len"][:1]), ("block_table", args["block_table"].t()),
               ("block_table", args["block_table"].long()), ("block_table", args["block_table"][:1]),
               ("block_table", args["block_table"][:, :0]), ("n_q", 7), ("n_q", 0), ("n_q", 9), ("n_kv", 4), ("n_kv", 0), ("head_dim", 32),
               ("page_tokens", 32), ("window", -1), ("max_new", -1)]
    refused(K.attention_tree, args, changes, list(args), ["out"])


def test_attention_tree_limits():
    """Heads of more than 256, pages of another size, more sequences than a launch lists."""
    from stratum_b200 import kernels as K

    def call(B=1, hd=64, page=64):
        q = torch.zeros(B, hd, device="cuda")
        cache = torch.zeros(1, 1, page, hd, device="cuda")
        table = torch.zeros(B, 1, dtype=torch.int32, device="cuda")
        K.attention_tree(q, cache, cache.clone(), torch.zeros(B, dtype=torch.int32, device="cuda"),
                         torch.ones(B, 1, dtype=torch.int64, device="cuda"), torch.arange(B + 1, dtype=torch.int32, device="cuda"),
                         torch.ones(B, dtype=torch.int32, device="cuda"), table, q.clone(), 1, 1, hd, page, 0, 1.0, 1)
        K.check_status()

    call(4096)
    call(hd=256)
    for wrong in (dict(B=4097), dict(hd=257), dict(page=128)):
        with pytest.raises(K.KernelError):
            call(**wrong)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_tree_of_columns_and_of_one_row(dtype):
    """q and out may be columns of one matrix; the distance between rows means nothing where there is one."""
    from stratum_b200 import kernels as K
    for old, new in (([70, 9], [5, 2]), ([70], [1])):
        b = TreeBatch(3, old, new, 8, 2, 64).round_to(dtype)
        T, W = sum(new), 512
        want = run_tree(b, dtype)[:, :W].clone()
        up = lambda x, t: torch.as_tensor(x).to(device="cuda", dtype=t)                  # noqa: E731
        both = torch.zeros(T, 2 * W + 24, dtype=dtype, device="cuda")
        q, out = both[:, :W], both[:, W:2 * W]
        if T == 1:
            q = torch.as_strided(both, (1, W), (3, 1))
        q.copy_(up(b.q, dtype))
        K.attention_tree(q, up(b.k, dtype), up(b.v, dtype), up(np.array(b.pos), torch.int32), up(b.mask(), torch.int64),
                         up(b.start, torch.int32), up(b.length, torch.int32), up(b.table, torch.int32), out, 8, 2, 64, 64, 0, b.scale,
                         max(new))
        K.check_status()
        assert torch.equal(out, want)
        assert float(both[:, 2 * W:].abs().sum()) == 0.0


def test_token_probs():
    from stratum_b200 import kernels as K
    wide = torch.randn(6, 300, device="cuda")
    args = dict(logits=torch.randn(6, 100, device="cuda"), temperature=torch.ones(6, device="cuda"), out=torch.zeros(6, 100, device="cuda"))
    changes = [("logits", args["logits"].bfloat16()), ("logits", args["logits"][:5]), ("logits", args["logits"][:, :99]),
               ("logits", wide[:, ::3]), ("logits", args["logits"][:1].expand(6, -1)), ("logits", args["logits"].cpu()),
               ("logits", args["logits"][0]), ("out", args["out"].double()), ("out", args["out"][:, :99]), ("temperature", args["temperature"][:5]),
               ("temperature", args["temperature"].double()), ("temperature", torch.ones(6, 2, device="cuda")[:, 0])]
    refused(K.token_probs, args, changes, list(args), ["out"])
    for a, b in ((wide[:, :100], wide[:, 50:150]), (wide[:5, :100], wide[1:, :100]), (wide[:, 100:200], wide[:, 99:199])):
        with pytest.raises(K.KernelError):
            K.token_probs(a, torch.ones(a.shape[0], device="cuda"), b)
    # in place, and columns of one matrix
    want = torch.softmax(wide[:, :100].double(), 1)
    K.token_probs(wide[:, :100], args["temperature"], wide[:, 150:250])
    K.token_probs(wide[:, :100], args["temperature"], wide[:, :100])
    for got in (wide[:, :100], wide[:, 150:250]):
        assert float((got.double() - want).abs().max()) < 4 * 2.0 ** -22


def test_verify_drafts():
    from stratum_b200 import kernels as K
    p = torch.softmax(torch.randn(5, 40, device="cuda"), 1)
    z = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")                       # noqa: E731
    args = dict(target=p, draft=p.flip(1).contiguous(), tokens=i32(1, 2, 3, 4, 5), parents=i32(-1, 0, 1, -1, 0), seq_start=i32(0, 3, 5),
                uniform=torch.rand(5, device="cuda"), path=z(5), n_kept=z(2), next_ids=z(2))
    changes = [("target", p.double()), ("target", p[:4]), ("target", p[:, ::2]), ("target", p.cpu()), ("target", p[:, :0]),
               ("draft", p[:, :39]), ("draft", p[:4]), ("draft", p.half()), ("tokens", args["tokens"].long()), ("tokens", args["tokens"][:4]),
               ("parents", args["parents"][1:]), ("parents", args["parents"].long()), ("uniform", args["uniform"].double()),
               ("uniform", args["uniform"][:4]), ("seq_start", i32(0, 5)), ("seq_start", args["seq_start"].long()), ("path", z(4)),
               ("path", z(5).long()), ("n_kept", z(3)), ("n_kept", z(2).long()), ("next_ids", z(3)), ("next_ids", z(2).float())]
    refused(K.verify_drafts, args, changes, list(args), ["path", "n_kept", "next_ids"])
    for name, other in (("path", "tokens"), ("path", "parents"), ("next_ids", "n_kept")):        # what is written is also read, or written twice
        with pytest.raises(K.KernelError):
            K.verify_drafts(**{**args, name: args[other]})
    n = K.VERIFY_MAX_NODES + 1
    with pytest.raises(K.KernelError):
        K.verify_drafts(torch.zeros(n, 4, device="cuda"), None, z(n), z(n), i32(0, n), torch.zeros(n, device="cuda"), z(n), z(1), z(1))


def test_keep_rows():
    from stratum_b200 import kernels as K
    f = lambda *s: torch.randn(*s, device="cuda")                                        # noqa: E731
    args = dict(k=f(2, 3, 2, 64, 8), v=f(2, 3, 2, 64, 8), block_table=i32(0, 1, 2, -1).view(2, 2), seq_start=i32(0, 4, 6),
                seq_len=i32(70, 6), path=i32(0, 2, 3, -1, 0, 1), n_kept=i32(0, 0))
    both = f(2, 2, 3, 2, 64, 8)
    changes = [("k", args["k"][0]), ("k", args["k"].transpose(1, 2)), ("k", args["k"][:, :0]), ("k", args["k"].cpu()), ("v", args["v"][:1]),
               ("v", args["v"][:, :2]), ("v", args["v"][:, :, :, :32].contiguous()), ("v", args["k"]), ("v", args["k"].view(torch.int32)),
               ("block_table", args["block_table"].t()), ("block_table", args["block_table"][:1]), ("block_table", args["block_table"].long()),
               ("block_table", args["block_table"][:, :0]), ("seq_start", i32(0, 4)), ("seq_start", args["seq_start"].long()),
               ("seq_len", i32(70)), ("seq_len", args["seq_len"].long()), ("path", args["path"].long()), ("n_kept", i32(1)),
               ("n_kept", args["n_kept"].long())]
    refused(K.keep_rows, args, changes, list(args), ["k", "v"])
    with pytest.raises(K.KernelError):
        K.copy_pages(args["k"], args["k"], [0], [1])
    K.copy_pages(both[0], both[1], [0], [1])                  # halves of one tensor have nothing in common
    assert torch.equal(both[:, :, 1], both[:, :, 0])
    K.check_status()
