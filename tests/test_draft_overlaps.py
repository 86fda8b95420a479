"""Memory that a call of drafted decoding would write while it is read: refused before anything runs.  (No GPU: the device check and
the launch are replaced.)"""
import pytest
import torch

from stratum_b200 import kernels as K


@pytest.fixture
def launches(monkeypatch):
    """The calls that would have been launched."""
    seen = []
    monkeypatch.setattr(K, "_one_device", lambda *a: None)
    monkeypatch.setattr(K, "_stream", lambda: 0)
    monkeypatch.setattr(K, "status_word", lambda: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(K, "_tree_plans", {(False, False, 64): (148, 32)})
    monkeypatch.setattr(K, "_fn", lambda lib, name, types: lambda *a: seen.append(name) or 0)
    return seen


def i32(n):
    return torch.zeros(n, dtype=torch.int32)


def verify_args(T=6, B=2, V=40):
    return dict(target=torch.zeros(T, V), draft=torch.zeros(T, V), tokens=i32(T), parents=i32(T), seq_start=i32(B + 1), uniform=torch.zeros(T),
                path=i32(T), n_kept=i32(B), next_ids=i32(B))


@pytest.mark.parametrize("shift", [-5, -1, 0, 1, 5])
@pytest.mark.parametrize("read", ["tokens", "parents", "uniform", "seq_start"])
@pytest.mark.parametrize("written", ["path", "n_kept", "next_ids"])
def test_verify_outputs_that_meet_an_input(launches, written, read, shift):
    args = verify_args()
    n, m = args[read].numel(), args[written].numel()
    buf = torch.zeros(40, dtype=args[read].dtype)
    args[read] = buf[10:10 + n]
    args[written] = buf.view(torch.int32)[10 + shift:10 + shift + m]
    meets = shift < n and shift + m > 0
    if meets:
        with pytest.raises(K.KernelError, match="memory of their own"):
            K.verify_drafts(**args)
    else:
        K.verify_drafts(**args)
    assert launches == ([] if meets else ["stratum_verify_drafts"])


@pytest.mark.parametrize("T", [6, 0])
@pytest.mark.parametrize("a,b", [("path", "n_kept"), ("n_kept", "next_ids"), ("next_ids", "path")])
def test_verify_outputs_that_meet_one_another(launches, a, b, T):
    args = verify_args(T)
    na, nb = args[a].numel(), args[b].numel()
    buf = i32(40)
    for shift in range(-8, 9):
        args[a], args[b] = buf[10:10 + na], buf[10 + shift:10 + shift + nb]
        launches.clear()
        if na and nb and shift < na and shift + nb > 0:
            with pytest.raises(K.KernelError, match="memory of their own"):
                K.verify_drafts(**args)
            assert not launches
        else:
            K.verify_drafts(**args)
            assert launches


@pytest.mark.parametrize("name", ["target", "draft"])
def test_verify_outputs_inside_a_row(launches, name):
    """Rows of 40 in a matrix of 60 columns: the columns between the rows are nobody's."""
    for at, meets in ((0, True), (34, True), (39, True), (40, False), (54, False), (55, True), (5 * 60 + 39, True), (5 * 60 + 40, False),
                      (61, True), (104, False)):
        args = verify_args()
        buf = torch.zeros(6 * 60 + 60)
        args[name] = buf[:360].view(6, 60)[:, :40]
        args["path"] = buf.view(torch.int32)[at:at + 6]
        launches.clear()
        if meets:
            with pytest.raises(K.KernelError, match="memory of their own"):
                K.verify_drafts(**args)
            assert not launches
        else:
            K.verify_drafts(**args)
            assert launches


def test_verify_takes_views_side_by_side(launches):
    """One buffer cut into the three outputs, inputs that are one another's views, a row without a distance."""
    args = verify_args()
    out = i32(10)
    args.update(path=out[:6], n_kept=out[6:8], next_ids=out[8:], parents=args["tokens"], draft=args["target"])
    K.verify_drafts(**args)
    one = verify_args(T=1, B=1)
    one["target"] = torch.as_strided(torch.zeros(200), (1, 40), (3, 1))
    K.verify_drafts(**one)
    K.verify_drafts(**{**verify_args(), "draft": None})
    assert len(launches) == 3


@pytest.mark.parametrize("in_place", [False, True])
def test_temperatures_inside_the_probabilities(launches, in_place):
    """out: 3 rows of 40 in a matrix of 50 columns."""
    for at, meets in ((0, True), (38, True), (40, False), (47, False), (48, True), (100, True), (138, True), (140, False)):
        buf = torch.zeros(200)
        out = buf[:150].view(3, 50)[:, :40]
        args = (out if in_place else torch.zeros(3, 40), buf[at:at + 3], out)
        launches.clear()
        if meets:
            with pytest.raises(K.KernelError, match="no part of out"):
                K.token_probs(*args)
            assert not launches
        else:
            K.token_probs(*args)
            assert launches


@pytest.mark.parametrize("name,dtype", [("k_cache", torch.float32), ("v_cache", torch.float32), ("token_pos", torch.int32),
                                        ("tree_mask", torch.int64), ("seq_start", torch.int32), ("seq_len", torch.int32),
                                        ("block_table", torch.int32)])
def test_attention_outputs_inside_what_is_read(launches, name, dtype):
    """out: 3 rows of 128 in a matrix of 160 columns."""
    shapes = dict(k_cache=(2, 2, 64, 64), v_cache=(2, 2, 64, 64), token_pos=(3,), tree_mask=(3, 1), seq_start=(3,), seq_len=(2,),
                  block_table=(2, 2))
    n = 1
    for x in shapes[name]:
        n *= x
    words = n * (2 if dtype == torch.int64 else 1)         # of 32 bits
    front = 2 * 16384
    for at in (0, 60, 126, 128, 130, 158, 160, 320 + 126, 320 + 128, -words, -2):
        meets = any(at < r * 160 + 128 and at + words > r * 160 for r in range(3))
        buf = torch.zeros(front + 480 + 16384)
        args = dict(q=torch.zeros(3, 128), out=buf[front:front + 480].view(3, 160)[:, :128], n_q=2, n_kv=2, head_dim=64, page_tokens=64,
                    window=0, scale=0.125, max_new=2)
        for other, shape in shapes.items():
            args[other] = torch.zeros(shape, dtype={"tree_mask": torch.int64}.get(other, torch.float32 if "cache" in other else torch.int32))
        args[name] = buf[front + at:front + at + words].view(dtype).view(shapes[name])
        launches.clear()
        if meets:
            with pytest.raises(K.KernelError, match="memory of its own"):
                K.attention_tree(**args)
            assert not launches
        else:
            K.attention_tree(**args)
            assert launches == ["stratum_attention_tree"]


@pytest.mark.parametrize("name", ["block_table", "seq_start", "seq_len", "path", "n_kept"])
@pytest.mark.parametrize("where", ["k", "v"])
def test_kept_rows_described_inside_the_cache(launches, where, name):
    shapes = dict(block_table=(2, 2), seq_start=(3,), seq_len=(2,), path=(6,), n_kept=(2,))
    n = shapes[name][0] * (shapes[name][1] if len(shapes[name]) > 1 else 1)
    size = 2 * 3 * 2 * 64 * 5                               # of keys and of values
    for at, meets in ((0, True), (size - 1, True), (size, False), (-n, False), (-n + 1, True), (size // 2, True)):
        buf = i32(size + 40)
        args = {k: i32(s) for k, s in shapes.items()}
        args[name] = buf[20 + at:20 + at + n].view(shapes[name])
        for kv in "kv":
            args[kv] = (buf[20:20 + size] if kv == where else i32(size)).view(2, 3, 2, 64, 5)
        launches.clear()
        if meets:
            with pytest.raises(K.KernelError, match="no part of the cache"):
                K.keep_rows(**args)
            assert not launches
        else:
            K.keep_rows(**args)
            assert launches == ["stratum_keep_rows"]
