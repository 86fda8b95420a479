"""Steps of drafted tokens through a model: trees against the plain oracle, the walk and the kept rows together as they are
used, sequences that go on as ordinary ones, forks."""
import json
import os

import numpy as np
import pytest
import torch

from draft_helpers import random_tree
from helpers import TINY, TOL, assert_close, load_plain, make_model_dir, plain_logits, rand_tokens
from plain import llama_plain as P

pytestmark = pytest.mark.gpu
DTYPES = ["float32", "bfloat16"]


@pytest.fixture(scope="module", params=[(n, d) for n in "ABCDEG" for d in DTYPES], ids=lambda p: f"{p[0]}-{p[1]}")
def setup(request, tmp_path_factory):
    from stratum_b200 import Stratum
    name, dtype = request.param
    path = make_model_dir(str(tmp_path_factory.mktemp(f"draft{name}_{dtype}")), TINY[name], seed=ord(name), dtype=dtype)
    cfg, w = load_plain(path)
    return name, dtype, cfg, w, Stratum(path, dtype=dtype, max_tokens=4096)


def line(tokens, tree, i):
    """The tokens from the first node down to node i."""
    out = []
    while i >= 0:
        out.append(tokens[i])
        i = tree[i]
    return out[::-1]


def check_trees(llm, plain, vocab, dtype, olds, news, seed):
    from stratum_b200 import DraftEntry, StepEntry
    rng = np.random.default_rng(seed)
    prompts = [rand_tokens(rng, n, vocab) for n in olds]
    slots = [llm.acquire() for _ in olds]
    if any(olds):
        llm.step([StepEntry(s, p) for s, p in zip(slots, prompts) if p])
    entries = [DraftEntry(s, rand_tokens(rng, n, vocab), random_tree(rng, n, 4)) for s, n in zip(slots, news)]
    logits, batch = llm.engine.run_drafts(entries)
    llm.engine.check_kernels()
    got, r = logits.cpu().numpy(), 0
    for s, p, e in zip(slots, prompts, entries):
        assert llm.engine.length(s) == len(p)
        for i in range(len(e.tokens)):
            ref = plain(p + line(e.tokens, e.parents, i))[-1]
            assert_close(got[r + i], ref, dtype, f"node {i} behind {len(p)}")
        r += len(e.tokens)
    llm.engine.cache.trim(slots)
    for s in slots:
        llm.release(s)
    llm.engine.cache.check()
    assert llm.engine.cache.tokens_held() == 0


def test_trees_against_the_plain_model(setup):
    name, dtype, cfg, w, llm = setup
    longest = cfg.get("max_position_embeddings", 512)
    plain = lambda toks: plain_logits(cfg, w, toks)      # noqa: E731
    check_trees(llm, plain, cfg["vocab_size"], dtype, [5, 0, 64, 33], [7, 3, 1, 12], 1)
    if longest >= 256:
        check_trees(llm, plain, cfg["vocab_size"], dtype, [130, 60], [20, 70], 2)
    check_trees(llm, plain, cfg["vocab_size"], dtype, [9], [1], 3)


def test_greedy_generation_with_drafts(setup):
    """Looked-up drafts of which some are right: the tokens are the greedy ones, whatever is drafted, and the sequence goes on
    by ordinary steps behind them."""
    from stratum_b200 import DraftEntry, StepEntry
    name, dtype, cfg, w, llm = setup
    rng = np.random.default_rng(7)
    V = cfg["vocab_size"]
    prompts = [rand_tokens(rng, n, V) for n in (9, 61, 1)]
    want = [r.tokens for r in llm.generate(prompts, max_new_tokens=40, stop_ids=())]
    if dtype == "float32":
        assert want[0][:8] == P.greedy_generate(cfg, w, prompts[0], 8)
    slots = [llm.acquire() for _ in prompts]
    first = llm.step([StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)]).argmax(1).tolist()
    out = [[t] for t in first]
    steps = kept = 0
    while any(len(o) < 30 for o in out):
        entries, live = [], [i for i, o in enumerate(out) if len(o) < 30]
        for i in live:
            n = int(rng.integers(1, 9))
            tree = random_tree(rng, n, 3)
            tokens = [out[i][-1]]
            depth = [0]
            for j in range(1, n):                          # right with a chance of two thirds where its parent is
                depth.append(depth[tree[j]] + 1)
                right = want[i][len(out[i]) - 1 + depth[j]] if len(out[i]) - 1 + depth[j] < 40 else 0
                tokens.append(right if rng.random() < 0.67 else int(rng.integers(0, V)))
            entries.append(DraftEntry(slots[i], tokens, tree))
        before = [llm.engine.length(e.slot) for e in entries]
        new = llm.draft_step(entries)
        steps += 1
        for i, e, t, b in zip(live, entries, new, before):
            assert 1 <= len(t) <= len(e.tokens) and llm.engine.length(e.slot) == b + len(t)
            kept += len(t) - 1
            out[i] += t
        llm.engine.cache.check()
    for o, ref in zip(out, want):
        same = next((k for k, (a, b) in enumerate(zip(o, ref)) if a != b), len(ref))
        # (in bfloat16 a near tie may fall the other way in a batch of another shape)
        assert same >= min(len(o), len(ref)) if dtype == "float32" else same >= 1
    assert kept > 0 and steps < 30
    # the rows that were moved are the sequence's own: an ordinary step behind them sees what the plain model sees
    got = llm.engine.step([StepEntry(s, [o[-1]], [0]) for s, o in zip(slots, out)]).cpu().numpy()
    for i in range(len(slots)):
        seq = prompts[i] + out[i]
        if len(seq) <= cfg.get("max_position_embeddings", 512):
            assert_close(got[i], plain_logits(cfg, w, seq)[-1], dtype, f"behind {len(seq)} tokens")
    for s in slots:
        llm.release(s)
    llm.engine.cache.check()


def test_drawn_tokens(setup):
    """Draws with a temperature, drafted from a distribution and looked up: fixed by the streams, the lengths follow."""
    from stratum_b200 import DraftEntry, SamplingParams, StepEntry
    from stratum_b200.sampling import Pcg32
    name, dtype, cfg, w, llm = setup
    rng = np.random.default_rng(9)
    V = cfg["vocab_size"]
    prompts = [rand_tokens(rng, n, V) for n in (12, 30)]
    params = SamplingParams(temperature=0.8, seed=3)
    draft = torch.softmax(torch.randn(13, V, device="cuda", generator=torch.Generator("cuda").manual_seed(1)), -1)
    drafts = [rand_tokens(rng, 6, V), rand_tokens(rng, 5, V)]
    results = []
    for _ in range(2):
        slots = [llm.acquire() for _ in prompts]
        llm.step([StepEntry(s, p) for s, p in zip(slots, prompts)])
        streams = [Pcg32(3, i) for i in range(2)]
        a = llm.draft_step([DraftEntry(s, [1] + d) for s, d in zip(slots, drafts)], params, streams, draft)
        b = llm.draft_step([DraftEntry(s, [t[-1]] + d[:2], [-1, 0, 0]) for s, t, d in zip(slots, a, drafts)], params, streams)
        assert [llm.engine.length(s) for s in slots] == [len(p) + len(x) + len(y) for p, x, y in zip(prompts, a, b)]
        assert all(0 <= t < V for x in a + b for t in x)
        results.append((a, b))
        for s in slots:
            llm.release(s)
    assert results[0] == results[1]


def test_errors_leave_sequences_as_they_were(setup):
    from stratum_b200 import DraftEntry, SamplingParams, StepEntry
    from stratum_b200.cache import CacheFull
    from stratum_b200.engine import StepError
    name, dtype, cfg, w, llm = setup
    s = llm.acquire()
    llm.step([StepEntry(s, [1, 2, 3])])
    held = llm.engine.cache.tokens_held()
    V = cfg["vocab_size"]
    for entry in (DraftEntry(s, []), DraftEntry(s, [V]), DraftEntry(s, [1, -1]), DraftEntry(s, [1, 2], [-1]), DraftEntry(s, [1, 2], [0, 0]),
                  DraftEntry(s, [1, 2], [-1, 1]), DraftEntry(s, [1, 2, 3], [-1, 0, -1]), DraftEntry(s + 1, [1]), DraftEntry(s, [1] * 1025)):
        with pytest.raises(StepError):
            llm.draft_step([entry])
    with pytest.raises(StepError):
        llm.draft_step([DraftEntry(s, [1]), DraftEntry(s, [2])])
    with pytest.raises(StepError):
        llm.draft_step([])
    for params in (SamplingParams(temperature=1.0, top_k=5), SamplingParams(temperature=1.0, top_p=0.9), SamplingParams(temperature=1.0)):
        with pytest.raises(ValueError):
            llm.draft_step([DraftEntry(s, [1])], params)
    with pytest.raises(ValueError):
        llm.draft_step([DraftEntry(s, [1, 2])], draft=torch.zeros(1, V, device="cuda"))
    other = llm.acquire()
    llm.engine.cache.reserve([other], [4096 - 64])
    with pytest.raises(CacheFull):
        llm.draft_step([DraftEntry(s, [1] * 100)])
    llm.release(other)
    with pytest.raises(Exception):                        # a draft the kernel refuses, behind the step that took pages for it
        llm.draft_step([DraftEntry(s, [1] * 100)], draft=torch.zeros(100, V, device="cuda", dtype=torch.bfloat16))
    assert llm.engine.length(s) == 3 and llm.engine.cache.tokens_held() == held
    logits, batch = llm.engine.run_drafts([DraftEntry(s, [5, 6])])
    llm.engine.step([StepEntry(s, [7])])                  # the sequence goes on without its drafts: they cannot be kept any more
    with pytest.raises(StepError):
        llm.engine.keep_drafts(batch, [1])
    llm.release(s)
    llm.engine.cache.check()


def test_forks_go_on_by_themselves(setup):
    from stratum_b200 import DraftEntry, StepEntry
    name, dtype, cfg, w, llm = setup
    rng = np.random.default_rng(11)
    V = cfg["vocab_size"]
    for n in (1, 64, 75):
        prompt = rand_tokens(rng, n, V)
        s = llm.acquire()
        llm.step([StepEntry(s, prompt)])
        forks = [s] + llm.fork(s, 2)
        tails = [rand_tokens(rng, k, V) for k in (3, 9, 5)]
        got = llm.engine.step([StepEntry(f, t, list(range(len(t)))) for f, t in zip(forks, tails)]).cpu().numpy()
        ref = np.concatenate([plain_logits(cfg, w, prompt + t)[n:] for t in tails])
        assert_close(got, ref, dtype, f"forks of {n}")
        llm.release(s)                                    # the others keep the pages they share
        llm.engine.cache.check()
        more = [rand_tokens(rng, 2, V) for _ in range(2)]
        logits, batch = llm.engine.run_drafts([DraftEntry(f, t) for f, t in zip(forks[1:], more)])
        got = logits.cpu().numpy()
        ref = np.concatenate([plain_logits(cfg, w, prompt + t + m)[-2:] for t, m in zip(tails[1:], more)])
        assert_close(got, ref, dtype, f"drafts of forks of {n}")
        for f in forks[1:]:
            llm.release(f)
        llm.engine.cache.check()
        assert llm.engine.cache.tokens_held() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_layers_with_and_without_a_window(tmp_path, dtype):
    """Layers whose windows differ, and sequences whose pages have been handed back behind them."""
    from stratum_b200 import Stratum
    from stratum_b200.engine.model import expected_tensors
    from stratum_b200.weights.random_init import _TORCH_DTYPES, random_tensors
    from stratum_b200.weights.safetensors_io import write_safetensors
    from test_windowed_layers_gpu import _define, _plain
    cfg = _define().from_dict({"architectures": ["ToyWindowedForCausalLM"], "hidden": 64, "inner": 96, "vocab": 97, "eps": 1e-5})
    tensors = random_tensors(expected_tensors(cfg), 5, 0.1, _TORCH_DTYPES[dtype])
    path = str(tmp_path / "windowed")
    os.makedirs(path)
    with open(os.path.join(path, "config.json"), "w") as f:
        json.dump(dict(cfg.to_dict(), torch_dtype=dtype), f)
    write_safetensors(os.path.join(path, "model.safetensors"), tensors)
    c, w = load_plain(path)
    llm = Stratum(path, dtype=dtype, max_tokens=2048)
    check_trees(llm, lambda toks: _plain(c, w, toks), 97, dtype, [150, 20, 0, 200], [50, 9, 80, 3], 4)


@pytest.mark.parametrize("family", ["vitinex", "mokatar", "dabodra", "getizen", "memipel", "nibelorn"])
def test_forks_of_models_with_states(tmp_path, family):
    """A fork has the state, the windows' pages and the embedding's last token too: it answers as the sequence it came from."""
    import importlib
    from stratum_b200 import DraftEntry, StepEntry, Stratum
    from stratum_b200.engine import StepError
    helpers = importlib.import_module(f"{family}_helpers")
    path = helpers.make(str(tmp_path / family), "A", "float32")[0]
    llm = Stratum(path, dtype="float32", max_tokens=1024, use_graphs=False)
    rng = np.random.default_rng(2)
    V = llm.model.vocab
    s = llm.acquire()
    llm.step([StepEntry(s, rand_tokens(rng, 70, V))])
    (f,) = llm.fork(s)
    for k in range(3):
        t = rand_tokens(rng, 2, V)
        a = llm.engine.step([StepEntry(s, t, [0, 1])])
        b = llm.engine.step([StepEntry(f, t, [0, 1])])
        assert torch.equal(a, b) and bool(a.abs().max() > 0)
    llm.engine.step([StepEntry(f, rand_tokens(rng, 3, V))])          # they part, and neither disturbs the other
    x = llm.engine.step([StepEntry(s, [1], [0])])
    (g,) = llm.fork(s)
    assert torch.equal(llm.engine.step([StepEntry(g, [2], [0])]), llm.engine.step([StepEntry(s, [2], [0])]))
    assert torch.isfinite(x).all()
    if not llm.model.takes_drafts():
        with pytest.raises(StepError):
            llm.draft_step([DraftEntry(s, [1, 2])])
    for slot in (s, f, g):
        llm.release(slot)
    llm.engine.cache.check()


def test_drafts_between_ordinary_steps(setup):
    """Ordinary steps (captured ones), steps of drafted tokens, forks and steps of several tokens in turn: a sequence goes on as if it
    had been decoded one token at a time, whoever joined or left meanwhile."""
    from stratum_b200 import DraftEntry, StepEntry
    name, dtype, cfg, w, llm = setup
    rng = np.random.default_rng(21)
    V = cfg["vocab_size"]
    prompts = [rand_tokens(rng, n, V) for n in (61, 5, 90)]
    want = [r.tokens for r in llm.generate(prompts, max_new_tokens=30, stop_ids=())]
    slots = [llm.acquire() for _ in prompts]
    have = [[t] for t in llm.step([StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)]).argmax(1).tolist()]
    drafted = 0
    for turn in range(30):
        live = [i for i in range(3) if len(have[i]) < 26]
        if not live:
            break
        if turn % 3 == 1:                                 # drafts: some right, some wrong
            entries = []
            for i in live:
                n = len(have[i])
                good = want[i][n:n + 2] if have[i] == want[i][:n] else [1, 2]
                entries.append(DraftEntry(slots[i], [have[i][-1], good[0], (good[-1] + 1) % V, good[-1]], [-1, 0, 1, 1]))
            for i, t in zip(live, llm.draft_step(entries)):
                have[i] += t
                drafted += len(t) - 1
        elif turn % 3 == 2:                               # another sequence comes and goes
            f = llm.fork(slots[live[0]])
            llm.draft_step([DraftEntry(f[0], rand_tokens(rng, 9, V))])
            llm.decode_step(f, [1])
            llm.release(f[0])
        else:
            for i, t in zip(live, llm.decode_step([slots[i] for i in live], [have[i][-1] for i in live])[0]):
                have[i].append(t)
    llm.engine.cache.check()
    for i, s in enumerate(slots):
        assert llm.engine.length(s) == len(prompts[i]) + len(have[i]) - 1
        # every token is the model's own pick behind the ones in front of it, as far as near-equal logits allow
        ref = plain_logits(cfg, w, prompts[i] + have[i][:-1])[len(prompts[i]) - 1:]
        span = np.abs(ref).max()
        for r, t in zip(ref, have[i]):
            assert r.max() - r[t] <= 2 * TOL[dtype] * span    # (the errors of two logits)
        llm.release(s)
    assert drafted > 0 and llm.engine.cache.tokens_held() == 0
