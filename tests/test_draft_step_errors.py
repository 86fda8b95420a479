"""A step of drafted tokens that fails leaves its random streams where they were (no GPU: the engine and the kernels are replaced)."""
import types

import pytest
import torch

from stratum_b200 import DraftEntry, SamplingParams, Stratum
from stratum_b200.engine import api
from stratum_b200.sampling import Pcg32

STAGES = ["run_drafts", "token_probs", "verify_drafts", "move_kept", "check_kernels"]


class Step:
    """A Stratum whose stage `fails` raises; `numbers`: what verify_drafts was given."""

    def __init__(self, monkeypatch):
        self.fails, self.numbers, self.trimmed = None, [], []
        slots = types.SimpleNamespace(is_live=lambda s: True)
        engine = types.SimpleNamespace(validate_drafts=lambda entries: None, run_drafts=self.run_drafts, keep_drafts=lambda batch, kept: None,
                                       move_kept=lambda *a: self.at("move_kept"), check_kernels=lambda: self.at("check_kernels"),
                                       cache=types.SimpleNamespace(slots=slots, trim=self.trimmed.append))
        self.llm = Stratum.__new__(Stratum)
        self.llm.engine = engine
        self.llm.model = types.SimpleNamespace(vocab=7, runtime=types.SimpleNamespace(device="cpu"))
        monkeypatch.setattr(api.K, "token_probs", lambda *a: self.at("token_probs"))
        monkeypatch.setattr(api.K, "verify_drafts", self.verify_drafts)

    def at(self, stage):
        if self.fails == stage:
            raise RuntimeError(stage)

    def run_drafts(self, entries):
        self.at("run_drafts")
        T = sum(len(e.tokens) for e in entries)
        return torch.zeros(T, 7), types.SimpleNamespace(token_ids=None, seq_start=None, drafts=types.SimpleNamespace(parent=None))

    def verify_drafts(self, target, draft, tokens, parents, start, uniform, path, kept, picked):
        self.at("verify_drafts")
        self.numbers.append(uniform.tolist())
        path.fill_(-1)
        kept.zero_()
        picked.fill_(3)


@pytest.mark.parametrize("stage", STAGES)
@pytest.mark.parametrize("shared", [False, True])
def test_streams_stay_where_they_were(monkeypatch, stage, shared):
    step = Step(monkeypatch)
    entries = [DraftEntry(0, [1, 2, 3]), DraftEntry(4, [5])]
    params = SamplingParams(temperature=0.7, seed=3)
    make = lambda: [Pcg32(3, 0)] * 2 if shared else [Pcg32(3, 0), Pcg32(3, 1)]           # noqa: E731
    streams, fresh = make(), make()
    step.fails = stage
    for _ in range(2):
        with pytest.raises(RuntimeError, match=stage):
            step.llm.draft_step(entries, params, streams)
    assert step.trimmed == [[0, 4]] * 2
    step.fails = None
    step.numbers.clear()
    assert step.llm.draft_step(entries, params, streams) == [[3], [3]]
    assert step.numbers == [[fresh[0].uniform() for _ in range(3)] + [fresh[1].uniform()]]
    assert [s.state for s in streams] == [s.state for s in fresh]         # a step that succeeds moves them on


def test_a_greedy_step_that_fails_needs_no_streams(monkeypatch):
    step = Step(monkeypatch)
    step.fails = "move_kept"
    with pytest.raises(RuntimeError, match="move_kept"):
        step.llm.draft_step([DraftEntry(2, [1, 2])])
    assert step.trimmed == [[2]]
