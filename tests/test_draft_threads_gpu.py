"""The first calls of a process, made by several threads at once on streams of their own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = r"""
import threading
import numpy as np
import torch
from draft_helpers import PAGE, TreeBatch, run_tree
from stratum_b200 import kernels as K
from stratum_b200.csrc import build

for name in ("attention_tree", "draft_verify"):
    build.load(name)                       # (what is raced for is the first launch, not the compiler)
K.status_word()
batches = [TreeBatch(3, [300, 70], [new, 2], 8, 2, hd).round_to(dt) for dt, hd, new in
           ((torch.bfloat16, 64, 5), (torch.bfloat16, 64, 40), (torch.bfloat16, 128, 5), (torch.bfloat16, 128, 40), (torch.float32, 128, 5))]
types = [torch.bfloat16] * 4 + [torch.float32]
T, V = 6, 128256
target = torch.softmax(torch.randn(T, V, device="cuda"), 1)
i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
tokens, parents, start, uniform = i32(1, 2, 3, 4, 5, 6), i32(-1, 0, 0, 1, 1, 2), i32(0, 6), torch.rand(T, device="cuda")
torch.cuda.synchronize()
gate, errors, results = threading.Barrier(8), [], [None] * 8

def work(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            gate.wait()
            out = [run_tree(b, dt) for b, dt in zip(batches, types)]
            probs = torch.empty(T, V, device="cuda")
            K.token_probs(target, torch.ones(T, device="cuda"), probs)
            path, kept, picked = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (T, 1, 1))
            K.verify_drafts(target, None, tokens, parents, start, uniform, path, kept, picked)
            torch.cuda.current_stream().synchronize()
            results[i] = out + [probs, path, kept, picked]
    except Exception as e:
        errors.append(repr(e))

threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
K.check_status()
assert not errors, errors
for r in results[1:]:
    assert all(torch.equal(a, b) for a, b in zip(results[0], r))
print("all alike")
"""


def test_first_calls_of_eight_threads():
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(here), here, os.environ.get("PYTHONPATH", "")]))
    run = subprocess.run([sys.executable, "-c", PROGRAM], env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "all alike" in run.stdout, run.stderr[-2000:]
