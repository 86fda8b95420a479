"""The launchers of drafted decoding opt into large shared memory and large clusters at every launch (no GPU: their sources)."""
import os
import re

import pytest

import stratum_b200

CSRC = os.path.join(os.path.dirname(stratum_b200.__file__), "csrc")


def bodies(text):
    """(name, body) of the functions that begin in the first column."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"^[A-Za-z_][^\n;={}]*?(\w+)\([^;{}]*\)\s*\{\n(.*?)^\}", text, re.M | re.S):
        yield m.group(1), m.group(2)


@pytest.mark.parametrize("name,functions", [("attention_tree", {"launch_tree_tc", "launch_tree_simple"}),
                                            ("draft_verify", {"launch_clusters", "resident_clusters"})])
def test_opt_ins_are_made_at_every_launch(name, functions):
    """The opt-in is the current device's, may fail once, and may be asked for by two threads at once: nothing that outlives a launch
    decides whether it is made."""
    with open(os.path.join(CSRC, name + ".cu")) as f:
        source = f.read()
    found = set()
    for function, body in bodies(source):
        if "cudaFuncSetAttribute" not in body:
            continue
        found.add(function)
        assert not re.search(r"\bstatic\b", body), function
        for guard in re.findall(r"if \(([^{};]*?)\)\s*\{?[^{}]*?cudaFuncSetAttribute", body):
            assert re.match(r"(cluster|C) > 8\b", guard), (function, guard)      # (sizes of this launch alone)
    assert found == functions


def test_what_is_kept_of_a_device_is_kept_for_that_device():
    """Of the answers of one device (SMs, resident clusters) the next one has no use, and a failure is no answer."""
    for name in ("draft_verify", "cache_move"):
        with open(os.path.join(CSRC, name + ".cu")) as f:
            source = re.sub(r"//[^\n]*", "", f.read())
        for kept in re.findall(r"^[ \t]+static (?!constexpr|const\b)([^;]*);", source, re.M):
            assert re.match(r"std::atomic<int> \w+\[64\]", kept), (name, kept)
