"""The forms that the cache operators' GPU tests mean to run are those the
library's plans choose, so that a change of the plans' constants cannot leave a
kernel without its test; and those tests' own definition of the eviction."""

from __future__ import annotations

import os
import subprocess
from pathlib import Path

import pytest
import torch

import cache_ops_ref as ref
import test_gpu_cache_forms as forms
import test_gpu_tree_small_weights as small

ROOT = Path(__file__).resolve().parents[1]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not found")
def test_tree_forms_are_the_plans(tmp_path):
    from SSA import ssa_tree_num_splits

    exe = tmp_path / "plans"
    cmd = [HIPCC, "-x", "hip", "--cuda-host-only", "-std=c++20", "-O1", "-I", str(ROOT / "luciole-1b_amd" / "csrc"),
           str(ROOT / "tests" / "host_addr" / "cache_plans.cpp"), "-o", str(exe)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stderr[-3000:]
    calls = [((B, Hq, Hk, cap, T, s), (rows, splits)) for (B, Hq, Hk, cap, T, _, s), (rows, splits) in forms.FORMS]
    calls += [((*c, 1), (rows, 1)) for c, rows in small.FORMS]
    lines = "".join("tree " + " ".join(map(str, c)) + "\n" for c, _ in calls)
    out = subprocess.run([str(exe)], input=lines, capture_output=True, text=True, timeout=60, check=True).stdout.split("\n")
    for (call, want), line in zip(calls, out):
        rows, _, splits = map(int, line.split())
        assert (rows, splits) == want, call
        assert ssa_tree_num_splits(*call[:5], call[5]) == splits, call  # of the built library too
    # every number of rows, several stages of keys each; the merge of few splits and of many
    assert {rows for _, (rows, _) in calls} == {32, 64, 128, 256}
    assert all(any(s > 8 for _, (r, s) in calls if r == rows) for rows in (32, 128, 256))
    for (B, _, _, _, _, lens, _), _ in forms.FORMS:
        assert len(lens) == B


@pytest.mark.parametrize("cap,lens,keep,sinks,recent", [
    (300, [300, 299, 120, 0, 1000], 120, 4, 30), (64, [64], 1, 0, 0), (64, [64, 63], 63, 63, 0),
    (200, [200], 100, 40, 60), (90, [90, 88], 89, 0, 7)])
def test_evicted_is_the_definition(cap, lens, keep, sinks, recent):
    w = forms._odd_weights(len(lens), 2, cap, cap, torch.device("cpu"))
    got = forms._evicted(lens, w, keep, sinks, recent)
    want = ref.evict(lens, w, keep, sinks, recent)
    assert got[0].tolist() == want[0] and torch.equal(got[2], want[2])
    assert torch.equal(got[1].view(torch.int32), want[1].view(torch.int32))
