"""Requests that branch in a model with a window, on the GPU."""

from __future__ import annotations

import pytest
import windowed_branches as windowed
from helpers import read_config

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("recorded", [False, True], ids=["eager", "recorded"])
def test_runs_of_neighbours_differ_between_groups_of_pages(recorded, model_folders, monkeypatch):
    from miniserve_amd import ops
    from miniserve_amd.engine import batch

    monkeypatch.setattr(batch, "SHARED_FRONT_KEYS", 256)
    folder, block_size = model_folders["c"]
    before = ops.attention_calls["shared"]
    runner = windowed.make_runner(folder, block_size, "bfloat16", device="cuda:0", recorded=recorded)
    branches = windowed.five_branches_and_three_pairs(runner, read_config(folder)["vocab_size"])
    found, allowed = windowed.worst(branches, folder, "bfloat16")
    assert found <= allowed, f"{found:.3e} > {allowed:.3e}"
    assert ops.attention_calls["shared"] > before
    if recorded:
        assert {key[2] for key in runner._decode_graphs if len(key) == 3} == {(1, 256)}


@pytest.mark.parametrize("recorded", [False, True], ids=["eager", "recorded"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_drafts_in_a_model_with_a_window(dtype, recorded, model_folders):
    folder, block_size = model_folders["c"]
    runner = windowed.make_runner(folder, block_size, dtype, device="cuda:0", recorded=recorded)
    branches = windowed.rounds_of_drafts(runner, read_config(folder)["vocab_size"], rounds=25, seed=31)
    found, allowed = windowed.worst(branches, folder, dtype)
    assert found <= allowed, f"{found:.3e} > {allowed:.3e}"
