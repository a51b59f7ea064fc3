"""Requests that branch in a model with a window, over the stand-ins for the kernels."""

from __future__ import annotations

import pytest
import torch_branching_kernels as kernels
import windowed_branches as windowed
from helpers import read_config
from test_cache_manager import Need, manager

from miniserve_amd.cache import CacheError, StepItem
from miniserve_amd.parts import KVCacheNeed


@pytest.mark.parametrize("recorded", [False, True], ids=["eager", "recorded"])
def test_runs_of_neighbours_differ_between_groups_of_pages(recorded, model_folders, monkeypatch):
    from miniserve_amd.engine import batch

    monkeypatch.setattr(batch, "SHARED_FRONT_KEYS", 256)
    kernels.install(monkeypatch, recordings=recorded)
    folder, block_size = model_folders["c"]
    runner = windowed.make_runner(folder, block_size, "bfloat16", device="cpu", recorded=recorded)
    branches = windowed.five_branches_and_three_pairs(runner, read_config(folder)["vocab_size"])
    found, allowed = windowed.worst(branches, folder, "bfloat16")
    assert found <= allowed, f"{found:.3e} > {allowed:.3e}"
    assert kernels.CALLS["attention_shared_prefix"] >= 3
    if recorded:
        assert {key[2] for key in runner._decode_graphs if len(key) == 3} == {(1, 256)}


@pytest.mark.parametrize("window,size", [(6, 4), (6, 3), (1, 2), (9, 8), (16, 4)])
def test_drafts_are_forgotten_at_every_place_of_a_window(window, size):
    """A token and nine drafts a step, cut back to every length from the token on: the pages that the
    window needs there are still held, and afterwards no page more than a request has that was never cut."""

    needs = [Need(0, KVCacheNeed(1, 8)), Need(1, KVCacheNeed(1, 8, window=window, block_size=size))]
    m = manager(needs, block_size=4, num_blocks=60, slots=3, max_len=200)
    m.admit("r")
    length = 0
    for turn in range(60):
        taken = turn * 7 % 10
        step = m.prepare_step([StepItem("r", length, length + 10, keep=length + 1)])
        assert sum(page >= 0 for page in step.sequences[0].block_tables[1]) <= m.capacity().most_pages_held(length + 10, 10)[1]
        m.commit_step(step)
        m.assert_invariants()
        if turn % 5 == 0:
            m.fork("r", ["x"])
        m.truncate("r", length + 1 + taken)
        length += 1 + taken
        m.assert_invariants()
        first = max(length - window + 1, 0) // size
        table = m.block_table("r", 1)
        assert table[:first] == (-1,) * min(first, len(table)) and all(page >= 0 for page in table[first:])
        if turn % 5 == 0:
            m.truncate("x", length - taken)        # the branch takes none of the drafts
            m.commit_step(m.prepare_step([StepItem("x", length - taken, length - taken + 3)]))
            m.assert_invariants()
            m.release("x")
        if length > 180:
            m.release("r")
            m.admit("r")
            length = 0
    with pytest.raises(CacheError, match="keep"):
        m.prepare_step([StepItem("r", length, length + 2, keep=length + 3)])
    m.release("r")
    assert m.capacity().free_blocks == m.num_blocks


def test_pages_kept_for_a_cut_are_given_back_by_the_next_step():
    m = manager([Need(0, KVCacheNeed(1, 8, window=4))], block_size=4, num_blocks=5, slots=2, max_len=100)
    m.admit("r")
    m.commit_step(m.prepare_step([StepItem("r", 0, 16, keep=1)]))
    assert m.block_table("r") == (0, 1, 2, 3)
    m.commit_step(m.prepare_step([StepItem("r", 16, 28, keep=17)]))      # four pages are held, three more needed, one is free
    assert m.block_table("r")[:3] == (-1, -1, -1) and m.capacity().free_blocks == (1,)
    m.truncate("r", 28)                                                  # nothing to forget: all were taken
    assert m.capacity().free_blocks == (4,)
    m.assert_invariants()


@pytest.mark.parametrize("recorded", [False, True], ids=["eager", "recorded"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_drafts_in_a_model_with_a_window(dtype, recorded, model_folders, monkeypatch):
    kernels.install(monkeypatch, recordings=recorded)
    folder, block_size = model_folders["c"]
    runner = windowed.make_runner(folder, block_size, dtype, device="cpu", recorded=recorded)
    branches = windowed.rounds_of_drafts(runner, read_config(folder)["vocab_size"], rounds=25, seed=31)
    found, allowed = windowed.worst(branches, folder, dtype)
    assert found <= allowed, f"{found:.3e} > {allowed:.3e}"
