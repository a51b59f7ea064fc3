"""How attention over a shared prefix cuts its work, against what the launcher takes."""

from __future__ import annotations

import random

import pytest
import torch


@pytest.fixture
def launch(monkeypatch):
    from miniserve_amd import ops

    monkeypatch.setattr(ops, "_decode_target", lambda: 512)
    ops.shared_prefix_launch.cache_clear()
    yield ops.shared_prefix_launch
    ops.shared_prefix_launch.cache_clear()


def taken(launch, sequences, tokens, groups, kv_heads, per_token, longest, dtype, *, max_query, max_sharing):
    """The cut for a batch, after the checks of the library's entry (attention_shared.hip)."""

    rows = sequences * tokens * per_token
    tile, shared_splits, own_tiles, own_splits = launch(rows, max_sharing, sequences, kv_heads, per_token, longest, longest, max_query, dtype, 64)
    assert own_tiles >= 1
    if shared_splits:
        shared_tiles = -(-rows // tile) if groups == 1 else rows // tile + groups
        units = -(-kv_heads * shared_splits // 8) * 8
        assert rows // tile + groups < 2**24 // shared_splits
        assert units * shared_tiles + sequences * own_tiles * own_splits * kv_heads < 2**22, "the batch is too large"
    assert sequences * own_tiles * max(own_splits, 1) < 2**22 // kv_heads, "the batch is too large"
    return own_tiles


@pytest.mark.parametrize("sequences,tokens,heads", [(1500, 1, 32), (500, 5, 64), (4000, 1, 64), (2, 4000, 64)])
def test_batches_without_bounds_are_taken(launch, sequences, tokens, heads):
    taken(launch, sequences, tokens, 1, 8, heads // 8, 4096, torch.bfloat16, max_query=sequences * tokens, max_sharing=1)


def test_batches_of_all_sizes_are_taken(launch):
    rng = random.Random(1)
    for _ in range(3000):
        sequences = round(4000 ** rng.random())
        tokens = round((8000 // sequences + 1) ** rng.random())
        groups = rng.randint(1, sequences)
        kv_heads, per_token = rng.choice([1, 2, 8, 16]), rng.choice([1, 2, 3, 8, 16])
        longest = rng.choice([1, 100, 5000, 100_000])
        for max_query in (tokens, sequences * tokens):
            for dtype in (torch.float32, torch.bfloat16):
                taken(launch, sequences, tokens, groups, kv_heads, per_token, longest, dtype, max_query=max_query, max_sharing=groups)


def test_a_few_sequences_get_a_workgroup_a_tile(launch):
    assert taken(launch, 64, 1, 1, 8, 8, 30_000, torch.bfloat16, max_query=1, max_sharing=1) == 1
    assert taken(launch, 16, 5, 1, 8, 2, 4_096, torch.bfloat16, max_query=5, max_sharing=1) == 1
    assert taken(launch, 4, 200, 1, 8, 4, 4_096, torch.bfloat16, max_query=200, max_sharing=1) == 50
