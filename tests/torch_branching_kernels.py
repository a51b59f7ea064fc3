"""Stand-ins, with torch on CPU tensors, for the kernels of requests that branch; see
``torch_kernels.py``, whose stand-ins they join."""

from __future__ import annotations

import plain_branching as plain
import torch
import torch_kernels

CALLS = {"attention_shared_prefix": 0, "copy_pages": 0, "verify_drafts": 0}


def attention_shared_prefix(q, key_pool, value_pool, *, block_table, query_start, context_lens, group_start, shared_lens, scale,
                            max_sharing=None, max_shared=None, max_own=None, max_query=None):
    """Each sequence over its own table, but the keys that its group shares over the table of
    the group's first sequence, and with the contract checked."""

    CALLS["attention_shared_prefix"] += 1
    page, table = key_pool.shape[2], block_table.clone()
    starts = group_start.tolist()
    assert starts == sorted(starts) and 0 <= starts[0] and starts[-1] <= block_table.shape[0]
    assert sum(length > 0 for length in shared_lens.tolist()) <= max_sharing
    for g, length in enumerate(shared_lens.tolist()):
        rows = range(starts[g], starts[g + 1])
        assert length % page == 0 and length <= max_shared
        for row in rows:
            brings = int(query_start[row + 1] - query_start[row])
            assert length <= int(context_lens[row]) - brings and brings <= max_query and int(context_lens[row]) - length <= max_own
            assert torch.equal(block_table[row, : length // page], block_table[rows[0], : length // page])
            table[row, : length // page] = block_table[rows[0], : length // page]
    return plain.attention_rows(q, key_pool, value_pool, table, query_start, context_lens, scale)[0].to(q.dtype)


def copy_pages(pools, source, destination):
    CALLS["copy_pages"] += 1
    assert len(source) == len(destination) == len(set(destination)) and not set(source) & set(destination)
    for pool in pools:
        assert pool.is_contiguous() and 0 <= min(*source, *destination) and max(*source, *destination) < pool.shape[1]
        pool[:, list(destination)] = pool[:, list(source)]


def verify_drafts(logits, row_start, draft_tokens, *, draft_probs=None, accept_uniform=None, draw_uniform=None, temperature=None):
    CALLS["verify_drafts"] += 1
    tokens, accepted = plain.verify(logits, row_start, draft_tokens, draft_probs, accept_uniform, draw_uniform, temperature)
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(accepted, dtype=torch.int32)


def install(monkeypatch, **options):
    from miniserve_amd import ops

    torch_kernels.install(monkeypatch, **options)
    for name in CALLS:
        CALLS[name] = 0
        monkeypatch.setattr(ops, name, globals()[name])
    monkeypatch.setattr(ops, "can_share_prefix", lambda head_dim, block_size: head_dim % 16 == 0 and head_dim <= 128 and block_size % 16 == 0)
