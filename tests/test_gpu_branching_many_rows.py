"""Attention over a shared prefix for batches of many sequences, without bounds on them."""

from __future__ import annotations

import pytest
import torch
from test_gpu_branching_kernels import attention_case, check_attention, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sequences,tokens,heads,kv_heads", [(1600, 1, 32, 8), (500, 5, 64, 8), (3000, 1, 4, 4)])
def test_many_sequences_without_bounds(ops, sequences, tokens, heads, kv_heads):  # noqa: F811
    members = [(tokens, tokens + i % 23) for i in range(sequences)]
    half = sequences // 2
    case = attention_case(torch.bfloat16, heads, kv_heads, 16, 16, [(48, members[:half]), (16, members[half:])], seed=sequences)
    check_attention(ops, case)
    check_attention(ops, case, max_query=tokens)
