"""Attention over a shared prefix with every size of tile and many parts, whatever the rule on the
work would choose: each walk against the plain implementation, and which one ran."""

from __future__ import annotations

import random

import pytest
import torch
from test_gpu_branching_kernels import DEVICE, attention_case, check_attention, ints, ops  # noqa: F401

pytestmark = pytest.mark.gpu

TILES = [16, 32, 64, 128]
TENSORS = ("q", "key_pool", "value_pool")


@pytest.fixture
def cut(ops, monkeypatch):  # noqa: F811
    """``cut(tile, shared parts, workgroups of a sequence's rows, own parts)``: from then on all calls
    are cut so; at the end every call must have reached the library with a cut that was asked for."""

    asked, launched = [], []

    def ask(tile, shared=1, own_tiles=1, own=1):
        asked.append((tile, shared, own_tiles, own))
        monkeypatch.setattr(ops, "shared_prefix_launch", lambda *sizes: (tile, shared, own_tiles, own))

    library_call = ops.call

    def call(name, *arguments):
        if name == "ms_attention_shared_prefix":
            launched.append(tuple(arguments[20:24]))
        return library_call(name, *arguments)

    monkeypatch.setattr(ops, "call", call)
    yield ask
    assert launched and set(launched) <= set(asked) and launched[-1] == asked[-1]


def call_attention(ops, case, **bounds):  # noqa: F811
    return ops.attention_shared_prefix(*(case[name] for name in TENSORS), **{k: v for k, v in case.items() if k not in TENSORS}, **bounds)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
def test_rows_around_the_tile_in_all_head_sizes(ops, cut, tile, dim):  # noqa: F811
    # one kv head, as many query heads: rows = sequences times heads
    for index, rows in enumerate((1, 15, tile - 1, tile, tile + 1, 2 * tile + 5)):
        heads = next(h for h in (4, 3, 5, 1) if rows % h == 0)
        page = (16, 32, 48)[(index + dim // 16) % 3]
        members = [(1, 1 + i % 5) for i in range(rows // heads)]
        for shared, parts in ((1, 1), (31, 1), (13 * page + 1, 2), (700, 1), (1024, 4)):
            cut(tile, parts)
            check_attention(ops, attention_case(torch.bfloat16, heads, 1, dim, page, [(shared, members)], seed=rows + shared))


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("shared", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 511, 513, 800])
def test_shared_lengths_around_pairs_rounds_and_parts(ops, cut, tile, shared):  # noqa: F811
    members = [(1, 1 + 7 * i % 40) for i in range(9)]
    for parts in (1, 2, 3):
        cut(tile, parts, 1, parts)
        check_attention(ops, attention_case(torch.bfloat16, 16, 2, 64, 32, [(shared, members)], seed=shared + parts))
    cut(tile, 2)
    check_attention(ops, attention_case(torch.bfloat16, 16, 2, 128, 64, [(shared, members)], seed=shared))


@pytest.mark.parametrize("tile", TILES)
def test_groups_of_all_sizes_and_empty_ones(ops, cut, tile):  # noqa: F811
    rng = random.Random(tile)
    cut(tile, 3, 2, 2)
    groups = [(rng.randint(0, 30) * 16, [(rng.randint(1, 3), rng.randint(3, 90)) for _ in range(rng.randint(1, 12))]) for _ in range(9)]
    check_attention(ops, attention_case(torch.bfloat16, 16, 2, 48, 16, groups, seed=3))
    # a group without sequences, one that shares nothing, sequences that bring nothing, some in no group, a token
    # whose context is empty, and rows before the first sequence and behind the last
    case = attention_case(torch.bfloat16, 24, 2, 80, 16, [(64, [(1, 4), (0, 9), (2, 30)]), (32, []), (0, [(1, 50), (1, 1)]), (48, [(0, 1)]),
                                                          (333, [(3, 5)] * 7)],
                          alone=[(1, 1), (3, 200), (0, 0), (2, 1)], spare_rows=3, seed=8)
    out = check_attention(ops, case)
    assert not bool(out[-3:].any()) and not bool(out[-5].any()) and bool(out[-4].any())
    later = {**case, "q": torch.cat([case["q"][:2], case["q"]]), "query_start": case["query_start"] + 2}
    moved = call_attention(ops, later)
    assert not bool(moved[:2].any()) and torch.equal(moved[2:], out)
    # more groups than a wave has lanes
    cut(tile, 2)
    check_attention(ops, attention_case(torch.bfloat16, 4, 2, 32, 16, [(16 * (1 + g % 3), [(1, 1 + g % 7)] * (1 + g % 2)) for g in range(131)], seed=4))


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("tokens", [2, 5, 9, 70])
def test_drafted_tokens(ops, cut, tile, tokens):  # noqa: F811
    members = [(tokens, tokens), (tokens, tokens + 30), (1, 9), (tokens, tokens + 1)]
    for own_tiles, own in ((1, 1), (3, 2)):
        cut(tile, 2, own_tiles, own)
        check_attention(ops, attention_case(torch.bfloat16, 8, 2, 96, 16, [(96, members), (304, members)], seed=tokens))


@pytest.mark.parametrize("tile", TILES)
def test_scores_far_from_zero_and_rows_that_rise_along_the_keys(ops, cut, tile):  # noqa: F811
    cut(tile, 2)
    for scale in (30.0, 300.0):
        check_attention(ops, attention_case(torch.bfloat16, 32, 2, 64, 16, [(400, [(1, 30), (4, 9), (1, 2)])], sharp=scale, seed=int(scale)))
    # keys grow along the sequence, so that the running maximum moves again and again
    case = attention_case(torch.bfloat16, 32, 2, 64, 16, [(640, [(1, 30), (2, 9), (1, 2)])], sharp=8.0, seed=1)
    for row, context in enumerate(case["context_lens"].tolist()):
        for entry in range(640 // 16 if row == 0 else 0):
            case["key_pool"][case["block_table"][row, entry].long()] *= 0.1 + entry / 20
    check_attention(ops, case)


@pytest.mark.parametrize("tile", TILES)
def test_a_poisoned_group_leaves_the_others_alone(ops, cut, tile):  # noqa: F811
    cut(tile, 2)
    case = attention_case(torch.bfloat16, 8, 2, 64, 16, [(160, [(1, 20), (1, 40)] * 9), (96, [(1, 3), (2, 9)])], seed=6)
    first = call_attention(ops, case)
    assert torch.equal(first, call_attention(ops, case))
    for row in (18, 19):
        for page in case["block_table"][row].tolist():
            case["key_pool"][page] = float("nan")
    poisoned = call_attention(ops, case)
    assert torch.equal(first[:18], poisoned[:18]) and bool(poisoned[18:].isnan().all())


@pytest.mark.parametrize("tile", TILES)
def test_recorded_calls_serve_other_groups(ops, cut, tile):  # noqa: F811
    cut(tile, 3, 1, 2)
    cases = [attention_case(torch.bfloat16, 16, 2, 128, 16, groups, seed=seed) for seed, groups in enumerate((
        [(64, [(1, 20)] * 9), (496, [(1, 3), (2, 9), (1, 1)])],
        [(640, [(1, 2), (2, 50)] + [(1, 8)] * 9), (16, [(1, 100)])],
        [(0, [(2, 200)]), (320, [(1, 1 + i) for i in range(11)])],
    ))]
    pages, width = max(c["key_pool"].shape[0] for c in cases), max(c["block_table"].shape[1] for c in cases)
    static = {
        "q": torch.empty_like(cases[0]["q"]),
        "key_pool": torch.empty(pages, *cases[0]["key_pool"].shape[1:], dtype=torch.bfloat16, device=DEVICE),
        "value_pool": torch.empty(pages, *cases[0]["value_pool"].shape[1:], dtype=torch.bfloat16, device=DEVICE),
        "block_table": torch.zeros(12, width, dtype=torch.int32, device=DEVICE),
        **{k: torch.empty_like(cases[0][k]) for k in ("query_start", "context_lens", "group_start", "shared_lens")},
        "scale": cases[0]["scale"],
    }

    def fill(case):
        for name, tensor in static.items():
            if name == "block_table":
                tensor.zero_()
                tensor[:, : case[name].shape[1]] = case[name]
            elif name != "scale":
                tensor[: case[name].shape[0]].copy_(case[name])

    fill(cases[0])
    call_attention(ops, static)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = call_attention(ops, static)
    for _ in range(2):
        for case in cases:
            fill(case)
            graph.replay()
            check_attention(ops, case, out=out)
            assert torch.equal(out, call_attention(ops, static))


@pytest.mark.parametrize("tile,dtype", [(16, torch.float32), *((tile, torch.bfloat16) for tile in TILES)])
def test_more_parts_than_a_wave_has_lanes(ops, cut, tile, dtype):  # noqa: F811
    # 64 parts of the shared keys and 64 of a sequence's own, all of them with keys, and the same with most of them empty
    keys = 128 if tile <= 32 else 256
    cut(tile, 64, 1, 64)
    check_attention(ops, attention_case(dtype, 4, 1, 32, 64, [(63 * keys + 17, [(1, 63 * 128 + 5), (1, 3)])], seed=tile))
    check_attention(ops, attention_case(dtype, 4, 1, 128, 64, [(200, [(1, 300), (1, 3)]), (16, [(1, 2)])], seed=tile))
    cut(tile, 40, 1, 30)
    check_attention(ops, attention_case(dtype, 4, 1, 48, 64, [(39 * keys + 1, [(1, 29 * 128 + 5), (2, 40 * 128)])], seed=tile))


@pytest.mark.parametrize("tile", TILES)
def test_pages_far_into_a_pool(ops, cut, tile):  # noqa: F811
    # offsets of elements past 2**31 and of bytes past 2**32
    cut(tile, 2)
    page, dim, kv_heads = 16, 128, 8
    pages = 2**31 // (kv_heads * page * dim) + 60
    small = attention_case(torch.bfloat16, 64, kv_heads, dim, page, [(240, [(1, 20), (1, 40)] * 9)], seed=10)
    count = small["key_pool"].shape[0]
    pages += count
    keys = torch.empty(pages, kv_heads, page, dim, dtype=torch.bfloat16, device=DEVICE)
    values = torch.empty(pages, kv_heads, dim, page, dtype=torch.bfloat16, device=DEVICE)
    keys[pages - count :] = small["key_pool"]
    values[pages - count :] = small["value_pool"]
    near = call_attention(ops, small)
    far = {**small, "key_pool": keys, "value_pool": values, "block_table": small["block_table"] + (pages - count)}
    assert torch.equal(near, call_attention(ops, far))
