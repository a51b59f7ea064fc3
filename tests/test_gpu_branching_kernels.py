"""The kernels for requests that branch, each alone against a plain implementation in 64
bits: attention over a shared prefix, copies of pages, the check of drafted tokens."""

from __future__ import annotations

import random

import plain_branching as plain
import pytest
import torch

pytestmark = pytest.mark.gpu

DEVICE = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from miniserve_amd import ops as module

    module.load()
    assert module.library_path().endswith("libminiserve_hip.so")
    return module


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


# ---- attention over a shared prefix ------------------------------------------------------

@pytest.fixture(params=["parts", "whole"])
def form(ops, request, monkeypatch):
    """Keys cut into parts that a second kernel joins, or a workgroup a sequence (where that is
    allowed at all): the rule decides by the keys' bytes, here every test runs both."""

    monkeypatch.setattr(ops, "WHOLE_BYTES", 0 if request.param == "parts" else 10**15)
    ops.shared_prefix_launch.cache_clear()
    yield request.param
    ops.shared_prefix_launch.cache_clear()


def attention_case(dtype, heads, kv_heads, dim, page, groups, *, alone=(), seed=0, spare_rows=0, sharp=2.5):
    """``groups``: per group (shared keys, [(tokens, keys behind the shared ones), ...]);
    ``alone``: (tokens, context) of sequences behind the last group.  What no sequence holds
    of the pools is NaN, and the tables name a page of NaN behind every sequence's last."""

    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    tables, brings, contexts, starts, shared = [], [], [], [0], []
    pages = [1]      # page 0 is nobody's

    def take(count):
        pages[0] += count
        return list(range(pages[0] - count, pages[0]))

    same = []        # (page of the group's first sequence, page of another, entries that are alike)
    for length, members in groups:
        whole, rest = divmod(length, page)
        front, edges = take(whole), []
        for tokens, behind in members:
            own = take(-(-(rest + behind) // page))
            if rest and own:
                edges.append(own[0])
            tables.append(front + own)
            brings.append(tokens)
            contexts.append(length + behind)
        same += [(edges[0], other, rest) for other in edges[1:]]
        starts.append(starts[-1] + len(members))
        shared.append(length)
    for tokens, context in alone:
        tables.append(take(-(-max(context, 0) // page)))
        brings.append(tokens)
        contexts.append(context)
    order = list(range(1, pages[0]))
    rng.shuffle(order)
    name = [0, *order]
    width = max(len(t) for t in tables) + 1
    table = torch.tensor([[name[p] for p in t] + [0] * (width - len(t)) for t in tables], dtype=torch.int32)
    keys = torch.randn(pages[0], kv_heads, page, dim, generator=gen)
    values = torch.randn(pages[0], kv_heads, dim, page, generator=gen)
    for a, b, count in same:
        keys[name[b], :, :count] = keys[name[a], :, :count]
        values[name[b], :, :, :count] = values[name[a], :, :, :count]
    used = torch.zeros(pages[0], page, dtype=torch.bool)
    for t, context in zip(tables, contexts):
        for position in range(max(context, 0)):
            used[name[t[position // page]], position % page] = True
    keys.permute(0, 2, 1, 3)[~used] = float("nan")
    values.permute(0, 3, 1, 2)[~used] = float("nan")
    query_start = [0]
    for t in brings:
        query_start.append(query_start[-1] + t)
    q = torch.randn(query_start[-1] + spare_rows, heads, dim, generator=gen) * sharp
    return {
        "q": q.to(dtype).to(DEVICE), "key_pool": keys.to(dtype).to(DEVICE), "value_pool": values.to(dtype).to(DEVICE),
        "block_table": table.to(DEVICE), "query_start": ints(query_start), "context_lens": ints(contexts),
        "group_start": ints(starts), "shared_lens": ints(shared), "scale": dim**-0.5,
    }


def check_attention(ops, case, out=None, **bounds):
    if out is None:
        out = ops.attention_shared_prefix(case["q"], case["key_pool"], case["value_pool"],
                                          **{k: v for k, v in case.items() if k not in ("q", "key_pool", "value_pool")}, **bounds)
    expected, spread, score = plain.attention_rows(case["q"], case["key_pool"], case["value_pool"], case["block_table"],
                                                   case["query_start"], case["context_lens"], case["scale"])
    bound = plain.attention_bound(expected, spread, score, case["q"].dtype, case["q"].shape[2], int(case["context_lens"].max()))
    error = (out.double().cpu() - expected).abs()
    assert out.dtype == case["q"].dtype and bool(torch.isfinite(out).all())
    worst = float((error / bound).max())
    assert worst <= 1, f"off by {worst:.2f} times what rounding allows"
    return out


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads", [(16, 8), (32, 8), (8, 1), (3, 3), (12, 4), (24, 1)])
def test_one_group_of_single_tokens(ops, dtype, heads, kv_heads):
    check_attention(ops, attention_case(dtype, heads, kv_heads, 64, 16, [(160, [(1, 1), (1, 16), (1, 17), (1, 40), (1, 3)])]))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("page", [16, 32, 48])
def test_head_sizes_and_pages(ops, dtype, dim, page):
    check_attention(ops, attention_case(dtype, 8, 2, dim, page, [(2 * page, [(1, 5), (1, 33)]), (page, [(1, 1), (2, 2), (1, 70)])]))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shared", [1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 500])
def test_shared_lengths_inside_pages_and_tiles(ops, dtype, shared):
    # a shared part that ends inside a page: the rows' own tables name a copy of that page, which goes on differently
    check_attention(ops, attention_case(dtype, 8, 4, 64, 32, [(shared, [(1, 1), (1, 20), (1, 64)])], seed=shared))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_groups_of_all_sizes(ops, dtype):
    rng = random.Random(5)
    groups = [(rng.randint(0, 20) * 16, [(rng.randint(1, 3), rng.randint(3, 90)) for _ in range(rng.randint(1, 5))]) for _ in range(9)]
    check_attention(ops, attention_case(dtype, 8, 2, 32, 16, groups, seed=3))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("rows", [16, 17, 33, 64, 65, 100, 128, 129, 200, 300])
@pytest.mark.parametrize("dim,page", [(64, 16), (80, 48), (128, 16), (112, 32), (32, 64)])
def test_rows_of_a_group_around_every_tile(ops, rows, dim, page):
    # one kv head, as many query heads: rows = sequences times heads
    heads = next(h for h in (4, 3, 5, 1) if rows % h == 0)
    members = [(1, 1 + i % 5) for i in range(rows // heads)]
    for shared in (page, 13 * page + 1, 700):
        check_attention(ops, attention_case(torch.bfloat16, heads, 1, dim, page, [(shared, members)], seed=rows + shared))


@pytest.mark.usefixtures("form")
def test_more_groups_than_a_wave_has_lanes(ops):
    groups = [(16 * (1 + g % 3), [(1, 1 + g % 7)] * (1 + g % 2)) for g in range(131)]
    check_attention(ops, attention_case(torch.bfloat16, 4, 2, 32, 16, groups, seed=4))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [2, 5, 8, 33, 70])
def test_drafted_tokens_see_each_other_causally(ops, dtype, tokens):
    members = [(tokens, tokens), (tokens, tokens + 30), (1, 9), (tokens, tokens + 1)]
    check_attention(ops, attention_case(dtype, 8, 4, 64, 16, [(96, members)], seed=tokens))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_groups_sequences_and_rows(ops, dtype):
    # a group without sequences, one that shares nothing, sequences that bring nothing, some in no group, a token whose
    # context is empty, and rows behind the last sequence
    case = attention_case(dtype, 8, 4, 48, 16, [(64, [(1, 4), (0, 9), (2, 30)]), (32, []), (0, [(1, 50), (1, 1)]), (48, [(0, 1)])],
                          alone=[(1, 1), (3, 200), (0, 0), (2, 1)], spare_rows=3, seed=8)
    out = check_attention(ops, case)
    assert not bool(out[-3:].any()) and not bool(out[-5].any()), "rows without keys are zero"
    assert bool(out[-4].any())


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_beyond_a_table_count_as_its_keys_and_rows_before_the_first_sequence_are_zero(ops, dtype):
    case = attention_case(dtype, 8, 4, 64, 16, [(64, [(1, 16), (1, 16)])], alone=[(1, 80)])
    case["block_table"] = case["block_table"][:, :5].contiguous()
    check_attention(ops, case)
    far = {**case, "context_lens": ints([10**6, 2**31 - 1, 81])}
    again = ops.attention_shared_prefix(**far, max_own=16)
    # (bounds only move rounding, and here they cut the work alike)
    assert torch.equal(again, ops.attention_shared_prefix(**case, max_own=16))
    same = case["block_table"].clone()
    same[1] = same[0]
    check_attention(ops, {**case, "block_table": same, "shared_lens": ints([2**31 - 1])})
    later = {**case, "q": torch.cat([case["q"][:2], case["q"]]), "query_start": case["query_start"] + 2}
    moved = ops.attention_shared_prefix(**later)
    assert not bool(moved[:2].any()) and torch.equal(moved[2:], ops.attention_shared_prefix(**case))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_parts_are_split_and_joined(ops, dtype):
    check_attention(ops, attention_case(dtype, 4, 1, 64, 64, [(3000, [(1, 2100), (1, 1)])], seed=2))
    check_attention(ops, attention_case(dtype, 8, 2, 32, 16, [(1600, [(1, 1 + i) for i in range(40)])], seed=2))


@pytest.mark.usefixtures("form")
def test_bounds_that_are_too_small_or_missing_change_nothing_but_speed(ops):
    case = attention_case(torch.bfloat16, 8, 2, 64, 16, [(320, [(9, 40), (20, 333), (1, 1)]), (16, [(3, 80)])], seed=1)
    check_attention(ops, case)
    check_attention(ops, case, max_sharing=0, max_shared=1, max_own=1, max_query=1)
    check_attention(ops, case, max_sharing=10**6, max_shared=10**6, max_own=10**6, max_query=10**6)
    check_attention(ops, case, max_shared=320, max_own=333, max_query=20)


@pytest.mark.usefixtures("form")
def test_scores_far_from_zero(ops):
    # sharp rows (one key carries everything) and scores of some hundreds: no overflow, no empty sum
    for scale in (30.0, 300.0):
        for dtype in DTYPES:
            check_attention(ops, attention_case(dtype, 8, 2, 64, 16, [(200, [(1, 30), (4, 9)])], sharp=scale, seed=int(scale)))


@pytest.mark.usefixtures("form")
def test_a_row_depends_only_on_its_sequence(ops):
    """Two calls on the same inputs give the same bits, and a poisoned group (NaN in all its
    keys) leaves the others alone."""

    case = attention_case(torch.bfloat16, 8, 2, 64, 16, [(160, [(1, 20), (1, 40)]), (96, [(1, 3), (2, 9)])], seed=6)
    call = lambda: ops.attention_shared_prefix(case["q"], case["key_pool"], case["value_pool"], **{  # noqa: E731
        k: v for k, v in case.items() if k not in ("q", "key_pool", "value_pool")})
    first = call()
    assert torch.equal(first, call())
    for row in (2, 3):
        for page in case["block_table"][row].tolist():
            case["key_pool"][page] = float("nan")
    poisoned = call()
    assert torch.equal(first[:2], poisoned[:2]) and bool(poisoned[2:].isnan().all())


@pytest.mark.usefixtures("form")
def test_recorded_call_serves_other_lengths_and_groups(ops):
    """A recorded call replayed with other groups, lengths and queries in the same tensors,
    another recorded call and eager ones in between."""

    cases = [
        attention_case(torch.bfloat16, 8, 2, 64, 16, [(64, [(1, 20), (1, 40)]), (96, [(1, 3), (2, 9)])], seed=6),
        attention_case(torch.bfloat16, 8, 2, 64, 16, [(160, [(1, 2), (2, 50), (1, 8)]), (16, [(1, 100)])], seed=7),
        attention_case(torch.bfloat16, 8, 2, 64, 16, [(0, [(2, 200)]), (112, [(1, 3), (1, 9), (1, 1)])], seed=8),
    ]
    pages, width = max(c["key_pool"].shape[0] for c in cases), max(c["block_table"].shape[1] for c in cases)
    static = {
        "q": torch.empty_like(cases[0]["q"]),
        "key_pool": torch.empty(pages, *cases[0]["key_pool"].shape[1:], dtype=torch.bfloat16, device=DEVICE),
        "value_pool": torch.empty(pages, *cases[0]["value_pool"].shape[1:], dtype=torch.bfloat16, device=DEVICE),
        "block_table": torch.zeros(4, width, dtype=torch.int32, device=DEVICE),
        **{k: torch.empty_like(cases[0][k]) for k in ("query_start", "context_lens", "group_start", "shared_lens")},
    }

    def fill(case):
        for name, tensor in static.items():
            if name == "block_table":
                tensor.zero_()
                tensor[:, : case[name].shape[1]] = case[name]
            else:
                tensor[: case[name].shape[0]].copy_(case[name])

    names = ("block_table", "query_start", "context_lens", "group_start", "shared_lens")
    call = lambda **bounds: ops.attention_shared_prefix(static["q"], static["key_pool"], static["value_pool"],  # noqa: E731
                                                        scale=cases[0]["scale"], **{k: static[k] for k in names}, **bounds)
    fill(cases[0])
    call()
    graphs = []
    for bounds in ({"max_shared": 160, "max_own": 200, "max_query": 2}, {}):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = call(**bounds)
        graphs.append((graph, out))
    for turn in range(2):
        for case in cases:
            fill(case)
            for graph, out in graphs:
                graph.replay()
                check_attention(ops, case, out=out)
            check_attention(ops, case, out=call())


@pytest.mark.usefixtures("form")
def test_on_another_stream(ops):
    case = attention_case(torch.bfloat16, 8, 2, 64, 16, [(160, [(1, 20), (1, 40)])], seed=9)
    names = {k: v for k, v in case.items() if k not in ("q", "key_pool", "value_pool")}
    here = ops.attention_shared_prefix(case["q"], case["key_pool"], case["value_pool"], **names)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        there = ops.attention_shared_prefix(case["q"], case["key_pool"], case["value_pool"], **names)
    stream.synchronize()
    assert torch.equal(here, there)


@pytest.mark.usefixtures("form")
def test_pages_far_into_a_pool(ops):
    # offsets of elements past 2**31 and of bytes past 2**32
    page, dim, kv_heads = 16, 128, 8
    pages = 2**31 // (kv_heads * page * dim) + 40
    small = attention_case(torch.bfloat16, 16, kv_heads, dim, page, [(64, [(1, 20), (1, 40)])], seed=10)
    count = small["key_pool"].shape[0]
    keys = torch.empty(pages, kv_heads, page, dim, dtype=torch.bfloat16, device=DEVICE)
    values = torch.empty(pages, kv_heads, dim, page, dtype=torch.bfloat16, device=DEVICE)
    keys[pages - count :] = small["key_pool"]
    values[pages - count :] = small["value_pool"]
    names = {k: v for k, v in small.items() if k not in ("q", "key_pool", "value_pool")}
    near = ops.attention_shared_prefix(small["q"], small["key_pool"], small["value_pool"], **names)
    names["block_table"] = small["block_table"] + (pages - count)
    assert torch.equal(near, ops.attention_shared_prefix(small["q"], keys, values, **names))


# ---- copies of pages ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8])
@pytest.mark.parametrize("shape", [(1, 9, 1), (3, 40, 2, 16, 64), (28, 30, 8, 16, 128), (2, 33, 3, 5, 7), (5, 2, 1031)])
def test_copy_pages(ops, dtype, shape):
    rng = random.Random(len(shape))
    pools = [(torch.rand(shape, device=DEVICE) * 200).to(dtype), (torch.rand(*shape, 3, device=DEVICE) * 200).to(dtype)]
    ids = rng.sample(range(shape[1]), shape[1])
    half = shape[1] // 2
    destination, source = ids[:half], [rng.choice(ids[half:]) for _ in range(half)]
    expected = [pool.clone() for pool in pools]
    for pool in expected:
        for a, b in zip(source, destination):
            pool[:, b] = pool[:, a]
    ops.copy_pages(pools, source, destination)
    assert all(torch.equal(pool, want) for pool, want in zip(pools, expected))


def test_copy_pages_more_than_one_launch_carries_and_more_pools(ops):
    pools = [torch.rand(2 + p, 2100, 24 + 4 * p, device=DEVICE).bfloat16() for p in range(5)]
    order = random.Random(1).sample(range(2100), 2100)
    destination, source = order[:1050], order[1050:]
    expected = [pool.clone() for pool in pools]
    for pool in expected:
        pool[:, destination] = pool[:, source]
    ops.copy_pages(pools, source, destination)
    assert all(torch.equal(pool, want) for pool, want in zip(pools, expected))


def test_copy_pages_from_views_at_odd_addresses_and_far_into_a_pool(ops):
    # a pool that begins two bytes past a 16-byte border
    flat = torch.rand(1 + 2 * 6 * 33, device=DEVICE).bfloat16()
    pool = flat[1:].view(2, 6, 33)
    want = flat.clone()
    want[1:].view(2, 6, 33)[:, 4] = want[1:].view(2, 6, 33)[:, 1]
    ops.copy_pages([pool], [1], [4])
    assert torch.equal(flat, want)
    # more than 4 GiB into a pool
    big = torch.zeros(2, 40, 64 << 20, dtype=torch.uint8, device=DEVICE)
    big[:, 39] = 7
    ops.copy_pages([big], [39], [38])
    assert bool((big[:, 38] == 7).all()) and not bool(big[:, :38].any())


def test_copy_pages_in_a_recorded_graph_and_on_another_stream(ops):
    pool = torch.rand(3, 8, 64, device=DEVICE)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.copy_pages([pool], [1, 2], [5, 6])
    for turn in range(3):
        pool.copy_(torch.rand(3, 8, 64, device=DEVICE))
        want = pool.clone()
        want[:, [5, 6]] = want[:, [1, 2]]
        graph.replay()
        assert torch.equal(pool, want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.copy_pages([pool], [0], [7])
    stream.synchronize()
    assert torch.equal(pool[:, 7], pool[:, 0])


# ---- drafted tokens ----------------------------------------------------------------------

def draft_case(drafts, vocab, *, temperature=0.8, probs=True, seed=0, agree=0.4):
    gen = torch.Generator().manual_seed(seed)
    starts = [0]
    for n in drafts:
        starts.append(starts[-1] + n + 1)
    logits = 3 * torch.randn(starts[-1], vocab, generator=gen)
    rows = [start + i for start, n in zip(starts, drafts) for i in range(n)]
    guess = logits[rows] + agree * torch.randn(len(rows), vocab, generator=gen)
    if isinstance(temperature, (int, float)):
        temperature = [temperature] * len(drafts)
    heat = torch.tensor([t or 1.0 for t, n in zip(temperature, drafts) for _ in range(n)])
    guess = torch.softmax(guess / heat[:, None], -1) if rows else guess
    cold = torch.tensor([t == 0 for t, n in zip(temperature, drafts) for _ in range(n)], dtype=torch.bool)
    tokens = torch.where(cold, guess.argmax(-1), torch.multinomial(guess, 1, generator=gen)[:, 0]) if rows else torch.zeros(0)
    return {"logits": logits, "row_start": torch.tensor(starts, dtype=torch.int32), "draft_tokens": tokens.int(),
            "draft_probs": guess if probs else None, "accept_uniform": torch.rand(len(rows), generator=gen),
            "draw_uniform": torch.rand(len(drafts), generator=gen), "temperature": torch.tensor(temperature)}


def run_verify(ops, case):
    sent = {k: None if v is None else v.to(DEVICE) for k, v in case.items()}
    return ops.verify_drafts(sent.pop("logits"), sent.pop("row_start"), sent.pop("draft_tokens"), **sent)


def check_verify(ops, case):
    tokens, accepted = run_verify(ops, case)
    want_tokens, want_accepted = plain.verify(**case)
    assert tokens.dtype == accepted.dtype == torch.int32
    assert accepted.tolist() == want_accepted
    assert tokens.tolist() == want_tokens
    return want_accepted


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4093, 4096, 4097, 8191, 32003, 151936])
def test_verify_drafts_vocabularies(ops, vocab, probs):
    drafts = [4, 0, 3, 1, 8] if vocab < 100000 else [3, 0, 2]
    taken = check_verify(ops, draft_case(drafts, vocab, seed=vocab, probs=probs))
    assert vocab > 4 or sum(taken) > 0


@pytest.mark.parametrize("temperature", [0.0, 0.05, 0.6, 1.0, 2.0])
def test_verify_drafts_temperatures(ops, temperature):
    for seed in range(4):
        check_verify(ops, draft_case([2, 5, 0, 1, 7, 3, 3], 5003, temperature=temperature, seed=seed, probs=seed % 2 == 0))


@pytest.mark.parametrize("requests,vocab", [(1100, 130), (400, 9001)])
def test_verify_drafts_of_many_requests(ops, requests, vocab):
    rng = random.Random(vocab)
    drafts = [rng.randint(0, 4) for _ in range(requests)]
    case = draft_case(drafts, vocab, temperature=[rng.choice([0.0, 0.7, 1.0]) for _ in drafts], seed=requests)
    for request in (3, requests - 1):      # these end with -1, at the first row that is reached
        case["logits"][int(case["row_start"][request])] = float("nan")
    taken = check_verify(ops, case)
    assert sum(taken) > requests // 2


def test_verify_drafts_greedy_and_sampled_requests_in_one_call(ops):
    case = draft_case([3, 3, 3, 0, 0, 6], 7001, temperature=[0.0, 0.7, 0.0, 0.0, 1.0, 0.0], agree=0.05, seed=2)
    taken = check_verify(ops, case)
    assert max(taken[0], taken[2], taken[5]) > 0
    # all greedy: no uniform numbers, no temperatures; ties go to the lowest index
    case["logits"][4, [17, 900, 6999]] = 50.0
    tokens, accepted = ops.verify_drafts(case["logits"].to(DEVICE), case["row_start"].to(DEVICE), case["draft_tokens"].to(DEVICE))
    want = plain.verify(case["logits"], case["row_start"], case["draft_tokens"], None, None, None, None)
    assert (tokens.tolist(), accepted.tolist()) == want


@pytest.mark.parametrize("vocab,drafts", [(1, [3, 0, 2]), (130, [0, 1] * 300), (5003, [0, 40, 7, 1, 5]), (151936, [2, 4])])
def test_verify_drafts_without_temperatures(ops, vocab, drafts):
    """All requests greedy, said by leaving the temperatures out: as with temperatures of 0."""

    case = draft_case(drafts, vocab, temperature=0.0, agree=0.02, seed=vocab)
    if len(drafts) == 5:
        case["logits"][int(case["row_start"][1]) + 3, 17] = float("inf")
    taken = check_verify(ops, case)
    sent = [case[name].to(DEVICE) for name in ("logits", "row_start", "draft_tokens")]
    tokens, accepted = ops.verify_drafts(*sent)
    assert accepted.tolist() == taken and max(taken) > 0
    assert torch.equal(tokens, run_verify(ops, case)[0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        again = ops.verify_drafts(*sent)
    for _ in range(3):
        again[0].fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again[0], tokens) and torch.equal(again[1], accepted)


def test_verify_drafts_all_taken_none_taken_and_only_next_tokens(ops):
    case = draft_case([4, 4], 999, seed=5)
    case["accept_uniform"][:] = 0.0
    assert check_verify(ops, case) == [4, 4]
    case["accept_uniform"][:] = 1.0 - 2**-24
    case["draft_tokens"][:] = case["logits"].argmin(-1)[0].int()
    case["draft_probs"][:, int(case["draft_tokens"][0])] = 0.9
    assert check_verify(ops, case) == [0, 0]
    check_verify(ops, draft_case([0] * 70, 513, seed=6))           # more requests than a wave has lanes
    check_verify(ops, draft_case([130], 257, seed=6, agree=0.0))   # one request with many drafts


def test_verify_drafts_extreme_uniform_numbers(ops):
    for draw in (0.0, 1.0 - 2**-24):
        for probs in (True, False):
            case = draft_case([2, 0, 3], 4501, seed=3, probs=probs)
            case["draw_uniform"][:] = draw
            check_verify(ops, case)


def test_verify_drafts_draft_that_is_the_target(ops):
    # p == q but for roundings: nearly every draft is taken; a residual of nothing falls back on p
    case = draft_case([6] * 8, 2000, temperature=1.0, agree=0.0, seed=4)
    assert sum(check_verify(ops, case)) >= 47
    # one token has all of the target's mass and of the draft's, which drafted another: the residual is nothing at all
    logits = torch.full((2, 300), -3e38)
    logits[:, 7] = 3e38
    probs = torch.zeros(1, 300)
    probs[0, 7] = 1.0
    case = {"logits": logits, "row_start": torch.tensor([0, 2], dtype=torch.int32), "draft_tokens": torch.tensor([9], dtype=torch.int32),
            "draft_probs": probs, "accept_uniform": torch.tensor([0.5]), "draw_uniform": torch.tensor([0.5]), "temperature": torch.ones(1)}
    assert check_verify(ops, case) == [0]


def test_verify_drafts_rows_that_are_not_finite(ops):
    for value in (float("nan"), float("inf"), float("-inf")):
        for temperature in (0.0, 0.9):
            case = draft_case([3, 3, 3, 0], 6007, temperature=temperature, seed=9, agree=0.0)
            case["accept_uniform"][:] = 0.0
            case["logits"][2, 6000] = value          # after two drafts of the first request
            case["logits"][4, 0] = value             # the first row of the second
            case["logits"][12, 5] = value            # the only row of the last
            tokens, accepted = run_verify(ops, case)
            want = plain.verify(**case)
            assert (tokens.tolist(), accepted.tolist()) == want
            assert accepted.tolist()[1] == 0 and tokens.tolist()[4] == -1 and tokens.tolist()[12] == -1


def test_verify_drafts_ids_outside_the_vocabulary_are_never_taken(ops):
    for probs in (True, False):
        for token in (-1, 1000, 2**31 - 1, -(2**31)):
            for temperature in (0.0, 1.0):
                case = draft_case([2, 2], 1000, temperature=temperature, probs=probs, seed=1, agree=0.0)
                case["accept_uniform"][:] = 0.0
                case["draft_tokens"][1] = token
                assert check_verify(ops, case)[0] <= 1


def test_verify_drafts_follows_the_targets_probabilities(ops):
    """Tokens that come out have the target's probabilities, whatever the draft proposes:
    20,000 requests of one draft over five tokens, counts within five standard deviations."""

    n, gen = 20000, torch.Generator().manual_seed(1)
    row = torch.tensor([0.1, 1.2, -0.4, 0.9, -1.5])
    p = torch.softmax(row.double(), 0)
    q = torch.tensor([0.5, 0.1, 0.1, 0.1, 0.2])
    case = {"logits": row.repeat(2 * n, 1), "row_start": torch.arange(0, 2 * n + 1, 2, dtype=torch.int32),
            "draft_tokens": torch.multinomial(q, n, replacement=True, generator=gen).int(), "draft_probs": q.repeat(n, 1),
            "accept_uniform": torch.rand(n, generator=gen), "draw_uniform": torch.rand(n, generator=gen), "temperature": torch.ones(n)}
    tokens, _ = run_verify(ops, case)
    counts = torch.bincount(tokens[0::2].cpu(), minlength=5).double()
    assert bool(((counts - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()), (counts, n * p)


def test_verify_drafts_recorded(ops):
    cases = [draft_case([3, 1, 2], 9001, seed=s) for s in range(3)]
    static = {k: v.to(DEVICE) for k, v in cases[0].items()}
    call = lambda: ops.verify_drafts(**static)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = call()
    for turn in range(2):
        for case in cases:
            for k, v in case.items():
                static[k].copy_(v)
            graph.replay()
            assert (out[0].tolist(), out[1].tolist()) == plain.verify(**case)
            assert (call()[0].tolist()) == plain.verify(**case)[0]


# ---- refusals ------------------------------------------------------------------------------

def test_refusals_of_the_gpu_side(ops):
    from miniserve_amd.ops import KernelError

    case = attention_case(torch.bfloat16, 8, 2, 64, 16, [(32, [(1, 4), (1, 5)])])
    names = {k: v for k, v in case.items() if k not in ("q", "key_pool", "value_pool")}

    def refused(match, *tensors, **changes):
        q, keys, values = tensors or (case["q"], case["key_pool"], case["value_pool"])
        with pytest.raises(KernelError, match=match):
            ops.attention_shared_prefix(q, keys, values, **{**names, **changes})

    refused("must be torch.bfloat16", case["q"], case["key_pool"].float(), case["value_pool"])
    refused("contiguous", case["q"].transpose(0, 1), case["key_pool"], case["value_pool"])
    refused("float32 or bfloat16", case["q"].half(), case["key_pool"].half(), case["value_pool"].half())
    refused("must have shape", case["q"], case["key_pool"], case["value_pool"].transpose(2, 3).contiguous())
    refused("not a multiple", case["q"][:, :7].contiguous(), case["key_pool"], case["value_pool"])
    refused("query_start must have shape", query_start=names["query_start"][:-1].contiguous())
    refused("context_lens must be torch.int32", context_lens=names["context_lens"].long())
    refused("shared_lens must have shape", shared_lens=ints([32, 32]))
    refused("at least one group", group_start=ints([0]), shared_lens=ints([]))
    refused("whole number", max_shared=-1)
    refused("whole number", max_sharing=True)
    refused("whole number", max_query=1.5)
    odd = attention_case(torch.bfloat16, 8, 2, 64, 16, [(32, [(1, 4)])])
    with pytest.raises(KernelError, match="head_dim 8"):
        ops.attention_shared_prefix(odd["q"][..., :8].contiguous(), odd["key_pool"][..., :8].contiguous(),
                                    odd["value_pool"][:, :, :8].contiguous(), **{k: v for k, v in odd.items() if k not in (
                                        "q", "key_pool", "value_pool")})
    with pytest.raises(KernelError, match="block_size 8"):
        ops.attention_shared_prefix(odd["q"], odd["key_pool"][:, :, :8].contiguous(), odd["value_pool"][..., :8].contiguous(),
                                    **{k: v for k, v in odd.items() if k not in ("q", "key_pool", "value_pool")})

    pool = torch.zeros(2, 5, 8, device=DEVICE)
    for match, pools, source, destination in [
        ("list of at least one", pool, [0], [1]), ("outside", [pool], [5], [1]), ("outside", [pool], [-1], [1]), ("outside", [pool], [1], [5]),
        ("outside", [pool, torch.zeros(2, 3, 8, device=DEVICE)], [4], [1]), ("two copies", [pool], [0, 1], [2, 2]),
        ("source of one copy", [pool], [0, 1], [1, 2]), ("source of one copy", [pool], [3], [3]), ("1 pages to 2", [pool], [0], [1, 2]),
        ("whole numbers", [pool], [0.0], [1]), ("whole numbers", [pool], [True], [2]), ("contiguous", [pool[:, :, ::2]], [0], [1]),
        ("calls>0", [torch.zeros(5, device=DEVICE)], [0], [1]), ("same memory", [pool, pool], [0], [1]),
        ("same memory", [pool[1:], pool.view(1, 10, 8)], [0], [1]), ("outside", [pool], [2**40], [1]),
        ("outside", [torch.zeros(1, pages, 4, device=DEVICE) for pages in (5, 5, 5, 5, 3)], [4], [1]),
    ]:
        with pytest.raises(KernelError, match=match):
            ops.copy_pages(pools, source, destination)
    ops.copy_pages([pool], [], [])

    good = {k: v.to(DEVICE) for k, v in draft_case([2, 1], 100).items()}
    for match, changes in [
        ("float32", {"logits": good["logits"].bfloat16()}), ("R>0", {"logits": good["logits"][:0]}),
        ("1 to 5 requests", {"row_start": ints([0])}), ("1 to 5 requests", {"row_start": ints(range(7))}),
        ("draft_tokens must have shape", {"draft_tokens": ints([1, 2])}), ("draft_probs must have shape", {"draft_probs": good["draft_probs"][:2]}),
        ("uniform numbers", {"draw_uniform": None}), ("uniform numbers", {"accept_uniform": None}),
        ("temperature must have shape", {"temperature": torch.ones(3, device=DEVICE)}), ("draw_uniform must be", {"draw_uniform": good["draw_uniform"].double()}),
        ("GPU", {"row_start": good["row_start"].cpu()}),
    ]:
        with pytest.raises(KernelError, match=match):
            ops.verify_drafts(**{**good, **changes})
