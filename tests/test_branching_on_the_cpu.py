"""Requests that branch, without a GPU: the cache manager's forks, cuts and moves; the step
function over the stand-ins for the kernels; drafted tokens through the sampler; and what
the entry points refuse before anything is launched."""

from __future__ import annotations

import random

import branching_run
import plain_branching as plain
import pytest
import torch
import torch_branching_kernels as kernels
from helpers import read_config, read_weights
from test_cache_manager import Need, manager

from miniserve_amd.cache import CacheError, OutOfPagesError, PageAllocator, StepItem
from miniserve_amd.parts import KVCacheNeed, StateNeed


def advance(m, **counts):
    r = m.prepare_step([StepItem(name, m.committed_tokens(name), m.committed_tokens(name) + n) for name, n in counts.items()])
    m.commit_step(r)
    return r


# ---- allocator ---------------------------------------------------------------------------

def test_pages_are_moved_with_their_owners():
    allocator = PageAllocator(6)
    allocator.allocate(5)
    allocator.retain([4])
    allocator.release([0, 1])
    allocator.move({4: 0, 3: 1})
    assert [allocator.refcount(p) for p in range(6)] == [2, 1, 1, 0, 0, 0] and allocator.free_ids() == (3, 4, 5)
    allocator.assert_invariants()
    assert allocator.allocate(1) == [3]
    for moves, error in (({5: 4}, RuntimeError), ({0: 1}, RuntimeError), ({0: 9}, ValueError), ({0: 4, 1: 4}, ValueError), ({9: 4}, IndexError)):
        before = [allocator.refcount(p) for p in range(6)], allocator.free_ids()
        with pytest.raises(error):
            allocator.move(moves)
        assert before == ([allocator.refcount(p) for p in range(6)], allocator.free_ids())


# ---- cache manager -----------------------------------------------------------------------

def test_a_fork_shares_whole_pages_and_copies_the_last():
    m = manager(num_blocks=10)
    m.admit("p")
    advance(m, p=10)
    assert m.fork("p", ["x", "y"]) == [1, 2]
    assert m.block_table("p") == (0, 1, 2) and m.block_table("x") == (0, 1, 3) and m.block_table("y") == (0, 1, 4)
    assert [m.allocators[0].refcount(p) for p in range(5)] == [3, 3, 1, 1, 1]
    assert m.fork_of("p") is m.fork_of("x") is m.fork_of("y") and m.fork_of("p").pages == (2,)
    assert m.capacity().held_blocks == {"p": (1,), "x": (1,), "y": (1,)}      # what each gives back when it goes
    m.assert_invariants()
    r = advance(m, x=1, p=1)
    assert [meta.slot_mappings[0][0] for meta in r.sequences] == [3 * 4 + 2, 2 * 4 + 2]
    m.release("p")
    m.assert_invariants()
    assert m.capacity().free_blocks == (6,)
    m.release("x")
    m.release("y")
    assert m.capacity().free_blocks == (10,) and m.capacity().free_slots == 4


def test_a_fork_at_a_pages_edge_or_of_an_empty_request():
    m = manager()
    m.admit("p")
    m.fork("p", ["e"])
    assert m.fork_of("e") is None and m.block_table("e") == ()
    advance(m, p=8)
    m.fork("p", ["x"])
    assert m.block_table("x") == (0, 1)
    advance(m, p=1, x=1)
    assert m.block_table("p") == (0, 1, 2) and m.block_table("x") == (0, 1, 3)
    m.assert_invariants()
    assert m.fork("p", []) == []


def test_a_fork_that_cannot_be_met_changes_nothing():
    m = manager(num_blocks=4, slots=4)
    m.admit("p")
    advance(m, p=10)
    before = m.capacity()
    with pytest.raises(OutOfPagesError):
        m.fork("p", ["x", "y"])
    with pytest.raises(CacheError, match="NO_FREE_SLOT"):
        m.fork("p", ["w", "x", "y", "z"])
    with pytest.raises(CacheError, match="twice"):
        m.fork("p", ["x", "x"])
    with pytest.raises(CacheError, match="already live"):
        m.fork("p", ["p"])
    with pytest.raises(CacheError, match="not live"):
        m.fork("q", ["x"])
    r = m.prepare_step([StepItem("p", 10, 11)])
    for call in (lambda: m.fork("p", ["x"]), lambda: m.truncate("p", 3)):
        with pytest.raises(CacheError, match="open step"):
            call()
    with pytest.raises(CacheError, match="open"):
        m.compact()
    m.abort_step(r)
    assert m.capacity() == before and m.fork_of("p") is None
    m.assert_invariants()


def test_a_cut_gives_pages_back_and_copies_one_that_others_hold():
    m = manager(num_blocks=10)
    m.admit("p")
    advance(m, p=10)
    m.fork("p", ["x"])
    advance(m, x=7)
    m.truncate("x", 13)
    assert m.committed_tokens("x") == 13 and len(m.block_table("x")) == 4
    m.truncate("x", 12)
    assert len(m.block_table("x")) == 3 and m.fork_of("x") is m.fork_of("p")
    m.truncate("x", 6)          # into the second shared page: a page of its own
    assert m.block_table("x")[0] == 0 and m.block_table("x")[1] not in m.block_table("p") and m.fork_of("x") is None
    m.assert_invariants()
    m.truncate("x", 4)          # at its edge: nothing is written into the shared page
    assert m.block_table("x") == (0,)
    m.truncate("x", 0)
    assert m.block_table("x") == ()
    m.assert_invariants()
    for wrong in (-1, 11, 1.0, None):
        with pytest.raises(CacheError):
            m.truncate("p", wrong)
    with pytest.raises(CacheError, match="not live"):
        m.truncate("q", 0)


def test_pages_that_a_branch_would_give_back_are_those_that_it_holds_alone():
    m = manager(num_blocks=10)
    m.admit("p")
    advance(m, p=10)
    assert m.capacity().held_blocks == {"p": (3,)}
    m.fork("p", ["x", "y"])
    assert m.capacity().held_blocks == {"p": (1,), "x": (1,), "y": (1,)}
    m.truncate("x", 4)          # no longer alike in all that was shared, and still on a page of the others
    assert m.fork_of("x") is None and m.capacity().held_blocks["x"] == (0,)
    m.release("p")
    m.release("y")
    assert m.capacity().held_blocks == {"x": (1,)}
    free = m.capacity().free_blocks
    m.release("x")
    assert m.capacity().free_blocks == (free[0] + 1,)


def test_a_cut_without_a_page_for_the_copy_changes_nothing():
    m = manager(num_blocks=3)
    m.admit("p")
    advance(m, p=8)
    m.fork("p", ["x"])
    advance(m, p=1)
    with pytest.raises(OutOfPagesError):
        m.truncate("x", 5)
    assert m.committed_tokens("x") == 8 and m.block_table("x") == (0, 1)
    m.assert_invariants()
    m.truncate("p", 5)          # its own third page goes first and serves the copy
    assert m.block_table("p") == (0, 2) and m.allocators[0].refcount(1) == 1
    m.assert_invariants()


def test_windows_and_state_limit_cuts():
    needs = [Need(0, KVCacheNeed(1, 16)), Need(1, KVCacheNeed(1, 16, window=6))]
    m = manager(needs, num_blocks=12)
    m.admit("p")
    advance(m, p=20)
    m.fork("p", ["x"])
    assert m.block_table("x", 1)[:3] == (-1, -1, -1)
    m.assert_invariants()
    m.truncate("x", 18)
    with pytest.raises(CacheError, match="window"):
        m.truncate("x", 16)      # position 16 sees keys from 11 on, their page is gone
    advance(m, p=9, x=3)
    m.assert_invariants()
    m.compact()
    m.assert_invariants()
    m.release("p")
    m.release("x")
    assert m.capacity().free_blocks == (12, 12)
    m = manager([Need(0, (KVCacheNeed(1, 16), StateNeed((3,))))])
    m.allocate_storage(torch.float32, "cpu")
    m.admit("p")
    advance(m, p=4)
    m.state_tensors[0][m.state_slot("p")] = torch.tensor([1.0, 2.0, 3.0])
    m.fork("p", ["x"])
    assert m.state_tensors[0][m.state_slot("x")].tolist() == [1.0, 2.0, 3.0]
    with pytest.raises(CacheError, match="state"):
        m.truncate("p", 3)
    m.truncate("p", 4)


@pytest.mark.parametrize("seed", range(6))
def test_random_branches_keep_their_contents(seed, monkeypatch):
    """Random forks, steps, aborted steps, cuts, moves and releases over two groups of
    different pages: what a request reads through its tables is always what it wrote."""

    from miniserve_amd import ops

    monkeypatch.setattr(ops, "copy_pages", kernels.copy_pages)
    rng = random.Random(seed)
    needs = [Need(0, KVCacheNeed(1, 2)), Need(1, KVCacheNeed(1, 2, block_size=3)), Need(2, KVCacheNeed(1, 2))]
    m = manager(needs, block_size=4, num_blocks=40, slots=7, max_len=60)
    m.allocate_storage(torch.float32, "cpu")
    for pool in m.page_pools():
        pool.fill_(float("nan"))
    texts: dict[str, list[int]] = {}
    serial, names, forks, cuts, moved = 0, 0, 0, 0, 0

    def write(r):
        nonlocal serial
        for meta in r.sequences:
            for group, slots in enumerate(meta.slot_mappings):
                size = m.block_sizes[group]
                for i, slot in enumerate(slots):
                    m.pools[group]["key"][:, slot // size, 0, slot % size] = float(serial + i)
                    m.pools[group]["value"][:, slot // size, 0, :, slot % size] = float(serial + i)
            texts.setdefault(meta.request_id, [])
            written = list(range(serial, serial + meta.after - meta.before))
            serial += len(written)
            yield meta.request_id, written

    for _ in range(500):
        live = list(m.live_requests())
        what = rng.choice(["admit", "step", "step", "step", "abort", "fork", "cut", "compact", "release"])
        try:
            if what == "admit" and len(live) < 6:
                names += 1
                m.admit(f"r{names}")
                texts[f"r{names}"] = []
            elif what in ("step", "abort") and live:
                chosen = rng.sample(live, rng.randint(1, len(live)))
                items = [StepItem(n, len(texts[n]), len(texts[n]) + rng.choice([1, 1, 1, 5, 9])) for n in chosen if len(texts[n]) < 50]
                if items:
                    r = m.prepare_step(items)
                    new = list(write(r))
                    if what == "step":
                        m.commit_step(r)
                        for name, written in new:
                            texts[name] += written
                    else:
                        m.abort_step(r)
            elif what == "fork" and live:
                source, children = rng.choice(live), [f"r{names + 1}", f"r{names + 2}"][: rng.randint(1, 2)]
                m.fork(source, children)
                names += len(children)
                for child in children:
                    texts[child] = list(texts[source])
                forks += 1
            elif what == "cut" and live:
                name = rng.choice(live)
                length = rng.randint(max(0, len(texts[name]) - 12), len(texts[name]))
                m.truncate(name, length)
                del texts[name][length:]
                cuts += 1
            elif what == "compact":
                moved += m.compact()
            elif what == "release" and live and rng.random() < 0.5:
                name = rng.choice(live)
                m.release(name)
                del texts[name]
        except (OutOfPagesError, CacheError) as error:
            assert isinstance(error, OutOfPagesError) or "NO_FREE_SLOT" in str(error)
        m.assert_invariants()
        for name, text in texts.items():
            assert m.committed_tokens(name) == len(text)
            for group, size in enumerate(m.block_sizes):
                table = m.block_table(name, group)
                assert len(table) == -(-len(text) // size)
                for pool in (m.pools[group]["key"][:, :, 0, :, 0], m.pools[group]["value"][:, :, 0, 0, :]):
                    if text:
                        got = pool[:, list(table)].flatten(1)[:, : len(text)]
                        assert torch.equal(got, torch.tensor(text).float().expand_as(got)), (what, name)
    assert forks > 10 and cuts > 10 and moved > 10


# ---- the step function over the stand-ins ------------------------------------------------

def make_runner(folder, block_size, dtype, **options):
    from miniserve_amd.config import EngineConfig
    from miniserve_amd.engine import ModelRunner

    config = EngineConfig(dtype=dtype, kv_block_size=block_size, num_kv_blocks=60, max_num_seqs=8, enable_chunked_prefill=True, **options)
    runner = ModelRunner.from_folder(folder, config, device="cpu")
    for pool in runner.cache.page_pools():
        pool.fill_(float("nan"))
    return runner


@pytest.mark.parametrize("recorded", [False, True], ids=["eager", "recorded"])
@pytest.mark.parametrize("name,dtype", [("a", "float32"), ("a", "bfloat16"), ("b", "bfloat16"), ("c", "bfloat16")])
def test_branches_follow_the_plain_implementation(name, dtype, recorded, model_folders, monkeypatch):
    from miniserve_amd.engine import batch

    monkeypatch.setattr(batch, "SHARED_FRONT_KEYS", 256)       # the plain implementation takes its time over longer prompts
    kernels.install(monkeypatch, recordings=recorded)
    folder, block_size = model_folders[name]
    runner = make_runner(folder, block_size, dtype, decode_graphs=recorded)
    config = read_config(folder)
    branches = branching_run.run(runner, config["vocab_size"], prompt=298)
    worst, allowed = branches.worst(read_weights(folder), config, dtype)
    assert worst <= allowed, f"{worst:.3e} > {allowed:.3e}"
    # tiny b has pages of eight keys, which the kernel does not take; 32-bit results must not hang on the batch
    assert (kernels.CALLS["attention_shared_prefix"] > 0) == (dtype == "bfloat16" and name != "b")
    assert kernels.CALLS["copy_pages"] >= 3
    if recorded:
        shared = [key for key in runner._decode_graphs if len(key) == 3]
        assert bool(shared) == (dtype == "bfloat16")


def test_runs_of_neighbours():
    from miniserve_amd.cache import Fork
    from miniserve_amd.engine.batch import Fronts, shared_fronts

    f, g = Fork((40, 3)), Fork((32, 40))
    #                       rows 0 and 1 share 640 keys, 2 to 4 nothing with a neighbour, 5 to 7 share 512
    contexts = [650, 660, 9, 20, 41, 600, 700, 530]
    assert shared_fronts([f, f, None, g, f, g, g, g], contexts, 0, 16) == Fronts([0, 2, 5, 8], [640, 0, 512], 2, 188)
    assert shared_fronts([None, f, f, f, None, g], [5, 641, 642, 643, 9, 7], 0, 16) == Fronts([0, 1, 4], [0, 640], 1, 9)
    assert shared_fronts([f, None, f, g], [641, 1, 641, 513], 0, 16) is None       # nobody next to its like
    assert shared_fronts([f, f, f], [50, 50, 50], 1, 16) is None                   # 48 keys: too few to pay
    assert shared_fronts([f, f], [641, 641], 0, 16) is None                        # less than half is spared
    assert shared_fronts([None, None], [900, 900], 0, 16) is None and shared_fronts([], [], 0, 16) is None
    rng = random.Random(3)
    for _ in range(300):
        forks = [rng.choice([None, f, f, g]) for _ in range(rng.randint(1, 20))]
        contexts = [rng.randint(641, 660) for _ in forks]
        fronts = shared_fronts(forks, contexts, 0, 16)
        if fronts is None:
            continue
        assert fronts.starts[0] == 0 and len(fronts.starts) == len(fronts.lens) + 1 <= 2 * fronts.runs + 1
        assert sum(length > 0 for length in fronts.lens) == fronts.runs and fronts.starts[-1] <= len(forks)
        shares = [0] * len(forks)
        for first, end, length in zip(fronts.starts, fronts.starts[1:], fronts.lens):
            assert end > first and (length == 0 or len({id(fork) for fork in forks[first:end]}) == 1)
            shares[first:end] = [length] * (end - first)
        for row, fork in enumerate(forks):
            like = fork is not None and any(0 <= near < len(forks) and forks[near] is fork for near in (row - 1, row + 1))
            assert shares[row] == (fork.pages[0] * 16 if like else 0)
        assert fronts.behind == max(context - length for context, length in zip(contexts, shares))


# ---- drafted tokens through the sampler ----------------------------------------------------

def test_drafted_tokens_take_numbers_from_the_requests_own_stream(monkeypatch):
    from miniserve_amd import ops
    from miniserve_amd.engine import SamplingParams
    from miniserve_amd.sampling import NonFiniteLogitsError, Sampler

    sent = []

    def verify(logits, row_start, draft_tokens, **rest):
        sent.append({"row_start": row_start.tolist(), "draft_tokens": draft_tokens.tolist(),
                     **{k: None if v is None else v.tolist() for k, v in rest.items() if k != "draft_probs"}})
        return kernels.verify_drafts(logits, row_start, draft_tokens, **rest)

    monkeypatch.setattr(ops, "verify_drafts", verify)
    gen = torch.Generator().manual_seed(2)
    logits = 2 * torch.randn(7, 50, generator=gen)
    best = logits.argmax(-1).tolist()
    sampler = Sampler()
    requests = [("g", SamplingParams(), [best[0], best[1], (best[2] + 1) % 50]), ("s", SamplingParams(temperature=0.7, seed=9), [3]),
                ("n", SamplingParams(temperature=1.1, seed=10), [])]
    staged = sampler.stage_drafts(logits, requests)
    assert sent[0]["row_start"] == [0, 4, 6, 7] and sent[0]["draft_tokens"] == [best[0], best[1], (best[2] + 1) % 50, 3]
    assert sent[0]["temperature"] == pytest.approx([0.0, 0.7, 1.1])
    assert staged[0].accepted == 2 and staged[0].token_ids == (best[0], best[1], best[2]) and staged[0].generator_state is None
    own = torch.Generator().manual_seed(9)
    numbers = [float(torch.rand((), generator=own, dtype=torch.float64)) for _ in range(2)]
    assert sent[0]["accept_uniform"][3] == pytest.approx(numbers[0]) and sent[0]["draw_uniform"][1] == pytest.approx(numbers[1])
    again = sampler.stage_drafts(logits, requests)          # nothing advances before the commit
    assert [s.token_ids for s in staged] == [s.token_ids for s in again]
    sampler.commit(staged)
    sampler.stage_drafts(logits, requests)
    third = float(torch.rand((), generator=own, dtype=torch.float64))
    assert sent[-1]["accept_uniform"][3] == pytest.approx(third)
    # a row that is not finite after two drafts that are taken
    bad = logits.clone()
    bad[2, 7] = float("nan")
    with pytest.raises(NonFiniteLogitsError):
        sampler.stage_drafts(bad, requests)
    bad = logits.clone()
    bad[3, 7] = float("nan")       # behind the draft that is not taken: never reached
    assert sampler.stage_drafts(bad, requests)[0].token_ids == staged[0].token_ids
    for wrong, match in (([("s", SamplingParams(temperature=1.0, top_p=0.9), [1])], "top-p"), ([("s", SamplingParams(temperature=1.0, top_k=4), [1])], "top-k"),
                         ([("s", SamplingParams(), [-1])], "non-negative"), ([("s", SamplingParams(), [logits.shape[1]])], "vocabulary"),
                         ([("s", SamplingParams(), []), ("s", SamplingParams(), [])], "named twice"), ([("s", SamplingParams(), [1, 2])], "rows of logits"), ([], "rows of logits")):
        with pytest.raises(ValueError, match=match):
            sampler.stage_drafts(logits[:2], wrong)


# ---- refusals that need no GPU -------------------------------------------------------------

def test_entry_points_refuse_tensors_that_are_not_on_the_gpu():
    from miniserve_amd import ops

    pool = torch.zeros(4, 2, 16, 16)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="GPU"):
        ops.attention_shared_prefix(torch.zeros(1, 2, 16), pool, pool, block_table=one[None], query_start=torch.zeros(2, dtype=torch.int32),
                                    context_lens=one, group_start=torch.zeros(2, dtype=torch.int32), shared_lens=one, scale=1.0)
    with pytest.raises(ops.KernelError, match="GPU"):
        ops.copy_pages([pool], [0], [1])
    with pytest.raises(ops.KernelError, match="list of at least one"):
        ops.copy_pages([], [0], [1])
    with pytest.raises(ops.KernelError, match="GPU"):
        ops.verify_drafts(torch.zeros(1, 5), torch.zeros(2, dtype=torch.int32), torch.zeros(0, dtype=torch.int32))


def test_the_cut_of_the_work_stays_within_what_the_kernel_takes(monkeypatch):
    from miniserve_amd import ops

    monkeypatch.setattr(ops, "_decode_target", lambda: 512)
    ops.shared_prefix_launch.cache_clear()
    rng, whole = random.Random(0), 0
    for _ in range(2000):
        sequences = rng.choice([1, 2, 7, 64, 500])
        groups = rng.randint(1, sequences)
        kv_heads, per_token, query = rng.choice([1, 2, 8]), rng.choice([1, 2, 3, 8, 24]), rng.choice([1, 2, 9, 70])
        longest = rng.choice([1, 100, 5000, 10**6])
        dtype = rng.choice([torch.float32, torch.bfloat16])
        launch = ops.shared_prefix_launch(sequences * query * per_token, groups, sequences, kv_heads, per_token, longest, longest, query, dtype,
                                          rng.choice([16, 64, 128]))
        tile, shared_splits, own_tiles, own_splits = launch
        if shared_splits == own_splits == 0:       # a workgroup a sequence
            whole += 1
            assert longest <= 100 and tile == 16 and own_tiles >= 1
            continue
        assert tile in ((16, 32, 64, 128) if dtype == torch.bfloat16 else (16,)) and 1 <= shared_splits <= 64 and 1 <= own_splits <= 64 and own_tiles >= 1
    assert 100 < whole < 1900
    ops.shared_prefix_launch.cache_clear()


def test_the_plain_check_of_drafted_tokens_by_hand():
    logits = torch.log(torch.tensor([[0.5, 0.3, 0.2], [0.1, 0.8, 0.1]]))
    probs = torch.tensor([[0.2, 0.7, 0.1]])
    start = torch.tensor([0, 2])
    one = lambda x: torch.tensor([x])  # noqa: E731
    # p(1) = 0.3 < 0.6 * 0.7: not taken; the residual is (0.3, 0, 0.1), its border at 0.75 of its mass
    assert plain.verify(logits, start, one(1), probs, one(0.6), one(0.74), one(1.0)) == ([0, -1], [0])
    assert plain.verify(logits, start, one(1), probs, one(0.6), one(0.76), one(1.0)) == ([2, -1], [0])
    # 0.4 * 0.7 < 0.3: taken, then the second row's own distribution
    assert plain.verify(logits, start, one(1), probs, one(0.4), one(0.05), one(1.0)) == ([1, 0], [1])
    assert plain.verify(logits, start, one(1), None, one(0.31), one(0.7), one(1.0)) == ([0, -1], [0])
    assert plain.verify(logits, start, one(0), None, None, None, None) == ([0, 1], [1])
