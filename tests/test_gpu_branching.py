"""Requests that branch, on the GPU: a fork, branches over their shared pages in eager and
recorded steps, drafted tokens, cuts and moves, against the plain implementation; and
generation with drafted tokens against generation one token at a time."""

from __future__ import annotations

import branching_run
import pytest
import torch
from helpers import random_tokens, read_config, read_weights

pytestmark = pytest.mark.gpu


def make_runner(folder, block_size, dtype, recorded):
    from miniserve_amd.config import EngineConfig
    from miniserve_amd.engine import ModelRunner

    runner = ModelRunner.from_folder(folder, EngineConfig(
        dtype=dtype, kv_block_size=block_size, num_kv_blocks=60, max_num_seqs=8, enable_chunked_prefill=True, decode_graphs=recorded))
    for pool in runner.cache.page_pools():
        pool.fill_(float("nan"))
    return runner


@pytest.mark.parametrize("recorded", [False, True], ids=["eager", "recorded"])
@pytest.mark.parametrize("name,dtype", [("a", "float32"), ("a", "bfloat16"), ("b", "bfloat16"), ("c", "float32"), ("c", "bfloat16")])
def test_branches_follow_the_plain_implementation(name, dtype, recorded, model_folders, monkeypatch):
    from miniserve_amd import ops
    from miniserve_amd.engine import batch

    monkeypatch.setattr(batch, "SHARED_FRONT_KEYS", 256)       # the plain implementation takes its time over longer prompts
    folder, block_size = model_folders[name]
    config = read_config(folder)
    before = dict(ops.attention_calls)
    runner = make_runner(folder, block_size, dtype, recorded)
    branches = branching_run.run(runner, config["vocab_size"], prompt=298)
    worst, allowed = branches.worst(read_weights(folder), config, dtype)
    assert worst <= allowed, f"{worst:.3e} > {allowed:.3e}"
    assert (ops.attention_calls["shared"] > before["shared"]) == (dtype == "bfloat16" and name != "b")
    if recorded:
        assert runner.graph_steps > 8 and any(len(key) == 3 for key in runner._decode_graphs) == (dtype == "bfloat16")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_engine_against_itself_drafted_tokens_change_no_greedy_token(dtype, model_folders):
    """Greedy generation in which every step brings three drafted tokens (right ones, wrong
    ones, and none) gives the tokens of generation one by one: in 32-bit the logits of a
    position do not hang on the cut of the work, so the tokens are the same; in bfloat16 each
    token is the best of its own step's row."""

    from miniserve_amd.engine import SamplingParams, StepEntry
    from miniserve_amd.sampling import Sampler

    folder, block_size = model_folders["a"]
    config = read_config(folder)
    runner = make_runner(folder, block_size, dtype, recorded=False)
    prompt, wanted = random_tokens(50, config["vocab_size"], 77), 40
    runner.admit("one")
    logits = runner.step([StepEntry("one", tuple(prompt), (len(prompt) - 1,))])
    one = [int(logits[0].argmax())]
    while len(one) < wanted + 8:
        one.append(int(runner.step([StepEntry("one", (one[-1],), (0,))])[0].argmax()))
    sampler, params = Sampler(), SamplingParams()
    runner.admit("many")
    logits = runner.step([StepEntry("many", tuple(prompt), (len(prompt) - 1,))])
    many, steps, taken = [int(logits[0].argmax())], 0, 0
    while len(many) < wanted:
        ahead = list(one[len(many) : len(many) + 3])
        if steps % 3 == 1:
            ahead[1] = (ahead[1] + 1) % config["vocab_size"]
        if steps % 5 == 4:
            ahead = []
        held = runner.cache.committed_tokens("many")
        logits = runner.step([StepEntry("many", (many[-1], *ahead), tuple(range(len(ahead) + 1)))])
        staged = sampler.stage_drafts(logits, [("many", params, ahead)])[0]
        best = logits.argmax(-1).tolist()
        assert staged.token_ids == tuple(best[: staged.accepted + 1]) and list(staged.token_ids[:-1]) == ahead[: staged.accepted]
        assert staged.accepted == len(ahead) or ahead[staged.accepted] != best[staged.accepted]
        runner.truncate("many", held + 1 + staged.accepted)
        many += staged.token_ids
        steps, taken = steps + 1, taken + staged.accepted
        runner.cache.assert_invariants()
    if dtype == "float32":
        assert many[:wanted] == one[:wanted] and taken > wanted // 2


def test_sampled_drafts_on_the_device_take_the_plain_choice(model_folders):
    """``Sampler.stage_drafts`` on the device against the same with the plain check in the kernel's place."""

    import plain_branching as plain
    from miniserve_amd import ops
    from miniserve_amd.engine import SamplingParams
    from miniserve_amd.sampling import Sampler

    gen = torch.Generator().manual_seed(5)
    logits = 2.5 * torch.randn(11, 3001, generator=gen)
    probs = torch.softmax(logits[[0, 1, 2, 4, 5, 6, 7, 9]] + 0.3 * torch.randn(8, 3001, generator=gen), -1)
    drafts = torch.multinomial(probs, 1, generator=gen)[:, 0].tolist()
    requests = [("a", SamplingParams(temperature=1.0, seed=1), drafts[:3]), ("b", SamplingParams(temperature=0.8, seed=2), drafts[3:7]),
                ("c", SamplingParams(), drafts[7:])]
    got = Sampler().stage_drafts(logits.cuda(), requests, probs.cuda())
    kernel = ops.verify_drafts
    try:
        def instead(rows, start, tokens, **rest):
            host = {k: v.cpu() for k, v in rest.items()}
            out = plain.verify(rows.cpu(), start.cpu(), tokens.cpu(), host["draft_probs"], host["accept_uniform"], host["draw_uniform"], host["temperature"])
            return torch.tensor(out[0], dtype=torch.int32), torch.tensor(out[1], dtype=torch.int32)

        ops.verify_drafts = instead
        want = Sampler().stage_drafts(logits.cuda(), requests, probs.cuda())
    finally:
        ops.verify_drafts = kernel
    assert [(s.token_ids, s.accepted) for s in got] == [(s.token_ids, s.accepted) for s in want]


def test_branches_in_steps_that_are_launched_ahead(model_folders, monkeypatch):
    """Four branches decode in recorded steps whose numbers are prepared, and which are launched,
    before the host has read the tokens of the step before; one such step is thrown away, and
    a branch is cut and another forked between them.  Greedy tokens, every row of logits
    against the plain implementation."""

    from miniserve_amd import ops
    from miniserve_amd.engine import StepEntry, batch

    monkeypatch.setattr(batch, "SHARED_FRONT_KEYS", 256)
    folder, block_size = model_folders["a"]
    config, weights = read_config(folder), read_weights(folder)
    runner = make_runner(folder, block_size, "bfloat16", recorded=True)
    branches = branching_run.Branches(runner, config["vocab_size"], seed=77)
    branches.admit("p")
    branches.step(p=290)
    branches.fork("p", "a", "b", "c")
    names = ["p", "a", "b", "c"]

    def keep(logits):
        for name, row in zip(names, logits.float().cpu()):
            branches.rows.append((list(branches.tokens[name]), row))
        return ops.sample_rows(logits.float().contiguous())

    def eager_tokens():
        tokens = {}
        for i, name in enumerate(names):
            tokens[name] = (17 * i + len(branches.tokens[name])) % config["vocab_size"]
            branches.tokens[name].append(tokens[name])
        return [StepEntry(name, (tokens[name],), (0,)) for name in names]

    chained = 0
    for part in range(3):
        tokens = keep(runner.step(eager_tokens()))
        for turn in range(4):
            prepared = runner.prepare_decode(names)
            assert prepared is not None
            runner.launch_chained(prepared, tokens)
            chosen = tokens.tolist()
            if turn == 3:
                runner.discard(prepared)
                break
            for name, token in zip(names, chosen):
                branches.tokens[name].append(token)
            tokens = keep(runner.step([StepEntry(name, (token,), (0,)) for name, token in zip(names, chosen)], prepared))
            chained += 1
        runner.cache.assert_invariants()
        if part == 0:
            branches.truncate("b", len(branches.tokens["b"]) - 2)
        if part == 1:
            branches.release("c")
            branches.fork("a", "d", "e")
            names = ["p", "b", "a", "d", "e"]    # two runs now
    keys = [key for key in runner._decode_graphs if len(key) == 3]
    assert runner.chained_steps == chained + 3 and keys and {key[2][0] for key in keys} == {1, 2}
    worst, allowed = branches.worst(weights, config, "bfloat16")
    assert worst <= allowed, f"{worst:.3e} > {allowed:.3e}"
