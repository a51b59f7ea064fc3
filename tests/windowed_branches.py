"""Requests that branch in a model whose second layer has a window and pages of its own size."""

from __future__ import annotations

import dataclasses

import branching_run
import plain_qwen3 as plain
import torch
from helpers import read_config, read_weights

WINDOW, WINDOW_PAGE = 40, 16


def make_runner(folder, block_size, dtype, *, device, recorded, max_num_seqs=12):
    from miniserve_amd.config import EngineConfig, load_config
    from miniserve_amd.engine import ModelRunner
    from miniserve_amd.parts.model import DecoderModel
    from miniserve_amd.weights import load_weights

    spec = load_config(folder).model_spec()
    second = spec.layers[1]
    mixer = dataclasses.replace(second.mixer, params={**second.mixer.params, "window": WINDOW, "block_size": WINDOW_PAGE})
    spec = dataclasses.replace(spec, layers=(spec.layers[0], dataclasses.replace(second, mixer=mixer), *spec.layers[2:]))
    model = DecoderModel(spec, dtype)
    tensors, _ = load_weights(folder, model.weight_specs(), dtype=model.dtype, device=device)
    config = EngineConfig(dtype=dtype, kv_block_size=block_size, num_kv_blocks=60, max_num_seqs=max_num_seqs,
                          enable_chunked_prefill=True, decode_graphs=recorded)
    runner = ModelRunner(model, tensors, config, device=device)
    assert [group.window for group in runner.cache.layout.groups] == [None, WINDOW]
    assert runner.cache.block_sizes == (block_size, WINDOW_PAGE)
    for pool in runner.cache.page_pools():
        pool.fill_(float("nan"))
    return runner


def worst(branches: branching_run.Branches, folder, dtype: str) -> tuple[float, float]:
    """As ``Branches.worst``, with the second layer's window."""

    config, weights = read_config(folder), read_weights(folder)
    windows = [None, WINDOW] + [None] * (config["num_hidden_layers"] - 2)
    if dtype == "bfloat16":
        weights = {k: v.to(torch.bfloat16).float() for k, v in weights.items()}
    histories = branches.histories + list(branches.tokens.values())
    exact = [plain.forward_logits(weights, config, tokens, windows=windows).float() for tokens in histories]
    allowed = 2e-5
    if dtype == "bfloat16":
        longest = max(range(len(histories)), key=lambda i: len(histories[i]))
        rounded = plain.forward_logits(weights, config, histories[longest], windows=windows, rd=torch.bfloat16).float()
        allowed = 3 * float((rounded - exact[longest]).abs().max())
    found = 0.0
    for tokens, row in branches.rows:
        index = next(i for i, history in enumerate(histories) if history[: len(tokens)] == tokens)
        error = float((row - exact[index][len(tokens) - 1]).abs().max())
        assert error == error, "a logit is not a number"
        found = max(found, error)
    return found, allowed


def five_branches_and_three_pairs(runner, vocab: int) -> branching_run.Branches:
    """Five neighbours share 256 keys, three pairs behind them 16 tokens each: a page of the window
    layer's, none of the other's, so that the two groups of pages have different runs of neighbours."""

    branches = branching_run.Branches(runner, vocab, seed=900)
    branches.admit("p")
    branches.step(p=270)
    branches.fork("p", "a", "b", "c", "d")
    names = ["p", "a", "b", "c", "d"]
    for pair in ("x", "y", "z"):
        branches.admit(pair)
        branches.step(**{pair: 20})
        branches.fork(pair, pair + "2")
        names += [pair, pair + "2"]
    for _ in range(3):
        branches.step(**{name: 1 for name in names})
    return branches


def rounds_of_drafts(runner, vocab: int, *, rounds: int, seed: int) -> branching_run.Branches:
    """Two requests that bring drafted tokens and lose some, or all, of them again, over several
    windows; a branch that is made before its parent's drafts are decided goes on beside it."""

    import random

    rng = random.Random(seed)
    branches = branching_run.Branches(runner, vocab, seed=seed)
    for name, prompt in (("p", 30), ("q", 61)):
        branches.admit(name)
        branches.step(**{name: prompt})
    for turn in range(rounds):
        counts = {name: 1 + rng.randint(0, 12) for name in branches.tokens}
        branches.step(**counts)
        if turn == rounds // 2:
            branches.fork("p", "x")
            counts["x"] = counts["p"]
        for name, count in counts.items():
            branches.truncate(name, len(branches.tokens[name]) - rng.choice((0, count - 1, rng.randint(0, count - 1))))
        if turn % 3 == 2:
            branches.step(**{name: 1 for name in branches.tokens})
    for name in list(branches.tokens):
        branches.release(name)
    assert runner.cache.capacity().free_blocks == runner.cache.num_blocks
    return branches
