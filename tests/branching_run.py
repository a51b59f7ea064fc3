"""A run of requests that branch, through ``ModelRunner``: one prompt, forked; branches that
go on side by side, with drafted tokens of which some are forgotten; a branch cut back into
what it shares; pages moved; a fork of a fork.  Tokens are given, and every row of logits is
compared with the plain implementation's for the tokens before it."""

from __future__ import annotations

import plain_qwen3 as plain
import torch
from helpers import random_tokens


class Branches:
    def __init__(self, runner, vocab: int, seed: int) -> None:
        self.runner, self.vocab, self.seed = runner, vocab, seed
        self.tokens: dict[str, list[int]] = {}
        self.histories: list[list[int]] = []
        self.rows: list[tuple[list[int], torch.Tensor]] = []

    def admit(self, name: str) -> None:
        self.runner.admit(name)
        self.tokens[name] = []

    def step(self, **counts: int) -> None:
        """A step in which each request brings so many further tokens; all logits are kept."""

        from miniserve_amd.engine import StepEntry

        entries = []
        for name, count in counts.items():
            self.seed += 1
            new = random_tokens(count, self.vocab, self.seed)
            self.tokens[name] += new
            entries.append(StepEntry(name, tuple(new), tuple(range(count))))
        logits = self.runner.step(entries).float().cpu().clone()
        at = 0
        for entry in entries:
            have = self.tokens[entry.request_id]
            for i in range(len(entry.token_ids)):
                self.rows.append((have[: len(have) - len(entry.token_ids) + i + 1], logits[at]))
                at += 1
        self.runner.cache.assert_invariants()

    def fork(self, name: str, *children: str) -> None:
        slots = self.runner.fork(name, children)
        assert slots == [self.runner.cache.state_slot(child) for child in children]
        for child in children:
            self.tokens[child] = list(self.tokens[name])
            assert self.runner.cache.committed_tokens(child) == len(self.tokens[name])
        self.runner.cache.assert_invariants()

    def truncate(self, name: str, length: int) -> None:
        self.histories.append(list(self.tokens[name]))
        del self.tokens[name][length:]
        self.runner.truncate(name, length)
        assert self.runner.cache.committed_tokens(name) == length
        self.runner.cache.assert_invariants()

    def release(self, name: str) -> None:
        self.histories.append(self.tokens.pop(name))
        self.runner.release(name)
        self.runner.cache.assert_invariants()

    def worst(self, weights, config, dtype: str, tolerance_f32: float = 2e-5) -> tuple[float, float]:
        """(largest error of any logit, what is allowed): bfloat16 is allowed three times the
        distance between the plain implementation with every intermediate rounded to
        bfloat16 and itself in 64 bits, on the same tokens."""

        histories = self.histories + list(self.tokens.values())
        reference = weights if dtype == "float32" else {k: v.to(torch.bfloat16).float() for k, v in weights.items()}
        exact = [plain.forward_logits(reference, config, tokens).float() for tokens in histories]
        allowed = tolerance_f32
        if dtype == "bfloat16":
            longest = max(range(len(histories)), key=lambda i: len(histories[i]))
            rounded = plain.forward_logits(reference, config, histories[longest], rd=torch.bfloat16).float()
            allowed = 3 * float((rounded - exact[longest]).abs().max())
        worst = 0.0
        for tokens, row in self.rows:
            index = next(i for i, history in enumerate(histories) if history[: len(tokens)] == tokens)
            error = float((row - exact[index][len(tokens) - 1]).abs().max())
            worst = max(worst, error) if error == error else float("nan")
            assert worst == worst, "a logit is not a number"
        return worst, allowed


def run(runner, vocab: int, prompt: int) -> Branches:
    branches = Branches(runner, vocab, seed=4000 + prompt)
    branches.admit("p")
    branches.admit("other")
    branches.step(p=prompt, other=19)
    branches.fork("p", "a", "b", "c")
    for _ in range(4):
        branches.step(p=1, a=1, b=1, c=1, other=1)
    branches.step(p=5, a=5, b=3, c=1)                      # drafted tokens behind the next one
    branches.truncate("a", len(branches.tokens["a"]) - 3)  # three of them not taken
    branches.truncate("p", len(branches.tokens["p"]) - 4)
    branches.step(a=1, b=1, p=2, c=1, other=1)
    branches.step(p=1, a=1, b=1, c=1)
    branches.truncate("b", prompt - 30)                    # into what it shares with the others
    branches.step(p=1, a=1, b=1, c=1)
    branches.release("other")
    branches.fork("a", "d")                                # a fork of a fork
    branches.step(a=1, d=1, p=1, c=1, b=1)
    branches.release("p")
    branches.release("c")
    moved = runner.compact()
    assert moved > 0 and runner.compact() == 0
    runner.cache.assert_invariants()
    for _ in range(3):
        branches.step(a=1, d=1, b=1)
    branches.step(b=40, a=1, d=4)
    for name in ("a", "d", "b"):
        branches.release(name)
    assert runner.cache.live_requests() == () and runner.cache.capacity().free_blocks == runner.cache.num_blocks
    return branches
