"""The check of drafted tokens where logits over the temperature are far from zero: every
temperature that a request may have, and every finite logit."""

from __future__ import annotations

import pytest
import torch
from test_gpu_branching_kernels import check_verify, draft_case, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def ends(case):
    """First rows of the requests and their number of drafts."""

    starts = case["row_start"].tolist()
    return [(first, end - first - 1) for first, end in zip(starts, starts[1:])]


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("temperature", [1e-3, 1e-6, 1e-9, 1e-12, 1e-14, 1e-15, 1e-16, 1e-17, 1e-18, 1e-19, 1e-20, 1e-21, 1e-22, 1e-30, 1e-37, 1e-44])
def test_temperatures_down_to_the_smallest(ops, temperature, probs):  # noqa: F811
    """One token a row has all of the mass, or a few equal ones share it: taken while drafted (with a
    uniform number below its share), drawn where another was drafted.  Uniform numbers come from a
    generator: none lies at a border, which are multiples of 1/3 and 1/2."""

    for seed in range(4):
        case = draft_case([2, 5, 0, 1, 7, 3, 3, 12], 5003, temperature=1.0, seed=seed, probs=probs)
        case["logits"] = case["logits"] + 10 * (seed - 1)
        best = case["logits"].argmax(-1)
        if seed % 2:
            for row in range(0, best.numel(), 3):
                case["logits"][row, [4099, 11, 2050][: 2 + row % 2]] = float(case["logits"][row].max()) + 1
        best = case["logits"].argmax(-1)
        draft = 0
        for first, drafts in ends(case):      # the best token is drafted, at every fourth place the one behind it
            for i in range(drafts):
                case["draft_tokens"][draft] = (int(best[first + i]) + (i % 4 == 3)) % 5003
                draft += 1
        case["temperature"][:] = temperature
        taken = check_verify(ops, case)
        if temperature < 1e-8 and not seed % 2:
            assert taken == [min(drafts, 3) for _, drafts in ends(case)], "the best token has all of the mass"


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("size", [1e8, 1e13, 1e16, 1e17, 1e18, 1e20, 1e25, 1e30, 3e37])
def test_logits_up_to_the_largest(ops, size, probs):  # noqa: F811
    for seed, temperature in enumerate((1.0, 0.3, 2.0)):
        case = draft_case([2, 5, 0, 1, 7, 3, 3], 5003, temperature=1.0, seed=seed, probs=probs)
        case["logits"] = (case["logits"] / case["logits"].abs().max() * size * 10).clamp(-3.4e38, 3.4e38)
        best, draft = case["logits"].argmax(-1), 0
        for first, drafts in ends(case):
            case["draft_tokens"][draft : draft + drafts] = best[first : first + drafts].int()
            draft += drafts
        case["temperature"][:] = temperature
        assert check_verify(ops, case) == [drafts for _, drafts in ends(case)]


def test_near_ties_at_small_temperatures(ops):  # noqa: F811
    # neighbours in 32 bits around 10, over a temperature of their distance: masses e^0, e^-0.95, e^-1.9, ...
    step = 2.0**-20
    for seed in range(6):
        case = draft_case([3, 2, 4, 0, 6], 4099, temperature=1.0, seed=seed, probs=seed % 2 == 0)
        gen = torch.Generator().manual_seed(100 + seed)
        rows, vocab = case["logits"].shape
        case["logits"] = 10 - step * torch.randint(0, 40, (rows, vocab), generator=gen)
        case["temperature"][:] = 1e-6
        check_verify(ops, case)
