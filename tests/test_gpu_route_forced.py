"""Scored routing with experts forced by a bias of +inf and taken out by one of
-inf, with expert groups: the group of a forced expert is on offer, whatever the
others in it, and groups of equal value go to the lowest index."""

import math

import pytest
import torch

from extend_nano_vllm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def route(bias, keep, top_k, how="top2", tokens=5, experts=32, groups=8, score="sigmoid"):
    g = torch.Generator(device=DEV).manual_seed(1)
    logits = torch.randn((tokens, experts), generator=g, device=DEV)
    return ops.route_scored_topk(logits, top_k, score=score, bias=bias, num_groups=groups,
                                 topk_groups=keep, group_score=how)[1]


@pytest.mark.parametrize("how", ["top2", "max"])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_a_forced_expert_alone_in_its_group(how, score):
    # Expert 21 forced, the rest of its group (20..23) taken out; two more forced experts
    # in group 2, whose value is +inf too: of three such groups the lowest indexes stay.
    bias = torch.zeros(32, device=DEV)
    bias[20:24] = -math.inf
    bias[21] = math.inf
    ids = route(bias, 1, 1, how, score=score)
    assert bool((ids == 21).all())
    bias[8], bias[9], bias[28] = math.inf, math.inf, math.inf
    ids = route(bias, 1, 2, how, score=score)  # group 2
    assert ids.tolist() == [[8, 9]] * 5
    ids = route(bias, 2, 3, how, score=score)  # groups 2 and 5, not 7
    assert ids.tolist() == [[8, 9, 21]] * 5
    ids = route(bias, 3, 4, how, score=score)
    assert ids.tolist() == [[8, 9, 21, 28]] * 5


@pytest.mark.parametrize("how", ["top2", "max"])
def test_groups_that_are_taken_out_come_last(how):
    bias = torch.full((32,), -math.inf, device=DEV)
    bias[12:16] = 0.0
    ids = route(bias, 1, 4, how)
    assert bool((ids.sort(-1).values == torch.arange(12, 16, device=DEV)).all())
