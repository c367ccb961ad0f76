"""Scored routing against a plain 64-bit implementation.

Ids have to be equal wherever 64 bits leave no doubt that 32 bits could have
another order: a row is left out when two neighbouring choice values (or group
values at the cut) differ by less than 1e-5 of their size plus 1e-6, some ten
times what fp32 scores and sums can be off by.  Equal logits with equal biases
are exact ties in both, and go to the lowest index.  Weights: fp32 arithmetic
and one bf16 store, so 2^-8 covers the store (2^-9) twice over."""

import math

import pytest
import torch

from extend_nano_vllm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain(logits, top_k, score="softmax", bias=None, num_groups=1, topk_groups=1,
          group_score="top2", renormalize=True, scale=1.0):
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    if score == "sigmoid":
        s = torch.sigmoid(x)
    else:
        top = x.amax(-1, keepdim=True)
        e = torch.where(x == top, 1.0, torch.exp(x - top))
        e = torch.where(top == -math.inf, 0.0, e)
        total = e.sum(-1, keepdim=True)
        s = torch.where(total > 0, e / total, 0.0)
    c = s if bias is None else s + bias.double()
    c = torch.where(c.isnan(), -math.inf, c)
    unsure = torch.zeros(x.size(0), dtype=torch.bool, device=x.device)

    def close(a, b):
        gap = (a - b).abs()
        return (gap > 0) & (gap < 1e-5 * (a.abs() + b.abs()) + 1e-6 * (bias is not None))

    if num_groups > 1:
        by = c.view(x.size(0), num_groups, -1)
        v = (by.amax(-1) if group_score == "max" or by.size(-1) == 1
             else by.topk(2, -1).values.sum(-1))
        order = v.sort(dim=-1, descending=True, stable=True)
        if topk_groups < num_groups:
            unsure |= close(order.values[:, topk_groups - 1], order.values[:, topk_groups])
        kept = torch.zeros_like(v, dtype=torch.bool).scatter_(1, order.indices[:, :topk_groups], True)
        kept = kept[..., None].expand_as(by).reshape(c.shape)
    else:
        kept = torch.ones_like(c, dtype=torch.bool)
    # Experts that are not on offer come after all others, -inf among them.
    first = c.sort(dim=-1, descending=True, stable=True).indices
    offered = kept.gather(1, first).to(torch.int8).sort(dim=-1, descending=True, stable=True).indices
    order = first.gather(1, offered)
    values = c.gather(1, order)
    n = min(top_k + 1, int(kept.sum(-1).min()))
    unsure |= close(values[:, :n - 1], values[:, 1:n]).any(-1)
    ids = order[:, :top_k]
    w = s.gather(1, ids)
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return w * scale, ids, ~unsure


def check(logits, top_k, least=0.9, **how):
    weights, ids = ops.route_scored_topk(logits, top_k, **how)
    ref_w, ref_ids, sure = plain(logits, top_k, **how)
    assert weights.dtype == torch.bfloat16 and ids.dtype == torch.int64
    # Enough rows are compared: all but a share, and one in a batch of a few.
    assert int(sure.sum()) >= int(least * sure.numel()) and bool(sure.any())
    assert torch.equal(ids[sure], ref_ids[sure])
    err = (weights.double() - ref_w).abs()[sure]
    assert bool((err <= 2.0 ** -8 * ref_w[sure].abs() + 1e-30).all())
    return weights, ids


def logits_of(tokens, experts, seed, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn((tokens, experts), generator=g, device=DEV) * 1.5).to(dtype)


def bias_of(experts, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(experts, generator=g, device=DEV) * 0.05


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("tokens,experts,top_k,groups,keep,how", [
    (1, 256, 8, 8, 4, "top2"), (5, 128, 8, 1, 1, "max"), (97, 160, 6, 8, 3, "max"),
    (33, 72, 3, 6, 2, "top2"), (300, 512, 10, 16, 5, "top2"), (64, 1024, 32, 32, 9, "max"),
    (9, 64, 1, 1, 1, "top2"), (7, 24, 12, 24, 12, "top2"), (3, 1, 1, 1, 1, "max"),
    (4, 40, 4, 20, 2, "top2"), (11, 33, 33 - 1, 1, 1, "max")])
def test_against_64_bits(tokens, experts, top_k, groups, keep, how, biased, score, dtype):
    logits = logits_of(tokens, experts, tokens + experts, dtype)
    check(logits, top_k, least=0.5, score=score, bias=bias_of(experts, 3) if biased else None,
          num_groups=groups, topk_groups=keep, group_score=how, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_large_batch_without_renormalising(score):
    check(logits_of(4099, 128, 1), 8, score=score, renormalize=False, scale=0.5)


def test_equal_values_go_to_the_lowest_index():
    logits = torch.zeros((3, 64), device=DEV)
    logits[1, 40:] = 1.0
    _, ids = check(logits, 4, score="sigmoid", num_groups=8, topk_groups=2)
    assert ids[0].tolist() == [0, 1, 2, 3] and ids[1].tolist() == [40, 41, 42, 43]
    coarse = (logits_of(500, 128, 2) * 2).round() / 2  # many ties in every row
    check(coarse, 8, score="softmax", num_groups=8, topk_groups=3, group_score="max")
    check(coarse.half(), 8, score="sigmoid", num_groups=8, topk_groups=3, group_score="top2")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_infinite_and_nan_logits(score):
    inf, nan = math.inf, math.nan
    logits = logits_of(6, 32, 5)
    logits[0] = -inf                      # nothing on offer
    logits[1, :30] = -inf                 # fewer finite ones than are chosen
    logits[2, 4] = inf
    logits[3, 5] = nan
    logits[4] = torch.finfo(torch.float32).min
    logits[5, 6:9] = inf
    weights, ids = check(logits, 4, least=0.8, score=score)
    assert ids[0].tolist() == [0, 1, 2, 3] and weights[0].tolist() == [0.0] * 4
    assert ids[2, 0] == 4
    assert 5 not in ids[3].tolist()
    # An expert taken out by its bias is chosen only when nothing else is left.
    bias = torch.zeros(32, device=DEV)
    bias[:16] = -inf
    _, ids = check(logits_of(40, 32, 6), 8, score=score, bias=bias)
    assert int(ids.min()) >= 16
    bias[20] = nan
    _, ids = check(logits_of(40, 32, 7), 8, score=score, bias=bias)
    assert not bool((ids == 20).any())


def test_strides_streams_graphs_and_no_tokens():
    wide = logits_of(12, 256, 8)
    check(wide[:, ::2], 8, score="sigmoid")
    check(wide[::3, :128], 8, score="sigmoid")
    w, ids = ops.route_scored_topk(wide[:0], 8)
    assert w.shape == (0, 8) and ids.shape == (0, 8)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.route_scored_topk(wide, 8, score="sigmoid", num_groups=8, topk_groups=4)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, ids = ops.route_scored_topk(wide, 8, score="sigmoid", num_groups=8, topk_groups=4)
    wide.copy_(logits_of(12, 256, 9))
    graph.replay()
    torch.cuda.synchronize()
    ref_w, ref_ids = ops.route_scored_topk(wide, 8, score="sigmoid", num_groups=8, topk_groups=4)
    assert torch.equal(ids, ref_ids) and torch.equal(w, ref_w)


def test_refusals():
    x = logits_of(2, 64, 1)
    with pytest.raises(ValueError, match="score function"):
        ops.route_scored_topk(x, 4, score="tanh")
    with pytest.raises(ValueError, match="group score"):
        ops.route_scored_topk(x, 4, group_score="mean")
    with pytest.raises(ValueError, match="top_k must be"):
        ops.route_scored_topk(x, 65)
    with pytest.raises(ValueError, match="divide"):
        ops.route_scored_topk(x, 4, num_groups=7)
    with pytest.raises(ValueError, match="topk_groups"):
        ops.route_scored_topk(x, 4, num_groups=8, topk_groups=9)
    with pytest.raises(ValueError, match="experts of topk_groups"):
        ops.route_scored_topk(x, 9, num_groups=8, topk_groups=1)
    with pytest.raises(NotImplementedError, match="top_k 40"):
        ops.route_scored_topk(x, 40)
    with pytest.raises(NotImplementedError, match="1024"):
        ops.route_scored_topk(logits_of(1, 1056, 1), 4)
    with pytest.raises(TypeError, match="bias"):
        ops.route_scored_topk(x, 4, bias=torch.zeros(63, device=DEV))
    with pytest.raises(TypeError, match="logits"):
        ops.route_scored_topk(x.double(), 4)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.route_scored_topk(x.cpu(), 4)
