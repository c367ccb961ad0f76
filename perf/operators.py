"""Cases of three operators of a mixture-of-experts layer that serves with 4-bit weights.

  route    scored routing: sigmoid or softmax scores, a selection bias, expert groups, top-k,
           renormalised weights
  experts  the routed experts' products (SwiGLU MLPs) with 4-bit weights and group scales
  linear   the dense product with 4-bit weights and group scales (a shared expert's projections)

A 4-bit weight is W[n, k] = scale[n, k // g] * (q[n, k] - zero[n, k // g]) with q in 0..15 and
zero = 8 where no zeros are given.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # One sequence's decode step of a 256-expert layer with sigmoid scores, a balance bias and
        # 8 groups of which 4 are kept: pure latency.
        _route("route-one", 1, 256, 8, "sigmoid", True, 8, 4, "top2", 2.5, "f32"),
        # A decode batch of the 128-expert layer with softmax scores and a bias, logits as the bf16
        # router projection leaves them (many equal logits).
        _route("route-decode", 64, 128, 8, "softmax", True, 1, 1, "max", 1.0, "bf16"),
        # A ragged chunk of a prompt: softmax scores, groups by their best expert, fp16 logits.
        _route("route-odd", 1031, 160, 6, "softmax", False, 8, 3, "max", 16.0, "f16"),
        # A full prefill chunk of 8192 tokens.
        _route("route-prefill", 8192, 256, 8, "sigmoid", True, 8, 4, "top2", 2.5, "f32"),
        # One sequence's decode step through the 128-expert layer (8 experts read).
        _experts("experts-one", 1, 2048, 768, 128, 8, 128, False),
        # A small decode batch of the 512-expert, top-10 layer: over a hundred experts, mostly one
        # row each.
        _experts("experts-few", 16, 2048, 512, 512, 10, 64, True),
        # An ordinary decode batch: nearly every expert is read for a few rows.
        _experts("experts-decode", 64, 2048, 768, 128, 8, 128, False),
        # A large, odd decode batch with small groups and zero points: ragged experts.
        _experts("experts-batch", 509, 2048, 768, 128, 8, 32, True),
        # A prefill chunk of 8192 tokens: bound by the matrix products.
        _experts("experts-prefill", 8192, 2048, 768, 128, 8, 128, False),
        # One token through a wide projection: the matrix-vector product.
        _linear("linear-one", 1, 8192, 4096, 128, False),
        # A few tokens, a width that fills no tile, small groups with zero points.
        _linear("linear-few", 17, 1000, 2048, 32, True),
        # A prefill chunk through a square projection.
        _linear("linear-prefill", 4096, 4096, 4096, 128, False),
    ]


def _route(name, tokens, experts, top_k, score, bias, groups, topk_groups, group_score, scale, dtype):
    return dict(name=name, op="route", tokens=tokens, experts=experts, top_k=top_k, score=score,
                bias=bias, groups=groups, topk_groups=topk_groups, group_score=group_score,
                scale=scale, dtype=dtype)


def _experts(name, tokens, hidden, inter, experts, top_k, group, zeros):
    return dict(name=name, op="experts", tokens=tokens, hidden=hidden, inter=inter, experts=experts,
                top_k=top_k, group=group, zeros=zeros)


def _linear(name, tokens, out, inner, group, zeros):
    return dict(name=name, op="linear", tokens=tokens, out=out, inner=inner, group=group, zeros=zeros)


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "linear"])
    if op == "route":
        experts, groups, topk_groups = rng.choice(
            [(256, 8, 4), (160, 8, 3), (128, 1, 1), (512, 1, 1), (64, 1, 1), (256, 16, 5), (72, 6, 2)])
        case = _route("", _log(rng, 1, 8192), experts, rng.choice([1, 2, 4, 6, 8, 10]),
                      rng.choice(["sigmoid", "softmax"]), rng.random() < 0.6, groups, topk_groups,
                      rng.choice(["max", "top2"]), rng.choice([1.0, 2.5, 16.0]),
                      rng.choice(["f32", "bf16", "f16"]))
    elif op == "experts":
        hidden, inter, experts, top_k = rng.choice(
            [(2048, 768, 128, 8), (2048, 512, 512, 10), (1024, 384, 32, 4)])
        case = _experts("", _log(rng, 1, 8192), hidden, inter, experts, top_k,
                        rng.choice([32, 64, 128]), rng.random() < 0.5)
    else:
        group = rng.choice([32, 64, 128])
        case = _linear("", _log(rng, 1, 4096), _log(rng, 64, 8192),
                       max(1, _log(rng, 256, 4096) // group) * group, group, rng.random() < 0.5)
        if case["tokens"] * case["out"] * case["inner"] > 1 << 36:
            case["tokens"] = (1 << 36) // (case["out"] * case["inner"])
    del case["name"]
    return case


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rand(shape, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _quantised(shape, group, zeros, g):
    """N(0, 0.02) weights [..., rows, k] rounded to 4 bits by groups of k: codes (one per byte), bf16
    scales and, where asked for, integer zero points."""
    w = _rand(shape, g).mul_(0.02).view(*shape[:-1], shape[-1] // group, group)
    if zeros:
        low, high = w.amin(-1, keepdim=True).clamp_(max=0), w.amax(-1, keepdim=True).clamp_(min=0)
        scale = ((high - low) / 15).bfloat16()
        zero = (-low / scale.float()).round_().clamp_(0, 15)
    else:
        scale = (w.abs().amax(-1, keepdim=True) / 7).bfloat16()
        zero = torch.full_like(scale, 8, dtype=torch.float32)
    codes = w.div_(scale.float()).round_().add_(zero).clamp_(0, 15).to(torch.uint8).view(shape)
    return codes, scale.squeeze(-1), zero.squeeze(-1).to(torch.uint8) if zeros else None


def _close(a, b, biased):
    """Whether two 64-bit scores are unequal and yet too near for 32 bits to order surely."""
    gap = (a - b).abs()
    return (gap > 0) & (gap < 4e-6 * (a.abs() + b.abs()) + (1e-6 if biased else 0.0))


def _choice64(case, logits, bias):
    """Scores and choice in 64 bits -> (scores, ids, rows whose choice 32 bits may not share)."""
    x = logits.double()
    score = 1 / (1 + torch.exp(-x)) if case["score"] == "sigmoid" else torch.softmax(x, -1)
    pick = score + bias.double() if bias is not None else score
    unsure = torch.zeros(x.shape[0], dtype=torch.bool, device=x.device)
    groups, keep = case["groups"], case["topk_groups"]
    if groups > 1:
        by = pick.view(x.shape[0], groups, -1)
        best = by.amax(-1) if case["group_score"] == "max" else by.topk(2, -1).values.sum(-1)
        order = best.sort(dim=-1, descending=True, stable=True)
        if keep < groups:
            unsure |= _close(order.values[:, keep - 1], order.values[:, keep], bias is not None)
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order.indices[:, :keep], True)
        pick = torch.where(kept[..., None], by, -math.inf).view_as(pick)
    order = pick.sort(dim=-1, descending=True, stable=True)
    k = case["top_k"]
    last = min(k + 1, pick.shape[1])
    unsure |= _close(order.values[:, :last - 1], order.values[:, 1:last], bias is not None).any(-1)
    return score, order.indices[:, :k], unsure


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "route":
        shape = (case["tokens"], case["experts"])
        bias = _rand((case["experts"],), g) * 0.05 if case["bias"] else None
        logits = (_rand(shape, g) * 1.5).to(_DTYPES[case["dtype"]])
        # A row whose choice hangs on the last bit of a 32-bit score has no answer that two orders of
        # summation share: such rows (one in some thousand) are drawn again.
        for _ in range(8):
            unsure = _choice64(case, logits, bias)[2]
            logits = torch.where(unsure[:, None], (_rand(shape, g) * 1.5).to(logits.dtype), logits)
        return {"case": case, "logits": logits, "bias": bias}
    if case["op"] == "linear":
        weight = _quantised((case["out"], case["inner"]), case["group"], case["zeros"], g)
        state = {"case": case, "x": _rand((case["tokens"], case["inner"]), g).bfloat16(), "weight": weight}
        if own:  # a program lays its weights out once, when it loads them
            state["packed"] = _ops().pack_w4(*weight)
        return state
    tokens, experts, hidden, inter = (case[n] for n in ("tokens", "experts", "hidden", "inter"))
    w13 = _quantised((experts, 2 * inter, hidden), case["group"], case["zeros"], g)
    w2 = _quantised((experts, hidden, inter), case["group"], case["zeros"], g)
    # Some experts are asked for more often than others, as in a trained layer.
    logits = _rand((tokens, experts), g) + 0.5 * _rand((experts,), g)
    top = torch.softmax(logits, -1).topk(case["top_k"], -1)
    state = {"case": case, "x": _rand((tokens, hidden), g).bfloat16(), "ids": top.indices,
             "weights": (top.values / top.values.sum(-1, keepdim=True)).bfloat16(),
             "w13": w13, "w2": w2,
             # Rows of the fullest expert: what the plain form's padded buffer has to hold.
             "most": int(torch.bincount(top.indices.view(-1), minlength=experts).max())}
    if own:
        state["packed"] = (_ops().pack_w4(*w13, layout="gate_up"), _ops().pack_w4(*w2))
    return state


def _ops():
    import extend_nano_vllm_b200

    return extend_nano_vllm_b200.ops


def run(state):
    case = state["case"]
    if own:
        if case["op"] == "route":
            return _ops().route_scored_topk(
                state["logits"], case["top_k"], score=case["score"], bias=state["bias"],
                num_groups=case["groups"], topk_groups=case["topk_groups"],
                group_score=case["group_score"], renormalize=True, scale=case["scale"])
        if case["op"] == "linear":
            return _ops().linear_w4(state["x"], state["packed"])
        return _ops().experts_w4(state["x"], state["ids"], state["weights"], *state["packed"])
    return {"route": _plain_route, "experts": _plain_experts, "linear": _plain_linear}[case["op"]](state)


def _plain_route(state):
    case, x = state["case"], state["logits"].float()
    if case["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        e = torch.exp(x - x.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    pick = score if state["bias"] is None else score + state["bias"]
    if case["groups"] > 1:
        by = pick.view(x.shape[0], case["groups"], -1)
        best = by.amax(-1) if case["group_score"] == "max" else by.topk(2, -1).values.sum(-1)
        first = best.sort(dim=-1, descending=True, stable=True).indices[:, :case["topk_groups"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, first, True)
        pick = torch.where(kept[..., None], by, -math.inf).view_as(pick)
    ids = pick.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
    weights = score.gather(1, ids)
    weights = weights / weights.sum(-1, keepdim=True) * case["scale"]
    return weights.bfloat16(), ids


def _dequantised(weight, group, dtype=torch.float32):
    codes, scale, zero = weight
    by = codes.view(*codes.shape[:-1], -1, group).to(dtype)
    by = by - (8 if zero is None else zero.to(dtype)[..., None])
    return by.mul_(scale.to(dtype)[..., None]).view(codes.shape)


def _plain_linear(state):
    w = _dequantised(state["weight"], state["case"]["group"])
    return (state["x"].float() @ w.T).bfloat16()


def _plain_experts(state):
    case, ids = state["case"], state["ids"].view(-1)
    rows = state["x"].float().repeat_interleave(case["top_k"], 0)
    if ids.numel() < case["experts"]:  # fewer routes than experts: each route's own weights
        part = lambda w: tuple(None if t is None else t[ids] for t in w)  # noqa: E731
        h = torch.bmm(_dequantised(part(state["w13"]), case["group"]), rows[..., None])[..., 0]
        gate, up = h.chunk(2, -1)
        act = gate / (1.0 + torch.exp(-gate)) * up
        y = torch.bmm(_dequantised(part(state["w2"]), case["group"]), act[..., None])[..., 0]
        y = y.view(case["tokens"], case["top_k"], -1) * state["weights"].float()[..., None]
        return y.sum(1).bfloat16()
    w13 = _dequantised(state["w13"], case["group"])
    # Each route's place among its expert's, and the rows in a buffer padded to the fullest expert.
    order = ids.sort(stable=True)
    first = torch.searchsorted(order.values, torch.arange(case["experts"], device=ids.device))
    place = torch.empty_like(ids)
    place[order.indices] = torch.arange(ids.numel(), device=ids.device) - first[order.values]
    padded = rows.new_zeros(case["experts"], state["most"], case["hidden"])
    padded[ids, place] = rows
    gate, up = torch.bmm(padded, w13.transpose(1, 2)).chunk(2, -1)
    act = gate / (1.0 + torch.exp(-gate)) * up
    del w13, rows, padded, gate, up
    y = torch.bmm(act, _dequantised(state["w2"], case["group"]).transpose(1, 2))[ids, place]
    y = y.view(case["tokens"], case["top_k"], -1) * state["weights"].float()[..., None]
    return y.sum(1).bfloat16()


def work(case):
    if case["op"] == "route":
        size = 4 if case["dtype"] == "f32" else 2
        tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": tokens * (experts * size + k * 10) + (experts * 4 if case["bias"] else 0),
                "flops": tokens * experts * 6}
    per_weight = 0.5 + (3 if case["zeros"] else 2) / case["group"]
    if case["op"] == "linear":
        m, n, k = case["tokens"], case["out"], case["inner"]
        return {"bytes": n * k * per_weight + 2 * m * (n + k), "flops": 2 * m * n * k}
    tokens, experts, k = case["tokens"], case["experts"], case["top_k"]
    weights = 3 * case["hidden"] * case["inter"]
    # The experts that the tokens' routes reach, as many as routes that fall evenly would.
    active = experts * (1 - (1 - k / experts) ** tokens)
    return {"bytes": active * weights * per_weight + tokens * (case["hidden"] * 4 + k * 10),
            "flops": 2 * tokens * k * weights}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        score, ids, _ = _choice64(case, state["logits"], state["bias"])
        weights = torch.gather(score, 1, ids)
        return weights / weights.sum(-1, keepdim=True) * case["scale"], ids
    if case["op"] == "linear":
        w = _dequantised(state["weight"], case["group"], torch.float64)
        return torch.einsum("mk,nk->mn", state["x"].double(), w)
    x, ids, weights = state["x"].double(), state["ids"], state["weights"].double()
    out = torch.zeros_like(x)
    part = lambda w, e: tuple(None if t is None else t[e] for t in w)  # noqa: E731
    for e in ids.unique().tolist():
        token, slot = torch.where(ids == e)
        h = x[token] @ _dequantised(part(state["w13"], e), case["group"], torch.float64).T
        gate, up = h.chunk(2, -1)
        y = (gate * torch.sigmoid(gate) * up) @ _dequantised(part(state["w2"], e), case["group"],
                                                              torch.float64).T
        out.index_add_(0, token, y * weights[token, slot][:, None])
    return out
