"""ExpertParallelMoE with scored routing and 4-bit weights: the layer against the
operators it is made of and against 64 bits.

Tolerance of the 64-bit comparison: the routed sum is off by its own bound
(bf16 act, fp32 sums: below 2^-7 of the largest output in these shapes) and the
shared expert adds three bf16 roundings of its chain, 2^-8 each, and the sum
one more; 2^-5 of the largest output covers them together."""

import pytest
import torch

import extend_nano_vllm_b200.workloads as wl
from extend_nano_vllm_b200 import ExpertParallelMoE, device_status, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(shared=None, capacity=None, seed=1, top_k=4):
    shape = wl.LayerShape("small", 256, 128, 32, top_k)
    layer = ExpertParallelMoE(shape.hidden, shape.intermediate, shape.num_experts, top_k, True,
                              expert_capacity_factor=capacity,
                              shared_expert_intermediate_size=shared)
    layer = layer.to(device=DEV, dtype=torch.bfloat16)
    w13, w2 = wl.expert_weights(shape, seed)
    with torch.no_grad():
        layer.gate.weight.copy_(wl.gate_weight(shape, seed).bfloat16() * 4)
        layer.gate_up_proj.copy_(w13)
        layer.down_proj.copy_(w2)
        if shared:
            g = torch.Generator().manual_seed(seed)
            for p in (layer.shared_expert.gate_up_proj.weight,
                      layer.shared_expert.down_proj.weight, layer.shared_expert_gate.weight):
                p.copy_(torch.randn(p.shape, generator=g) * 0.02)
    return layer


def bias(experts=32):
    return torch.randn(experts, generator=torch.Generator().manual_seed(3)) * 0.05


def back(codes, scales, zeros):
    by = codes.double().unflatten(-1, (scales.size(-1), -1))
    z = 8.0 if zeros is None else zeros.double()[..., None]
    return ((by - z) * scales.double()[..., None]).flatten(-2)


@pytest.mark.parametrize("tokens", [1, 3, 17, 200])
def test_scored_routing_with_bf16_experts(tokens):
    layer = make()
    layer.set_scored_routing("sigmoid", bias(), 8, 4, "top2", 2.5)
    x = wl.hidden_states(tokens, 256, 5, DEV)
    weights, ids = ops.route_scored_topk(layer.gate(x), 4, score="sigmoid", bias=bias().cuda(),
                                         num_groups=8, topk_groups=4, scale=2.5)
    out, local = layer._execute_local(x, weights, ids)
    assert local == tokens * 4
    # The layer's own forward packs in the same way: equal bit for bit.
    assert torch.equal(layer(x), out)
    assert layer.total_assignment_count == tokens * 4
    assert torch.equal(layer._route(x)[1], ids)


@pytest.mark.parametrize("shared", [None, 128, 96])
@pytest.mark.parametrize("tokens,zeros", [(1, False), (9, True), (150, False)])
def test_w4_layer(tokens, zeros, shared):
    layer = make(shared)
    w13 = [ops.quantize_w4(w, 32, zeros) for w in layer.gate_up_proj.detach()]
    w2 = [ops.quantize_w4(w, 32, zeros) for w in layer.down_proj.detach()]
    if shared:
        s13 = back(*ops.quantize_w4(layer.shared_expert.gate_up_proj.weight.detach(), 32, zeros))
        s2 = back(*ops.quantize_w4(layer.shared_expert.down_proj.weight.detach(), 32, zeros))
    before = layer.expert_parameter_bytes
    layer.set_scored_routing("sigmoid", bias(), 8, 4, "top2", 2.5)
    layer.quantize_w4(32, zeros)
    assert layer.expert_parameter_bytes < 0.4 * before
    x = wl.hidden_states(tokens, 256, 6, DEV)
    out = layer(x)
    assert out.shape == x.shape and out.dtype == torch.bfloat16
    weights, ids = layer._route(x)
    xd = x.double()
    ref = torch.zeros_like(xd)
    for e in range(32):
        token, slot = torch.where(ids == e)
        gate, up = (xd[token] @ back(*w13[e]).T).chunk(2, -1)
        y = (gate * torch.sigmoid(gate) * up) @ back(*w2[e]).T
        ref.index_add_(0, token, y * weights[token, slot].double()[:, None])
    if shared:
        gate, up = (xd @ s13.T).chunk(2, -1)
        gated = torch.sigmoid(layer.shared_expert_gate(x).double())
        ref += gated * ((gate * torch.sigmoid(gate) * up) @ s2.T)
    assert float((out.double() - ref).abs().max()) <= 2.0 ** -5 * float(ref.abs().max())
    assert layer.dispatch_assignment_count == tokens * 4
    assert torch.equal(layer(x.view(1, tokens, 256)).view_as(out), out)
    assert device_status() == 0


def test_w4_layer_with_capacity_counts_and_drops():
    layer = make(capacity=0.5)
    layer.quantize_w4(64)
    x = wl.hidden_states(64, 256, 7, DEV)
    weights, ids = ops.route_topk(layer.gate(x), 4, True)
    packed = ops.pack_routes(ids.view(-1), weights.view(-1), 32, 32, capacity=layer._capacity(64))
    dropped = int(packed.counters[3])
    assert dropped > 0
    out = layer(x)
    assert layer.dropped_assignment_count == dropped
    assert layer.dispatch_assignment_count == 64 * 4 - dropped
    assert torch.equal(out, ops.experts_w4(x, ids, weights, *layer._w4))


def test_w4_layer_in_a_graph_and_after_a_move():
    layer = make(shared=96)
    layer.set_scored_routing("softmax", None, 8, 4, "max")
    with pytest.raises(ValueError, match="multiple of the group size"):
        layer.quantize_w4(128)  # the shared expert's 96 k; nothing has changed
    layer.quantize_w4(32)
    x = wl.hidden_states(24, 256, 8, DEV)
    first = layer(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer(x)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    moved = layer.to("cpu").to(DEV)
    assert torch.equal(moved(x), first)


def test_w4_layer_refuses_loading_and_relocating():
    layer = make()
    layer.quantize_w4(64)
    with pytest.raises(RuntimeError, match="4-bit"):
        layer.load_expert_weight(0, "down_proj", torch.zeros(256, 128))
    placed = ExpertParallelMoE(256, 128, 32, 4, True, dynamic_placement=True).to(
        device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        for p in placed.parameters():
            p.normal_(0, 0.02)
    placed.quantize_w4(64)
    with pytest.raises(NotImplementedError, match="relocated"):
        placed.relocate_experts([0] * 32)
