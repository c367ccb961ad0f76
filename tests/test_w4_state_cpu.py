"""What a layer with scored routing and 4-bit weights keeps through device and
dtype moves and through calls that are refused, without a GPU.  Packing is
replaced by a stand-in that keeps the shapes; nothing is computed."""

import pytest
import torch

from extend_nano_vllm_b200 import _lib, ops
from extend_nano_vllm_b200.moe import ExpertParallelMoE


@pytest.mark.parametrize("move", [lambda m: m.to(torch.bfloat16), lambda m: m.half(),
                                  lambda m: m.bfloat16().float(), lambda m: m.double(),
                                  lambda m: m.to("cpu", torch.bfloat16),
                                  lambda m: torch.nn.ModuleList([m]).to(torch.bfloat16)[0]])
def test_the_selection_bias_keeps_its_values(move):
    layer = ExpertParallelMoE(64, 32, 8, 2, True)
    # A large offset and small differences: one value in bf16 and in fp16.
    bias = torch.linspace(5.0, 5.001, 8)
    assert bias.unique().numel() == 8 and bias.bfloat16().unique().numel() == 1
    layer.set_scored_routing("sigmoid", bias)
    moved = move(layer)
    assert moved.route_bias.dtype == torch.float32
    assert torch.equal(moved.route_bias, bias)
    assert "route_bias" in dict(moved.named_buffers())


def test_the_selection_bias_follows_the_device():
    layer = ExpertParallelMoE(64, 32, 8, 2, True)
    layer.set_scored_routing("sigmoid", torch.zeros(8))
    layer.to("meta", torch.bfloat16)
    assert layer.route_bias.device.type == "meta" and layer.route_bias.dtype == torch.float32
    assert ExpertParallelMoE(64, 32, 8, 2, True).to(torch.bfloat16).route_bias is None


@pytest.fixture
def packed_by_shape(monkeypatch):
    """ops.pack_w4 without a GPU: the shapes and flags of a packed weight."""
    def pack(codes, scales, zeros=None, *, layout="rows"):
        rows, k = codes.shape[-2:]
        flags = ((_lib.W4_ZEROS if zeros is not None else 0)
                 | (_lib.W4_GATE_UP if layout == "gate_up" else 0))
        matrices = codes.size(0) if codes.dim() == 3 else 1
        group = k // scales.size(-1)
        size = _lib.LIB.b200moe_w4_bytes(matrices, rows, k, group, flags)
        return ops.W4Weight(torch.zeros(size, dtype=torch.uint8), matrices, rows, k, group, flags)
    monkeypatch.setattr(ops, "pack_w4", pack)


def layer_of(shared=None, **kw):
    layer = ExpertParallelMoE(64, 32, 8, 2, True, shared_expert_intermediate_size=shared, **kw)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0.0, 0.02, generator=torch.Generator().manual_seed(p.numel()))
    return layer.bfloat16()


@pytest.mark.parametrize("shared", [32, 64])
def test_a_shared_expert_with_4_bits_alone(packed_by_shape, shared):
    layer = layer_of(shared)
    before = layer.gate_up_proj.detach().clone(), layer.down_proj.detach().clone()
    layer.shared_expert.quantize_w4(32)
    x = torch.empty(3, 64, dtype=torch.bfloat16)
    x_on_gpu = type("OnGpu", (), {"is_cuda": True})()
    assert not layer._fused_shared(x) and not layer._fused_shared(x_on_gpu)
    moved = layer.to(torch.bfloat16).float().bfloat16()
    assert torch.equal(moved.gate_up_proj, before[0]) and torch.equal(moved.down_proj, before[1])


def state(layer):
    shared = layer.shared_expert
    return ({n: p.detach().clone() for n, p in layer.named_parameters()}, layer._w4,
            shared and shared._w4)


def same(a, b):
    return (a[0].keys() == b[0].keys() and all(torch.equal(v, b[0][n]) for n, v in a[0].items())
            and a[1:] == b[1:])


@pytest.mark.parametrize("shared", [None, 32, 64])
def test_a_refused_rounding_leaves_the_layer_as_it_was(packed_by_shape, shared):
    layer = layer_of(shared)
    layer.fp64_combine = True
    before = state(layer)
    with pytest.raises(NotImplementedError, match="FP64"):
        layer.quantize_w4(32)
    assert same(state(layer), before)
    layer.fp64_combine = False
    with pytest.raises(ValueError, match="multiple of the group size"):
        layer.quantize_w4(64)  # the routed experts' 32 k
    assert same(state(layer), before)
    layer.quantize_w4(32)
    assert layer._w4 is not None and (shared is None or layer.shared_expert._w4 is not None)


@pytest.mark.parametrize("fails", range(4))
def test_a_packing_that_fails_leaves_the_layer_as_it_was(packed_by_shape, monkeypatch, fails):
    layer, pack, calls = layer_of(64), ops.pack_w4, []

    def failing(*args, **kw):
        calls.append(args)
        if len(calls) == fails + 1:
            raise torch.OutOfMemoryError("no memory")
        return pack(*args, **kw)

    monkeypatch.setattr(ops, "pack_w4", failing)
    before = state(layer)
    with pytest.raises(torch.OutOfMemoryError):
        layer.quantize_w4(32)
    assert same(state(layer), before)


@pytest.mark.parametrize("shared", [32, 64])
def test_rounding_one_part_after_the_other_and_twice(packed_by_shape, shared):
    layer = layer_of(shared)
    layer.shared_expert.quantize_w4(32)
    held = layer.shared_expert._w4
    layer.quantize_w4(32)
    assert layer._w4 is not None and layer.shared_expert._w4 is held
    before = state(layer)
    for again in (layer, layer.shared_expert):
        with pytest.raises(RuntimeError, match="4-bit weights already"):
            again.quantize_w4(32)
    assert same(state(layer), before)


def filled(layer, seed):
    g = torch.Generator().manual_seed(seed)
    for holder in (layer, layer.shared_expert):
        for weight in (holder and holder._w4) or ():
            weight.data.copy_(torch.randint(0, 256, weight.data.shape, generator=g))
    return layer


def packed_of(layer):
    return [w for holder in (layer, layer.shared_expert) for w in (holder and holder._w4) or ()]


@pytest.mark.parametrize("shared", [None, 32, 64])
@pytest.mark.parametrize("into_rounded", [False, True])
def test_saved_and_loaded(packed_by_shape, tmp_path, shared, into_rounded):
    layer = layer_of(shared)
    layer.quantize_w4(32)
    filled(layer, 1)
    torch.save(torch.nn.ModuleDict({"mlp": layer}).state_dict(), tmp_path / "layer.pt")
    other = layer_of(shared)
    if into_rounded:
        other.quantize_w4(32)
        filled(other, 2)
        kept = [w.data.data_ptr() for w in packed_of(other)]
    with torch.no_grad():
        other.gate.weight.zero_()
    torch.nn.ModuleDict({"mlp": other}).load_state_dict(torch.load(tmp_path / "layer.pt"))
    assert torch.equal(other.gate.weight, layer.gate.weight)
    assert len(packed_of(other)) == (2 if shared is None else 4)
    for a, b in zip(packed_of(layer), packed_of(other)):
        assert torch.equal(a.data, b.data) and a.data.data_ptr() != b.data.data_ptr()
        assert (a.matrices, a.rows, a.k, a.group, a.flags) == (b.matrices, b.rows, b.k, b.group,
                                                              b.flags)
    if into_rounded:  # in place, so that captured graphs keep their pointers
        assert [w.data.data_ptr() for w in packed_of(other)] == kept
    assert other.gate_up_proj.numel() == 0
    other.to(torch.bfloat16)


def test_loading_what_does_not_fit_raises(packed_by_shape):
    rounded, plain = layer_of(32), layer_of(32)
    saved = plain.state_dict()
    assert not any("w4" in name for name in saved)
    plain.load_state_dict(saved)
    rounded.quantize_w4(32)
    with pytest.raises(RuntimeError, match="size mismatch"):
        rounded.load_state_dict(saved)  # bf16 weights into a rounded layer
    packed = rounded.state_dict()
    wider = ExpertParallelMoE(64, 64, 8, 2, True, shared_expert_intermediate_size=32)
    with torch.no_grad():
        wider.gate_up_proj.fill_(1.0)
    before = state(wider)
    with pytest.raises(RuntimeError, match="w13 must be"):
        wider.load_state_dict(packed)
    assert wider._w4 is None and torch.equal(before[0]["gate_up_proj"], wider.gate_up_proj)
    missing = {n: t for n, t in packed.items() if n != "w4_w2"}
    with pytest.raises(RuntimeError, match="w4_w2"):
        rounded.load_state_dict(missing)
    with pytest.raises(RuntimeError, match="w4_w13"):
        layer = layer_of(32)
        layer.quantize_w4(32)
        layer.load_state_dict({n: t for n, t in packed.items() if "w4" not in n})
    short = dict(packed)
    short["w4_w2"] = short["w4_w2"][:-1]
    with pytest.raises(RuntimeError, match="w4_w2"):
        rounded.load_state_dict(short)


def test_loading_into_a_layer_on_meta(packed_by_shape):
    layer = layer_of(64)
    layer.quantize_w4(32)
    saved = filled(layer, 3).state_dict()
    with torch.device("meta"):
        fresh = ExpertParallelMoE(64, 32, 8, 2, True, shared_expert_intermediate_size=64)
    torch.nn.ModuleDict({"mlp": fresh}).load_state_dict(
        {f"mlp.{n}": t for n, t in saved.items()}, assign=True)
    for a, b in zip(packed_of(layer), packed_of(fresh)):
        assert b.data.device.type == "cpu" and torch.equal(a.data, b.data)
    other = filled(layer_of(64), 4)
    other.quantize_w4(32)
    other.load_state_dict(saved, assign=True)
    assert all(torch.equal(a.data, b.data) for a, b in zip(packed_of(layer), packed_of(other)))


def test_hooks_see_and_change_the_state_dict_that_is_loaded(packed_by_shape):
    # A hook of the layer that renames what an older version saved for a part of it.
    for rounded in (False, True):
        layer, other = layer_of(64), layer_of(64)
        if rounded:
            layer.quantize_w4(32)
        saved = layer.state_dict()
        saved["shared_expert_gate.old"] = saved.pop("shared_expert_gate.weight")

        def rename(module, state_dict, prefix, *rest):
            state_dict[f"{prefix}shared_expert_gate.weight"] = state_dict.pop(
                f"{prefix}shared_expert_gate.old")

        other.register_load_state_dict_pre_hook(rename)
        with torch.no_grad():
            other.shared_expert_gate.weight.zero_()
        other.load_state_dict(saved)
        assert torch.equal(other.shared_expert_gate.weight, layer.shared_expert_gate.weight)
