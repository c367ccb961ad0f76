"""A layer whose shared expert alone has 4-bit weights, at the routed experts'
width (where the bf16 shared expert runs as one more routed expert) and at
another.  Expected: the routed output plus the gated shared expert, each from the
same kernels, so bit for bit."""

import pytest
import torch

from extend_nano_vllm_b200 import ExpertParallelMoE, device_status

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(shared):
    layer = ExpertParallelMoE(256, 128, 16, 4, True, shared_expert_intermediate_size=shared)
    layer = layer.to(device=DEV, dtype=torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(shared)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0.0, 0.05, generator=g)
    return layer


@pytest.mark.parametrize("shared", [128, 96])
@pytest.mark.parametrize("tokens", [1, 9, 130])
def test_forward_and_moves(shared, tokens):
    layer = make(shared)
    x = torch.randn((tokens, 256), generator=torch.Generator(device=DEV).manual_seed(tokens),
                    device=DEV).bfloat16()
    with torch.no_grad():
        layer(x)  # the fused form, where it applies
        layer.shared_expert.quantize_w4(32)
        want = layer._forward_local(x) + torch.sigmoid(layer.shared_expert_gate(x)) * \
            layer.shared_expert(x)
        assert torch.equal(layer(x), want)
        assert torch.equal(layer.to("cpu").to(device=DEV, dtype=torch.bfloat16)(x), want)
    assert device_status() == 0


@pytest.mark.parametrize("tokens", [1, 130])
def test_routed_experts_with_4_bits_beside_a_bf16_shared_expert(tokens):
    from extend_nano_vllm_b200 import ops

    layer = make(128)
    x = torch.randn((tokens, 256), generator=torch.Generator(device=DEV).manual_seed(1),
                    device=DEV).bfloat16()
    with torch.no_grad():
        shared = layer.shared_expert(x)
        w13 = ops.pack_w4(*ops.quantize_w4(layer.gate_up_proj.detach(), 64), layout="gate_up")
        layer.set_w4_weights(w13, ops.pack_w4(*ops.quantize_w4(layer.down_proj.detach(), 64)))
        assert torch.equal(layer.shared_expert(x), shared)
        want = layer._forward_local(x) + torch.sigmoid(layer.shared_expert_gate(x)) * shared
        assert torch.equal(layer(x), want)
        assert torch.equal(layer.to("cpu").to(DEV)(x), want)
    assert device_status() == 0


def test_rounding_in_two_steps_is_rounding_in_one():
    x = torch.randn((40, 256), generator=torch.Generator(device=DEV).manual_seed(2),
                    device=DEV).bfloat16()
    with torch.no_grad():
        one, two = make(128), make(128)
        one.quantize_w4(64)
        two.shared_expert.quantize_w4(64)
        two.quantize_w4(64)
        assert torch.equal(one(x), two(x))
        with pytest.raises(RuntimeError, match="4-bit weights already"):
            two.quantize_w4(64)
        assert torch.equal(one(x), two(x))


@pytest.mark.parametrize("shared", [128, 96])
def test_a_saved_layer_computes_the_same(shared, tmp_path):
    x = torch.randn((40, 256), generator=torch.Generator(device=DEV).manual_seed(3),
                    device=DEV).bfloat16()
    with torch.no_grad():
        layer = make(shared)
        layer.quantize_w4(32, zeros=True)
        want = layer(x)
        torch.save(layer.state_dict(), tmp_path / "layer.pt")
        saved = torch.load(tmp_path / "layer.pt", map_location="cpu")
        fresh = ExpertParallelMoE(256, 128, 16, 4, True, shared_expert_intermediate_size=shared)
        fresh = fresh.to(device=DEV, dtype=torch.bfloat16)
        fresh.load_state_dict(saved)
        assert torch.equal(fresh(x), want)
        again = make(shared)
        again.quantize_w4(32, zeros=True)
        for weight in (*again._w4, *again.shared_expert._w4):
            weight.data.zero_()
        again.load_state_dict(saved)
        assert torch.equal(again(x), want)
