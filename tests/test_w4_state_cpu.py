"""What a layer with scored routing and 4-bit weights keeps through device and
dtype moves and through calls that are refused, without a GPU.  Packing is
replaced by a stand-in that keeps the shapes; nothing is computed."""

import pytest
import torch

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
