"""4-bit weights and scored routing without a GPU: rounding, sizes of the
layout, and what the C entry points and the layer refuse before the device is
touched."""

import ctypes

import pytest
import torch

from extend_nano_vllm_b200 import _lib, ops
from extend_nano_vllm_b200.moe import ExpertParallelMoE

NULL = ctypes.c_void_p(0)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_rounding_is_to_the_nearest_code(group, zeros):
    g = torch.Generator().manual_seed(group)
    w = torch.randn((3, 16, 256), generator=g, dtype=torch.float32) * 0.02
    w[0, 0] = 0
    codes, scales, zero = ops.quantize_w4(w, group, zeros)
    assert codes.dtype == torch.uint8 and int(codes.max()) <= 15
    assert scales.shape == (3, 16, 256 // group) and scales.dtype == torch.bfloat16
    assert (zero is None) != zeros
    s = scales.double().repeat_interleave(group, -1)
    z = 8.0 if zero is None else zero.double().repeat_interleave(group, -1)
    back = (codes.double() - z) * s
    # No other code of the group is nearer (fp32 division and ties: a hair).
    for step in (-1, 1):
        other = (codes.double() + step - z) * s
        allowed = (codes.double() + step >= 0) & (codes.double() + step <= 15)
        nearer = (other - w.double()).abs() < (back - w.double()).abs() - 1e-6 * s.abs()
        assert not bool((nearer & allowed).any())
    assert bool((back[0, 0] == 0).all())


def test_rounding_refusals():
    with pytest.raises(ValueError, match="group size 16"):
        ops.quantize_w4(torch.zeros(4, 64), 16)
    with pytest.raises(ValueError, match="multiple of the group size"):
        ops.quantize_w4(torch.zeros(4, 96), 64)


def test_layout_sizes():
    size = _lib.LIB.b200moe_w4_bytes
    # Tiles of 128 rows, blocks of 128 k: 8192 bytes of codes, 256 of scales and
    # 128 of zero points per group and tile.
    assert size(1, 128, 128, 128, 0) == 8192 + 256
    assert size(1, 129, 128, 128, 0) == 2 * (8192 + 256)
    assert size(1, 1, 32, 32, 0) == 8192 + 4 * 256
    assert size(3, 256, 320, 64, _lib.W4_ZEROS) == 3 * 2 * 3 * (8192 + 2 * 384)
    # A gate/up tile holds 64 features of each.
    assert size(2, 2 * 96, 256, 128, _lib.W4_GATE_UP) == 2 * 2 * 2 * (8192 + 256)
    for bad in ((0, 128, 128, 128, 0), (1, 0, 128, 128, 0), (1, 128, 128, 16, 0),
                (1, 128, 100, 32, 0), (1, 129, 128, 128, _lib.W4_GATE_UP)):
        assert size(*bad) == -1


def test_entry_points_refuse_without_a_device():
    with pytest.raises(ValueError, match="top_k"):
        _lib.call("b200moe_route_scored_topk", NULL, _lib.F32, 4, 8, 9, 0, NULL, 1, 1, 0, 1, 1.0,
                  NULL, NULL, NULL)
    with pytest.raises(ValueError, match="divide"):
        _lib.call("b200moe_route_scored_topk", NULL, _lib.F32, 4, 8, 2, 0, NULL, 3, 1, 0, 1, 1.0,
                  NULL, NULL, NULL)
    with pytest.raises(ValueError, match="score function"):
        _lib.call("b200moe_route_scored_topk", NULL, _lib.F32, 4, 8, 2, 7, NULL, 1, 1, 0, 1, 1.0,
                  NULL, NULL, NULL)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call("b200moe_route_scored_topk", NULL, _lib.F32, 4, 8, 2, 0, NULL, 1, 1, 0, 1, 1.0,
                  NULL, NULL, NULL)
    with pytest.raises(ValueError, match="group size"):
        _lib.call("b200moe_w4_linear", NULL, 1, 8, 64, NULL, 48, 0, NULL, NULL)
    with pytest.raises(ValueError, match="multiple of the group size"):
        _lib.call("b200moe_w4_linear", NULL, 1, 8, 96, NULL, 64, 0, NULL, NULL)
    with pytest.raises(ValueError, match="plain row order"):
        _lib.call("b200moe_w4_linear", NULL, 1, 8, 64, NULL, 64, _lib.W4_GATE_UP, NULL, NULL)
    with pytest.raises(ValueError, match="zero points"):
        _lib.call("b200moe_w4_pack", ctypes.c_void_p(16), ctypes.c_void_p(16), NULL, 1, 8, 64, 64,
                  _lib.W4_ZEROS, ctypes.c_void_p(16), NULL)
    with pytest.raises(ValueError, match="gate_up row order"):
        _lib.call("b200moe_w4_experts", NULL, 1, 64, 64, NULL, NULL, 1, 4, NULL, 64, 0, NULL, 64,
                  0, NULL, 0, NULL, NULL)
    with pytest.raises(ValueError, match="workspace"):
        p = ctypes.c_void_p(4096)
        _lib.call("b200moe_w4_experts", p, 1, 64, 64, p, p, 1, 4, p, 64, _lib.W4_GATE_UP, p, 64,
                  0, p, 16, p, NULL)


def test_workspace_and_launches():
    ws = _lib.LIB.b200moe_w4_experts_workspace
    assert ws(2, 256, 128, 8, 64) == 16 * 128 * 2      # route by route: act alone
    assert ws(0, 256, 128, 8, 64) == 0 and ws(-1, 256, 128, 8, 64) == -1
    assert ws(3, 256, 128, 8, 64) >= 24 * 256 * 4      # fp32 rows of the down product
    launches = _lib.LIB.b200moe_w4_experts_launches
    assert [launches(t, 8, 64) for t in (0, 2, 3, 64, 65, 1024, 1025)] == [0, 2, 4, 4, 5, 5, 6]


def test_layer_refusals():
    layer = ExpertParallelMoE(64, 32, 8, 2, True, ep_rank=0, ep_size=2)
    with pytest.raises(NotImplementedError, match="one EP rank"):
        layer.quantize_w4(32)
    with pytest.raises(ValueError, match="score function"):
        layer.set_scored_routing("softplus")
    with pytest.raises(ValueError, match="divide"):
        layer.set_scored_routing(num_groups=3)
    with pytest.raises(ValueError, match="topk_groups"):
        layer.set_scored_routing(num_groups=4, topk_groups=5)
    with pytest.raises(ValueError, match="experts of topk_groups"):
        ExpertParallelMoE(64, 32, 8, 4, True).set_scored_routing(num_groups=4, topk_groups=1)
    with pytest.raises(ValueError, match="one value per expert"):
        layer.set_scored_routing(bias=torch.zeros(7))
    layer.set_scored_routing(bias=torch.zeros(8, dtype=torch.bfloat16))
    assert layer.route_bias.dtype == torch.float32
    assert layer.to(torch.bfloat16).route_bias.dtype == torch.float32
    assert "route_bias" not in layer.state_dict()
    one = ExpertParallelMoE(64, 32, 8, 2, True)
    fake = ops.W4Weight(torch.empty(0, dtype=torch.uint8), 8, 64, 64, 32, 0)
    with pytest.raises(ValueError, match="gate_up"):
        one.set_w4_weights(fake, fake)
