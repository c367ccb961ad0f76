"""Experts with fp16 scales (every kernel of both engines: few routes, streamed
rows, tcgen05 tiles), and with scales that only one of the two types holds.

The bounds are those of the bf16-scale tests: W = s (q - z) is exact in 64 bits;
fp32 sums of k terms are off by at most about k 2^-24 sum |x w|; act and the result
are stored in bf16 (2^-9 each, covered twice over by 2^-8)."""

import pytest
import torch

from extend_nano_vllm_b200 import device_status, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = 2.0 ** -8


def parts_of(shape, group, zeros, seed, dtype, span=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 16, shape, generator=g, device=DEV, dtype=torch.uint8)
    per = (*shape[:-1], shape[-1] // group)
    scales = ((torch.rand(per, generator=g, device=DEV) * 0.02 + 1e-3) * span).to(dtype)
    zero = torch.randint(0, 16, per, generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return codes, scales, zero


def exact(codes, scales, zeros):
    by = codes.double().unflatten(-1, (scales.size(-1), -1))
    z = 8.0 if zeros is None else zeros.double()[..., None]
    return ((by - z) * scales.double()[..., None]).flatten(-2)


@pytest.mark.parametrize("dtypes", [(torch.float16, torch.float16),
                                    (torch.float16, torch.bfloat16),
                                    (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("tokens", [1, 4, 33, 300])
def test_experts(tokens, group, zeros, dtypes):
    hidden, inter, experts, top_k = 384, 256, 16, 4
    p13 = parts_of((experts, 2 * inter, hidden), group, zeros, group, dtypes[0])
    p2 = parts_of((experts, hidden, inter), group, not zeros, group + 1, dtypes[1])
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x = torch.randn((tokens, hidden), generator=g, device=DEV).bfloat16()
    top = torch.rand((tokens, experts), generator=g, device=DEV).topk(top_k, -1)
    ids, weights = top.indices, (top.values / top.values.sum(-1, keepdim=True)).bfloat16()
    out = ops.experts_w4(x, ids, weights, ops.pack_w4(*p13, layout="gate_up"), ops.pack_w4(*p2))
    a, b = exact(*p13), exact(*p2)
    ref, room = torch.zeros_like(x, dtype=torch.float64), torch.zeros_like(x, dtype=torch.float64)
    for e in range(experts):
        token, slot = torch.where(ids == e)
        xt, w = x[token].double(), weights[token, slot].double()[:, None]
        gate, up = (xt @ a[e].T).chunk(2, -1)
        off_gate, off_up = (hidden * 2.0 ** -24 * (xt.abs() @ a[e].abs().T)).chunk(2, -1)
        silu = gate * torch.sigmoid(gate)
        act = silu * up
        # The slope of silu is below 1.1; fast exp and division: 2^-19 of act.
        off = (BF16 + 2.0 ** -19) * act.abs() + 1.1 * off_gate * up.abs() + silu.abs() * off_up
        ref.index_add_(0, token, act @ b[e].T * w)
        room.index_add_(0, token, (off + inter * 2.0 ** -24 * act.abs()) @ b[e].abs().T * w)
    assert bool(((out.double() - ref).abs() <= BF16 * ref.abs() + room).all())
    assert device_status() == 0


@pytest.mark.parametrize("dtype,span", [(torch.float16, 2.0 ** -14), (torch.float16, 2.0 ** 20),
                                        (torch.bfloat16, 2.0 ** -60), (torch.bfloat16, 2.0 ** 60)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 16, 40, 130])
def test_linear_with_small_and_large_scales(m, group, dtype, span):
    # fp16 subnormals and its largest values; bf16 far from 1.
    p = parts_of((200, 256), group, True, m, dtype, span)
    x = torch.randn((m, 256), generator=torch.Generator(device=DEV).manual_seed(m),
                    device=DEV).bfloat16()
    out, w = ops.linear_w4(x, ops.pack_w4(*p)), exact(*p)
    ref, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    assert bool(((out.double() - ref).abs() <= BF16 * ref.abs() + 256 * 2.0 ** -24 * size).all())
    assert device_status() == 0
