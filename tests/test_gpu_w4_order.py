"""4-bit weights that are packed or updated by the kernel right before the product
that reads them: the products wait for it like for any other operand.  Every
comparison is exact, with the same product of weights that were finished long
before."""

import pytest
import torch

from extend_nano_vllm_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def codes_of(shape, group, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 16, shape, generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.rand((*shape[:-1], shape[-1] // group), generator=g, device=DEV) * 0.02 + 1e-3
    return codes, scales.bfloat16()


@pytest.mark.parametrize("m", [1, 12, 40, 200])
def test_linear_right_after_packing_and_updating(m):
    n, k, group = 4096, 2048, 64
    g = torch.Generator(device=DEV).manual_seed(m)
    x = torch.randn((m, k), generator=g, device=DEV).bfloat16()
    parts = [codes_of((n, k), group, seed) for seed in range(4)]
    finished = [ops.pack_w4(*p) for p in parts]
    torch.cuda.synchronize()
    want = [ops.linear_w4(x, w) for w in finished]
    torch.cuda.synchronize()
    live = ops.pack_w4(*parts[0])
    got = []
    for turn in range(12):
        if turn % 2:
            live.data.copy_(finished[turn % 4].data)
            got.append(ops.linear_w4(x, live))
        else:
            got.append(ops.linear_w4(x, ops.pack_w4(*parts[turn % 4])))
    for turn, out in enumerate(got):
        assert torch.equal(out, want[turn % 4]), f"turn {turn}"


@pytest.mark.parametrize("tokens", [1, 24, 300])
def test_experts_right_after_packing_and_updating(tokens):
    experts, hidden, inter, top_k, group = 16, 512, 256, 4, 64
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x = torch.randn((tokens, hidden), generator=g, device=DEV).bfloat16()
    top = torch.rand((tokens, experts), generator=g, device=DEV).topk(top_k, -1)
    ids, weights = top.indices, top.values.bfloat16()
    parts = [(codes_of((experts, 2 * inter, hidden), group, seed),
              codes_of((experts, hidden, inter), group, 10 + seed)) for seed in range(2)]
    finished = [(ops.pack_w4(*a, layout="gate_up"), ops.pack_w4(*b)) for a, b in parts]
    torch.cuda.synchronize()
    want = [ops.experts_w4(x, ids, weights, *w) for w in finished]
    torch.cuda.synchronize()
    live = ops.pack_w4(*parts[0][0], layout="gate_up"), ops.pack_w4(*parts[0][1])
    for turn in range(8):
        for part, source in zip(live, finished[turn % 2]):
            part.data.copy_(source.data)
        assert torch.equal(ops.experts_w4(x, ids, weights, *live), want[turn % 2]), f"turn {turn}"
        fresh = ops.pack_w4(*parts[turn % 2][0], layout="gate_up"), ops.pack_w4(*parts[turn % 2][1])
        assert torch.equal(ops.experts_w4(x, ids, weights, *fresh), want[turn % 2]), f"turn {turn}"
