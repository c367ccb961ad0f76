"""The products with 4-bit weights against 64-bit results on the same codes,
scales and zero points.

Tolerances.  W = s (q - z) is exact in 64 bits, and the kernels sum integers
times bf16 values in fp32: over k terms the error is at most about
k * 2^-24 * sum |x w| (every rounding at its worst), and one bf16 store adds
2^-9 of the result.  experts_w4 also stores act in bf16 (2^-9 of each act value,
carried through the second product) and its fp32 exp and division are good to
some units in 2^-23, far below that."""

import pytest
import torch

from extend_nano_vllm_b200 import device_status, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = 2.0 ** -8  # twice the largest relative error of one bf16 store


def weight(shape, group, zeros, seed, scale_dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 16, shape, generator=g, device=DEV, dtype=torch.uint8)
    per_group = (*shape[:-1], shape[-1] // group)
    scales = (torch.rand(per_group, generator=g, device=DEV) * 0.02 + 1e-3).to(scale_dtype)
    zero = (torch.randint(0, 16, per_group, generator=g, device=DEV, dtype=torch.uint8)
            if zeros else None)
    return codes, scales, zero


def exact(codes, scales, zeros):
    by = codes.double().unflatten(-1, (scales.size(-1), -1))
    z = 8.0 if zeros is None else zeros.double()[..., None]
    return ((by - z) * scales.double()[..., None]).flatten(-2)


def activations(shape, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).bfloat16()


def check_linear(x, packed, w, out=None):
    out = ops.linear_w4(x, packed) if out is None else out
    k = x.size(-1)
    ref = x.double().reshape(-1, k) @ w.T
    size = x.double().abs().reshape(-1, k) @ w.abs().T
    err = (out.double().reshape(ref.shape) - ref).abs()
    assert bool((err <= BF16 * ref.abs() + k * 2.0 ** -24 * size).all())
    assert device_status() == 0


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 16, 17, 63, 130, 300])
def test_linear_rows(m, group, zeros):
    parts = weight((200, 384), group, zeros, seed=m + group)
    check_linear(activations((m, 384), m), ops.pack_w4(*parts), exact(*parts))


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (7, 96, 32), (128, 128, 128), (129, 192, 64),
                                       (1000, 2048, 32), (257, 4224, 128), (64, 8320, 64),
                                       (96, 12320, 32)])
@pytest.mark.parametrize("m", [1, 9, 33])
def test_linear_shapes(m, n, k, group):
    parts = weight((n, k), group, n % 2 == 1, seed=n)
    check_linear(activations((m, k), n), ops.pack_w4(*parts), exact(*parts))


@pytest.mark.parametrize("group,zeros", [(128, False), (64, True), (32, True)])
@pytest.mark.parametrize("m,n,k", [(128, 38016, 128), (200, 19328, 384), (513, 7816, 320),
                                   (1000, 4744, 1152)])
def test_linear_many_tiles(m, n, k, group, zeros):
    # Enough 128-row tiles that two CTAs work on a pair of weight tiles: an odd
    # number of tiles, ragged rows and features, k inside a block.
    if k % group:
        pytest.skip("k is not a multiple of this group size")
    parts = weight((n, k), group, zeros, seed=n)
    check_linear(activations((m, k), n), ops.pack_w4(*parts), exact(*parts))


@pytest.mark.parametrize("m", [1, 40])
def test_linear_fp16_scales(m):
    parts = weight((140, 256), 64, True, seed=3, scale_dtype=torch.float16)
    check_linear(activations((m, 256), 4), ops.pack_w4(*parts), exact(*parts))


@pytest.mark.parametrize("m", [1, 21])
def test_linear_codes_and_zeros_at_their_ends(m):
    codes = torch.zeros((130, 256), device=DEV, dtype=torch.uint8)
    codes[:, ::2] = 15
    scales = torch.full((130, 8), 0.5, device=DEV).bfloat16()
    scales[5] = 0
    zeros = torch.zeros((130, 8), device=DEV, dtype=torch.uint8)
    zeros[::3] = 15
    check_linear(activations((m, 256), 5), ops.pack_w4(codes, scales, zeros),
                 exact(codes, scales, zeros))


def test_linear_shapes_of_x_strides_and_streams():
    parts = weight((72, 160), 32, False, seed=9)
    packed, w = ops.pack_w4(*parts), exact(*parts)
    base = activations((6, 4, 320), 10)
    check_linear(base[:, :, ::2], packed, w)                     # strided
    check_linear(base.view(-1)[3:3 + 160 * 5].view(5, 160), packed, w)  # off a 16-byte address
    empty = ops.linear_w4(base[:0, :, :160], packed)
    assert empty.shape == (0, 4, 72)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = ops.linear_w4(base[0, :, :160], packed)
    stream.synchronize()
    check_linear(base[0, :, :160], packed, w, out)


@pytest.mark.parametrize("m", [1, 30])
def test_linear_infinite_and_nan_rows_stay_apart(m):
    # A row of x with NaN or infinities must not reach the other rows.
    parts = weight((150, 256), 128, False, seed=11)
    x = activations((m + 2, 256), 12)
    x[0, 3] = float("nan")
    x[1, 7] = float("inf")
    out = ops.linear_w4(x, ops.pack_w4(*parts))
    check_linear(x[2:], ops.pack_w4(*parts), exact(*parts), out[2:])
    assert bool(out[0].isnan().all())


def routed(tokens, experts, top_k, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    scores = torch.rand((tokens, experts), generator=g, device=DEV)
    top = scores.topk(top_k, -1)
    return top.indices, (top.values / top.values.sum(-1, keepdim=True)).bfloat16()


def check_experts(x, ids, weights, parts13, parts2, packed=None):
    w13, w2 = packed or (ops.pack_w4(*parts13, layout="gate_up"), ops.pack_w4(*parts2))
    out = ops.experts_w4(x, ids, weights, w13, w2)
    experts, hidden, inter = parts2[0].shape
    ref = torch.zeros_like(x, dtype=torch.float64)
    size = torch.zeros_like(ref)
    for e in range(experts):
        token, slot = torch.where(ids == e)
        if not token.numel():
            continue
        part = lambda w: tuple(None if t is None else t[e] for t in w)  # noqa: E731
        a, b = exact(*part(parts13)), exact(*part(parts2))
        xt = x[token].double()
        gate, up = (xt @ a.T).chunk(2, -1)
        # What fp32 sums over `hidden` terms can be off by, through the product.
        mag = xt.abs() @ a.abs().T
        slack = hidden * 2.0 ** -24 * mag
        act = gate * torch.sigmoid(gate) * up
        off = (BF16 * act.abs() + 1.1 * slack[:, :inter] * up.abs()
               + slack[:, inter:] * (gate * torch.sigmoid(gate)).abs()
               + 2.0 ** -19 * act.abs())
        wgt = weights[token, slot].double()[:, None]
        ref.index_add_(0, token, act @ b.T * wgt)
        size.index_add_(0, token, (off @ b.abs().T + inter * 2.0 ** -24 * (act.abs() @ b.abs().T))
                        * wgt)
    err = (out.double() - ref).abs()
    assert bool((err <= BF16 * ref.abs() + size).all())
    assert device_status() == 0
    return out


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("tokens", [1, 2, 3, 8, 33, 130, 700])
def test_experts(tokens, group, zeros):
    hidden, inter, experts, top_k = 256, 128, 16, 4
    parts13 = weight((experts, 2 * inter, hidden), group, zeros, seed=group)
    parts2 = weight((experts, hidden, inter), group, not zeros, seed=group + 1)
    ids, weights = routed(tokens, experts, top_k, tokens)
    check_experts(activations((tokens, hidden), tokens), ids, weights, parts13, parts2)


@pytest.mark.parametrize("hidden,inter,experts,top_k,tokens", [
    (96, 32, 3, 1, 1), (96, 32, 3, 1, 50), (160, 96, 8, 8, 5), (512, 224, 40, 6, 61),
    (1056, 352, 5, 3, 200), (128, 64, 512, 10, 16), (320, 160, 2, 2, 515)])
def test_experts_odd_shapes(hidden, inter, experts, top_k, tokens):
    parts13 = weight((experts, 2 * inter, hidden), 32, True, seed=hidden)
    parts2 = weight((experts, hidden, inter), 32, False, seed=inter)
    ids, weights = routed(tokens, experts, top_k, tokens)
    check_experts(activations((tokens, hidden), 1), ids, weights, parts13, parts2)


@pytest.mark.parametrize("group,zeros", [(128, False), (32, True)])
@pytest.mark.parametrize("hidden,inter,experts,top_k,tokens", [
    (1152, 640, 4, 2, 1000), (640, 128, 8, 2, 4100), (2048, 384, 6, 3, 1030)])
def test_experts_prefill(hidden, inter, experts, top_k, tokens, group, zeros):
    # Hundreds of rows per expert: whole tiles, part tiles, pairs of CTAs, and
    # (with 4100 tokens and two routes each) the packing of many routes.
    parts13 = weight((experts, 2 * inter, hidden), group, zeros, seed=hidden)
    parts2 = weight((experts, hidden, inter), group, False, seed=inter)
    ids, weights = routed(tokens, experts, top_k, tokens)
    ids[7] = experts  # a token that was dropped
    check_experts(activations((tokens, hidden), 1), ids, weights, parts13, parts2)


@pytest.mark.parametrize("group,zeros", [(128, False), (64, True), (32, True)])
@pytest.mark.parametrize("hidden,inter,experts,top_k,tokens", [
    (640, 256, 4, 4, 9), (384, 1280, 3, 2, 16),       # few experts, passes of 16 rows
    (384, 256, 32, 4, 40), (384, 256, 32, 4, 48),     # five and six rows on average
    (256, 2304, 16, 4, 24), (256, 384, 64, 2, 130)])  # long rows; four rows on average
def test_experts_of_few_rows(hidden, inter, experts, top_k, tokens, group, zeros):
    parts13 = weight((experts, 2 * inter, hidden), group, zeros, seed=hidden)
    parts2 = weight((experts, hidden, inter), group, not zeros, seed=inter)
    packed = ops.pack_w4(*parts13, layout="gate_up"), ops.pack_w4(*parts2)
    ids, weights = routed(tokens, experts, top_k, tokens)
    x = activations((tokens, hidden), 1)
    check_experts(x, ids, weights, parts13, parts2, packed)
    ids[:, 0], ids[:, 1] = 1, 2  # two experts with every token: passes over them
    for s in range(2, top_k):
        ids[:, s] = experts
    check_experts(x, ids, weights, parts13, parts2, packed)


@pytest.mark.parametrize("tokens", [2, 90])
def test_experts_dropped_routes_and_one_full_expert(tokens):
    hidden, inter, experts, top_k = 128, 128, 8, 2
    parts13 = weight((experts, 2 * inter, hidden), 64, False, seed=1)
    parts2 = weight((experts, hidden, inter), 64, True, seed=2)
    ids, weights = routed(tokens, experts, top_k, 3)
    ids[0] = experts       # a token whose routes were all dropped
    ids[1, 1] = experts
    out = check_experts(activations((tokens, hidden), 4), ids, weights, parts13, parts2)
    assert bool((out[0] == 0).all())
    ids[:, 0] = 5          # every token to one expert
    ids[:, 1] = 6
    check_experts(activations((tokens, hidden), 5), ids, weights, parts13, parts2)
    ids[:] = experts       # nothing left at all
    out = check_experts(activations((tokens, hidden), 6), ids, weights, parts13, parts2)
    assert bool((out == 0).all())


def test_experts_no_tokens():
    parts13 = weight((4, 128, 64), 64, False, seed=1)
    parts2 = weight((4, 64, 64), 64, False, seed=2)
    out = ops.experts_w4(activations((0, 64), 0), torch.empty((0, 2), device=DEV, dtype=torch.int64),
                         torch.empty((0, 2), device=DEV, dtype=torch.bfloat16),
                         ops.pack_w4(*parts13, layout="gate_up"), ops.pack_w4(*parts2))
    assert out.shape == (0, 64)


@pytest.mark.parametrize("tokens", [1, 48, 300])
def test_experts_repeat_bit_for_bit_and_replay_in_a_graph(tokens):
    hidden, inter, experts, top_k = 512, 256, 24, 4
    parts13 = weight((experts, 2 * inter, hidden), 128, False, seed=1)
    parts2 = weight((experts, hidden, inter), 128, False, seed=2)
    packed = ops.pack_w4(*parts13, layout="gate_up"), ops.pack_w4(*parts2)
    ids, weights = routed(tokens, experts, top_k, 3)
    x = activations((tokens, hidden), 4)
    first = check_experts(x, ids, weights, parts13, parts2, packed)
    for _ in range(3):
        assert torch.equal(first, ops.experts_w4(x, ids, weights, *packed))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.experts_w4(x, ids, weights, *packed)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.experts_w4(x, ids, weights, *packed)
    other_ids, other_weights = routed(tokens, experts, top_k, 7)
    ids.copy_(other_ids)
    weights.copy_(other_weights)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, check_experts(x, ids, weights, parts13, parts2, packed))


@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_then_linear_is_near_the_weight(zeros):
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn((96, 256), generator=g, device=DEV) * 0.02
    w[3] = 0
    codes, scales, zero = ops.quantize_w4(w, 64, zeros)
    # Rounding to the nearest code is off by half a step, and a bf16 scale
    # (2^-9) shifts the end codes by at most 15 * 2^-9 of a step more.
    step = scales.double().repeat_interleave(64, -1)
    assert bool(((exact(codes, scales, zero) - w.double()).abs()
                 <= step * (0.5 + (0.5 if zeros else 0) + 15 * 2.0 ** -8) + 1e-9).all())
    check_linear(activations((3, 256), 2), ops.pack_w4(codes, scales, zero),
                 exact(codes, scales, zero))


def test_refusals():
    codes, scales, zero = weight((64, 128), 64, True, seed=1)
    x = activations((2, 128), 1)
    packed = ops.pack_w4(codes, scales, zero)
    with pytest.raises(TypeError, match="codes"):
        ops.pack_w4(codes.int(), scales)
    with pytest.raises(TypeError, match="scales"):
        ops.pack_w4(codes, scales.float())
    with pytest.raises(ValueError, match="scales"):
        ops.pack_w4(codes, scales[:32])
    with pytest.raises(TypeError, match="zeros"):
        ops.pack_w4(codes, scales, zero[:, :1])
    with pytest.raises(ValueError, match="layout"):
        ops.pack_w4(codes, scales, layout="columns")
    with pytest.raises(ValueError, match="groups of 16"):
        ops.pack_w4(codes, scales.repeat(1, 4))
    with pytest.raises(ValueError, match="even number of rows"):
        ops.pack_w4(codes[:63], scales[:63], layout="gate_up")
    with pytest.raises(TypeError, match="bf16 activations"):
        ops.linear_w4(x.half(), packed)
    with pytest.raises(ValueError, match="k = 128"):
        ops.linear_w4(x[:, :64], packed)
    with pytest.raises(ValueError, match="rows"):
        ops.linear_w4(x, ops.pack_w4(codes, scales, layout="gate_up"))
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.linear_w4(x.cpu(), packed)
    w13 = ops.pack_w4(*weight((4, 128, 128), 64, False, seed=2), layout="gate_up")
    w2 = ops.pack_w4(*weight((4, 128, 64), 64, False, seed=3))
    ids, weights = routed(2, 4, 2, 1)
    with pytest.raises(TypeError, match="expert_ids"):
        ops.experts_w4(x, ids.int(), weights, w13, w2)
    with pytest.raises(TypeError, match="route_weights"):
        ops.experts_w4(x, ids, weights.float(), w13, w2)
    with pytest.raises(ValueError, match="gate_up"):
        ops.experts_w4(x, ids, weights, w2, w13) if w2.k == 128 else ops.experts_w4(
            x, ids, weights, ops.pack_w4(*weight((4, 128, 128), 64, False, seed=2)), w2)
    with pytest.raises(ValueError, match="w2 must be"):
        ops.experts_w4(x, ids, weights, w13, ops.pack_w4(*weight((3, 128, 64), 64, False, seed=3)))
