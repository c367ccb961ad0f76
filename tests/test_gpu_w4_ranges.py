"""Codes and zero points outside 0..15 are refused, and recorded on the device
where the host cannot look."""

import pytest
import torch

from extend_nano_vllm_b200 import _lib, device_status, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def parts(rows=130, k=192, group=64):
    g = torch.Generator(device=DEV).manual_seed(1)
    codes = torch.randint(0, 16, (rows, k), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.full((rows, k // group), 0.5, device=DEV).bfloat16()
    zeros = torch.randint(0, 16, scales.shape, generator=g, device=DEV, dtype=torch.uint8)
    return codes, scales, zeros


@pytest.mark.parametrize("which,name", [(0, "codes"), (2, "zeros")])
@pytest.mark.parametrize("value", [16, 128, 255])
def test_values_above_15_are_refused(which, name, value):
    p = parts()
    p[which][129, -1] = value
    with pytest.raises(ValueError, match=f"{name} must be 0..15, got {value}"):
        ops.pack_w4(*p)
    assert device_status() == 0


@pytest.mark.parametrize("which", [None, 0, 2])
@pytest.mark.parametrize("flags", [0, _lib.W4_GATE_UP])
def test_the_c_call_records_them(which, flags):
    p = parts()
    if which is not None:
        p[which][129, -1] = 16
    flags |= _lib.W4_ZEROS
    out = torch.empty(_lib.LIB.b200moe_w4_bytes(1, 130, 192, 64, flags), device=DEV,
                      dtype=torch.uint8)
    _lib.call("b200moe_w4_pack", *(ops._p(t) for t in p), 1, 130, 192, 64, flags, ops._p(out),
              ops._stream(out))
    assert device_status(clear=True) == (0 if which is None else 2)
    assert device_status() == 0


def test_packing_under_capture():
    p = parts()
    want = ops.pack_w4(*p)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.pack_w4(*p)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        packed = ops.pack_w4(*p)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(packed.data, want.data)
