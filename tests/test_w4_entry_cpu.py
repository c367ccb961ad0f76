"""Pointers that the C entry points of the 4-bit products would fault on are
refused before the device is touched."""

import ctypes

import pytest

from extend_nano_vllm_b200 import _lib


def experts(**at):
    p = {name: 1 << 20 for name in ("x", "ids", "weights", "w13", "w2", "workspace", "out")}
    p.update({name: (1 << 20) + off for name, off in at.items()})
    p = {name: ctypes.c_void_p(v) for name, v in p.items()}
    # No workspace: a call whose pointers are in order stops there.
    _lib.call("b200moe_w4_experts", p["x"], 3, 64, 64, p["ids"], p["weights"], 8, 8, p["w13"], 64,
              _lib.W4_GATE_UP, p["w2"], 64, 0, p["workspace"], 0, p["out"], None)


@pytest.mark.parametrize("name,off", [("x", 2), ("w13", 8), ("w2", 4), ("workspace", 8),
                                      ("out", 2), ("out", 8), ("ids", 4), ("weights", 1)])
def test_experts(name, off):
    with pytest.raises(ValueError, match="aligned"):
        experts(**{name: off})


def test_a_call_in_order_gets_past_the_pointers():
    with pytest.raises(ValueError, match="workspace needs"):
        experts()
    with pytest.raises(ValueError, match="workspace needs"):
        experts(ids=8, weights=2)


@pytest.mark.parametrize("x,w,out", [(2, 0, 0), (0, 8, 0), (0, 0, 1)])
def test_linear(x, w, out):
    at = [ctypes.c_void_p((1 << 20) + off) for off in (x, w, out)]
    with pytest.raises(ValueError, match="aligned"):
        _lib.call("b200moe_w4_linear", at[0], 1, 8, 64, at[1], 64, 0, at[2], None)


def test_more_experts_than_a_packing_takes():
    size = _lib.LIB.b200moe_w4_experts_workspace(3, 64, 64, 8, 4097)
    at = ctypes.c_void_p(1 << 20)
    with pytest.raises(ValueError, match="4096"):
        _lib.call("b200moe_w4_experts", at, 3, 64, 64, at, at, 8, 4097, at, 64, _lib.W4_GATE_UP,
                  at, 64, 0, at, size, at, None)
