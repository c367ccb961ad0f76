"""The stages of the tcgen05 product with 4-bit weights, without a GPU.

Two groups of warps decode alternate blocks of k, and a wait on a stage goes by
the parity of its use.  Use u of a stage and use u - 2 have the same parity, so a
group may ask for use u only when it knows that use u - 1 has landed.  What the
group that decodes block b knows: its own earlier blocks b - 2, b - 4, ... landed,
and so did every block up to b - 2 - (operand stages), whose products had ended
when it took the operand stage of block b - 2."""

import ctypes
import itertools

import pytest

from extend_nano_vllm_b200 import _lib

GROUPS = 2


def stages(product, rows, group, flags, split):
    code, operand = ctypes.c_int(), ctypes.c_int()
    _lib.call("b200moe_w4_ring_stages", product, rows, group, flags, split, ctypes.byref(code),
              ctypes.byref(operand))
    return code.value, operand.value


def configurations():
    for product, rows, group, flags, split in itertools.product(
            range(3), (32, 64, 128), (32, 64, 128), (0, _lib.W4_ZEROS), (1, 2, 4)):
        if (split - 1) * rows <= 112:
            yield product, rows, group, flags, split


@pytest.mark.parametrize("product,rows,group,flags,split", list(configurations()))
def test_a_wait_cannot_pass_on_an_older_use(product, rows, group, flags, split):
    code, operand = stages(product, rows, group, flags, split)
    assert code >= GROUPS and operand >= GROUPS
    for block in range(2 * code, 6 * code):
        landed = set(range(block % GROUPS, block, GROUPS))
        landed.update(range(block - GROUPS - operand + 1))
        assert block - code in landed, f"block {block}: {code} stages, {operand} of operands"
        # The operand stages: use u - 1 of block's stage is that of block - operand, and the
        # group saw the products of every block up to block - 2 - operand end.
        assert block - 2 * operand <= block - GROUPS - operand


def test_refusals():
    for bad, message in (((3, 64, 32, 0, 1), "product"), ((0, 16, 32, 0, 1), "tile of 16"),
                         ((0, 64, 16, 0, 1), "group size"), ((0, 128, 32, 0, 2), "clusters"),
                         ((0, 32, 32, 0, 3), "clusters")):
        with pytest.raises(ValueError, match=message):
            stages(*bad)
