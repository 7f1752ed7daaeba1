"""Which stacks of experts are registered (no device is touched): none whose
layout kernel's 32-bit offsets in a tile would not hold, and none so wide that
every call would decline it."""
import ctypes

import pytest

WIDEST = 523744  # (2^24 - 1) / 1025 column ranges of 32, less one


def status(q8, experts, rows, cols):
    fn = q8.lib().llmcp_q8_test_expert_stack
    fn.argtypes, fn.restype = [ctypes.c_int64] * 3, ctypes.c_int
    return fn(experts, rows, cols)


@pytest.mark.parametrize("experts,rows,cols", [
    (1, 8, 32), (1024, 768, 2560), (4, 16, 45056), (1, 8, WIDEST // 32 * 32), (1, WIDEST // 8 * 8, 32)])
def test_taken(q8, experts, rows, cols):
    assert status(q8, experts, rows, cols) == q8.OK


# a tile's values of 2 KiB per 128 of cols: 2^31 bytes at 2^27, where the
# expert's copy (2.28 GB) stays below 4 GiB
@pytest.mark.parametrize("experts,rows,cols", [
    (1, 8, 1 << 27), (1, 8, (1 << 27) - 32), (2, 16, (1 << 27) + 4096), (1, 8, WIDEST + 32),
    (1, WIDEST + 8, 32), (1, 1 << 30, 32), (1, 1 << 40, 32), (1, 8, 1 << 40), (1, 1 << 20, 8192),
    (0, 8, 32), (1025, 8, 32), (1, 12, 32), (1, 8, 48)])
def test_declined(q8, experts, rows, cols):
    assert status(q8, experts, rows, cols) == q8.DECLINED


@pytest.mark.parametrize("cols", [32, 128, 2560, WIDEST])
def test_offsets_in_a_tile_of_a_taken_stack(q8, cols):
    """What the layout kernel computes in int: the scales' place behind a
    tile's values, and the last of them."""
    steps = (cols // 32 + 3) // 4
    assert status(q8, 1, 8, cols) == q8.OK
    assert steps * 2048 + steps * 128 < 1 << 31
