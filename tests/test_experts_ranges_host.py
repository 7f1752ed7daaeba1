"""How the experts' products divide an expert's columns over workgroups (no
device is touched)."""
import ctypes

import numpy as np
import pytest


def ranges(q8, slots, experts, rows, widest, dual=False, forced=0):
    """(slots per tile, planned, workgroups side by side, ranges of each)."""
    fn = q8.lib().llmcp_q8_test_expert_ranges
    fn.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_int32] * 2 + [ctypes.c_void_p] * 3
    out = (ctypes.c_int32 * 3)()
    at = [ctypes.addressof(out) + 4 * i for i in range(3)]
    repeat = fn(slots, experts, rows, widest, int(dual), forced, *at)
    return out[0], bool(out[1]), out[2], repeat


def columns(tile_rows, dual):
    return (32 if dual else 64) * (1 if tile_rows <= 16 else 2)


def test_ranges_cover_the_columns(q8):
    """Every workgroup has a range with columns, and together they have all;
    so with every forced count."""
    rng = np.random.default_rng(0)
    for _ in range(3000):
        slots, experts = (int(2 ** rng.uniform(0, 15)) for _ in range(2))
        experts = min(experts, 1024)
        rows = 8 * int(2 ** rng.uniform(0, 11))
        dual, forced = bool(rng.random() < 0.5), int(rng.choice([0, 0, 1, 2, 3, 7, 1000]))
        tile, _, n, repeat = ranges(q8, slots, experts, rows, max(rows, 64), dual, forced)
        groups = -(-rows // columns(tile, dual))
        assert n >= 1 and repeat >= 1
        assert (n - 1) * repeat < groups <= n * repeat
        if forced:
            assert repeat <= forced


@pytest.mark.parametrize("slots,experts,rows,widest,dual,tile,repeat", [
    (128, 128, 2560, 2560, False, 4, 2),       # 16 tokens of 8: down
    (128, 128, 768, 2560, True, 4, 1),         # their gate and up
    (128, 128, 1536, 2560, True, 4, 3),        # twice as wide
    (32768, 128, 2560, 2560, False, 64, 2),    # 4096 tokens of 8: down
    (32768, 128, 768, 2560, True, 64, 1),
    (640, 32, 2560, 2560, False, 32, 1)])
def test_ranges_of_sizes(q8, slots, experts, rows, widest, dual, tile, repeat):
    """On 256 CUs."""
    got = ranges(q8, slots, experts, rows, widest, dual)
    assert (got[0], got[3]) == (tile, repeat)
