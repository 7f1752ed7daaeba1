"""Expert products whose workgroups take several column ranges one after another
(chosen for many tiles, forced here on small ones): the ring of weights carried
from one range to the next, the h rows and their Q8_1 written once per range, a
last workgroup with fewer ranges than the others, slots without an expert.
Bit for bit the linear of each slot's expert (Q8Matmul.cpp:204-223)."""
import ctypes

import numpy as np
import pytest

from test_experts_ranges_host import columns, ranges
from test_gpu_experts import (Stack, by_slot, choices, expert_mlp_case, from_type, mlp_reference,
                              run_linear, same, slot_rows, to_type)

pytestmark = pytest.mark.gpu


@pytest.fixture
def forced(ctx, q8):
    fn = q8.lib().llmcp_q8_test_ctx_expert_repeat
    fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_int32], ctypes.c_int
    assert fn(ctx.handle, -1) == q8.EINVAL

    def force(n):
        assert fn(ctx.handle, n) == q8.OK
    yield force
    force(0)


# (tokens, top_k, experts, slots per tile, whether planned): each kernel, with the
# slots found by the workgroups and by the plan
KINDS = [(6, 2, 16, 4, False), (150, 2, 256, 4, True), (12, 2, 8, 8, False), (300, 2, 200, 8, True),
         (40, 2, 10, 16, False), (200, 2, 50, 16, True), (60, 2, 6, 32, True), (150, 2, 5, 64, True)]


# K of one step (one block, and ragged), of several with a ragged end, and of
# more steps than a wave's ring holds
@pytest.mark.parametrize("k", [32, 96, 544, 1056])
@pytest.mark.parametrize("m,top_k,e,tile,planned", KINDS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_over_ranges(ctx, q8, oracle, forced, m, top_k, e, tile, planned, k, dtype):
    rng = np.random.default_rng(m + e + k)
    # seven ranges, the last of eight columns
    n = 6 * columns(tile, False) + 8 if e < 100 or k == 96 else 2 * columns(tile, False) + 8
    st = Stack(ctx, oracle, rng, e, n, k)
    act = ("none", "silu", "sigmoid", "softplus")[k // 32 % 4]
    try:
        ids = choices(rng, m, top_k, e, masked=0.2)
        ids[0] = -1
        x = rng.standard_normal((m, k)).astype(np.float32)
        if dtype == "bf16":
            x = oracle.bf16_bits_to_f32(oracle.f32_to_bf16_bits(x))
        ref = by_slot(ids, lambda i, r: oracle.linear(r, st.p4[i], n, activation=act, epilogue=ctx.epilogue),
                      slot_rows(x, ids, False), n)
        if dtype == "bf16":
            ref = oracle.bf16_bits_to_f32(oracle.f32_to_bf16_bits(ref))
        for force in (0, 2, 3, 1000):
            forced(force)
            assert ranges(q8, ids.size, e, n, k, False, force)[:2] == (tile, planned)
            repeat = ranges(q8, ids.size, e, n, k, False, force)[3]
            assert (repeat > 1) == (force > 0)
            assert same(run_linear(ctx, oracle, st, x, ids, False, act, dtype), ref), force
        assert ctx.check_flag() == 0
    finally:
        st.release()


@pytest.mark.parametrize("h", [32, 96, 544, 1056])
@pytest.mark.parametrize("m,top_k,e,tile,planned", KINDS)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_mlp_over_ranges(ctx, q8, oracle, forced, m, top_k, e, tile, planned, h, dtype):
    rng = np.random.default_rng(m + e + h)
    # five ranges of gate and up, the last of half as many columns
    f = 4 * columns(tile, True) + max(32, columns(tile, True) // 2)
    if e > 100:
        f, h = min(f, 2 * columns(tile, True) + 32), min(h, 544)
    gate, up, down, ids, p, x, r = expert_mlp_case(ctx, oracle, rng, m, top_k, e, h, f, dtype, 0.2)
    try:
        ids[0] = -1
        xd, idd, pd, rd = (to_type(ctx, oracle, x, dtype), ctx.to_device(ids), ctx.to_device(p),
                           to_type(ctx, oracle, r, dtype))
        _, ref, bound = mlp_reference(oracle, ctx.epilogue, x, ids, p, gate, up, down, r, dtype)
        et = np.uint16 if dtype == "bf16" else np.uint32
        plain = None
        for force in (0, 2, 3, 1000):
            forced(force)
            got = ranges(q8, ids.size, e, f, max(f, h), True, force)
            assert got[:2] == (tile, planned) and (got[3] > 1) == (force > 0)
            yd = ctx.to_device(np.full(m * h, 7, et))
            ctx.expert_mlp(xd, idd, pd, m, top_k, gate.t, up.t, down.t, yd, residual=rd, dtype=dtype)
            bits = ctx.to_host(yd, (m, h), et)
            plain = bits if plain is None else plain
            assert np.array_equal(bits, plain), force
            assert (np.abs(from_type(ctx, oracle, yd, (m, h), dtype).astype(np.float64) - ref) <= bound).all()
    finally:
        for s in (gate, up, down):
            s.release()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_mlp_takes_several_ranges_by_itself(ctx, q8, oracle, dtype):
    """As wide an MLP as takes three ranges of gate and up per workgroup without
    being forced, on 256 CUs."""
    rng = np.random.default_rng(9)
    m, top_k, e, h, f = 16, 8, 128, 32, 1536
    assert ranges(q8, m * top_k, e, f, f, True) == (4, False, 16, 3)
    gate, up, down, ids, p, x, r = expert_mlp_case(ctx, oracle, rng, m, top_k, e, h, f, dtype)
    try:
        yd = ctx.alloc(m * h * 4)
        ctx.expert_mlp(to_type(ctx, oracle, x, dtype), ctx.to_device(ids), ctx.to_device(p), m, top_k,
                       gate.t, up.t, down.t, yd, residual=to_type(ctx, oracle, r, dtype), dtype=dtype)
        _, ref, bound = mlp_reference(oracle, ctx.epilogue, x, ids, p, gate, up, down, r, dtype)
        y = from_type(ctx, oracle, yd, (m, h), dtype).astype(np.float64)
        assert (np.abs(y - ref) <= bound).all()
    finally:
        for s in (gate, up, down):
            s.release()
