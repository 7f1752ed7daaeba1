"""Rows of infinities, NaN, subnormal and huge values through the expert
products: each slot the bits that the linear of its expert gives on that row by
itself, whatever the rows beside it hold; and such values where a slot has no
expert.  And a stack whose copy passes 32 bits."""
import numpy as np
import pytest

from test_gpu_experts import Stack, choices, from_type, to_type
from test_gpu_experts_ranges import KINDS

pytestmark = pytest.mark.gpu


def alike(a, b):
    """The same bits, NaNs alike."""
    return ((a.view(np.uint8) == b.view(np.uint8)).reshape(a.shape + (-1,)).all(-1) | (np.isnan(a) & np.isnan(b))).all()


def odd_rows(rng, m, k):
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[1::7, rng.integers(0, k, 3)] = np.inf
    x[2::7, rng.integers(0, k, 3)] = -np.inf
    x[3::7, rng.integers(0, k, 3)] = np.nan
    x[4::7] *= np.float32(1e-41)
    x[5::7] *= np.float32(1e36)
    x[5::7, :32] *= np.float32(1e-30)
    return x


@pytest.mark.parametrize("m,top_k,e,tile,planned", KINDS + [(1, 2, 4, 4, False)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_of_odd_rows(ctx, oracle, m, top_k, e, tile, planned, dtype):
    rng = np.random.default_rng(m + e)
    n, k = 72, 160
    st = Stack(ctx, oracle, rng, e, n, k)
    single = [ctx.upload_p4(p, n, k) for p in st.p4[:min(e, 24)]]
    try:
        ids = choices(rng, m, top_k, min(e, 24), masked=0.1)
        if m > 8:
            ids[:8] = rng.integers(0, 2, (8, top_k))  # tiles of odd rows beside each other
        x = odd_rows(rng, m * top_k, k)
        et = np.uint16 if dtype == "bf16" else np.float32
        with np.errstate(invalid="ignore"):
            xb = oracle.f32_to_bf16_bits(x) if dtype == "bf16" else x
        xd = ctx.to_device(xb)
        yd = ctx.to_device(np.full((ids.size, n), 7, et))
        ctx.expert_linear(xd, ctx.to_device(ids), m, top_k, st.t, yd, per_slot=True, dtype=dtype)
        y = from_type(ctx, oracle, yd, (ids.size, n), dtype)
        want = np.zeros((ids.size, n), np.float32)
        for i in sorted(set(ids.ravel().tolist()) - {-1}):
            at = np.flatnonzero(ids == i)
            zd = ctx.alloc(at.size * n * 4)
            ctx.linear(ctx.to_device(np.ascontiguousarray(xb[at])), single[i], zd, at.size, mode="prefill" if at.size > 1 else "decode", dtype=dtype)
            want[at] = from_type(ctx, oracle, zd, (at.size, n), dtype)
        assert alike(y, want)
        assert not y[ids.ravel() < 0].any()
    finally:
        st.release()
        for w in single:
            ctx.release(w)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_mlp_of_odd_rows(ctx, oracle, dtype):
    """One at a time, a few, many: the same bits for every token."""
    rng = np.random.default_rng(5)
    m, top_k, e, h, f = 98, 3, 24, 160, 96
    stacks = [Stack(ctx, oracle, rng, e, n, k) for n, k in ((f, h), (f, h), (h, f))]
    names = [s.t for s in stacks]
    size = 2 if dtype == "bf16" else 4
    try:
        ids = choices(rng, m, top_k, e, masked=0.2)
        with np.errstate(invalid="ignore"):
            xd = to_type(ctx, oracle, odd_rows(rng, m, h), dtype)
        p = rng.standard_normal((m, top_k)).astype(np.float32)
        idd, pd, yd = ctx.to_device(ids), ctx.to_device(p), ctx.alloc(m * h * size)
        ctx.expert_mlp(xd, idd, pd, m, top_k, *names, yd, dtype=dtype)
        want = from_type(ctx, oracle, yd, (m, h), dtype)
        assert np.isfinite(want[::7]).all() and np.isfinite(want[6::7]).all()
        for n in (1, 3, 14, 49):
            for first in range(0, m - n + 1, n):
                ctx.expert_mlp(xd.ptr + first * h * size, idd.ptr + first * top_k * 4, pd.ptr + first * top_k * 4,
                               n, top_k, *names, yd, dtype=dtype)
                assert alike(from_type(ctx, oracle, yd, (n, h), dtype), want[first:first + n]), (n, first)
    finally:
        for s in stacks:
            s.release()


@pytest.mark.parametrize("m", [1, 6, 40, 200])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_mlp_without_experts_beside_odd_values(ctx, oracle, m, dtype):
    """Slots without an expert: neither their rows nor their weights count."""
    rng = np.random.default_rng(m)
    top_k, e, h, f = 4, 6, 64, 32
    stacks = [Stack(ctx, oracle, rng, e, n, k) for n, k in ((f, h), (f, h), (h, f))]
    try:
        ids = choices(rng, m, top_k, e, masked=0.5)
        ids[::3] = -1
        x, r = (rng.standard_normal((m, h)).astype(np.float32) for _ in range(2))
        p = rng.standard_normal((m, top_k)).astype(np.float32)
        clean = p.copy()
        p[ids < 0], clean[ids < 0] = np.nan, 0.0
        plain = x.copy()
        x[::3] = np.nan
        ys = []
        for a, w in ((x, p), (plain, clean)):
            yd = ctx.alloc(m * h * 4)
            with np.errstate(invalid="ignore"):
                xd = to_type(ctx, oracle, a, dtype)
            ctx.expert_mlp(xd, ctx.to_device(ids), ctx.to_device(w), m, top_k, *[s.t for s in stacks], yd,
                           residual=to_type(ctx, oracle, r, dtype), dtype=dtype)
            ys.append(from_type(ctx, oracle, yd, (m, h), dtype))
        assert np.isfinite(ys[0]).all() and np.array_equal(ys[0], ys[1])
        rb = oracle.bf16_bits_to_f32(oracle.f32_to_bf16_bits(r)) if dtype == "bf16" else r
        assert np.array_equal(ys[0][::3], rb[::3])
    finally:
        for s in stacks:
            s.release()


def test_stack_past_32_bits(ctx, q8):
    """A stack of 5.1 GB: experts at its end, by the kernels of few slots and of
    many, against the same bytes registered as one tensor each."""
    e, n, k = 96, 2048, 24576
    p4, _ = ctx.synthesize_p4(3, e * n, k)
    t = ctx.register_device_experts_p4(p4, e, n, k)
    each = n * k // 32 * 34

    class At:
        ptr = p4.ptr + (e - 1) * each
    last = ctx.register_device_p4(At, n, k)
    try:
        rng = np.random.default_rng(1)
        x = ctx.to_device(rng.standard_normal((70, k)).astype(np.float32))
        want = ctx.alloc(70 * n * 4)
        ctx.linear(x, last, want, 70, mode="prefill")
        want = ctx.to_host(want, (70, n), np.uint32)
        for m, top_k in ((1, 1), (3, 1), (70, 1), (70, 5)):
            ids = rng.integers(-1, e, (m, top_k)).astype(np.int32)
            ids[:, 0] = e - 1
            yd = ctx.alloc(m * top_k * n * 4)
            ctx.expert_linear(x, ctx.to_device(ids), m, top_k, t, yd)
            y = ctx.to_host(yd, (m, top_k, n), np.uint32)
            assert np.array_equal(y[:, 0], want[:m]), (m, top_k)
    finally:
        ctx.release(last)
        ctx.release(t)
