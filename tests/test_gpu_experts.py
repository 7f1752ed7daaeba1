"""The mixture-of-experts entries: llmcp_q8_route, llmcp_q8_expert_linear and
llmcp_q8_expert_mlp.  A slot's result must be bit for bit what the linear
with its expert's weight gives (Q8Matmul.cpp:204-223, Q8Scalar.cpp:192-199,
restated by the oracle); sums over slots are compared in float64 with bounds
counted in roundings."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8  # half a step of f32, of bf16


def same(a, b):
    return np.array_equal(np.asarray(a, np.float32).view(np.uint32),
                          np.asarray(b, np.float32).view(np.uint32))


class Stack:
    """`e` experts' weights [n, k], on the host and registered."""

    def __init__(self, ctx, oracle, rng, e, n, k, scale=0.02):
        self.ctx, self.n, self.k = ctx, n, k
        self.p4 = [oracle.pack_q8_0_p4((rng.standard_normal((n, k)) * scale).astype(np.float32))
                   for _ in range(e)]
        self.t = ctx.upload_experts_p4(np.concatenate(self.p4), e, n, k)

    def release(self):
        self.ctx.release(self.t)


def choices(rng, m, k, e, masked=0.0, only=None):
    """Distinct experts per token (of `only`, if given), some -1."""
    pool = np.arange(e) if only is None else np.asarray(only)
    ids = np.stack([rng.choice(pool, k, replace=len(pool) < k) for _ in range(m)]).astype(np.int32)
    ids[rng.random(ids.shape) < masked] = -1
    return ids


def by_slot(ids, f, x, n):
    """Rows f(expert, rows of x) put together by slot; zero without one."""
    ids = ids.ravel()
    y = np.zeros((ids.size, n), np.float32)
    for e in sorted(set(ids.tolist()) - {-1}):
        at = np.flatnonzero(ids == e)
        y[at] = f(e, x[at])
    return y


def slot_rows(x, ids, per_slot):
    return x if per_slot else np.repeat(x, ids.shape[1], axis=0)


def run_linear(ctx, oracle, st, x, ids, per_slot, act, dtype):
    m, top_k = ids.shape
    bits, wide = oracle.f32_to_bf16_bits, oracle.bf16_bits_to_f32
    xd = ctx.to_device(bits(x) if dtype == "bf16" else x)
    et = np.uint16 if dtype == "bf16" else np.float32
    yd = ctx.to_device(np.full((ids.size, st.n), 0xFFFF if dtype == "bf16" else np.nan, et))
    ctx.expert_linear(xd, ctx.to_device(ids), m, top_k, st.t, yd, per_slot=per_slot,
                      activation=act, dtype=dtype)
    y = ctx.to_host(yd, (ids.size, st.n), et)
    return wide(y) if dtype == "bf16" else y


# (tokens, top_k, experts, n, k): few slots (each workgroup finds its own) in
# tiles of 16, 32 and 64, more slots (sorted first) in the same, column ranges
# that end inside a tile of 16 and inside a workgroup, K of one block and of
# ragged steps and stages
@pytest.mark.parametrize("m,top_k,e,n,k", [
    (1, 1, 1, 8, 32), (1, 8, 16, 72, 96), (1, 4, 4, 200, 2560), (3, 2, 5, 136, 544),
    (2, 1, 1024, 16, 64), (40, 2, 6, 104, 160), (64, 4, 3, 264, 512), (31, 8, 8, 72, 672),
    (100, 3, 64, 40, 224), (300, 1, 1, 136, 96), (257, 2, 40, 24, 1056), (200, 4, 128, 16, 64),
    (500, 2, 9, 152, 288)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_expert_linear_bitwise(ctx, oracle, m, top_k, e, n, k, dtype):
    rng = np.random.default_rng(m * 131 + n + k)
    st = Stack(ctx, oracle, rng, e, n, k)
    per_slot = (m + top_k) % 2 == 0
    act = ("none", "silu", "sigmoid", "softplus")[(m + n // 8) % 4]
    try:
        ids = choices(rng, m, top_k, e, masked=0.2 if m > 1 else 0.0)
        x = rng.standard_normal((ids.size if per_slot else m, k)).astype(np.float32)
        x[0, :32] = 0.0
        x = oracle.bf16_bits_to_f32(oracle.f32_to_bf16_bits(x)) if dtype == "bf16" else x
        got = run_linear(ctx, oracle, st, x, ids, per_slot, act, dtype)
        ref = by_slot(ids, lambda i, r: oracle.linear(r, st.p4[i], n, activation=act,
                                                      epilogue=ctx.epilogue),
                      slot_rows(x, ids, per_slot), n)
        if dtype == "bf16":
            ref = oracle.bf16_bits_to_f32(oracle.f32_to_bf16_bits(ref))
        assert same(got, ref)
        assert ctx.check_flag() == 0
    finally:
        st.release()


# (tokens, top_k, experts, n, k): rows too wide for sixteen, eight and any of
# them in a workgroup's LDS; a plan of more slots than are sorted through LDS,
# of the most experts, and of a slot more than a workgroup looks over itself
@pytest.mark.parametrize("m,top_k,e,n,k", [
    (40, 2, 8, 24, 8192), (12, 1, 2, 16, 16416), (3, 2, 4, 16, 45056), (17000, 2, 5, 8, 32),
    (32768, 1, 3, 8, 32), (32769, 1, 70, 8, 32), (400, 4, 1024, 8, 32), (257, 1, 300, 8, 32),
    (256, 1, 200, 8, 32), (250, 1, 100, 24, 64)])
def test_expert_linear_limits(ctx, oracle, m, top_k, e, n, k):
    rng = np.random.default_rng(m + k)
    st = Stack(ctx, oracle, rng, e, n, k)
    try:
        ids = rng.integers(-1, e, (m, top_k)).astype(np.int32)
        x = rng.standard_normal((m, k)).astype(np.float32)
        got = run_linear(ctx, oracle, st, x, ids, False, "none", "f32")
        assert same(got, by_slot(ids, lambda i, r: oracle.linear(r, st.p4[i], n, epilogue=ctx.epilogue),
                                 slot_rows(x, ids, False), n))
    finally:
        st.release()


@pytest.mark.parametrize("m,top_k,e,only", [
    (60, 4, 64, [5]), (60, 4, 64, [0, 63, 7, 8]), (400, 2, 32, [31]), (400, 2, 32, [3, 3, 9])])
def test_expert_linear_uneven(ctx, oracle, m, top_k, e, only):
    """Every slot on one expert or a few, the same twice for one token, and the
    other experts without a row."""
    rng = np.random.default_rng(m + only[0])
    st = Stack(ctx, oracle, rng, e, 40, 128)
    try:
        ids = choices(rng, m, top_k, e, only=only)
        x = rng.standard_normal((m, 128)).astype(np.float32)
        got = run_linear(ctx, oracle, st, x, ids, False, "none", "f32")
        assert same(got, by_slot(ids, lambda i, r: oracle.linear(r, st.p4[i], 40, epilogue=ctx.epilogue),
                                 slot_rows(x, ids, False), 40))
    finally:
        st.release()


@pytest.mark.parametrize("m", [5, 300])
def test_expert_linear_without_experts(ctx, oracle, m):
    """All slots empty: rows of zeros; ids that are neither an expert nor -1
    count as empty and set the context's flag."""
    rng = np.random.default_rng(m)
    st = Stack(ctx, oracle, rng, 4, 40, 64)
    try:
        x = rng.standard_normal((m, 64)).astype(np.float32)
        ids = np.full((m, 2), -1, np.int32)
        assert not run_linear(ctx, oracle, st, x, ids, False, "sigmoid", "f32").any()
        assert ctx.check_flag() == 0
        ids[m // 2] = [4, 2]
        ids[0] = [1, -2]
        ids[m - 1] = [2 ** 31 - 1, -2 ** 31]
        got = run_linear(ctx, oracle, st, x, ids, False, "none", "f32")
        clean = np.where((ids < 0) | (ids > 3), -1, ids)
        assert same(got, by_slot(clean, lambda i, r: oracle.linear(r, st.p4[i], 40, epilogue=ctx.epilogue),
                                 slot_rows(x, ids, False), 40))
        assert ctx.check_flag() == 1
        assert ctx.check_flag() == 0
    finally:
        st.release()


@pytest.mark.parametrize("m", [7, 200])
def test_expert_linear_against_float64(ctx, oracle, m):
    """B blocks: a rounding of each scale product, and one (fma) or two per
    step of the chain, each at most U32 of the sum of magnitudes."""
    rng = np.random.default_rng(m)
    e, n, k = 6, 56, 416
    st = Stack(ctx, oracle, rng, e, n, k)
    try:
        ids = choices(rng, m, 3, e)
        x = rng.standard_normal((m, k)).astype(np.float32)
        got = run_linear(ctx, oracle, st, x, ids, False, "none", "f32").astype(np.float64)
        qa, sa = oracle.quantize_act_q8_1(x)
        a = qa.reshape(m, -1, 32).astype(np.float64) * sa.astype(np.float64)[:, :, None]
        for s, i in enumerate(ids.ravel()):
            qs, d = oracle.unpack_q8_0_p4(st.p4[i], n, k)
            w = qs.reshape(n, -1, 32) * oracle.f16_bits_to_f32(d).astype(np.float64)[:, :, None]
            dots = np.einsum("bi,nbi->nb", a[s // 3], w)
            bound = (k // 32 + 3) * U32 * np.abs(dots).sum(1)
            assert (np.abs(got[s] - dots.sum(1)) <= bound).all()
    finally:
        st.release()


def test_expert_linear_strides_and_alignment(ctx, q8, oracle):
    """Rows with a stride, from and to addresses of 4 B alignment; values
    between the output's rows stay."""
    rng = np.random.default_rng(3)
    m, top_k, e, n, k, ldx, ldy = 21, 2, 3, 40, 96, 101, 43
    st = Stack(ctx, oracle, rng, e, n, k)
    try:
        ids = choices(rng, m, top_k, e)
        x = rng.standard_normal((m, ldx)).astype(np.float32)
        xd, yd = ctx.alloc(m * ldx * 4 + 4), ctx.to_device(np.full(1 + m * top_k * ldy, 7.0, np.float32))
        q8.check(q8.lib().llmcp_q8_memcpy_h2d(ctx.handle, xd.ptr + 4, x.ctypes.data, x.nbytes))
        idd = ctx.to_device(ids)
        xi = q8.f32_memref(xd.ptr + 4, m, k, row_stride=ldx)
        yo = q8.f32_memref(yd.ptr + 4, m * top_k, n, row_stride=ldy)
        q8.check(q8.lib().llmcp_q8_expert_linear(
            ctx.handle, ctypes.byref(xi), idd.ptr, top_k, ctypes.byref(st.t.memref()),
            ctypes.byref(yo), 0))
        y = ctx.to_host(yd, (1 + m * top_k * ldy,), np.float32)
        assert y[0] == 7.0
        y = y[1:].reshape(m * top_k, ldy)
        assert (y[:, n:] == 7.0).all()
        assert same(y[:, :n], by_slot(ids, lambda i, r: oracle.linear(r, st.p4[i], n, epilogue=ctx.epilogue),
                                      np.repeat(x[:, :k], top_k, axis=0), n))
    finally:
        st.release()


# ------------------------------------------------------------------ MLP --

def mlp_reference(oracle, ep, x, ids, p, gate, up, down, residual, dtype):
    """(h rows by slot as stored, y in float64 from them, its error bound)."""
    bits, wide = oracle.f32_to_bf16_bits, oracle.bf16_bits_to_f32
    rnd = (lambda v: wide(bits(v))) if dtype == "bf16" else (lambda v: v)
    m, top_k = ids.shape
    xs = np.repeat(x, top_k, axis=0)
    f, n = gate.n, down.n
    g = by_slot(ids, lambda i, r: oracle.linear(r, gate.p4[i], f, activation="silu", epilogue=ep), xs, f)
    u = by_slot(ids, lambda i, r: oracle.linear(r, up.p4[i], f, epilogue=ep), xs, f)
    h = rnd(rnd(g) * rnd(u))
    o = rnd(by_slot(ids, lambda i, r: oracle.linear(r, down.p4[i], n, epilogue=ep), h, n))
    w = np.ones(ids.shape, np.float32) if p is None else p
    terms = o.reshape(m, top_k, n).astype(np.float64) * w[:, :, None]
    r = np.zeros((m, n)) if residual is None else residual.astype(np.float64)
    y = r + terms.sum(1)
    # an FMA rounding per slot on a partial sum, then the store's
    size = np.abs(r) + np.abs(terms).sum(1)
    bound = (top_k + 1) * U32 * size + (U16 * (np.abs(y) + top_k * U32 * size) if dtype == "bf16" else 0)
    return h, y, bound


def expert_mlp_case(ctx, oracle, rng, m, top_k, e, h, f, dtype, masked=0.0, residual=True,
                    weights=True, only=None):
    gate, up = Stack(ctx, oracle, rng, e, f, h), Stack(ctx, oracle, rng, e, f, h)
    down = Stack(ctx, oracle, rng, e, h, f)
    bits, wide = oracle.f32_to_bf16_bits, oracle.bf16_bits_to_f32
    ids = choices(rng, m, top_k, e, masked=masked, only=only)
    p = rng.random((m, top_k)).astype(np.float32) if weights else None
    x = rng.standard_normal((m, h)).astype(np.float32) * 4
    r = rng.standard_normal((m, h)).astype(np.float32) if residual else None
    if dtype == "bf16":
        x, r = wide(bits(x)), wide(bits(r)) if residual else None
    return gate, up, down, ids, p, x, r


def to_type(ctx, oracle, a, dtype):
    return None if a is None else ctx.to_device(oracle.f32_to_bf16_bits(a) if dtype == "bf16" else a)


def from_type(ctx, oracle, buf, shape, dtype):
    if dtype == "bf16":
        return oracle.bf16_bits_to_f32(ctx.to_host(buf, shape, np.uint16))
    return ctx.to_host(buf, shape, np.float32)


@pytest.mark.parametrize("m,top_k,e,h,f,masked", [
    (1, 1, 1, 32, 32, 0.0), (1, 8, 12, 2560, 96, 0.0), (1, 12, 20, 96, 160, 0.2), (1, 32, 40, 64, 32, 0.0),
    (3, 2, 40, 96, 64, 0.3), (5, 2, 40, 96, 64, 0.0), (11, 2, 40, 96, 64, 0.0), (1, 8, 12, 160, 224, 0.4),
    (2, 3, 4, 96, 64, 0.0), (16, 4, 24, 256, 96, 0.0), (60, 4, 3, 128, 160, 0.3),
    (33, 8, 9, 64, 32, 0.0), (150, 2, 7, 96, 192, 0.1), (300, 1, 1, 64, 96, 0.0),
    (130, 4, 100, 32, 64, 0.9)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_expert_mlp(ctx, oracle, m, top_k, e, h, f, masked, dtype):
    rng = np.random.default_rng(m * 17 + h + f)
    residual, weights = (m + f) % 3 != 0, m != 2
    gate, up, down, ids, p, x, r = expert_mlp_case(ctx, oracle, rng, m, top_k, e, h, f, dtype,
                                                   masked, residual, weights)
    try:
        yd = ctx.alloc(m * h * 4)
        ctx.expert_mlp(to_type(ctx, oracle, x, dtype), ctx.to_device(ids),
                       ctx.to_device(p) if weights else None, m, top_k, gate.t, up.t, down.t, yd,
                       residual=to_type(ctx, oracle, r, dtype), dtype=dtype)
        y = from_type(ctx, oracle, yd, (m, h), dtype).astype(np.float64)
        _, ref, bound = mlp_reference(oracle, ctx.epilogue, x, ids, p, gate, up, down, r, dtype)
        assert (np.abs(y - ref) <= bound).all()
        empty = (ids < 0).all(1)
        if empty.any():  # a token without an expert: its residual
            assert np.array_equal(y[empty], r[empty] if residual else np.zeros((empty.sum(), h)))
    finally:
        for s in (gate, up, down):
            s.release()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad", [0, 3, 4])
def test_expert_mlp_many_rows(ctx, q8, oracle, pad, dtype):
    """Enough rows that the sum takes eight bf16 columns per thread, residual
    and output with rows apart: the bits of calls on a few rows each."""
    rng = np.random.default_rng(pad)
    m, top_k, e, h, f = 4100, 3, 6, 1024, 32
    stacks = [Stack(ctx, oracle, rng, e, n, k) for n, k in ((f, h), (f, h), (h, f))]
    size, et = (2, np.uint16) if dtype == "bf16" else (4, np.float32)
    try:
        x, r = (rng.standard_normal((m, n)).astype(np.float32) for n in (h, h + pad))
        ids = choices(rng, m, top_k, e, masked=0.2)
        w = rng.standard_normal((m, top_k)).astype(np.float32)
        xd, rd = to_type(ctx, oracle, x, dtype), to_type(ctx, oracle, r, dtype)
        idd, wd = ctx.to_device(ids), ctx.to_device(w)
        fill = np.full((m, h + pad), 7, et)
        yd, part = ctx.to_device(fill), ctx.to_device(fill)
        names = [ctypes.byref(s.t.memref()) for s in stacks]

        def call(y, first, n):
            at = lambda buf, row: buf.ptr + first * row  # noqa: E731
            rows = [q8.f32_memref(at(b, k * size), n, h, k) for b, k in
                    ((xd, h), (rd, h + pad), (y, h + pad))]
            q8.check(getattr(q8.lib(), "llmcp_q8_expert_mlp" + ("_bf16" if dtype == "bf16" else ""))(
                ctx.handle, ctypes.byref(rows[0]), at(idd, 4 * top_k), at(wd, 4 * top_k), top_k, *names,
                ctypes.byref(rows[1]), ctypes.byref(rows[2])))
        call(yd, 0, m)
        for first in range(0, m, 400):
            call(part, first, min(400, m - first))
        a, b = (ctx.to_host(v, (m, h + pad), et) for v in (yd, part))
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
        assert (a[:, h:] == 7).all() and np.isfinite(from_type(ctx, oracle, yd, (m, h + pad), dtype)).all()
    finally:
        for s in stacks:
            s.release()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("e,top_k,h,f", [(40, 4, 160, 96), (3, 5, 96, 64), (12, 9, 2560, 192)])
def test_expert_mlp_alone_and_in_batches(ctx, q8, oracle, e, top_k, h, f, dtype):
    """A token's bits do not depend on the tokens beside it: one at a time, a
    few, many (each size has kernels of its own), rows as they are, at odd
    addresses or as Q8_1, and the output over the input."""
    rng = np.random.default_rng(e)
    m = 90
    gate, up, down, ids, p, x, _ = expert_mlp_case(ctx, oracle, rng, m, top_k, e, h, f, dtype, 0.1)
    size, et = (2, np.uint16) if dtype == "bf16" else (4, np.float32)
    try:
        bits = oracle.f32_to_bf16_bits(x) if dtype == "bf16" else np.ascontiguousarray(x, np.float32)
        xd, idd, pd, yd = ctx.to_device(bits), ctx.to_device(ids), ctx.to_device(p), ctx.alloc(m * h * size)
        stacks = (gate.t, up.t, down.t)
        ctx.expert_mlp(xd, idd, pd, m, top_k, *stacks, yd, dtype=dtype)
        want = ctx.to_host(yd, (m, h), et).view(np.uint8)
        for n in (1, 3, 17):
            for first in range(0, m - n + 1, 6 if n == 1 else n):
                ctx.expert_mlp(xd.ptr + first * h * size, idd.ptr + first * top_k * 4,
                               pd.ptr + first * top_k * 4, n, top_k, *stacks, yd, dtype=dtype)
                got = ctx.to_host(yd, (n, h), et).view(np.uint8)
                assert np.array_equal(got, want[first:first + n]), (n, first)
        odd = ctx.to_device(np.concatenate([bits.ravel()[:1], bits.ravel()]))
        q, s = ctx.alloc(m * h), ctx.alloc(m * h // 8)
        ctx.quantize(ctx.to_device(np.ascontiguousarray(x, np.float32)), m, h, q, s)
        for n in (1, 17, m):
            for rows in (odd.ptr + size, q8.Q8Rows(q, s, n, h)):
                ctx.expert_mlp(rows, idd, pd, n, top_k, *stacks, yd, dtype=dtype)
                assert np.array_equal(ctx.to_host(yd, (n, h), et).view(np.uint8), want[:n]), n
            over = ctx.to_device(bits)
            ctx.expert_mlp(over, idd, pd, n, top_k, *stacks, over, dtype=dtype)
            assert np.array_equal(ctx.to_host(over, (n, h), et).view(np.uint8), want[:n]), n
    finally:
        for st in (gate, up, down):
            st.release()


# H of several passes of a wave's ring (an odd number of steps, whole passes),
# rows of more pieces than are asked for at once, F of several rings; H past
# what the LDS of one token's kernels holds
@pytest.mark.parametrize("e,top_k,h,f", [(2, 3, 4480, 1056), (2, 2, 5120, 64), (3, 9, 160, 2208),
                                         (1, 2, 2592, 800), (2, 1, 23040, 32), (1, 1, 32768, 32)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_expert_mlp_one_wide_token(ctx, q8, oracle, e, top_k, h, f, dtype):
    rng = np.random.default_rng(h + f)
    gate, up, down, ids, p, x, r = expert_mlp_case(ctx, oracle, rng, 1, top_k, e, h, f, dtype)
    try:
        _, ref, bound = mlp_reference(oracle, ctx.epilogue, x, ids, p, gate, up, down, r, dtype)
        q, s, yd = ctx.alloc(h), ctx.alloc(h // 8), ctx.alloc(h * 4)
        ctx.quantize(ctx.to_device(np.ascontiguousarray(x, np.float32)), 1, h, q, s)
        for rows in (to_type(ctx, oracle, x, dtype), q8.Q8Rows(q, s, 1, h)):
            ctx.expert_mlp(rows, ctx.to_device(ids), ctx.to_device(p), 1, top_k, gate.t, up.t, down.t, yd,
                           residual=to_type(ctx, oracle, r, dtype), dtype=dtype)
            y = from_type(ctx, oracle, yd, (1, h), dtype).astype(np.float64)
            assert (np.abs(y - ref) <= bound).all()
    finally:
        for st in (gate, up, down):
            st.release()


def test_swiglu_rounds_as_the_oracle_over_the_gate_s_range(ctx, oracle):
    """bf16: silu of gate sums of every size and of both signs, those next to
    a rounding of bf16 among them, through one expert whose down weights
    pick single columns of h apart."""
    rng = np.random.default_rng(77)
    h, f, m, dtype = 64, 64, 400, "bf16"
    gate, up = Stack(ctx, oracle, rng, 1, f, h, 0.3), Stack(ctx, oracle, rng, 1, f, h, 0.3)
    down = Stack(ctx, oracle, rng, 1, h, f)
    bits, wide = oracle.f32_to_bf16_bits, oracle.bf16_bits_to_f32
    try:
        x = rng.standard_normal((m, h)) * 10.0 ** rng.uniform(-44, 3, (m, 1))
        x = wide(bits(x.astype(np.float32)))
        ids = np.zeros((m, 1), np.int32)
        yd = ctx.alloc(m * h * 2)
        ctx.expert_mlp(to_type(ctx, oracle, x, dtype), ctx.to_device(ids), None, m, 1, gate.t, up.t,
                       down.t, yd, dtype=dtype)
        _, ref, bound = mlp_reference(oracle, ctx.epilogue, x, ids, None, gate, up, down, None, dtype)
        fine = np.isfinite(ref)
        y = from_type(ctx, oracle, yd, (m, h), dtype)
        assert np.array_equal(np.isfinite(y), fine)
        # one slot of weight 1: the sum is o itself, already bf16
        assert np.array_equal(y[fine], ref[fine].astype(np.float32))
    finally:
        for s in (gate, up, down):
            s.release()


@pytest.mark.parametrize("m", [1, 3, 90])
def test_expert_mlp_in_place_and_rows(ctx, q8, oracle, m):
    """The output in the residual's memory, and the input as Q8_1 rows: the
    same bits."""
    rng = np.random.default_rng(m)
    top_k, e, h, f, dtype = 4, 6, 96, 64, "bf16"
    gate, up, down, ids, p, x, r = expert_mlp_case(ctx, oracle, rng, m, top_k, e, h, f, dtype)
    try:
        idd, pd = ctx.to_device(ids), ctx.to_device(p)
        xd, rd, yd = to_type(ctx, oracle, x, dtype), to_type(ctx, oracle, r, dtype), ctx.alloc(m * h * 2)
        ctx.expert_mlp(xd, idd, pd, m, top_k, gate.t, up.t, down.t, yd, residual=rd, dtype=dtype)
        want = ctx.to_host(yd, (m, h), np.uint16)
        ctx.expert_mlp(xd, idd, pd, m, top_k, gate.t, up.t, down.t, rd, residual=rd, dtype=dtype)
        assert np.array_equal(ctx.to_host(rd, (m, h), np.uint16), want)
        qa, sa = oracle.quantize_act_q8_1(x)
        rows = q8.Q8Rows(ctx.to_device(qa), ctx.to_device(sa), m, h)
        rd = to_type(ctx, oracle, r, dtype)
        ctx.expert_mlp(rows, idd, pd, m, top_k, gate.t, up.t, down.t, yd, residual=rd, dtype=dtype)
        assert np.array_equal(ctx.to_host(yd, (m, h), np.uint16), want)
    finally:
        for s in (gate, up, down):
            s.release()


@pytest.mark.parametrize("m,top_k", [(1, 4), (80, 4)])
def test_expert_mlp_replayed(ctx, oracle, m, top_k):
    """One captured graph replayed on new rows and other choices of experts,
    with eager calls of other sizes in between: every replay the eager bits."""
    rng = np.random.default_rng(m)
    e, h, f, dtype = 5, 128, 96, "bf16"
    gate, up, down, ids, p, x, r = expert_mlp_case(ctx, oracle, rng, m, top_k, e, h, f, dtype)
    try:
        xd, rd, yd = to_type(ctx, oracle, x, dtype), to_type(ctx, oracle, r, dtype), ctx.alloc(m * h * 2)
        idd, pd, zd = ctx.to_device(ids), ctx.to_device(p), ctx.alloc(m * h * 2)
        call = lambda y, n=m: ctx.expert_mlp(xd, idd, pd, n, top_k, gate.t, up.t, down.t, y,  # noqa: E731
                                             residual=rd, dtype=dtype)
        call(yd)
        ctx.sync()
        ctx.graph_begin()
        call(yd)
        g = ctx.graph_end()
        for i in range(5):
            new = oracle.f32_to_bf16_bits(rng.standard_normal((m, h)).astype(np.float32))
            ids = choices(rng, m, top_k, e, masked=0.3 * (i % 2), only=[i] if i == 3 else None)
            ctx.sync()
            for buf, a in ((xd, new), (idd, ids)):
                from llmcp_amd import check, lib
                check(lib().llmcp_q8_memcpy_h2d(ctx.handle, buf.ptr, a.ctypes.data, a.nbytes))
            ctx.graph_launch(g)
            got = ctx.to_host(yd, (m, h), np.uint16)
            if m > 1:
                call(zd, m // 2)
            call(zd)
            assert np.array_equal(got, ctx.to_host(zd, (m, h), np.uint16)), i
        ctx.graph_destroy(g)
    finally:
        for s in (gate, up, down):
            s.release()


# ---------------------------------------------------------------- route --

def route_reference(logits, top_k, normalize, scale):
    """float64, and the bound of the weights' error."""
    l = np.asarray(logits, np.float64)
    m, e = l.shape
    ids, w, tol = np.full((m, top_k), -1, np.int32), np.zeros((m, top_k)), np.zeros((m, top_k))
    for t in range(m):
        ok = [i for i in range(e) if l[t, i] > -np.inf]  # neither NaN nor -inf
        order = sorted(ok, key=lambda i: (-l[t, i], i))[:top_k]
        if not order:
            continue
        top = l[t, order[0]]
        p = {i: 1.0 if l[t, i] == top else np.exp(l[t, i] - top) for i in ok}
        total = sum(p[i] for i in (order if normalize else ok))
        for j, i in enumerate(order):
            ids[t, j], w[t, j] = i, p[i] / total * scale
            # the exponent's difference and exp in f32, e additions, a
            # division and the scale; exp below f32's normal range
            d = 0.0 if l[t, i] == top else min(abs(l[t, i] - top), 200.0)
            most = max([0.0] + [min(abs(l[t, k] - top), 200.0) for k in ok if l[t, k] != top])
            tol[t, j] = w[t, j] * U32 * (d + most + e + 5) + abs(scale) * 2.0 ** -149
    return ids, w, tol


def run_route(ctx, oracle, l, top_k, normalize, scale, dtype):
    m, e = l.shape
    ids, w = ctx.to_device(np.full((m, top_k), 99, np.int32)), ctx.alloc(m * top_k * 4)
    ctx.route(to_type(ctx, oracle, l, dtype), m, e, top_k, ids, w, normalize=normalize,
              scale=scale, dtype=dtype)
    return ctx.to_host(ids, (m, top_k), np.int32), ctx.to_host(w, (m, top_k), np.float32)


@pytest.mark.parametrize("m,e,top_k", [(1, 1, 1), (1, 128, 8), (3, 5, 5), (6, 63, 3), (9, 64, 32),
                                       (5, 65, 7), (70, 129, 8), (4, 257, 16), (3, 1024, 32),
                                       (2, 1000, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("normalize", [False, True])
def test_route(ctx, oracle, m, e, top_k, dtype, normalize):
    rng = np.random.default_rng(m + e * 7 + top_k)
    l = (rng.standard_normal((m, e)) * 3).astype(np.float32)
    if m > 1:
        l[0] = np.round(l[0])                       # many ties
        l[1, rng.random(e) < 0.5] = -np.inf         # masked
    if dtype == "bf16":
        l = oracle.bf16_bits_to_f32(oracle.f32_to_bf16_bits(l))
    ids, w = run_route(ctx, oracle, l, top_k, normalize, 1.5, dtype)
    ri, rw, tol = route_reference(l, top_k, normalize, 1.5)
    assert np.array_equal(ids, ri)
    assert (np.abs(w - rw) <= tol).all()


@pytest.mark.parametrize("normalize", [False, True])
def test_route_special_logits(ctx, oracle, normalize):
    inf, nan, low = np.inf, np.nan, np.finfo(np.float32).min
    rows = np.array([
        [-inf] * 6,                          # nothing left
        [nan] * 6,
        [nan, -inf, 1.0, nan, -inf, -inf],   # one left
        [inf, 0.0, inf, 1.0, -inf, nan],     # infinite ones share
        [low] * 6,                           # the type's lowest is a value
        [low, 0.0, low, -0.0, low, 0.0],     # zeros of both signs tie
        [1e38, -1e38, 3e38, 0.0, 88.0, -104.0],
        [0.0, -87.4, -95.0, -103.0, -104.5, -200.0],
    ], np.float32)
    ids, w = run_route(ctx, oracle, rows, 4, normalize, 1.0, "f32")
    ri, rw, tol = route_reference(rows, 4, normalize, 1.0)
    assert np.array_equal(ids, ri)
    assert (np.abs(w - rw) <= tol).all()
    assert (w[:2] == 0).all() and w[2, 0] == 1.0


# ------------------------------------------- the operators in one block --

@pytest.mark.parametrize("m", [1, 6, 150])
def test_block_end_to_end(ctx, q8, oracle, m):
    """A block as a model runs it, bf16: residual add + norm with rows of
    Q8_1, the router's linear, the choice, the experts with the residual."""
    rng = np.random.default_rng(m)
    h, f, e, top_k, dtype = 256, 96, 16, 4, "bf16"
    bits, wide = oracle.f32_to_bf16_bits, oracle.bf16_bits_to_f32
    gate, up, down, _, _, x, r = expert_mlp_case(ctx, oracle, rng, m, top_k, e, h, f, dtype)
    rw = oracle.pack_q8_0_p4((rng.standard_normal((e, h)) * 0.05).astype(np.float32))
    router = ctx.upload_p4(rw, e, h)
    try:
        nw = bits((rng.standard_normal(h) * 0.1).astype(np.float32))
        total, normed, logits = ctx.alloc(m * h * 2), ctx.alloc(m * h * 2), ctx.alloc(m * e * 2)
        rows = q8.Q8Rows(ctx.alloc(m * h), ctx.alloc(m * h // 8), m, h)
        ids, w, y = ctx.alloc(m * top_k * 4), ctx.alloc(m * top_k * 4), ctx.alloc(m * h * 2)
        ctx.add_rmsnorm(to_type(ctx, oracle, x, dtype), to_type(ctx, oracle, r, dtype),
                        ctx.to_device(nw), total, m, h, normed=normed, quantized=rows,
                        zero_centered=True, dtype=dtype)
        ctx.linear(normed, router, logits, m, dtype=dtype)
        ctx.route(logits, m, e, top_k, ids, w, dtype=dtype)
        ctx.expert_mlp(rows, ids, w, m, top_k, gate.t, up.t, down.t, y, residual=total, dtype=dtype)
        s = wide(ctx.to_host(total, (m, h), np.uint16))
        assert np.array_equal(bits(s), bits(x + r))
        n = wide(ctx.to_host(normed, (m, h), np.uint16))
        # each step from the rows that the step before stored
        l = wide(bits(oracle.linear(n, rw, e, epilogue=ctx.epilogue)))
        assert same(wide(ctx.to_host(logits, (m, e), np.uint16)), l)
        ri, rp, tol = route_reference(l, top_k, True, 1.0)
        got_w = ctx.to_host(w, (m, top_k), np.float32)
        assert np.array_equal(ctx.to_host(ids, (m, top_k), np.int32), ri)
        assert (np.abs(got_w - rp) <= tol).all()
        _, ref, bound = mlp_reference(oracle, ctx.epilogue, n, ri, got_w, gate, up, down, s, dtype)
        assert (np.abs(wide(ctx.to_host(y, (m, h), np.uint16)) - ref) <= bound).all()
    finally:
        ctx.release(router)
        for st in (gate, up, down):
            st.release()


def test_two_contexts_streams_and_graphs(ctx, q8, oracle):
    """Two contexts with the same weights on streams of their own, and two
    graphs of one context that share its workspace, replayed in turn."""
    rng = np.random.default_rng(12)
    e, h, f, top_k, dtype = 6, 96, 64, 3, "bf16"
    gate, up, down, _, _, _, _ = expert_mlp_case(ctx, oracle, rng, 4, top_k, e, h, f, dtype)
    cases, refs = [], []
    for m in (1, 100):
        ids, x = choices(rng, m, top_k, e), rng.standard_normal((m, h)).astype(np.float32)
        xb = oracle.f32_to_bf16_bits(x)
        cases.append((m, ctx.to_device(xb), ctx.to_device(ids), ctx.alloc(m * h * 2)))
        _, ref, bound = mlp_reference(oracle, ctx.epilogue, oracle.bf16_bits_to_f32(xb), ids, None,
                                      gate, up, down, None, dtype)
        refs.append((ref, bound))
    other = q8.Context(0)
    try:
        other.set_platform(ctx.platform)
        stacks = [other.upload_experts_p4(np.concatenate(s.p4), e, s.n, s.k) for s in (gate, up, down)]

        def call(c, st, i, y=None):
            m, x, ids, out = cases[i]
            c.expert_mlp(x, ids, None, m, top_k, *st, y or out, dtype=dtype)
        own = [s.t for s in (gate, up, down)]
        for i in (1, 0):
            call(ctx, own, i)
        ctx.sync()
        graphs = []
        for i in (0, 1):
            ctx.graph_begin()
            call(ctx, own, i)
            graphs.append(ctx.graph_end())
        outs = [other.alloc(cases[i][0] * h * 2) for i in (0, 1)]
        for rep in range(4):
            for i in ((0, 1), (1, 0))[rep % 2]:
                ctx.graph_launch(graphs[i])
                call(other, stacks, 1 - i, outs[1 - i])
        for c, bufs in ((ctx, [cases[0][3], cases[1][3]]), (other, outs)):
            for buf, case, (ref, bound) in zip(bufs, cases, refs):
                y = oracle.bf16_bits_to_f32(c.to_host(buf, (case[0], h), np.uint16))
                assert (np.abs(y - ref) <= bound).all()
        for g in graphs:
            ctx.graph_destroy(g)
    finally:
        other.close()
        for s in (gate, up, down):
            s.release()


# ------------------------------------------------------ registry, errors --

def test_stacks_are_for_expert_entries_alone(ctx, q8, oracle):
    rng = np.random.default_rng(4)
    st = Stack(ctx, oracle, rng, 3, 16, 64)
    plain = ctx.upload_p4(oracle.pack_q8_0_p4(np.ones((48, 64), np.float32)), 48, 64)
    buf = ctx.alloc(1 << 16)
    try:
        w = q8.Weight(ctx, st.t.key, 48, 64)  # the same bytes as one tensor
        with pytest.raises(q8.Declined, match="stack of experts"):
            ctx.linear(buf, w, buf, 1)
        with pytest.raises(q8.Declined, match="stack of experts"):
            ctx.embedding(buf, 1, w, buf)
        with pytest.raises(q8.Declined, match="not a stack"):
            ctx.expert_linear(buf, buf, 1, 1, q8.Experts(ctx, plain.key, 3, 16, 64), buf)
        assert q8.lib().llmcp_q8_device_bytes(ctx.handle, st.t.key) >= 3 * 16 * 68
    finally:
        st.release()
        ctx.release(plain)
    with pytest.raises(q8.Q8Error, match="not an uploaded"):
        ctx.expert_linear(buf, buf, 1, 1, st.t, buf)


def test_registering_stacks_refuses(ctx, q8, oracle):
    host = np.zeros(1 << 16, np.uint8)
    for e, n, k in ((0, 8, 32), (1025, 8, 32), (2, 12, 32), (2, 8, 48), (1, 0, 32), (-1, 8, 32),
                    (1, 1 << 20, 8192)):
        with pytest.raises(q8.Declined):
            ctx.upload_experts_p4(host, e, n, k)
        with pytest.raises(q8.Declined):
            ctx.register_device_experts_p4(ctx.alloc(64), e, n, k)
    with q8.Context(0) as c:
        c.set_weight_budget(4096)
        with pytest.raises(q8.Q8Error) as err:
            c.upload_experts_p4(host, 8, 16, 128)
        assert err.value.code == q8.ENOMEM


def test_registered_from_device_equals_uploaded(ctx, oracle):
    rng = np.random.default_rng(5)
    st = Stack(ctx, oracle, rng, 3, 24, 96)
    dev = ctx.to_device(np.concatenate(st.p4))
    t = ctx.register_device_experts_p4(dev, 3, 24, 96)
    try:
        x, ids = rng.standard_normal((4, 96)).astype(np.float32), choices(rng, 4, 2, 3)
        a = run_linear(ctx, oracle, st, x, ids, False, "none", "f32")
        yd = ctx.alloc(8 * 24 * 4)
        ctx.expert_linear(ctx.to_device(x), ctx.to_device(ids), 4, 2, t, yd)
        assert same(ctx.to_host(yd, (8, 24), np.float32), a)
    finally:
        st.release()
        ctx.release(t)


def test_expert_entries_refuse(ctx, q8, oracle):
    rng = np.random.default_rng(6)
    st, odd = Stack(ctx, oracle, rng, 3, 32, 64), Stack(ctx, oracle, rng, 3, 40, 64)
    down, two = Stack(ctx, oracle, rng, 3, 64, 32), Stack(ctx, oracle, rng, 2, 64, 32)
    buf, L = ctx.alloc(1 << 16), q8.lib()
    ref = ctypes.byref
    try:
        def linear(x, ids, k, w, y, act=0):
            return L.llmcp_q8_expert_linear(ctx.handle, ref(x), ids, k, ref(w), ref(y), act)
        mr, w = q8.f32_memref, st.t.memref()
        ok = (mr(buf.ptr, 2, 64), buf.ptr, 2, w, mr(buf.ptr + 4096, 4, 32))
        for i, bad, code in ((0, mr(buf.ptr, 2, 96), q8.DECLINED), (0, mr(buf.ptr, 3, 64), q8.DECLINED),
                             (1, None, q8.EINVAL), (2, 0, q8.DECLINED), (2, 33, q8.DECLINED),
                             (2, 3, q8.DECLINED), (4, mr(buf.ptr, 4, 40), q8.DECLINED),
                             (4, mr(buf.ptr, 5, 32), q8.DECLINED)):
            args = list(ok)
            args[i] = bad
            assert linear(*args) == code, (i, code)
        assert linear(*ok, act=4) == q8.DECLINED
        assert linear(*ok[:4], mr(buf.ptr, 4, 32)) == q8.EINVAL  # over its own input
        assert linear(mr(buf.ptr, 0, 64), buf.ptr, 2, w, mr(buf.ptr, 0, 32)) == q8.OK
        mlp = lambda x, y, wg, wu, wd, k=2, r=None: L.llmcp_q8_expert_mlp(  # noqa: E731
            ctx.handle, ref(x), buf.ptr, None, k, ref(wg.t.memref()), ref(wu.t.memref()),
            ref(wd.t.memref()), ref(r) if r is not None else None, ref(y))
        x, y = mr(buf.ptr, 2, 64), mr(buf.ptr + 4096, 2, 64)
        assert mlp(x, y, odd, odd, down) == q8.DECLINED   # F % 32
        assert mlp(x, y, st, odd, down) == q8.DECLINED
        assert mlp(x, y, st, st, two) == q8.DECLINED      # 3 experts and 2
        assert mlp(x, y, st, st, st) == q8.DECLINED
        assert mlp(mr(buf.ptr, 3, 64), y, st, st, down) == q8.DECLINED
        assert mlp(x, y, st, st, down, r=mr(buf.ptr, 1, 64)) == q8.DECLINED
        assert mlp(x, y, st, st, down, k=40) == q8.DECLINED
        assert mlp(mr(buf.ptr, 0, 64), mr(buf.ptr, 0, 64), st, st, down) == q8.OK
        rows = q8.MemRefRows(buf.ptr + 8, buf.ptr, 2, 64)  # values off by 8 B
        assert L.llmcp_q8_expert_mlp_rows(
            ctx.handle, ref(rows), buf.ptr, None, 2, ref(st.t.memref()), ref(st.t.memref()),
            ref(down.t.memref()), None, ref(y)) == q8.DECLINED
        logits = mr(buf.ptr, 2, 8)
        route = lambda l, k, i=buf.ptr, p=buf.ptr: L.llmcp_q8_route(  # noqa: E731
            ctx.handle, ref(l), k, 1, 1.0, i, p)
        assert route(logits, 0) == route(logits, 9) == q8.DECLINED
        assert route(mr(buf.ptr, 1, 1025), 2) == route(mr(buf.ptr, 1, 64), 33) == q8.DECLINED
        assert route(logits, 2, i=None) == route(logits, 2, p=None) == q8.EINVAL
        assert route(mr(buf.ptr, 0, 8), 2) == q8.OK
    finally:
        for s in (st, odd, down, two):
            s.release()
