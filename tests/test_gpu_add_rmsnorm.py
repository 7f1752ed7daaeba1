"""llmcp_q8_add_rmsnorm: the residual's addition, the norm with its sum of
squares in float64, and the normed rows' Q8_1 (Q8Decode.cpp:83-120)."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8  # half a step of f32, of bf16


def make(rng, oracle, m, h, dtype, scale=3.0):
    x, r = ((rng.standard_normal((m, h)) * scale).astype(np.float32) for _ in range(2))
    w = (rng.standard_normal(h) * 0.2 + 0.5).astype(np.float32)
    if dtype == "bf16":
        x, r, w = (oracle.bf16_bits_to_f32(oracle.f32_to_bf16_bits(a)) for a in (x, r, w))
    return x, r, w


def put(ctx, oracle, a, dtype):
    return ctx.to_device(oracle.f32_to_bf16_bits(a) if dtype == "bf16" else a)


def get(ctx, oracle, buf, shape, dtype):
    if dtype == "bf16":
        return oracle.bf16_bits_to_f32(ctx.to_host(buf, shape, np.uint16))
    return ctx.to_host(buf, shape, np.float32)


def stored(oracle, a, dtype):
    a = np.asarray(a, np.float32)
    return oracle.bf16_bits_to_f32(oracle.f32_to_bf16_bits(a)) if dtype == "bf16" else a


def same(a, b):
    a, b = np.asarray(a, np.float32), np.asarray(b, np.float32)
    nan = np.isnan(a)
    return np.array_equal(nan, np.isnan(b)) and np.array_equal(a[~nan].view(np.uint32),
                                                               b[~nan].view(np.uint32))


def check_rows(ctx, oracle, x, r, w, eps, zc, dtype, s, y, q, sc):
    """The sum bit for bit; the norm within a rounding of rstd and of each
    product (and the store's) of float64's; the Q8_1 that of the stored rows."""
    total = stored(oracle, x + r, dtype)
    assert same(s, total)
    t = total.astype(np.float64)
    ww = (w + np.float32(1.0)).astype(np.float64) if zc else w.astype(np.float64)
    ref = t / np.sqrt((t * t).mean(1, keepdims=True) + float(np.float32(eps))) * ww
    rel = (1 + U32) ** 3 - 1 + 1e-12
    bound = np.abs(ref) * (rel + (U16 * (1 + rel) if dtype == "bf16" else 0)) + 3 * 2.0 ** -149
    assert (np.abs(y - ref) <= bound).all()
    qa, sa = oracle.quantize_act_q8_1(y)
    assert np.array_equal(q, qa) and same(sc, sa)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,h", [(1, 32), (1, 2560), (3, 96), (5, 512), (2, 544), (70, 2208),
                                 (2, 8192), (2, 8224), (1, 16384), (1, 16416), (2, 32768)])
@pytest.mark.parametrize("zc", [False, True])
def test_add_rmsnorm(ctx, q8, oracle, m, h, dtype, zc):
    rng = np.random.default_rng(m * 5 + h)
    x, r, w = make(rng, oracle, m, h, dtype)
    if m > 1:
        x[1], r[1] = 0.0, 0.0   # a row of zeros: rstd = 1 / sqrt(eps)
    esz = 2 if dtype == "bf16" else 4
    s, y = ctx.alloc(m * h * esz), ctx.alloc(m * h * esz)
    rows = q8.Q8Rows(ctx.alloc(m * h), ctx.alloc(m * h // 8), m, h)
    ctx.add_rmsnorm(put(ctx, oracle, x, dtype), put(ctx, oracle, r, dtype), put(ctx, oracle, w, dtype),
                    s, m, h, normed=y, quantized=rows, eps=1e-5, zero_centered=zc, dtype=dtype)
    check_rows(ctx, oracle, x, r, w, 1e-5, zc, dtype, get(ctx, oracle, s, (m, h), dtype),
               get(ctx, oracle, y, (m, h), dtype), ctx.to_host(rows.values, (m, h), np.int8),
               ctx.to_host(rows.scales, (m, h // 32), np.float32))


def test_extreme_rows(ctx, q8, oracle):
    """Subnormal rows, rows whose f32 sum of squares would overflow, one large
    value among tiny ones; rows with infinities or NaN give what the formula
    gives, and their Q8_1 the quantizer's."""
    h = 256
    x = np.zeros((6, h), np.float32)
    x[0] = 1e-40
    x[1] = np.linspace(-3e38, 3e38, h)
    x[2] = 1e-20
    x[2, 7] = 1e20
    x[3, 9] = np.inf
    x[4, 9] = np.nan
    x[5] = 2.0 ** -80
    r, w = np.zeros_like(x), np.ones(h, np.float32)
    s, y = ctx.alloc(x.nbytes), ctx.alloc(x.nbytes)
    rows = q8.Q8Rows(ctx.alloc(x.size), ctx.alloc(x.size // 8), 6, h)
    ctx.add_rmsnorm(ctx.to_device(x), ctx.to_device(r), ctx.to_device(w), s, 6, h, normed=y,
                    quantized=rows, eps=1e-30)
    got = ctx.to_host(y, (6, h), np.float32)
    q, sc = ctx.to_host(rows.values, (6, h), np.int8), ctx.to_host(rows.scales, (6, h // 32), np.float32)
    fine = [0, 1, 2, 5]
    check_rows(ctx, oracle, x[fine], r[fine], w, 1e-30, False, "f32",
               ctx.to_host(s, (6, h), np.float32)[fine], got[fine], q[fine], sc[fine])
    # inf: rstd 0, so zeros and inf * 0; NaN: a row of NaN
    assert np.isnan(got[3, 9]) and not got[3, :9].any() and np.isnan(got[4]).all()
    assert not q[3].any() and not q[4].any() and not sc[3].any() and not sc[4].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("which", ["sum in x", "sum in r", "normed in x", "normed only", "quantized only"])
def test_outputs_in_place_and_alone(ctx, q8, oracle, dtype, which):
    rng = np.random.default_rng(8)
    m, h = 9, 160
    x, r, w = make(rng, oracle, m, h, dtype)
    xd, rd, wd = (put(ctx, oracle, a, dtype) for a in (x, r, w))
    esz = 2 if dtype == "bf16" else 4
    s, y = ctx.alloc(m * h * esz), ctx.alloc(m * h * esz)
    rows = q8.Q8Rows(ctx.alloc(m * h), ctx.alloc(m * h // 8), m, h)
    ctx.add_rmsnorm(xd, rd, wd, s, m, h, normed=y, quantized=rows, dtype=dtype)
    want = (get(ctx, oracle, s, (m, h), dtype), get(ctx, oracle, y, (m, h), dtype),
            ctx.to_host(rows.values, (m, h), np.int8), ctx.to_host(rows.scales, (m, h // 32), np.float32))
    s2 = {"sum in x": xd, "sum in r": rd}.get(which, ctx.alloc(m * h * esz))
    y2 = xd if which == "normed in x" else None if which == "quantized only" else ctx.alloc(m * h * esz)
    q2 = None if which == "normed only" else q8.Q8Rows(ctx.alloc(m * h), ctx.alloc(m * h // 8), m, h)
    ctx.add_rmsnorm(xd, rd, wd, s2, m, h, normed=y2, quantized=q2, dtype=dtype)
    assert same(get(ctx, oracle, s2, (m, h), dtype), want[0])
    if y2 is not None:
        assert same(get(ctx, oracle, y2, (m, h), dtype), want[1])
    if q2 is not None:
        assert np.array_equal(ctx.to_host(q2.values, (m, h), np.int8), want[2])
        assert same(ctx.to_host(q2.scales, (m, h // 32), np.float32), want[3])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_and_unaligned_rows(ctx, q8, oracle, dtype):
    """Rows of odd strides from odd addresses give the bits of dense ones, and
    what lies between the rows stays."""
    rng = np.random.default_rng(9)
    m, h, ld = 4, 96, 99
    et = np.uint16 if dtype == "bf16" else np.float32
    esz = np.dtype(et).itemsize
    x, r, w = make(rng, oracle, m, h, dtype)
    raw = lambda a: oracle.f32_to_bf16_bits(a) if dtype == "bf16" else a  # noqa: E731
    dense = [ctx.alloc(m * h * esz) for _ in range(2)]
    wd = put(ctx, oracle, w, dtype)
    ctx.add_rmsnorm(put(ctx, oracle, x, dtype), put(ctx, oracle, r, dtype), wd, dense[0], m, h,
                    normed=dense[1], dtype=dtype)

    def strided(a):
        b = np.full(1 + m * ld, 5, et)
        if a is not None:
            b[1:].reshape(m, ld)[:, :h] = raw(a)
        return ctx.to_device(b)
    bufs = [strided(a) for a in (x, r, None, None)]
    views = [q8.f32_memref(b.ptr + esz, m, h, row_stride=ld) for b in bufs]
    entry = getattr(q8.lib(), "llmcp_q8_add_rmsnorm" + ("_bf16" if dtype == "bf16" else ""))
    wv = q8.i8_memref(wd.ptr, h)
    q8.check(entry(ctx.handle, ctypes.byref(views[0]), ctypes.byref(views[1]), ctypes.byref(wv), 1e-6, 0,
                   ctypes.byref(views[2]), ctypes.byref(views[3]), None))
    for b, d in zip(bufs[2:], dense):
        got = ctx.to_host(b, (1 + m * ld,), et)
        assert got[0] == 5 and (got[1:].reshape(m, ld)[:, h:] == 5).all()
        assert np.array_equal(got[1:].reshape(m, ld)[:, :h], ctx.to_host(d, (m, h), et))


def test_add_rmsnorm_refuses(ctx, q8):
    buf, L, ref = ctx.alloc(1 << 20), q8.lib(), ctypes.byref
    mr = q8.f32_memref

    def call(x, r, w, s, n, q):
        opt = lambda d: None if d is None else ref(d)  # noqa: E731
        return L.llmcp_q8_add_rmsnorm(ctx.handle, ref(x), ref(r), opt(w), 1e-6, 0, ref(s), opt(n), opt(q))
    a = lambda i, m=2, h=64: mr(buf.ptr + (i << 14), m, h)  # noqa: E731
    w = q8.i8_memref(buf.ptr, 64)
    q = q8.MemRefRows(buf.ptr + (5 << 14), buf.ptr + (6 << 14), 2, 64)
    assert call(a(1), a(2), w, a(3), a(4), q) == q8.OK
    assert call(a(1), a(2), w, a(3), None, None) == q8.EINVAL
    assert call(a(1), a(2), w, a(3), a(3), None) == q8.EINVAL
    assert call(a(1), a(2), None, a(3), a(4), None) == q8.EINVAL
    assert call(a(1), a(2, 3), w, a(3), a(4), None) == q8.DECLINED
    assert call(a(1), a(2), w, a(3, 2, 32), a(4), None) == q8.DECLINED
    assert call(a(1), a(2), w, a(3), a(4, 1), None) == q8.DECLINED
    assert call(a(1), a(2), q8.i8_memref(buf.ptr, 32), a(3), a(4), None) == q8.DECLINED
    assert call(a(1), a(2), q8.i8_memref(buf.ptr + 4, 64), a(3), a(4), None) == q8.DECLINED
    h48 = q8.i8_memref(buf.ptr, 48)
    assert call(a(1, 2, 48), a(2, 2, 48), h48, a(3, 2, 48), a(4, 2, 48), None) == q8.DECLINED
    wide = 32800
    assert call(a(1, 1, wide), a(1, 1, wide), q8.i8_memref(buf.ptr, wide), a(1, 1, wide),
                a(16, 1, wide), None) == q8.DECLINED
    for bad in (q8.MemRefRows(None, buf.ptr, 2, 64), q8.MemRefRows(buf.ptr, None, 2, 64)):
        assert call(a(1), a(2), w, a(3), a(4), bad) == q8.EINVAL
    for bad in (q8.MemRefRows(buf.ptr + 8, buf.ptr, 2, 64), q8.MemRefRows(buf.ptr, buf.ptr, 3, 64)):
        assert call(a(1), a(2), w, a(3), a(4), bad) == q8.DECLINED
    assert call(a(1, 0), a(2, 0), w, a(3, 0), a(4, 0), None) == q8.OK
