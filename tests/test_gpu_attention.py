"""llmcp_q8_attention against its definition in float64, with a bound counted in
roundings: scores of D products summed in f32, exponentials and sums of f32,
and for bf16 rows the probabilities' and the result's rounding to bf16."""
import numpy as np
import pytest

from kv_reference import F32, Cache, rows_of, same

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8  # half a step of f32, of bf16


def reference(q, k, v, scale, first, bf16):
    """(o, bound) of the rows q [n, heads, dim] at the positions from `first`
    over k, v [keys, kv heads, dim]."""
    n, heads, dim = q.shape
    keys, kvh = k.shape[:2]
    out, bound = np.zeros((2, n, heads, dim))
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    sees = np.arange(keys)[None, :] <= (first + np.arange(n))[:, None]
    for h in range(heads):
        g = h // (heads // kvh)
        with np.errstate(all="ignore"):
            s = np.where(sees, scale * (q[:, h] @ k[:, g].T), -np.inf)
            most = np.where(sees, abs(scale) * (np.abs(q[:, h]) @ np.abs(k[:, g]).T), 0)
            if keys == 0:
                continue
            top = s.max(-1, keepdims=True)
            e = np.where(sees, np.exp(s - np.where(np.isneginf(top), 0, top)), 0)
            p = e / np.where(e.sum(-1, keepdims=True) == 0, 1, e.sum(-1, keepdims=True))
            vg = np.where(sees.any(0)[:, None], v[:, g], 0)
            out[:, h] = p @ vg
            # a score's error, from its products' sum and the scaling
            es = (dim + 8) * U32 * most.max(-1, initial=0, keepdims=True)
            # of a weight: twice that, the exponential and rescalings, the sums
            ep = 2 * es + (keys + 64) * U32 + 2.0 ** -20 + (U16 if bf16 else 0)
            bound[:, h] = ep * (p @ np.abs(vg)) + (U16 if bf16 else U32) * np.abs(out[:, h]) + 1e-37
    return out, bound


def run(q8, ctx, oracle, c, ns, lengths, q, dtype, scale, pad=0, sees=None):
    """The call's rows [sum ns + pad, heads, dim] and the check of those of
    every sequence."""
    starts = np.concatenate([[0], np.cumsum(ns)])
    rows = int(starts[-1]) + pad
    bits = oracle.f32_to_bf16_bits(q) if dtype == "bf16" else q
    y = ctx.to_device(np.full(q.shape, 7, bits.dtype))
    ctx.attention(ctx.to_device(bits), c.cache(), c.batch(starts, lengths), y, rows, q.shape[1],
                  scale=scale, dtype=dtype)
    got = ctx.to_host(y, q.shape, bits.dtype)
    assert (got[starts[-1]:] == 7).all()
    wide = oracle.bf16_bits_to_f32(got) if dtype == "bf16" else got
    for s, n in enumerate(ns):
        k, v = c.values(oracle, s, 0, max(0, min(lengths[s], c.width * c.page)))
        if sees is not None:
            k, v = k[sees[s]], v[sees[s]]
        a = starts[s]
        want, bound = reference(q[a:a + n], k, v, scale, lengths[s] - n, dtype == "bf16")
        err = np.abs(wide[a:a + n] - want)
        assert (err <= bound).all(), (s, float((err / bound).max()))
    return wide


def filled(q8, ctx, oracle, rng, lengths, page, kvh, dim, fmt, scale=1.0, **kw):
    c = Cache(q8, ctx, rng, lengths, page, kvh, dim, fmt, **kw)
    for s, n in enumerate(lengths):
        n = min(n, c.width * page)
        c.put(oracle, s, 0, *(rng.standard_normal((n, kvh, dim)).astype(F32) * scale
                              for _ in range(2)))
    c.upload()
    return c


# (rows, lengths, page, heads, kv heads, dim): single tokens of short, odd and long
# contexts; chunks that start at the first key and in the middle, whose tiles end
# inside a group and inside a step of keys; sequences without rows, without
# keys, with fewer keys than rows; many sequences; many heads of one kv head
SHAPES = [
    ([1], [1], 16, 4, 4, 64), ([1], [33], 32, 16, 4, 256), ([1], [1000], 1000, 16, 4, 256),
    ([1] * 5, [7, 300, 1, 129, 64], 48, 8, 2, 128), ([3, 0, 9], [3, 50, 200], 20, 6, 2, 64),
    ([40], [40], 7, 8, 8, 128), ([17, 65], [17, 170], 64, 12, 3, 64), ([23], [23], 16, 16, 4, 256),
    ([6, 5, 4], [0, 3, 4], 5, 2, 1, 64), ([2, 1], [600, 1500], 128, 24, 1, 64),
    ([1] * 67 + [0, 4], [5 * i + 1 for i in range(67)] + [9, 11], 16, 2, 2, 64),
    ([150], [400], 33, 4, 2, 128), ([130], [130], 64, 4, 1, 256), ([1], [4096], 256, 3, 1, 128),
    ([333, 1], [333, 700], 24, 4, 4, 64)]


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(q8, ctx, oracle, shape, dtype, fmt):
    ns, lengths, page, heads, kvh, dim = SHAPES[shape]
    rng = np.random.default_rng(100 + shape)
    c = filled(q8, ctx, oracle, rng, lengths, page, kvh, dim, fmt)
    _, q = rows_of(oracle, rng, sum(ns) + 2, heads, dim, dtype, 2.0)
    run(q8, ctx, oracle, c, ns, lengths, q, dtype, dim ** -0.5, pad=2)
    assert ctx.check_flag() == 0


@pytest.fixture
def forced(q8, ctx):
    """Forces the kernel (1: tiles of 16 rows, 2: of 128) and the parts of the
    keys on the context; undone afterwards."""
    yield lambda kernel, splits=0: q8.check(
        q8.lib().llmcp_q8_test_ctx_attention(ctx.handle, kernel, splits))
    q8.check(q8.lib().llmcp_q8_test_ctx_attention(ctx.handle, 0, 0))


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("kernel,splits", [(1, 1), (1, 5), (2, 1), (2, 3)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_each_kernel(q8, ctx, oracle, forced, shape, kernel, splits, fmt):
    ns, lengths, page, heads, kvh, dim = SHAPES[shape]
    rng = np.random.default_rng(300 + shape)
    c = filled(q8, ctx, oracle, rng, lengths, page, kvh, dim, fmt)
    _, q = rows_of(oracle, rng, sum(ns) + 2, heads, dim, "bf16", 2.0)
    forced(kernel, splits)
    run(q8, ctx, oracle, c, ns, lengths, q, "bf16", dim ** -0.5, pad=2)
    assert ctx.check_flag() == 0


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("ns,lengths,page,heads,kvh,dim", [
    ([1100], [1100], 64, 16, 4, 64), ([700, 500], [900, 500], 40, 16, 2, 128),
    ([1050], [1300], 1300, 16, 4, 256), ([1030, 3, 0], [1030, 40, 7], 16, 16, 16, 64)])
def test_long_chunks(q8, ctx, oracle, ns, lengths, page, heads, kvh, dim, fmt):
    rng = np.random.default_rng(23)
    c = filled(q8, ctx, oracle, rng, lengths, page, kvh, dim, fmt)
    _, q = rows_of(oracle, rng, sum(ns), heads, dim, "bf16", 2.0)
    run(q8, ctx, oracle, c, ns, lengths, q, "bf16", dim ** -0.5)


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("kernel", [1, 2])
def test_growing_scores(q8, ctx, oracle, forced, kernel, fmt):
    """Scores that rise by hundreds along the keys, and fall: the running
    maximum moves at every step, or never again."""
    rng = np.random.default_rng(29)
    n, length, dim = 70, 390, 64
    q = np.abs(rows_of(oracle, rng, n, 2, dim, "bf16", 1.0)[1])
    for sign in (1.0, -1.0):
        c = Cache(q8, ctx, rng, [length], 16, 1, dim, fmt)
        k = np.abs(rng.standard_normal((length, 1, dim))).astype(F32)
        k *= (sign * np.linspace(-3, 3, length)).astype(F32)[:, None, None]
        c.put(oracle, 0, 0, k, rng.standard_normal((length, 1, dim)).astype(F32))
        c.upload()
        forced(kernel, 2)
        run(q8, ctx, oracle, c, [n], [length], q, "bf16", 4.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_scales(q8, ctx, oracle, dtype, fmt, scale):
    """Flat, negative and nearly one-hot softmax."""
    rng = np.random.default_rng(7)
    c = filled(q8, ctx, oracle, rng, [90, 300], 16, 2, 128, fmt)
    _, q = rows_of(oracle, rng, 21, 6, 128, dtype, 2.0)
    run(q8, ctx, oracle, c, [20, 1], [90, 300], q, dtype, scale)


@pytest.mark.parametrize("n", [1, 40, 200])
@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("kernel", [1, 2])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_odd_values_out_of_sight(q8, ctx, oracle, forced, n, fmt, kernel, dim):
    """Infinities and NaN at positions that a row does not see leave it alone:
    behind the last key, in the chunk's later rows, on no page; the rows that
    see them are NaN or infinite."""
    forced(kernel)
    rng = np.random.default_rng(n)
    length, kvh, page = 260, 2, 16
    c = filled(q8, ctx, oracle, rng, [length + 30], page, kvh, dim, fmt)
    k, v = (rng.standard_normal((1, kvh, dim)).astype(F32) for _ in range(2))
    odd = length - 5 if n > 1 else length + 3
    k[0, 0, 3], v[0, 0, 9], v[0, 1, 7] = np.nan, np.inf, np.nan
    c.put(oracle, 0, odd, k, v)
    c.table[0, 3] = -1  # positions 48 .. 63
    c.upload()
    q = rows_of(oracle, rng, n, 4, dim, "bf16", 2.0)[1]
    starts = [0, n]
    y = ctx.to_device(np.zeros(q.shape, np.uint16))
    ctx.attention(ctx.to_device(oracle.f32_to_bf16_bits(q)), c.cache(), c.batch(starts, [length]), y,
                  n, 4, scale=0.2, dtype="bf16")
    got = oracle.bf16_bits_to_f32(ctx.to_host(y, q.shape, np.uint16))
    sees_odd = length - n + np.arange(n) >= odd
    kk, vv = c.values(oracle, 0, 0, length)
    keep = np.ones(length, bool)
    keep[48:64] = False
    first = length - n
    for i in range(n):
        if sees_odd[i]:
            assert not np.isfinite(got[i, 0]).all()
            assert np.isnan(got[i, 2:, 7] if fmt == "bf16" else got[i, 2:]).all()
            continue
        use = keep.copy()
        use[first + i + 1:] = False
        want, bound = reference(q[i:i + 1], kk[use], vv[use], 0.2, length, True)
        assert (np.abs(got[i] - want[0]) <= bound[0]).all()


@pytest.mark.parametrize("kernel", [1, 2])
def test_rows_without_sight(q8, ctx, oracle, forced, kernel):
    """No page at all, no key, and scores of -inf alone give zeros."""
    forced(kernel)
    rng = np.random.default_rng(3)
    c = filled(q8, ctx, oracle, rng, [40, 40, 8], 8, 1, 64, "bf16")
    c.table[0, :] = -1
    bits, q = rows_of(oracle, rng, 5, 2, 64, "bf16")
    c.k[c.table[2, 0], 0, :8, 1] = 0xFF80  # -inf
    bits[4, :, 1] = 0x3F80
    c.upload()
    y = ctx.to_device(np.full(q.shape, 7, np.uint16))
    ctx.attention(ctx.to_device(bits), c.cache(), c.batch([0, 2, 4, 5], [40, 0, 8]), y, 5, 2,
                  scale=0.1, dtype="bf16")
    assert (ctx.to_host(y, q.shape, np.uint16) == 0).all()
    assert ctx.check_flag() == 0


def test_bad_pages_are_flagged(q8, ctx, oracle):
    rng = np.random.default_rng(4)
    c = filled(q8, ctx, oracle, rng, [100], 10, 1, 128, "q8")
    c.table[0, 2], c.table[0, 7] = c.pages, -2
    sees = np.ones(100, bool)
    sees[20:30] = sees[70:80] = False
    _, q = rows_of(oracle, rng, 1, 3, 128, "f32", 2.0)
    run(q8, ctx, oracle, c, [1], [100], q, "f32", 0.1, sees=[sees])
    assert ctx.check_flag() == 1


def test_lengths_past_the_table(q8, ctx, oracle):
    rng = np.random.default_rng(9)
    c = filled(q8, ctx, oracle, rng, [64], 16, 2, 64, "bf16", width=4)
    _, q = rows_of(oracle, rng, 3, 4, 64, "bf16", 2.0)
    run(q8, ctx, oracle, c, [3], [2 ** 31 - 1], q, "bf16", 0.125)
    run(q8, ctx, oracle, c, [3], [66], q, "bf16", 0.125)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_views(q8, ctx, oracle, dtype):
    """Queries as a part of a linear's rows, the output with a stride."""
    rng = np.random.default_rng(11)
    n, heads, kvh, dim = 19, 4, 2, 64
    c = filled(q8, ctx, oracle, rng, [50], 16, kvh, dim, "bf16")
    wide = (heads + 2 * kvh) * dim + 8
    bits, x = rows_of(oracle, rng, n, 1, wide, dtype, 2.0)
    d, y = ctx.to_device(bits), ctx.to_device(np.zeros((n, wide), bits.dtype))
    e = bits.dtype.itemsize
    ctx.attention(d.ptr + 8 * e, c.cache(), c.batch([0, n]), y.ptr + 16 * e, n, heads, scale=0.125,
                  strides=(wide, wide), dtype=dtype)
    got = ctx.to_host(y, (n, wide), bits.dtype)
    assert (got[:, :16] == 0).all() and (got[:, 16 + heads * dim:] == 0).all()
    got = got[:, 16:16 + heads * dim].reshape(n, heads, dim)
    dense = np.ascontiguousarray(bits.reshape(n, wide)[:, 8:8 + heads * dim])
    y2 = ctx.to_device(np.zeros((n, heads, dim), bits.dtype))
    ctx.attention(ctx.to_device(dense), c.cache(), c.batch([0, n]), y2, n, heads, scale=0.125,
                  dtype=dtype)
    assert same(got, ctx.to_host(y2, (n, heads, dim), bits.dtype))


def test_a_sequence_does_not_depend_on_the_others(q8, ctx, oracle):
    """The same bits whatever the other sequences hold and wherever its pages are."""
    rng = np.random.default_rng(13)
    results = []
    k, v = (rng.standard_normal((700, 2, 128)).astype(F32) for _ in range(2))
    bits, q = rows_of(oracle, rng, 3, 8, 128, "bf16", 2.0)
    for other in (5, 650):
        c = filled(q8, ctx, oracle, rng, [other, 700, 700], 16, 2, 128, "q8", width=44)
        c.put(oracle, 1, 0, k, v)
        c.upload()
        y = ctx.to_device(np.zeros(q.shape, np.uint16))
        ctx.attention(ctx.to_device(bits), c.cache(), c.batch([0, 1, 2, 3], [other, 700, 3]), y, 3,
                      8, dtype="bf16")
        results.append(ctx.to_host(y, q.shape, np.uint16)[1])
    assert same(*results)


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
def test_decoding_replayed(q8, ctx, oracle, fmt):
    """A captured step of a cache write and attention, replayed as the
    sequences grow, eager work between the replays."""
    rng = np.random.default_rng(17)
    heads, kvh, dim, page = 16, 4, 256, 32
    c = filled(q8, ctx, oracle, rng, [300, 40], page, kvh, dim, fmt)
    _, k = rows_of(oracle, rng, 2, kvh, dim, "bf16")
    _, v = rows_of(oracle, rng, 2, kvh, dim, "bf16")
    _, q = rows_of(oracle, rng, 2, heads, dim, "bf16", 2.0)
    kd, vd, qd = (ctx.to_device(oracle.f32_to_bf16_bits(x)) for x in (k, v, q))
    y = ctx.to_device(np.zeros(q.shape, np.uint16))
    cache, batch = c.cache(), c.batch([0, 1, 2], [1, 1])
    keep = c.keep

    def calls():
        ctx.kv_write(kd, vd, cache, batch, 2, dtype="bf16")
        ctx.attention(qd, cache, batch, y, 2, heads, scale=0.0625, dtype="bf16")
    calls()
    ctx.graph_begin()
    calls()
    graph = ctx.graph_end()
    for s in range(2):
        c.put(oracle, s, 0, k[s:s + 1], v[s:s + 1])
    for lengths in ([2, 1], [17, 40], [300, 33]):
        host = np.asarray(lengths, np.int32)
        q8.check(q8.lib().llmcp_q8_memcpy_h2d(ctx.handle, keep[1].ptr, host.ctypes.data, 8))
        ctx.graph_launch(graph)
        got = ctx.to_host(y, q.shape, np.uint16)
        for s in range(2):
            c.put(oracle, s, lengths[s] - 1, k[s:s + 1], v[s:s + 1])
        eager = run(q8, ctx, oracle, c, [1, 1], lengths, q, "bf16", 0.0625)
        assert same(oracle.bf16_bits_to_f32(got), eager)
    ctx.graph_destroy(graph)
