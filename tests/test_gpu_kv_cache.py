"""llmcp_q8_kv_write and llmcp_q8_kv_read against a numpy restatement: bf16 by
rounding to nearest even, Q8 with the scale max|x| / 127 and q = rne(x * (1 /
scale)) in f32, bit for bit."""
import numpy as np
import pytest

from kv_reference import F32, Cache, narrow, rows_of, same

pytestmark = pytest.mark.gpu

# (rows, lengths, page, heads, dim): one row; pages of one slot, of odd size, one
# page per sequence; sequences without rows, without keys, with fewer keys than
# rows; more sequences than a wave looks at together
SHAPES = [
    ([1], [1], 16, 4, 256), ([1], [257], 64, 4, 256), ([5, 0, 3], [5, 9, 40], 1, 2, 64),
    ([7, 33, 1], [50, 33, 96], 48, 3, 128), ([4, 6, 2], [0, 3, 1], 5, 1, 64),
    ([1] * 70 + [0] * 60 + [2, 3], list(range(1, 71)) + [3] * 60 + [7, 3], 13, 2, 64),
    ([300], [1000], 1000, 8, 128)]


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_write_and_read(q8, ctx, oracle, shape, dtype, fmt):
    ns, lengths, page, heads, dim = SHAPES[shape]
    rng = np.random.default_rng(shape)
    c = Cache(q8, ctx, rng, lengths, page, heads, dim, fmt)
    starts = np.concatenate([[0], np.cumsum(ns)])
    rows = int(starts[-1]) + 2  # two behind the last sequence
    (kb, k), (vb, v) = (rows_of(oracle, rng, rows, heads, dim, dtype, 3.0) for _ in range(2))
    k[0, 0], kb[0, 0] = 0, 0
    ctx.kv_write(ctx.to_device(kb), ctx.to_device(vb), c.cache(), c.batch(starts), rows, dtype=dtype)
    for s, n in enumerate(ns):
        c.put(oracle, s, lengths[s] - n, k[starts[s]:starts[s] + n], v[starts[s]:starts[s] + n])
    for got, want in zip(c.download(), (c.k, c.v, c.ks, c.vs)):
        assert same(got, want)
    out = [ctx.to_device(np.full((rows, heads, dim), 7, kb.dtype)) for _ in range(2)]
    ctx.kv_read(c.cache(), c.batch(starts), out[0], out[1], rows, dtype=dtype)
    for j in range(2):
        got = ctx.to_host(out[j], (rows, heads, dim), kb.dtype)
        assert (got[starts[-1]:] == 7).all()
        for s, n in enumerate(ns):
            want = narrow(oracle, c.values(oracle, s, lengths[s] - n, lengths[s])[j], dtype)
            assert same(got[starts[s]:starts[s] + n], want)
    assert ctx.check_flag() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_views(q8, ctx, oracle, dtype):
    """Keys and values as parts of one linear's rows."""
    rng = np.random.default_rng(3)
    heads, dim, n = 2, 64, 9
    c = Cache(q8, ctx, rng, [20], 8, heads, dim, "q8")
    wide = 3 * heads * dim + 16
    xb, x = rows_of(oracle, rng, n, 1, wide, dtype)
    d = ctx.to_device(xb)
    e = xb.dtype.itemsize
    at = (heads * dim, 2 * heads * dim + 8)
    ctx.kv_write(d.ptr + at[0] * e, d.ptr + at[1] * e, c.cache(), c.batch([0, n]), n,
                 strides=(wide, wide), dtype=dtype)
    k, v = (x.reshape(n, wide)[:, a:a + heads * dim].reshape(n, heads, dim) for a in at)
    c.put(oracle, 0, 11, k, v)
    for got, want in zip(c.download(), (c.k, c.v, c.ks, c.vs)):
        assert same(got, want)


def test_extreme_rows(q8, ctx, oracle):
    """Rows of infinities, NaN, subnormal and huge values."""
    rng = np.random.default_rng(5)
    heads, dim, n = 1, 64, 12
    k = rng.standard_normal((n, heads, dim)).astype(F32)
    k[0, 0, 5] = np.inf
    k[1, 0, 6] = -np.inf
    k[2, 0, 7] = np.nan
    k[3] *= F32(1e-44)
    k[4] *= F32(2.0 ** -121)
    k[5, 0] = 0
    k[6, 0] = 3.4e38
    k[7, 0] = 0
    k[7, 0, 3] = F32(2.0 ** -118)
    k[8, 0] = 0
    k[8, 0, 3] = np.nextafter(F32(2.0 ** -118), F32(0))
    k[9, 0] = np.linspace(-127, 127, dim).astype(F32) / 2  # ties of the rounding
    k[9, 0, 0] = 127
    k[10, 0] = -0.0
    c = Cache(q8, ctx, rng, [n], 4, heads, dim, "q8")
    ctx.kv_write(ctx.to_device(k), ctx.to_device(k[::-1]), c.cache(), c.batch([0, n]), n)
    c.put(oracle, 0, 0, k, k[::-1])
    for got, want in zip(c.download(), (c.k, c.v, c.ks, c.vs)):
        assert same(got, want)
    out = [ctx.to_device(k) for _ in range(2)]
    ctx.kv_read(c.cache(), c.batch([0, n]), out[0], out[1], n)
    got = ctx.to_host(out[0], k.shape, F32)
    assert np.isnan(got[:3]).all() and np.isfinite(got[3:]).all()


def test_bad_pages_and_bounds(q8, ctx, oracle):
    """Ids that are no page are skipped and flagged, -1 is skipped; bounds of
    rows outside 0 .. rows are cut; positions past the table have no slot."""
    rng = np.random.default_rng(6)
    heads, dim = 2, 64
    c = Cache(q8, ctx, rng, [24, 16], 4, heads, dim, "bf16", width=5)
    c.table[0, 1], c.table[0, 2], c.table[1, 0] = -1, c.pages, -7
    n = 30
    kb, k = rows_of(oracle, rng, n, heads, dim, "bf16")
    starts, lengths = [-3, 24, 999], [24, 6]
    assert ctx.check_flag() == 0
    ctx.kv_write(ctx.to_device(kb), ctx.to_device(kb), c.cache(), c.batch(starts, lengths), n,
                 dtype="bf16")
    assert ctx.check_flag() == 1
    c.put(oracle, 0, 0, k[:24], k[:24])
    c.put(oracle, 1, 0, k[24:], k[24:])
    for got, want in zip(c.download(), (c.k, c.v)):
        assert same(got, want)
    out = [ctx.to_device(np.full(kb.shape, 9, np.uint16)) for _ in range(2)]
    ctx.kv_read(c.cache(), c.batch(starts, lengths), out[0], out[1], n, dtype="bf16")
    assert ctx.check_flag() == 1
    got = ctx.to_host(out[1], kb.shape, np.uint16)
    want = np.concatenate([c.values(oracle, 0, 0, 24)[1], c.values(oracle, 1, 0, 6)[1]])
    assert same(got, oracle.f32_to_bf16_bits(want))


def test_replayed_with_new_lengths(q8, ctx, oracle):
    """A captured write takes the lengths of the replay."""
    rng = np.random.default_rng(8)
    heads, dim = 4, 256
    c = Cache(q8, ctx, rng, [50, 70], 16, heads, dim, "q8")
    kb, k = rows_of(oracle, rng, 2, heads, dim, "bf16")
    d = ctx.to_device(kb)
    out = [ctx.to_device(np.zeros(kb.shape, np.uint16)) for _ in range(2)]
    batch = c.batch([0, 1, 2], [1, 2])
    cache = c.cache()

    def calls():
        ctx.kv_write(d, d, cache, batch, 2, dtype="bf16")
        ctx.kv_read(cache, batch, out[0], out[1], 2, dtype="bf16")
    calls()
    ctx.graph_begin()
    calls()
    graph = ctx.graph_end()
    c.put(oracle, 0, 0, k[:1], k[:1])
    c.put(oracle, 1, 1, k[1:], k[1:])
    for step in range(3):
        lengths = [5 + 17 * step, 30 + 16 * step]
        host = np.asarray(lengths, np.int32)
        q8.check(q8.lib().llmcp_q8_memcpy_h2d(ctx.handle, c.keep[1].ptr, host.ctypes.data, 8))
        ctx.graph_launch(graph)
        for s in range(2):
            c.put(oracle, s, lengths[s] - 1, k[s:s + 1], k[s:s + 1])
        for got, want in zip(c.download(), (c.k, c.v, c.ks, c.vs)):
            assert same(got, want)
        want = np.concatenate([c.values(oracle, s, lengths[s] - 1, lengths[s])[0] for s in range(2)])
        assert same(ctx.to_host(out[0], kb.shape, np.uint16), oracle.f32_to_bf16_bits(want))
    ctx.graph_destroy(graph)
