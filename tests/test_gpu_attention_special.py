"""llmcp_q8_attention with infinities and NaN among the keys and values that rows
see, with scores that leave f32, and where the low bits of f32 rows decide.

What is expected comes row by row from the definition in float64 over the keys
that the row sees, with IEEE's rules for infinities: a score of -inf is a weight
of 0, one of +inf or NaN makes the row NaN, an infinite value that has a weight
makes its column infinite.  Finite results keep to the bound of
test_gpu_attention.py."""
import numpy as np
import pytest

from kv_reference import F32, Cache, rows_of
from test_gpu_attention import filled, forced, reference  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of f32

# (dtype, kernel, splits): f32 rows always take tiles of 16
KINDS = [("f32", 0, 0), ("f32", 1, 3), ("bf16", 1, 1), ("bf16", 1, 3), ("bf16", 2, 1), ("bf16", 2, 2)]


@pytest.fixture(autouse=True)
def once(ctx):
    if ctx.platform != "aarch64":
        pytest.skip("the same kernels on either platform")


def some(n):
    """Rows of n that are looked at, those around the middle and the ends among them."""
    return sorted({i for i in range(n) if i % 7 == 0 or abs(i - n // 2) < 3 or n - i < 4})


def attend(q8, ctx, oracle, c, ns, lengths, q, dtype, scale):
    """Rows q (values of dtype) [sum ns, heads, dim] through the call, as f32."""
    bits = oracle.f32_to_bf16_bits(q) if dtype == "bf16" else q
    y = ctx.to_device(np.full(q.shape, 7, bits.dtype))
    ctx.attention(ctx.to_device(bits), c.cache(), c.batch(np.concatenate([[0], np.cumsum(ns)]), lengths),
                  y, q.shape[0], q.shape[1], scale=scale, dtype=dtype)
    got = ctx.to_host(y, q.shape, bits.dtype)
    return oracle.bf16_bits_to_f32(got) if dtype == "bf16" else got


@pytest.mark.parametrize("page", [16, 20, 64])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 75])
@pytest.mark.parametrize("kind", KINDS)
def test_infinite_keys(q8, ctx, oracle, forced, kind, n, dim, page):
    """Keys whose score is -inf have no weight, wherever they stand; one whose
    score is +inf makes the rows that see it NaN; the other kv head's rows keep
    their values.  The queries fit bf16, so f32 rows have parts that are 0."""
    dtype, kernel, splits = kind
    forced(kernel, splits)
    rng = np.random.default_rng(dim + n)
    length = 400
    c = filled(q8, ctx, oracle, rng, [length], page, 2, dim, "bf16")
    _, q = rows_of(oracle, rng, n, 4, dim, "bf16", 2.0)
    q[:, :, 1], q[:, 1, 1] = 1.0, 1.5
    lowest = [3, 40, 41, 200, 319, length - n, length - 1]
    for at in lowest:
        c.k[c.table[0, at // page], 0, at % page, 1] = 0xFF80
    c.upload()
    kk, vv = c.values(oracle, 0, 0, length)
    keep = np.ones(length, bool)
    keep[lowest] = False
    got = attend(q8, ctx, oracle, c, [n], [length], q, dtype, 0.2)
    for i in some(n):
        use = np.arange(length) <= length - n + i
        want, bound = reference(q[i:i + 1, 2:], kk[use, 1:], vv[use, 1:], 0.2, length, dtype == "bf16")
        assert (np.abs(got[i, 2:] - want[0]) <= bound[0]).all()
        use &= keep
        want, bound = reference(q[i:i + 1, :2], kk[use, :1], vv[use, :1], 0.2, length, dtype == "bf16")
        assert (np.abs(got[i, :2] - want[0]) <= bound[0]).all()
    at = length - (n + 1) // 2
    c.k[c.table[0, at // page], 0, at % page, 1] = 0x7F80
    c.upload()
    again = attend(q8, ctx, oracle, c, [n], [length], q, dtype, 0.2)
    sees = length - n + np.arange(n) >= at
    assert np.isnan(again[sees, :2]).all()
    assert np.array_equal(again[:, 2:], got[:, 2:]) and np.array_equal(again[~sees], got[~sees])


@pytest.mark.parametrize("kind", KINDS)
def test_scores_of_minus_infinity_alone(q8, ctx, oracle, forced, kind):
    """Give zeros, also of f32 rows whose values fit bf16."""
    dtype, kernel, splits = kind
    forced(kernel, splits)
    rng = np.random.default_rng(5)
    c = filled(q8, ctx, oracle, rng, [200, 200], 16, 1, 64, "bf16")
    c.k[c.table[0], 0, :, 1] = 0xFF80
    c.upload()
    _, q = rows_of(oracle, rng, 4, 2, 64, "bf16")
    q[:, :, 1] = 1.0
    got = attend(q8, ctx, oracle, c, [2, 2], [200, 200], q, dtype, 0.1)
    assert (got[:2] == 0).all() and np.isfinite(got).all() and (got[2:] != 0).all()


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("page", [16, 20, 64])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 75])
@pytest.mark.parametrize("kind", KINDS)
def test_odd_values(q8, ctx, oracle, forced, kind, n, dim, page, fmt):
    """Infinite and NaN values, seen by all rows and by some: an infinity keeps
    its sign, in its column and head alone (of a Q8 row with one, whose values
    read back as NaN, in all columns); all else keeps to the bound."""
    dtype, kernel, splits = kind
    forced(kernel, splits)
    rng = np.random.default_rng(dim + n)
    length, kvh = 400, 3
    c = filled(q8, ctx, oracle, rng, [length + 30], page, kvh, dim, fmt)
    _, q = rows_of(oracle, rng, n, 6, dim, dtype, 1.0)
    clean_k, clean_v = c.values(oracle, 0, 0, length)
    # (position, kv head, column, value); the two of kv head 0's column 9 meet
    odd = [(37, 0, 9, np.inf), (length - n // 2 - 1, 0, 20, -np.inf), (length - 2, 0, 9, -np.inf),
           (length - 1, 1, 0, np.inf), (length - n, 1, dim - 1, np.nan), (length, 2, 4, np.inf)]
    if fmt == "q8":
        odd = [o for o in odd if o[0] != 37]
    for at, h, col, x in odd:
        slot = c.table[0, at // page], h, at % page
        if fmt == "bf16":
            c.v[slot][col] = {np.inf: 0x7F80, -np.inf: 0xFF80}.get(x, 0x7FC0)
        else:
            c.vs[slot] = np.nan
    c.upload()
    got = attend(q8, ctx, oracle, c, [n], [length], q, dtype, 0.05)
    for i in some(n):
        last = length - n + i
        want, bound = reference(q[i:i + 1], clean_k[:last + 1], clean_v[:last + 1], 0.05, length, dtype == "bf16")
        expect, loose = want[0].copy(), bound[0].copy()
        for at, h, col, x in odd:
            if at <= last:
                here = np.s_[2 * h:2 * h + 2, col] if fmt == "bf16" else np.s_[2 * h:2 * h + 2]
                value = x if fmt == "bf16" else np.nan
                with np.errstate(invalid="ignore"):
                    expect[here] = expect[here] + value
        fine = np.isfinite(expect)
        assert np.array_equal(got[i][~fine], expect[~fine].astype(F32), equal_nan=True)
        assert (np.abs(got[i][fine] - expect[fine]) <= loose[fine]).all()


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("scale", [1e30, -1e30, 1e38, 3e37, 100.0, -1e4])
@pytest.mark.parametrize("kind", KINDS)
def test_scores_past_f32(q8, ctx, oracle, forced, kind, scale, fmt):
    """A score that f32 has no number for counts as infinite: above, the row is
    NaN; below, the key has no weight.  Queries and keys of one value each, so that
    q . k is exact: 127 * 2^20, which 1e30 takes to 1.3e38 (times log2 e 1.9e38),
    a number still, and the others past 3.4e38."""
    dtype, kernel, splits = kind
    forced(kernel, splits)
    rng = np.random.default_rng(8)
    length, n, dim = 300, 40, 64
    sign = 1.0 if scale > 0 else -1.0
    c = Cache(q8, ctx, rng, [length], 16, 1, dim, fmt)
    k = np.zeros((length, 1, dim), F32)
    k[::3, 0, 5] = -127.0 * 2.0 ** 10 * sign  # scores of -inf
    k[270, 0, 5] = 127.0 * 2.0 ** 10 * sign   # of +inf where q is positive
    v = rng.standard_normal((length, 1, dim)).astype(F32)
    c.put(oracle, 0, 0, k, v)
    c.upload()
    q = np.zeros((n, 2, dim), F32)
    q[:, 0, 5] = 2.0 ** 10
    got = attend(q8, ctx, oracle, c, [n], [length], q, dtype, scale)
    _, vv = c.values(oracle, 0, 0, length)
    for i in range(n):
        last = length - n + i
        even = np.zeros((1, 1, dim), F32)
        use = np.arange(length) <= last
        want, bound = reference(even, np.zeros((use.sum(), 1, dim)), vv[use], 1.0, length, dtype == "bf16")
        assert (np.abs(got[i, 1] - want[0, 0]) <= bound[0, 0]).all()
        if last >= 270 and abs(scale) > 1e30:
            assert np.isnan(got[i, 0]).all()
            continue
        if last >= 270:  # that key alone
            assert (np.abs(got[i, 0] - vv[270, 0]) <= (2.0 ** -7 if dtype == "bf16" else 2 * U32) * np.abs(vv[270, 0])).all()
            continue
        use &= k[:, 0, 5] == 0
        want, bound = reference(even, np.zeros((use.sum(), 1, dim)), vv[use], 1.0, length, dtype == "bf16")
        assert (np.abs(got[i, 0] - want[0, 0]) <= bound[0, 0]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-38, 1e-45])
def test_scales_next_to_zero(q8, ctx, oracle, forced, kind, scale):
    """A scale of 0 weighs every key alike, however large q . k; 0 times an
    infinite one is NaN.  q . k is 2^127 here, so a scale of 1e-38 or 1e-45 still
    gives scores of 1.7 and 2.4e-7."""
    dtype, kernel, splits = kind
    forced(kernel, splits)
    rng = np.random.default_rng(9)
    length, n, dim = 150, 36, 64
    c = Cache(q8, ctx, rng, [length], 32, 2, dim, "bf16")
    k = np.zeros((length, 2, dim), F32)
    k[::2, :, 3] = 2.0 ** 64
    v = rng.standard_normal((length, 2, dim)).astype(F32)
    c.put(oracle, 0, 0, k, v)
    c.k[c.table[0, 0], 1, 7, 3] = 0x7F80
    c.upload()
    q = np.zeros((n, 4, dim), F32)
    q[:, :, 3] = 2.0 ** 63
    got = attend(q8, ctx, oracle, c, [n], [length], q, dtype, scale)
    kk, vv = c.values(oracle, 0, 0, length)
    want, bound = reference(q[:, :2], kk[:, :1], vv[:, :1], float(F32(scale)), length - n, dtype == "bf16")
    assert (np.abs(got[:, :2] - want) <= bound).all()
    assert np.isnan(got[:, 2:]).all()


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("page", [16, 20])
def test_low_bits_of_f32_queries_decide(q8, ctx, oracle, page, fmt):
    """q's values differ from 1 + 2^-8 by a few 2^-17 and meet keys of +-2^17 c, so
    that a score is what the last 8 of q's 24 bits say; all products and sums are
    exact in f32.  With the leading 16 bits alone every weight would be the same."""
    rng = np.random.default_rng(21)
    length, n, dim = 90, 3, 64
    c = Cache(q8, ctx, rng, [length], page, 1, dim, fmt)
    k = np.zeros((length, 1, dim), F32)
    at = rng.integers(0, dim // 2, length)
    size = rng.integers(1, 3, length).astype(F32) * F32(2.0 ** 17)
    for j in range(length):
        k[j, 0, 2 * at[j]], k[j, 0, 2 * at[j] + 1] = size[j], -size[j]
    v = rng.standard_normal((length, 1, dim)).astype(F32)
    c.put(oracle, 0, 0, k, v)
    c.upload()
    kk, vv = c.values(oracle, 0, 0, length)
    q = np.full((n, 2, dim), 1 + 2.0 ** -8, F32)
    q[:, :, ::2] += rng.integers(0, 4, (n, 2, dim // 2)).astype(F32) * F32(2.0 ** -17)
    got = attend(q8, ctx, oracle, c, [n], [length], q, "f32", 0.5)
    # exact scores but for their scale (and of Q8 a step's rounding, in kk): a
    # rounding each for scale, scale * log2 e, a Q8 scale and the product, and the
    # exponential's, the sums' and the result's
    for i in range(n):
        seen = length - n + i + 1
        for h in range(2):
            s = 0.5 * (kk[:seen, 0].astype(np.float64) @ q[i, h].astype(np.float64))
            p = np.exp(s - s.max())
            p /= p.sum()
            want = p @ vv[:seen, 0].astype(np.float64)
            ep = (8 * np.abs(s).max() + seen + 64) * U32
            assert (np.abs(got[i, h] - want) <= ep * (p @ np.abs(vv[:seen, 0])) + U32 * np.abs(want)).all()
            flat = vv[:seen, 0].mean(0)
            assert np.abs(flat - want).max() > 0.05  # (what the leading 16 bits alone give)


@pytest.mark.parametrize("page", [16, 20])
def test_low_bits_of_f32_weights_decide(q8, ctx, oracle, page):
    """Two keys of weights 1 and 1 - d, d a few 2^-19, with values +-V: the result is
    V d / 2 next to V.  Two parts of a weight hold 16 bits, which would be off by up
    to 2^-17 V."""
    length, dim = 2, 64
    rng = np.random.default_rng(22)
    c = Cache(q8, ctx, rng, [length], page, 1, dim, "bf16")
    k, v = np.zeros((2, length, 1, dim), F32)
    k[1, 0, 0] = -1.0
    v[0], v[1] = 1024.0, -1024.0
    c.put(oracle, 0, 0, k, v)
    c.upload()
    q = np.zeros((1, 12, dim), F32)
    d = (np.arange(12) + 0.37) * 2.0 ** -19
    q[0, :, 0] = d.astype(F32)
    got = attend(q8, ctx, oracle, c, [1], [length], q, "f32", 1.0)
    p = np.exp(-d.astype(F32).astype(np.float64))
    want = 1024.0 * (1 - p) / (1 + p)
    # a step of f32 (2^-23) for each of the exponential, the rounded exponent and
    # the sums, of weights next to 1
    bound = 1024.0 * 4 * 2.0 ** -23 / 2
    assert (np.abs(got[0] - want[:, None]) <= bound).all()
    two = (np.floor(p * 2.0 ** 16) / 2.0 ** 16)
    assert (np.abs(1024.0 * (1 - two) / (1 + two) - want) > bound).sum() > 6


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ns,lengths", [
    ([260] + [1] * 9, [700] + [7 * i + 30 for i in range(9)]),
    ([1] * 40 + [150], [11 * i + 1 for i in range(40)] + [150]),
    ([1, 900, 0, 1, 2], [1300, 1000, 50, 3, 2])])
def test_a_prompt_among_single_rows(q8, ctx, oracle, ns, lengths, dtype, fmt):
    """One call of a chunk of many rows and sequences of one row, either way around."""
    from test_gpu_attention import run
    rng = np.random.default_rng(31)
    c = filled(q8, ctx, oracle, rng, lengths, 32, 2, 64, fmt)
    _, q = rows_of(oracle, rng, sum(ns), 8, 64, dtype, 2.0)
    run(q8, ctx, oracle, c, ns, lengths, q, dtype, 0.125)


@pytest.mark.parametrize("at", [20, 140, 195])
@pytest.mark.parametrize("kind", KINDS)
def test_nan_without_weight(q8, ctx, oracle, forced, kind, at):
    """A Q8 row of NaN values whose key is seen and whose weight is 0 in f32 (its
    score is 200 below the others) makes its rows NaN wherever it stands, as 0 times
    NaN does; rows that do not see it keep their values."""
    dtype, kernel, splits = kind
    forced(kernel, splits)
    rng = np.random.default_rng(at)
    length, n, dim, page = 200, 40, 64, 64
    c = Cache(q8, ctx, rng, [length], page, 1, dim, "q8")
    k = np.zeros((length, 1, dim), F32)
    k[at, 0, 0] = -200.0
    v = rng.standard_normal((length, 1, dim)).astype(F32)
    c.put(oracle, 0, 0, k, v)
    c.vs[c.table[0, at // page], 0, at % page] = np.nan
    c.upload()
    q = np.zeros((n, 2, dim), F32)
    q[:, :, 0] = 1.0
    got = attend(q8, ctx, oracle, c, [n], [length], q, dtype, 1.0)
    sees = length - n + np.arange(n) >= at
    assert np.isnan(got[sees]).all()
    if not sees.all():
        kk, vv = c.values(oracle, 0, 0, at)
        want, bound = reference(q[~sees], kk, vv, 1.0, length - n, dtype == "bf16")
        assert (np.abs(got[~sees] - want) <= bound).all()
