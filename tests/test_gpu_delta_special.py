"""The delta rule with decays that grow the state, infinities and NaN in each of its
inputs, and values that leave f32 on the way: rows before stay as they are, other
columns, heads and sequences too, in chunks as row after row."""
import numpy as np
import pytest

import delta_reference as ref

pytestmark = pytest.mark.gpu

F32 = np.float32
BITS = {"nan": 0x7FC0, "inf": 0x7F80, "-inf": 0xFF80}
KH, VH, KD, VD = 2, 4, 64, 32


@pytest.fixture(autouse=True)
def once(ctx):
    if ctx.platform != "aarch64":
        pytest.skip("the same kernels on either platform")


class Call:
    """Two sequences of n rows, dense inputs (f32 arrays; bf16 bits `odd` set
    afterwards)."""

    def __init__(self, oracle, seed, n, dtype, kd=KD):
        rng = np.random.default_rng(seed)
        self.oracle, self.n, self.dtype, self.kd = oracle, n, dtype, kd
        shape = {"q": (2 * n, KH, kd), "k": (2 * n, KH, kd), "v": (2 * n, VH, VD)}
        self.x = {a: ref.bf16(rng.standard_normal(s)) for a, s in shape.items()}
        self.x["decay"] = (-0.1 * rng.random((2 * n, VH))).astype(F32)
        self.x["beta"] = rng.random((2 * n, VH)).astype(F32)
        self.state = rng.standard_normal((2, VH, kd, VD)).astype(F32)
        self.eps, self.scale = 1e-6, 0.125

    def run(self, q8, ctx):
        n = self.n
        narrow = self.oracle.f32_to_bf16_bits if self.dtype == "bf16" else (lambda a: a)
        d = [ctx.to_device(narrow(self.x[a])) for a in "qkv"]
        d += [ctx.to_device(self.x[a]) for a in ("decay", "beta")]
        shape, kind = (2 * n, VH, VD), np.uint16 if self.dtype == "bf16" else F32
        y, after = ctx.to_device(np.zeros(shape, kind)), ctx.to_device(self.state)
        ctx.delta_rule(*d, y, 2 * n, KH, VH, self.kd, VD, state=ctx.to_device(self.state),
                       new_state=after, row_starts=ctx.to_device(np.asarray([0, n, 2 * n], np.int32)),
                       sequences=2, scale=self.scale, eps=self.eps, dtype=self.dtype)
        got = ctx.to_host(y, shape, kind)
        wide = self.oracle.bf16_bits_to_f32(got) if self.dtype == "bf16" else got
        return wide, ctx.to_host(after, self.state.shape, F32)

    def exact(self, seq, rows, dtype=np.float64):
        """(o, last state) of the sequence's first `rows` rows, and outputs' magnitudes."""
        a = seq * self.n
        x = [self.x[name][a:a + rows] for name in ("q", "k", "v", "decay", "beta")]
        args = (*x, self.state[seq], self.scale, self.eps)
        with np.errstate(all="ignore"):
            o, s, _, _ = ref.rows(*args, dtype)
            return o, s, ref.magnitudes(*args)

    def check(self, y, seq, rows, **at):
        """The sequence's first `rows` rows: half a step of bf16, or (f32, and what
        the sums make of bf16 rows) 2^-13 of the magnitudes."""
        o, _, most = self.exact(seq, rows)
        got = y[seq * self.n:seq * self.n + rows]
        where = np.s_[:, at.get("heads", slice(None)), at.get("columns", slice(None))]
        assert np.isfinite(got[where]).all()
        assert (ref.output_share(got, o, most)[where] <= 1).all()


# chunks from 10 rows per sequence on of bf16, else row after row
CASES = [("bf16", 150), ("bf16", 8), ("f32", 40)]


@pytest.mark.parametrize("dtype,n", CASES)
@pytest.mark.parametrize("rise", [3.0, 100.0])
def test_rows_before_a_growing_decay(q8, ctx, oracle, dtype, n, rise):
    """A log decay of 100 takes the state out of f32 from its row on, and one of 3
    grows it: rows before, other heads and the other sequence hold."""
    c = Call(oracle, 3, n, dtype)
    row = n // 3
    c.x["decay"][row, 1] = rise
    y, s = c.run(q8, ctx)
    heads = np.arange(VH) != 1
    c.check(y, 0, n, heads=heads)
    c.check(y, 0, row if rise > 50 else n)
    c.check(y, 1, n)
    assert np.isfinite(s[0, heads]).all() and np.isfinite(s[1]).all()
    if rise > 50:
        assert not np.isfinite(s[0, 1]).any()


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("rise", [0.125, 0.5, 2.0])
@pytest.mark.parametrize("dtype,n", CASES)
def test_growing_states_that_are_written_over(q8, ctx, oracle, dtype, n, rise, zero):
    """Log decays above 0 in every row, where the one key dim that keys and queries
    have is written over by each row (beta 1): the state is the row's value however
    far the running sum of the decays is, and the output is exact to a few steps of
    f32 times the growth of one row."""
    c = Call(oracle, 4, n, dtype)
    c.eps, c.scale = None, 1.0
    for a in "qk":
        c.x[a][:] = 0
        c.x[a][:, :, 3] = 1
    c.x["decay"][:], c.x["beta"][:] = rise, 1
    c.state[:] = 0 if zero else c.state
    # (dims without a key would grow without bound)
    c.state[:, :, np.arange(KD) != 3] = 0
    y, s = c.run(q8, ctx)
    tol = 8 * 2.0 ** -24 * np.exp(rise) * (np.abs(c.x["v"]).max() + np.abs(c.state).max())
    half = 2.0 ** -8 if dtype == "bf16" else 0
    assert (np.abs(y - c.x["v"]) <= tol + half * np.abs(c.x["v"])).all()
    for i in range(2):
        assert (np.abs(s[i, :, 3] - c.x["v"][(i + 1) * n - 1]) <= tol).all()
        assert (s[i, :, np.arange(KD) != 3] == 0).all()


@pytest.mark.parametrize("dtype,n", CASES)
def test_small_growth_keeps_its_digits(q8, ctx, oracle, dtype, n):
    """Decays on both sides of 0 that add up to a little."""
    c = Call(oracle, 5, n, dtype)
    rng = np.random.default_rng(6)
    c.x["decay"][:] = 0.02 * rng.standard_normal((2 * n, VH))
    y, s = c.run(q8, ctx)
    for i in range(2):
        c.check(y, i, n)
        _, exact, _ = c.exact(i, n)
        _, f32, _ = c.exact(i, n, F32)
        # (an exponential off by a step per row, or twice per chunk of 64)
        chunked = dtype == "bf16" and n > 9
        most = np.exp(np.abs(c.x["decay"][i * n:(i + 1) * n]).sum(0)) * ref.rms(exact)
        assert ref.share(s[i], exact, f32, chunked, most, 6 if chunked else n).max() <= 1


@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("where", ["q", "k", "v", "decay", "beta", "state"])
@pytest.mark.parametrize("dtype,n", CASES)
def test_odd_inputs(q8, ctx, oracle, dtype, n, where, value):
    """One infinity or NaN, of key head 0 (value heads 0 and 1) or value head 1:
    rows before it, the other heads, the other sequence and, of a value or a
    state's element, the other columns keep their values; a query's leaves the rows
    after it and the state alone too."""
    if where == "decay" and value == "-inf":
        pytest.skip("a decay to nothing, not an odd value")
    c = Call(oracle, 7, n, dtype)
    base_y, base_s = c.run(q8, ctx)
    row = {150: 74, 8: 3, 40: 17}[n]
    clean = {a: x.copy() for a, x in c.x.items()}
    states = c.state.copy()
    x = {"nan": np.nan, "inf": np.inf, "-inf": -np.inf}[value]
    heads = [0, 1] if where in "qk" else [1]
    at = {"q": (row, 0, 9), "k": (row, 0, 9), "v": (row, 1, 5), "decay": (row, 1), "beta": (row, 1)}
    if where == "state":
        c.state[0, 1, 20, 5] = x
        row = 0
    else:
        c.x[where][at[where]] = x
    y, s = c.run(q8, ctx)
    c.x, c.state = clean, states
    others = np.array([h not in heads for h in range(VH)])
    assert np.array_equal(y[:, others], base_y[:, others]) and np.array_equal(y[n:], base_y[n:])
    assert np.array_equal(s[0, others], base_s[0, others]) and np.array_equal(s[1], base_s[1])
    c.check(y, 0, row)
    if where in ("v", "state"):
        columns = np.arange(VD) != 5
        assert np.array_equal(y[..., columns], base_y[..., columns])
        assert np.array_equal(s[..., columns], base_s[..., columns])
        assert not np.isfinite(y[row:n, 1, 5]).any() and not np.isfinite(s[0, 1, :, 5]).all()
    elif where == "q":
        assert not np.isfinite(y[row, heads]).any()
        o, exact, most = c.exact(0, n)
        later = ref.output_share(y[row + 1:n], o[row + 1:], most[row + 1:])
        assert (later <= 1).all()
        assert ref.share(s[0], exact, c.exact(0, n, F32)[1], False, ref.rms(c.state[0]) + 1, n).max() <= 1
    else:
        assert not np.isfinite(y[row + 1:n, heads]).any() and not np.isfinite(s[0, heads]).all((1, 2)).any()


@pytest.mark.parametrize("dtype,n", CASES)
@pytest.mark.parametrize("kind", ["beta", "difference", "sum"])
def test_what_leaves_f32_on_the_way(q8, ctx, oracle, dtype, n, kind):
    """Finite inputs whose u is infinite: by beta times a value, by the difference of
    a large value and the state's, by the sum of a key with a state's column.  The
    rows before and the other columns keep their values."""
    c = Call(oracle, 11, n, dtype)
    row = {150: 42, 8: 3, 40: 17}[n]
    if kind == "beta":
        c.x["v"][row, 1, 5], c.x["beta"][row, 1] = 3e38, 2.0
    elif kind == "difference":
        c.x["v"][row, 1, 5], c.x["v"][row + 1, 1, 5] = 3e38, -3e38
        c.x["k"][row + 1] = c.x["k"][row]
        c.x["beta"][row:row + 2, 1], c.x["decay"][row:row + 2, 1] = 1.0, 0.0
    else:
        # keys and queries of one dim each, large states where they are not
        c.eps = None
        for a in "qk":
            c.x[a][:] = 0
            for i in range(2 * n):
                c.x[a][i, :, i % n % 40] = 1
        c.x["k"][row, 0] = 0
        c.x["k"][row, 0, 48:60] = 1
        c.state[0, 1, 48:60, 5], c.x["decay"][:n, 1] = 2e38, 0.0
    c.x["v"] = ref.bf16(c.x["v"])
    y, s = c.run(q8, ctx)
    c.check(y, 0, row)
    c.check(y, 0, n, heads=np.arange(VH) != 1)
    c.check(y, 0, n, columns=np.arange(VD) != 5)
    c.check(y, 1, n)
    assert not np.isfinite(y[n - 1, 1, 5]) or kind == "sum"
    assert not np.isfinite(s[0, 1, :, 5]).all()


@pytest.mark.parametrize("n", [150])
def test_rows_of_an_odd_column(q8, ctx, oracle, n):
    """In a chunk with a NaN among the values, the rows before it in its column come
    from the row-by-row form: next to the chunk form's, within both's roundings."""
    c = Call(oracle, 13, n, "bf16", kd=128)
    base, _ = c.run(q8, ctx)
    c.x["v"][100, 2, 5] = np.nan
    y, _ = c.run(q8, ctx)
    c.x["v"][100, 2, 5] = 0
    c.check(y, 0, 100)
    assert np.isnan(y[100:n, 2, 5]).all()
    _, _, most = c.exact(0, 100)
    step = 2 * 2.0 ** -8 * np.abs(base[:100]) + 2.0 ** -13 * most
    assert (np.abs(y[:100] - base[:100]) <= step).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ns", [[200] + [1] * 30, [1] * 6 + [300], [1, 0, 90, 1, 1, 64]])
def test_a_prompt_among_single_rows(q8, ctx, oracle, ns, dtype):
    """One call of a prompt and sequences of one row, in either form."""
    from test_gpu_delta_rule import Case
    c = Case(oracle, np.random.default_rng(17), ns, 1, 2, KD, VD, dtype, pad=2).upload(ctx)
    c.call(ctx, 0.125, 1e-6)
    c.check(ctx, 0.125, 1e-6, *c.results(ctx))
