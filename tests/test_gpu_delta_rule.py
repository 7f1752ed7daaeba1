"""llmcp_q8_delta_rule against its definition in float64, row after row.

The bound: with every |k| <= 1 after the norm (or near it without) and a, beta in
[0, 1], a row's update contracts, so an error made in one row does not grow.  The
errors of n rows of sums over key_dim products in f32 add up to about n *
(key_dim + 16) * 2^-24 of the largest state or value met, at worst all with one
sign; the output's rounding to its type comes on top."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32 = np.float32
U32, U16 = 2.0 ** -24, 2.0 ** -8  # half a step of f32, of bf16


def reference(q, k, v, decay, beta, state, scale, eps):
    """o [rows, heads, value dim], the last state and, per head, the largest
    magnitude that the sums meet."""
    q, k, v, decay, beta, s = (x.astype(np.float64) for x in (q, k, v, decay, beta, state))
    if eps is not None:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + eps) for x in (q, k))
    per = v.shape[1] // q.shape[1]
    q, k = np.repeat(q * scale, per, 1), np.repeat(k, per, 1)
    o, most = np.zeros(v.shape), np.abs(s).max((1, 2), initial=0)
    for t in range(v.shape[0]):
        s = s * np.exp(decay[t])[:, None, None]
        u = beta[t][:, None] * (v[t] - np.einsum("hkv,hk->hv", s, k[t]))
        s = s + k[t][:, :, None] * u[:, None, :]
        o[t] = np.einsum("hkv,hk->hv", s, q[t])
        most = np.maximum(most, np.maximum(np.abs(s).sum(1).max(1), np.abs(v[t]).max(1)))
    return o, s, most


class Case:
    def __init__(self, oracle, rng, ns, kh, vh, kd, vd, dtype, pad=0, fresh=False, first=0,
                 strength=1.0):
        self.oracle, self.ns, self.kh, self.vh, self.kd, self.vd = oracle, ns, kh, vh, kd, vd
        self.dtype = dtype
        self.starts = first + np.concatenate([[0], np.cumsum(ns)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + pad
        wide = 2 * kh * kd + vh * vd
        x = rng.standard_normal((self.rows, wide)).astype(F32)
        self.bits = oracle.f32_to_bf16_bits(x) if dtype == "bf16" else x
        self.x = oracle.bf16_bits_to_f32(self.bits) if dtype == "bf16" else x
        self.decay = (-strength * rng.random((self.rows, vh)) ** 3).astype(F32)
        self.beta = rng.random((self.rows, vh)).astype(F32)
        self.state = (None if fresh else
                      rng.standard_normal((len(ns), vh, kd, vd)).astype(F32))

    def parts(self):
        a, b = self.kh * self.kd, 2 * self.kh * self.kd
        return (self.x[:, :a].reshape(-1, self.kh, self.kd), self.x[:, a:b].reshape(-1, self.kh, self.kd),
                self.x[:, b:].reshape(-1, self.vh, self.vd))

    def upload(self, ctx):
        self.d = ctx.to_device(self.bits)
        e, wide = self.bits.itemsize, self.bits.shape[1]
        self.q, self.k = self.d.ptr, self.d.ptr + self.kh * self.kd * e
        self.v = self.k + self.kh * self.kd * e
        self.dd, self.db = ctx.to_device(self.decay), ctx.to_device(self.beta)
        self.ds = None if self.state is None else ctx.to_device(self.state)
        self.dst = ctx.to_device(self.starts)
        self.shape = (len(self.ns), self.vh, self.kd, self.vd)
        self.after = ctx.to_device(np.full(self.shape, np.nan, F32))
        self.y = ctx.to_device(np.full((self.rows, self.vh, self.vd), 7, self.bits.dtype))
        self.strides = (wide, wide, wide)
        return self

    def call(self, ctx, scale, eps, state="own", new_state=None):
        ctx.delta_rule(self.q, self.k, self.v, self.dd, self.db, self.y, self.rows, self.kh, self.vh,
                       self.kd, self.vd, state=self.ds if state == "own" else state,
                       new_state=new_state or self.after, row_starts=self.dst,
                       sequences=len(self.ns), scale=scale, eps=eps, strides=self.strides,
                       dtype=self.dtype)

    def results(self, ctx, new_state=None):
        y = ctx.to_host(self.y, (self.rows, self.vh, self.vd), self.bits.dtype)
        s = ctx.to_host(new_state or self.after, self.shape, F32)
        return y, s

    def check(self, ctx, scale, eps, y, s):
        assert (y[:self.starts[0]] == 7).all() and (y[self.starts[-1]:] == 7).all()
        wide = self.oracle.bf16_bits_to_f32(y) if self.dtype == "bf16" else y
        for i, n in enumerate(self.ns):
            a, b = self.starts[i], self.starts[i + 1]
            start = (np.zeros(self.shape[1:], F32) if self.state is None else self.state[i])
            q, k, v = self.parts()
            o, last, most = reference(q[a:b], k[a:b], v[a:b], self.decay[a:b], self.beta[a:b], start,
                                      scale, eps)
            if n == 0:
                assert np.array_equal(s[i], start)
                continue
            tol = (n + 1) * (self.kd + 16) * U32 * most
            err = np.abs(s[i] - last)
            assert (err <= tol[:, None, None]).all(), float((err / tol[:, None, None]).max())
            reach = np.abs(scale) * (1 if eps is not None else np.abs(q[a:b]).sum(-1).max())
            bound = (tol * reach)[None, :, None] + (U16 if self.dtype == "bf16" else 2 * U32) * np.abs(o)
            err = np.abs(wide[a:b] - o)
            assert (err <= bound + 1e-37).all(), float((err / (bound + 1e-37)).max())


# (rows, key heads, value heads, key dim, value dim): single rows; sequences
# without rows, of one, of odd lengths around whole chunks; dims of both kinds;
# more sequences than a wave looks at together
SHAPES = [
    ([1], 16, 32, 128, 128), ([1] * 5, 2, 6, 64, 48), ([3, 0, 2], 1, 2, 128, 16),
    ([31, 33, 0, 1, 32], 2, 2, 64, 64), ([63, 65, 64], 2, 4, 128, 128), ([17], 3, 3, 64, 160),
    ([200], 1, 3, 128, 64), ([129, 5], 4, 4, 64, 32), ([2] * 70 + [66], 1, 1, 64, 16),
    ([511], 1, 2, 128, 32), ([96, 0, 130, 7], 1, 2, 128, 112)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("eps", [1e-6, None])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_delta_rule(q8, ctx, oracle, shape, eps, dtype):
    ns, kh, vh, kd, vd = SHAPES[shape]
    rng = np.random.default_rng(shape)
    c = Case(oracle, rng, ns, kh, vh, kd, vd, dtype, pad=shape % 3, fresh=shape % 2 == 1,
             first=shape % 4)
    if eps is None:  # rows near length 1 by themselves
        a = 2 * kh * kd
        c.x[:, :a] *= F32(kd ** -0.5)
        c.bits = oracle.f32_to_bf16_bits(c.x) if dtype == "bf16" else c.x
        c.x = oracle.bf16_bits_to_f32(c.bits) if dtype == "bf16" else c.x
        length = np.sqrt((c.x[:, :a].reshape(-1, 2 * kh, kd) ** 2).sum(-1))
        c.beta /= F32(max(1.0, float(length.max()) ** 2))  # (beta |k|^2 <= 1: rows contract)
    c.upload(ctx).call(ctx, kd ** -0.5, eps)
    c.check(ctx, kd ** -0.5, eps, *c.results(ctx))


@pytest.mark.parametrize("n", [1, 40, 150])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_state_in_place(q8, ctx, oracle, n, dtype):
    rng = np.random.default_rng(n)
    c = Case(oracle, rng, [n, 0, 2], 2, 4, 128, 64, dtype).upload(ctx)
    c.call(ctx, 0.1, 1e-6, new_state=c.ds)
    inplace = c.results(ctx, c.ds)
    c.check(ctx, 0.1, 1e-6, *inplace)
    c.upload(ctx).call(ctx, 0.1, 1e-6)
    apart = c.results(ctx)
    assert np.array_equal(inplace[0], apart[0]) and np.array_equal(inplace[1], apart[1])


@pytest.mark.parametrize("n", [5, 140])
def test_one_sequence_without_starts(q8, ctx, oracle, n):
    rng = np.random.default_rng(1)
    c = Case(oracle, rng, [n], 2, 2, 64, 64, "bf16").upload(ctx)
    c.dst = None
    c.call(ctx, 0.3, 1e-6)
    c.check(ctx, 0.3, 1e-6, *c.results(ctx))


def test_no_rows(q8, ctx, oracle):
    """A call without rows hands the states on."""
    rng = np.random.default_rng(2)
    c = Case(oracle, rng, [0, 0], 1, 2, 64, 32, "bf16", pad=1).upload(ctx)
    c.rows = 0
    c.call(ctx, 0.3, 1e-6)
    assert np.array_equal(ctx.to_host(c.after, c.shape, F32), c.state)
    c.call(ctx, 0.3, 1e-6, state=None)
    assert (ctx.to_host(c.after, c.shape, F32) == 0).all()


@pytest.mark.parametrize("lowest", [-np.inf, np.finfo(F32).min, -200.0])
@pytest.mark.parametrize("n", [9, 130])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decays_to_nothing(q8, ctx, oracle, n, lowest, dtype):
    """A decay of the lowest value forgets the state before it and nothing
    else."""
    rng = np.random.default_rng(n)
    c = Case(oracle, rng, [n], 1, 2, 128, 32, dtype)
    c.decay[n // 2], c.decay[n // 2 + 3, 1] = lowest, lowest
    c.decay[n // 3, 0] = lowest
    c.upload(ctx).call(ctx, 0.1, 1e-6)
    c.check(ctx, 0.1, 1e-6, *c.results(ctx))


@pytest.mark.parametrize("strength", [0.0, 3.0, 40.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strong_and_no_decay(q8, ctx, oracle, strength, dtype):
    rng = np.random.default_rng(4)
    c = Case(oracle, rng, [200], 2, 4, 64, 32, dtype, strength=strength)
    c.upload(ctx).call(ctx, 0.125, 1e-6)
    c.check(ctx, 0.125, 1e-6, *c.results(ctx))


@pytest.mark.parametrize("n", [6, 150])
def test_odd_values_stay_in_their_head_and_sequence(q8, ctx, oracle, n):
    """A NaN in one head's value reaches the rows from its own on in its column
    alone; other heads and sequences are untouched, rows of another sequence in the
    same call among them."""
    rng = np.random.default_rng(6)
    c = Case(oracle, rng, [n, n], 2, 2, 64, 32, "bf16")
    a = 2 * 2 * 64
    row = n // 2
    c.upload(ctx).call(ctx, 0.125, 1e-6)
    clean = c.results(ctx)
    c.bits[row, a + 5] = 0x7FC0  # value 5 of head 0
    c.upload(ctx).call(ctx, 0.125, 1e-6)
    y, s = c.results(ctx)
    nan = (y & 0x7FFF) > 0x7F80
    assert nan[row:n, 0, 5].all()
    assert not nan[n:].any() and not nan[:n, 1].any() and not nan[:row].any()
    others = np.ones(32, bool)
    others[5] = False
    assert np.array_equal(y[:, :, others], clean[0][:, :, others])
    assert np.array_equal(s[1], clean[1][1]) and np.array_equal(s[0, 1], clean[1][0, 1])


def test_bounds_are_cut(q8, ctx, oracle):
    rng = np.random.default_rng(12)
    c = Case(oracle, rng, [10, 90], 1, 2, 64, 32, "bf16").upload(ctx)
    c.dst = ctx.to_device(np.asarray([-5, 10, 2 ** 31 - 1], np.int32))
    c.call(ctx, 0.125, 1e-6)
    c.check(ctx, 0.125, 1e-6, *c.results(ctx))


@pytest.mark.parametrize("n", [1, 7, 100])
def test_replayed(q8, ctx, oracle, n):
    """A captured step on a state in place, replayed with eager work between."""
    rng = np.random.default_rng(n)
    c = Case(oracle, rng, [n], 2, 4, 128, 128, "bf16").upload(ctx)
    start = c.state.copy()
    c.call(ctx, 0.1, 1e-6, new_state=c.ds)
    ctx.graph_begin()
    c.call(ctx, 0.1, 1e-6, new_state=c.ds)
    graph = ctx.graph_end()
    other = Case(oracle, rng, [n], 2, 4, 128, 128, "bf16").upload(ctx)
    other.call(ctx, 0.1, 1e-6)
    other.check(ctx, 0.1, 1e-6, *other.results(ctx))
    for _ in range(3):
        start = ctx.to_host(c.ds, c.shape, F32)
        ctx.graph_launch(graph)
        y, s = c.results(ctx, c.ds)
        c.state = start
        c.check(ctx, 0.1, 1e-6, y, s)
        other.call(ctx, 0.1, 1e-6)
    ctx.graph_destroy(graph)


@pytest.mark.parametrize("inplace", [False, True])
def test_more_chunks_than_the_workspace_holds(q8, ctx, oracle, inplace):
    """1024 heads leave room for 8 chunks at a time: sequences that end, begin and
    go on in a later window, and one without rows."""
    if ctx.platform != "aarch64":
        pytest.skip("the same kernels on either platform")
    rng = np.random.default_rng(31)
    c = Case(oracle, rng, [530, 0, 40, 200], 1, 1024, 64, 16, "bf16").upload(ctx)
    if inplace:
        c.call(ctx, 0.125, 1e-6, new_state=c.ds)
        c.check(ctx, 0.125, 1e-6, *c.results(ctx, c.ds))
    else:
        c.call(ctx, 0.125, 1e-6)
        c.check(ctx, 0.125, 1e-6, *c.results(ctx))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_descending_starts_stay_in_bounds(q8, ctx, oracle, dtype):
    """Bounds that descend give every other sequence all rows: nothing behind
    the states and the output is touched."""
    rng = np.random.default_rng(37)
    c = Case(oracle, rng, [40] * 30, 1, 1, 64, 16, dtype)
    c.rows, c.starts = 40, np.asarray([0, 40] * 15 + [0], np.int32)
    c.upload(ctx)
    guard = ctx.to_device(np.full((31,) + c.shape[1:], 5, F32))
    y = ctx.to_device(np.full((44, 1, 16), 7, c.bits.dtype))
    c.y = y
    c.call(ctx, 0.125, 1e-6, new_state=guard)
    assert (ctx.to_host(guard, (31,) + c.shape[1:], F32)[30] == 5).all()
    assert (ctx.to_host(y, (44, 1, 16), c.bits.dtype)[40:] == 7).all()
