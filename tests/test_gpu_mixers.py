"""The token mixers as a model uses them: between the norm's linears and the
output projection, a prompt first and then single tokens by a replayed graph,
with the state they carry; on other streams and in two contexts at once.  Each
mixer is checked against its definition on the rows that the linears in front of
it left, and what follows it against the same calls apart."""
import numpy as np
import pytest

from kv_reference import F32, Cache, same
from test_gpu_attention import reference as attention_reference
from test_gpu_attention import filled
from test_gpu_delta_rule import Case as DeltaCase
from test_gpu_delta_rule import reference as delta_reference

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8  # half a step of f32, of bf16
H, PROMPT, STEPS = 256, 70, 3


def weight(ctx, oracle, rng, n, k):
    return ctx.upload_p4(oracle.pack_q8_0_p4((rng.standard_normal((n, k)) * 0.05).astype(F32)), n, k)


class Layer:
    """Buffers of up to PROMPT rows and the weights of one mixer layer."""

    def __init__(self, ctx, oracle, rng, widths, out):
        self.ctx, self.oracle = ctx, oracle
        self.norm = ctx.to_device(oracle.f32_to_bf16_bits((rng.standard_normal(H) * 0.1 + 1).astype(F32)))
        self.w = [weight(ctx, oracle, rng, n, H) for n in widths]
        self.wo = weight(ctx, oracle, rng, H, out)
        self.x = ctx.alloc(PROMPT * H * 2)
        self.normed, self.y = ctx.alloc(PROMPT * H * 2), ctx.alloc(PROMPT * H * 2)
        self.parts = [ctx.alloc(PROMPT * n * 2) for n in widths]
        self.widths, self.out = widths, out

    def put(self, q8, bits):
        q8.check(q8.lib().llmcp_q8_memcpy_h2d(self.ctx.handle, self.x.ptr, bits.ctypes.data, bits.nbytes))

    def front(self, m):
        self.ctx.rmsnorm_linear_group(self.x, self.norm, self.normed, self.w, self.parts, m, dtype="bf16")

    def back(self, mixed, m):
        self.ctx.linear_add(mixed, self.wo, self.x, self.y, m, mode="decode" if m == 1 else "prefill",
                            dtype="bf16")

    def rows(self, buf, m, n):
        return self.oracle.bf16_bits_to_f32(self.ctx.to_host(buf, (m, n), np.uint16))

    def check_back(self, mixed, m):
        """The layer's output is what the same call gives on the mixer's rows."""
        got = self.ctx.to_host(self.y, (m, H), np.uint16)
        again = self.ctx.to_device(np.zeros((m, H), np.uint16))
        copy = self.ctx.to_device(self.ctx.to_host(mixed, (m, self.out), np.uint16))
        self.ctx.linear_add(copy, self.wo, self.x, again, m, mode="decode" if m == 1 else "prefill",
                            dtype="bf16")
        assert same(got, self.ctx.to_host(again, (m, H), np.uint16))

    def release(self):
        for w in self.w + [self.wo]:
            self.ctx.release(w)


def inputs(oracle, rng, m):
    return oracle.f32_to_bf16_bits(rng.standard_normal((m, H)).astype(F32))


@pytest.mark.parametrize("fmt", ["bf16", "q8"])
def test_attention_layer(q8, ctx, oracle, fmt):
    rng = np.random.default_rng(41)
    heads, kvh, dim = 4, 2, 64
    layer = Layer(ctx, oracle, rng, [heads * dim, kvh * dim, kvh * dim], heads * dim)
    c = Cache(q8, ctx, rng, [PROMPT + STEPS], 32, kvh, dim, fmt)
    mixed = ctx.alloc(PROMPT * heads * dim * 2)
    cache = c.cache()

    def check(m, length):
        q, k, v = (layer.rows(b, m, n) for b, n in zip(layer.parts, layer.widths))
        c.put(oracle, 0, length - m, k.reshape(m, kvh, dim), v.reshape(m, kvh, dim))
        want, bound = attention_reference(q.reshape(m, heads, dim), *c.values(oracle, 0, 0, length),
                                          dim ** -0.5, length - m, True)
        got = layer.rows(mixed, m, heads * dim).reshape(m, heads, dim)
        assert (np.abs(got - want) <= bound).all()
        layer.check_back(mixed, m)

    def calls(m, batch):
        layer.front(m)
        ctx.kv_write(layer.parts[1], layer.parts[2], cache, batch, m, dtype="bf16")
        ctx.attention(layer.parts[0], cache, batch, mixed, m, heads, dtype="bf16")
        layer.back(mixed, m)

    try:
        layer.put(q8, inputs(oracle, rng, PROMPT))
        calls(PROMPT, c.batch([0, PROMPT], [PROMPT]))
        check(PROMPT, PROMPT)
        batch = c.batch([0, 1], [PROMPT + 1])
        lengths = c.keep[1]
        layer.put(q8, inputs(oracle, rng, 1))
        calls(1, batch)
        ctx.graph_begin()
        calls(1, batch)
        graph = ctx.graph_end()
        for step in range(STEPS):
            layer.put(q8, inputs(oracle, rng, 1))
            host = np.asarray([PROMPT + 1 + step], np.int32)
            q8.check(q8.lib().llmcp_q8_memcpy_h2d(ctx.handle, lengths.ptr, host.ctypes.data, 4))
            ctx.graph_launch(graph)
            check(1, PROMPT + 1 + step)
        ctx.graph_destroy(graph)
        assert ctx.check_flag() == 0
    finally:
        layer.release()


def test_delta_layer(q8, ctx, oracle):
    """The linear-attention layer with its gated norm; log decay and beta come
    from the host here."""
    rng = np.random.default_rng(43)
    kh, vh, kd, vd = 1, 2, 64, 64
    wide = 2 * kh * kd + vh * vd
    layer = Layer(ctx, oracle, rng, [wide, vh * vd], vh * vd)
    gate_w = ctx.to_device((rng.standard_normal(vd) * 0.1 + 1).astype(F32))
    state = np.zeros((1, vh, kd, vd), F32)
    ds = ctx.to_device(state)
    mixed, gated = ctx.alloc(PROMPT * vh * vd * 2), ctx.alloc(PROMPT * vh * vd * 2)
    dd, db = ctx.alloc(PROMPT * vh * 4), ctx.alloc(PROMPT * vh * 4)

    def gates(m):
        g, b = -(rng.random((m, vh)) ** 2).astype(F32), rng.random((m, vh)).astype(F32)
        for buf, x in ((dd, g), (db, b)):
            q8.check(q8.lib().llmcp_q8_memcpy_h2d(ctx.handle, buf.ptr, x.ctypes.data, x.nbytes))
        return g, b

    def calls(m):
        layer.front(m)
        p = layer.parts[0].ptr
        ctx.delta_rule(p, p + kh * kd * 2, p + 2 * kh * kd * 2, dd, db, mixed, m, kh, vh, kd, vd,
                       state=ds, new_state=ds, strides=(wide, wide, wide), dtype="bf16")
        ctx.gated_rmsnorm(mixed, layer.parts[1], gate_w, gated, m, vh * vd, vd, dtype="bf16")
        layer.back(gated, m)

    def check(m, g, b, before):
        x = layer.rows(layer.parts[0], m, wide)
        a = kh * kd
        o, last, most = delta_reference(x[:, :a].reshape(m, kh, kd), x[:, a:2 * a].reshape(m, kh, kd),
                                        x[:, 2 * a:].reshape(m, vh, vd), g, b, before[0], kd ** -0.5, 1e-6)
        tol = (m + 1) * (kd + 16) * U32 * most
        after = ctx.to_host(ds, state.shape, F32)
        assert (np.abs(after[0] - last) <= tol[:, None, None]).all()
        got = layer.rows(mixed, m, vh * vd).reshape(m, vh, vd)
        assert (np.abs(got - o) <= (tol * kd ** -0.5)[None, :, None] + U16 * np.abs(o) + 1e-37).all()
        layer.check_back(gated, m)
        return after

    try:
        layer.put(q8, inputs(oracle, rng, PROMPT))
        g, b = gates(PROMPT)
        calls(PROMPT)
        before = check(PROMPT, g, b, state)
        layer.put(q8, inputs(oracle, rng, 1))
        g, b = gates(1)
        calls(1)
        before = check(1, g, b, before)
        ctx.graph_begin()
        calls(1)
        graph = ctx.graph_end()
        for _ in range(STEPS):
            layer.put(q8, inputs(oracle, rng, 1))
            g, b = gates(1)
            ctx.graph_launch(graph)
            before = check(1, g, b, before)
        ctx.graph_destroy(graph)
    finally:
        layer.release()


def test_other_streams(q8, ctx, oracle):
    """Calls on a stream of the caller's, whose workspaces the calls before it on
    the context's own stream still use."""
    rng = np.random.default_rng(47)
    n, heads, kvh, dim = 3, 8, 2, 128
    c = filled(q8, ctx, oracle, rng, [900], 32, kvh, dim, "q8")
    bits = oracle.f32_to_bf16_bits(rng.standard_normal((n, heads, dim)).astype(F32))
    q, cache, batch = ctx.to_device(bits), c.cache(), c.batch([0, n])
    ys = [ctx.to_device(np.zeros((n, heads, dim), np.uint16)) for _ in range(4)]
    other = q8.Context(0)
    stream = q8.lib().llmcp_q8_ctx_stream(other.handle)
    try:
        for i, y in enumerate(ys):
            q8.check(q8.lib().llmcp_q8_ctx_set_stream(ctx.handle, stream if i % 2 else None))
            ctx.attention(q, cache, batch, y, n, heads, dtype="bf16")
        ctx.sync()
    finally:
        q8.check(q8.lib().llmcp_q8_ctx_set_stream(ctx.handle, None))
        ctx.sync()
        other.close()
    out = [ctx.to_host(y, (n, heads, dim), np.uint16) for y in ys]
    assert all(same(o, out[0]) for o in out)


def test_two_contexts_at_once(q8, ctx, oracle):
    """Each context has its own workspaces: calls of two in flight together give
    what they give alone."""
    rng = np.random.default_rng(53)
    with q8.Context(0) as other:
        runs = []
        for at in (ctx, other):
            c = DeltaCase(oracle, rng, [200, 90], 2, 4, 64, 64, "bf16").upload(at)
            a = filled(q8, at, oracle, rng, [1500], 64, 2, 64, "bf16")
            bits = oracle.f32_to_bf16_bits(rng.standard_normal((2, 8, 64)).astype(F32))
            y = at.to_device(np.zeros((2, 8, 64), np.uint16))
            runs.append((at, c, at.to_device(bits), a.cache(), a.batch([0, 2]), y, a))
        alone = []
        for together in (False, True):
            for at, c, q, cache, batch, y, _ in runs:
                c.call(at, 0.125, 1e-6)
                at.attention(q, cache, batch, y, 2, 8, dtype="bf16")
                if not together:
                    at.sync()
            for i, (at, c, q, cache, batch, y, _) in enumerate(runs):
                got = c.results(at) + (at.to_host(y, (2, 8, 64), np.uint16),)
                if not together:
                    alone.append(got)
                else:
                    assert all(same(a, b) for a, b in zip(got, alone[i]))


def test_refusals(q8, ctx, oracle):
    """What only a context can refuse: shapes that do not meet, outputs over
    inputs; nothing is launched."""
    rng = np.random.default_rng(59)
    c = Cache(q8, ctx, rng, [20], 16, 2, 64, "bf16")
    cache, batch = c.cache(), c.batch([0, 4])
    x, y = ctx.alloc(1 << 16), ctx.alloc(1 << 16)

    def refused(code, f, *args, **kw):
        with pytest.raises(q8.Q8Error) as e:
            f(*args, **kw)
        assert e.value.code == code
    refused(q8.DECLINED, ctx.attention, x, cache, batch, y, 4, 3, dtype="bf16")  # 3 heads over 2
    refused(q8.EINVAL, ctx.attention, x, cache, batch, x, 4, 4, dtype="bf16")
    refused(q8.EINVAL, ctx.kv_read, cache, batch, x, x, 4, dtype="bf16")
    for scale in (np.nan, np.inf, -np.inf):
        refused(q8.EINVAL, ctx.attention, x, cache, batch, y, 4, 4, scale=scale, dtype="bf16")
    refused(q8.DECLINED, ctx.attention, x.ptr + 2, cache, batch, y, 4, 4, dtype="bf16")
    wrong = Cache(q8, ctx, rng, [20], 16, 2, 128, "bf16").cache()
    wrong.head_dim = 96
    refused(q8.DECLINED, ctx.kv_write, x, y, wrong, batch, 4, dtype="bf16")
    g, s = ctx.alloc(4096), ctx.alloc(1 << 20)
    args = (x, y, x, g, g)
    for kw, code in (({"key_dim": 32}, q8.DECLINED), ({"value_dim": 24}, q8.DECLINED),
                     ({"value_heads": 3}, q8.DECLINED), ({"sequences": 2}, q8.DECLINED),
                     ({"new_state": None}, q8.EINVAL), ({"value_dim": 2048}, q8.DECLINED),
                     ({"new_state": s.ptr + 4}, q8.DECLINED),
                     ({"strides": (1 << 22, None, None)}, q8.DECLINED)):
        full = {"rows": 4, "key_heads": 2, "value_heads": 2, "key_dim": 64, "value_dim": 32,
                "new_state": s, "dtype": "bf16"}
        full.update(kw)
        refused(code, ctx.delta_rule, *args, ctx.alloc(1 << 16), **full)
    refused(q8.EINVAL, ctx.delta_rule, x, y, x, g, g, x, 4, 2, 2, 64, 32, new_state=s, dtype="bf16")


@pytest.mark.parametrize("n", [150, 1])
@pytest.mark.parametrize("fmt", ["bf16", "q8"])
def test_caches_above_4_gib(q8, ctx, oracle, fmt, n):
    """Pages whose bytes lie past 32 bits: written, read back and attended."""
    if ctx.platform != "aarch64":
        pytest.skip("the same kernels on either platform")
    rng = np.random.default_rng(61)
    kvh, dim, page, length = 4, 256, 64, 200
    pages = 40000 if fmt == "bf16" else 80000  # 5.2 GB of keys, as much of values
    each = pages * kvh * page * dim * (2 if fmt == "bf16" else 1)
    assert each > 1 << 32
    bufs = [ctx.alloc(each) for _ in range(2)]
    scales = [ctx.alloc(pages * kvh * page * 4) for _ in range(2)] if fmt == "q8" else [None, None]
    cache = q8.KVCache(*bufs, pages, page, kvh, dim, key_scales=scales[0], value_scales=scales[1])
    table = np.asarray([[pages - 1, 0, pages - 3, pages // 2 + 9000]], np.int32)
    keep = [ctx.to_device(np.asarray(a, np.int32)) for a in ([0, length], [length], table, [0, n])]
    fill = q8.KVBatch(keep[0], keep[1], keep[2], 1, 4)
    kb, vb, qb = (oracle.f32_to_bf16_bits(rng.standard_normal(shape).astype(F32))
                  for shape in ((length, kvh, dim), (length, kvh, dim), (n, 16, dim)))
    ctx.kv_write(ctx.to_device(kb), ctx.to_device(vb), cache, fill, length, dtype="bf16")
    out = [ctx.to_device(np.zeros(kb.shape, F32)) for _ in range(2)]
    ctx.kv_read(cache, fill, out[0], out[1], length)
    k, v = (ctx.to_host(o, kb.shape, F32) for o in out)
    for got, bits in ((k, kb), (v, vb)):
        want = oracle.bf16_bits_to_f32(bits)
        step = 0 if fmt == "bf16" else np.abs(want).max(-1, keepdims=True) / 127 * (0.5 + 2.0 ** -10)
        assert (np.abs(got - want) <= step).all()
    y = ctx.to_device(np.zeros(qb.shape, np.uint16))
    ctx.attention(ctx.to_device(qb), cache, q8.KVBatch(keep[3], keep[1], keep[2], 1, 4), y, n, 16,
                  dtype="bf16")
    want, bound = attention_reference(oracle.bf16_bits_to_f32(qb), k, v, dim ** -0.5, length - n, True)
    got = oracle.bf16_bits_to_f32(ctx.to_host(y, qb.shape, np.uint16))
    assert (np.abs(got - want) <= bound).all()
    for b in bufs + [s for s in scales if s]:
        b.free()
