"""The rows' scales in the expert products: d = RN(max|x| / 127), a division
(Q8Decode.cpp:83-120), and no multiplication by the rounded 1/127, which gives
another f32 for one block in twenty-four.  Every block here is one of those, and
holds a value that the two scales put on different steps."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of f32


def steps_of(v, d):
    inv = np.float32(1.0) / d
    return np.rint(v * inv)


def rows_at_borders(rng, m, k):
    """f32 rows [m, k], their (steps, scales) by division, and by multiplication."""
    n = m * k // 32
    c = np.float32(1.0) / np.float32(127.0)
    top, border = np.zeros(0, np.float32), np.zeros(0, np.float32)
    while top.size < n:
        a = rng.uniform(1.0, 4.0, 20000).astype(np.float32)
        d, p = a / np.float32(127.0), a * c
        s = rng.integers(1, 126, a.size).astype(np.float32)
        v = (s + np.float32(0.5)) * d
        for _ in range(4):  # the floats around the border between two steps
            hit = (d != p) & (steps_of(v, d) != steps_of(v, p))
            top, border = np.concatenate([top, a[hit]]), np.concatenate([border, v[hit]])
            v = np.nextafter(v, np.float32(0.0))
    top, border = top[:n], border[:n]
    x = (rng.uniform(-0.99, 0.99, (n, 32)).astype(np.float32) * top[:, None]).astype(np.float32)
    x[:, 3], x[:, 17] = top, -border
    d, p = top / np.float32(127.0), top * c
    by = [(steps_of(x, s[:, None]).astype(np.float64), s.astype(np.float64)) for s in (d, p)]
    return x.reshape(m, k), by


# (tokens, top_k, experts): rows quantized by the workgroups that read them, by
# a launch in front, beside the plan (tiles of 32 and of 64 slots)
@pytest.mark.parametrize("m,top_k,e", [(3, 1, 16), (12, 2, 8), (160, 4, 32), (120, 2, 3)])
def test_expert_linear_scales_by_division(ctx, oracle, m, top_k, e):
    """Against 64 bits: a rounding of each scale product and one (fma) or two per
    step of the chain of B blocks, each at most U32 of the sum of magnitudes."""
    rng = np.random.default_rng(m * 7 + e)
    n, k = 40, 768
    x, ((q, d), (q2, p)) = rows_at_borders(rng, m, k)
    qa, sa = oracle.quantize_act_q8_1(x)
    assert np.array_equal(qa.reshape(q.shape), q) and np.array_equal(sa.ravel(), d)
    assert (q != q2).any(1).all() and (d != p).all()
    p4 = [oracle.pack_q8_0_p4((rng.standard_normal((n, k)) * 0.02).astype(np.float32)) for _ in range(e)]
    t = ctx.upload_experts_p4(np.concatenate(p4), e, n, k)
    try:
        ids = rng.integers(0, e, (m, top_k)).astype(np.int32)
        yd = ctx.alloc(m * top_k * n * 4)
        ctx.expert_linear(ctx.to_device(x), ctx.to_device(ids), m, top_k, t, yd)
        got = ctx.to_host(yd, (m * top_k, n), np.float32).astype(np.float64)
        far = 0
        for s, i in enumerate(ids.ravel()):
            qs, dw = oracle.unpack_q8_0_p4(p4[i], n, k)
            w = qs.reshape(n, -1, 32) * oracle.f16_bits_to_f32(dw).astype(np.float64)[:, :, None]
            at = slice(s // top_k * (k // 32), (s // top_k + 1) * (k // 32))
            dots, other = (np.einsum("bi,nbi->nb", a[at] * b[at, None], w) for a, b in ((q, d), (q2, p)))
            bound = (k // 32 + 3) * U32 * np.abs(dots).sum(1)
            assert (np.abs(got[s] - dots.sum(1)) <= bound).all()
            far += (np.abs(other.sum(1) - dots.sum(1)) > bound).sum()
        assert far > got.size // 2  # the other scales would not have passed
    finally:
        ctx.release(t)


@pytest.mark.parametrize("m", [1, 2, 20, 200])
def test_expert_mlp_scales_by_division(ctx, q8, oracle, m):
    """f32 rows and the same rows quantized here: the same bits."""
    rng = np.random.default_rng(m)
    top_k, e, h, f = 4, 24, 256, 64
    x, ((q, d), _) = rows_at_borders(rng, m, h)
    stacks = []
    try:
        for n, k in ((f, h), (f, h), (h, f)):
            w = [oracle.pack_q8_0_p4((rng.standard_normal((n, k)) * 0.1).astype(np.float32)) for _ in range(e)]
            stacks.append(ctx.upload_experts_p4(np.concatenate(w), e, n, k))
        ids = ctx.to_device(rng.integers(-1, e, (m, top_k)).astype(np.int32))
        rows = q8.Q8Rows(ctx.to_device(q.astype(np.int8).reshape(m, h)),
                         ctx.to_device(d.astype(np.float32).reshape(m, h // 32)), m, h)
        ys = []
        for src in (ctx.to_device(x), rows):
            yd = ctx.alloc(m * h * 4)
            ctx.expert_mlp(src, ids, None, m, top_k, *stacks, yd)
            ys.append(ctx.to_host(yd, (m, h), np.uint32))
        assert np.array_equal(*ys) and ys[0].any()
    finally:
        for t in stacks:
            ctx.release(t)
