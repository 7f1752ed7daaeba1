"""The gated delta rule in numpy, for bounds on the kernels' errors: the
definition in float64 with the magnitudes that an output is summed from, the
same steps row after row in float32, and the chunks' formulas in float32, as the
kernel has them or with a mistake planted."""
import numpy as np

F32 = np.float32
CHUNK = 64


def by_head(q, k, per):
    return np.repeat(q, per, 1), np.repeat(k, per, 1)


def rows(q, k, v, decay, beta, state, scale, eps, dtype):
    """(o [n, heads, value dim], the last state, U, the state before every row) row
    after row in dtype; q and k [n, key heads, key dim]."""
    q, k, v, decay, beta, s = (np.asarray(x, dtype) for x in (q, k, v, decay, beta, state))
    scale = dtype(scale)
    if eps is not None:
        q, k = (x * (dtype(1) / np.sqrt((x * x).sum(-1, keepdims=True) + dtype(eps))) for x in (q, k))
    q, k = by_head(q * scale, k, v.shape[1] // q.shape[1])
    o, us, before = np.zeros(v.shape, dtype), np.zeros(v.shape, dtype), []
    for t in range(v.shape[0]):
        before.append(s)
        s = s * np.exp(decay[t].astype(np.float64)).astype(dtype)[:, None, None]
        u = beta[t][:, None] * (v[t] - np.matmul(k[t][:, None, :], s)[:, 0])
        s = s + k[t][:, :, None] * u[:, None, :]
        o[t], us[t] = np.matmul(q[t][:, None, :], s)[:, 0], u
    return o, s, us, before


def magnitudes(q, k, v, decay, beta, state, scale, eps):
    """Of each output, the sum of what the chunk form adds up for it, without
    signs: exp(G_i) |q_i| |S0| + sum over j of |A_ij| |u_j|."""
    q, k, decay = (np.asarray(x, np.float64) for x in (q, k, decay))
    _, _, us, before = rows(q, k, v, decay, beta, state, scale, eps, np.float64)
    if eps is not None:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + eps) for x in (q, k))
    q, k = by_head(q * scale, k, us.shape[1] // q.shape[1])
    out = np.zeros(us.shape)
    for a in range(0, len(us), CHUNK):
        b = min(a + CHUNK, len(us))
        for h in range(us.shape[1]):
            g = np.cumsum(decay[a:b, h])
            low = np.tril(np.ones((b - a, b - a), bool))
            e = np.where(low, np.exp(np.where(low, g[:, None] - g[None, :], 0)), 0)
            out[a:b, h] = (np.exp(g)[:, None] * (np.abs(q[a:b, h]) @ np.abs(before[a][h])) +
                           np.abs(e * (q[a:b, h] @ k[a:b, h].T)) @ np.abs(us[a:b, h]))
    return out


def parts(x, n):
    """x as n values of 8 bits (each the leading ones of what is left)."""
    out = []
    for _ in range(n):
        top = (np.asarray(x, F32).view(np.uint32) & np.uint32(0xffff0000)).view(F32)
        out.append(top)
        x = x - top
    return out


def chunks(q, k, v, decay, beta, state, scale, eps, plant=None):
    """(o, last state) by the chunks' formulas in float32, o not rounded to bf16.
    plant: "state" keeps the state as bf16 from chunk to chunk, "reset" drops it,
    "sums" has the decays' running sums in float32, "s0", "u" one part less of S0
    towards U, of U towards the state, "o s0", "o u", "o a" one less towards the
    output."""
    less = lambda name, n: n - 1 if plant == name else n
    q, k, v, decay, beta, s = (np.array(x, F32) for x in (q, k, v, decay, beta, state))
    qn, kn = (np.ones(x.shape[:2], F32) if eps is None else
              F32(1) / np.sqrt((x * x).sum(-1, dtype=F32) + F32(eps)) for x in (q, k))
    qn = qn * F32(scale)
    per = v.shape[1] // q.shape[1]
    o = np.zeros(v.shape, F32)
    for h in range(v.shape[1]):
        kh = h // per
        state = s[h]
        for a in range(0, len(v), CHUNK):
            b = min(a + CHUNK, len(v))
            kc, qc, knc, qnc, bc = k[a:b, kh], q[a:b, kh], kn[a:b, kh], qn[a:b, kh], beta[a:b, h]
            g = np.cumsum(decay[a:b, h].astype(F32 if plant == "sums" else np.float64))
            low = np.tril(np.ones((b - a, b - a), bool))
            e = np.where(low, np.exp(np.where(low, g[:, None] - g[None, :], 0).astype(F32)), F32(0))
            eg, ek = np.exp(g.astype(F32)), np.exp((g[-1] - g).astype(F32))
            lm = np.tril((bc * knc)[:, None] * knc[None] * (e * (kc @ kc.T)), -1)
            am = qnc[:, None] * knc[None] * (e * (qc @ kc.T))
            t = np.eye(b - a, dtype=F32)
            for i in range(1, b - a):
                t[i, :i] = -(lm[i, :i] @ t[:i, :i])
            t = t * bc[None]
            x = v[a:b, h] - (eg * knc)[:, None] * sum(kc @ p for p in parts(state, less("s0", 3)))
            u = t @ x
            q0 = sum(qc @ p for p in parts(state, less("o s0", 2)))
            ap, up = parts(am, less("o a", 2)), parts(u, less("o u", 2))
            au = ap[0] @ up[0]
            if len(up) > 1:
                au = au + ap[0] @ up[1]
            if len(ap) > 1:
                au = au + ap[1] @ up[0]
            o[a:b, h] = au + (eg * qnc)[:, None] * q0
            add = sum(kc.T @ p for p in parts(u * (ek * knc)[:, None], less("u", 3)))
            state = (0 if plant == "reset" else eg[-1] * state) + add
            if plant == "state":
                w = np.asarray(state, F32).view(np.uint32).astype(np.uint64)
                state = ((w + 0x7fff + (w >> 16 & 1)).astype(np.uint32) & np.uint32(0xffff0000)).view(F32)
        s[h] = state
    return o, s


def rms(x):
    return np.sqrt((np.asarray(x, np.float64) ** 2).mean((-2, -1)))


def share(got, exact, f32, chunked, carried=0.0, exps=0):
    """The root mean square of a head's f32 errors as a share of what is allowed:
    that of the same steps in float32 row after row, twice where the kernel goes
    row after row too (its sums are taken in another order), and half a step of
    the value.  Chunks may not be worse than one time: a row's step rounds sums
    over key_dim products, a chunk's for 64 rows those and sums over 64 rows.

    The exponentials add to that where decays are not 0.  One is off by up to a
    step of f32, 2^-23 of its value, the same in a whole state and so with one sign:
    S_t = a_t P_t S_{t-1} + .. with a_t <= 1 and P_t = I - beta k k^T of norm <= 1
    changes by e_t a_t P_t S_{t-1}, which later rows do not enlarge.  `exps` of
    them (a row's each, of chunks one per chunk) add up to at most exps * 2^-23 *
    the largest state that is carried, or what outputs are summed from."""
    allowed = (1 if chunked else 2) * rms(f32 - exact) + 2.0 ** -24 * rms(exact)
    return rms(got - exact) / (allowed + exps * 2.0 ** -23 * carried + 1e-37)


def largest_state(args):
    """The largest root mean square of a head's state over the rows, per head."""
    _, last, _, before = rows(*args, np.float64)
    return np.max([rms(s) for s in before + [last]], 0)


def output_share(y, exact, most):
    """The worst error of bf16 outputs as a share of what is allowed: half a step of
    the result, 2^-13 of `most` (a part less of S0, A and U each: 2^-15 for S0, 2^-15
    for the part of A and of U each and 2^-14 for the product of their second parts)."""
    return np.abs(y - exact) / (2.0 ** -8 * np.abs(exact) + 2.0 ** -13 * most + 1e-37)


class Rows:
    """Rows of one sequence for the bounds: `kind` "long" has hundreds of rows and a
    state that decays little and is written weakly, so that what is carried from
    chunk to chunk matters; "keep" has no decay at all; "reset" has decays of -5000
    among small ones, whose sums float32 does not hold; "cancel" has one-hot keys and
    queries that add up states of nearly opposite values, so that the outputs are
    small next to what they are summed from."""
    KINDS = ("long", "keep", "reset", "cancel")

    def __init__(self, rng, kind, key_dim, n=None):
        self.kind, self.eps, self.scale = kind, 1e-6, key_dim ** -0.5
        n = self.n = n or {"long": 450, "keep": 330, "reset": 200, "cancel": 64}[kind]
        self.kh, self.vh, self.kd, self.vd = 1, 2, key_dim, 32
        self.q, self.k = (bf16(rng.standard_normal((n, 1, key_dim))) for _ in range(2))
        self.v = bf16(rng.standard_normal((n, 2, 32)))
        self.state = rng.standard_normal((2, key_dim, 32)).astype(F32)
        self.decay = np.zeros((n, 2), F32)
        if kind == "long":
            self.decay[:] = -2e-3 * rng.random((n, 2))
            self.beta = (0.1 * rng.random((n, 2))).astype(F32)
        elif kind == "keep":
            self.beta = (0.3 * rng.random((n, 2))).astype(F32)
        elif kind == "reset":
            self.decay[:] = -0.02 * rng.random((n, 2))
            self.decay[::70] = -5000.0
            self.beta = rng.random((n, 2)).astype(F32)
        else:
            self.eps, self.scale = None, 1.0
            half = key_dim // 2
            self.state[:, half:] = -self.state[:, :half] * F32(1 + 2.0 ** -11)
            self.decay[:] = -0.01 * rng.random((n, 2))
            self.beta = np.zeros((n, 2), F32)
            self.q[:], self.k[:], self.v[:] = 0, 0, 0
            # rows 0 .. 31: keys of both halves, which take the same share of both;
            # then the queries over a pair each, some met by a key and some not
            for i in range(32):
                self.k[i, 0, i // 2 + (half if i % 2 else 0)] = 1
                self.beta[i] = 0.37
            for i in range(32, n):
                self.q[i, 0, i - 32], self.q[i, 0, i - 32 + half] = 1, 1

    def exps(self, chunked):
        return 0 if self.kind == "keep" else -(-self.n // CHUNK) if chunked else self.n

    def args(self):
        return self.q, self.k, self.v, self.decay, self.beta, self.state, self.scale, self.eps


def bf16(x):
    w = np.asarray(x, F32).view(np.uint32).astype(np.uint64)
    return ((w + 0x7fff + (w >> 16 & 1)).astype(np.uint32) & np.uint32(0xffff0000)).view(F32)
