"""A paged key/value cache on the device and what it should hold, for the tests of
the cache's entries and of attention."""
import numpy as np

F32 = np.float32


class Cache:
    """A cache on the device whose memory starts as NaN (bf16, scales) or -128
    (int8), and the sequences' pages in shuffled order."""

    def __init__(self, q8, ctx, rng, lengths, page, heads, dim, fmt, extra=2, width=None):
        self.q8, self.ctx, self.page, self.heads, self.dim, self.fmt = q8, ctx, page, heads, dim, fmt
        self.lengths = [int(n) for n in lengths]
        need = [-(-max(n, 0) // page) for n in self.lengths]
        self.width = width or max(1, max(need))
        need = [min(n, self.width) for n in need]
        self.pages = sum(need) + extra
        order = rng.permutation(self.pages)
        self.table = np.full((len(need), self.width), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (self.pages, heads, page, dim)
        if fmt == "q8":
            self.k = np.full(shape, -128, np.int8)
            self.ks = np.full(shape[:3], np.nan, F32)
            self.v, self.vs = self.k.copy(), self.ks.copy()
        else:
            self.k = np.full(shape, 0x7FC0, np.uint16)
            self.v, self.ks, self.vs = self.k.copy(), None, None
        self.upload()

    def upload(self):
        c = self.ctx
        self.dk, self.dv = c.to_device(self.k), c.to_device(self.v)
        self.dks, self.dvs = ((None, None) if self.ks is None else
                              (c.to_device(self.ks), c.to_device(self.vs)))

    def cache(self):
        return self.q8.KVCache(self.dk, self.dv, self.pages, self.page, self.heads, self.dim,
                               key_scales=self.dks, value_scales=self.dvs)

    def batch(self, starts, lengths=None, table=None):
        self.keep = [self.ctx.to_device(np.asarray(a, np.int32)) for a in
                     (starts, self.lengths if lengths is None else lengths,
                      self.table if table is None else table)]
        return self.q8.KVBatch(*self.keep, len(starts) - 1, self.width)

    def download(self):
        c, shape = self.ctx, self.k.shape
        out = [c.to_host(b, shape, self.k.dtype) for b in (self.dk, self.dv)]
        if self.ks is not None:
            out += [c.to_host(b, shape[:3], F32) for b in (self.dks, self.dvs)]
        return out

    def put(self, oracle, seq, position, k, v):
        """The expected memory after rows [n, heads, dim] from `position` on."""
        for i in range(k.shape[0]):
            p = position + i
            if p < 0 or p >= self.width * self.page:
                continue
            page = self.table[seq, p // self.page]
            if page < 0 or page >= self.pages:
                continue
            for x, values, scales in ((k[i], self.k, self.ks), (v[i], self.v, self.vs)):
                if scales is None:
                    values[page, :, p % self.page] = oracle.f32_to_bf16_bits(x)
                else:
                    values[page, :, p % self.page], scales[page, :, p % self.page] = quantize(x)

    def values(self, oracle, seq, lo, hi):
        """What the positions stand for (f32; zeros without a slot)."""
        out = np.zeros((2, hi - lo, self.heads, self.dim), F32)
        for p in range(max(lo, 0), min(hi, self.width * self.page)):
            page = self.table[seq, p // self.page]
            if page < 0 or page >= self.pages:
                continue
            for j, (values, scales) in enumerate(((self.k, self.ks), (self.v, self.vs))):
                x = values[page, :, p % self.page]
                out[j, p - lo] = (oracle.bf16_bits_to_f32(x) if scales is None else
                                  x.astype(F32) * scales[page, :, p % self.page][:, None])
        return out


def quantize(x):
    """int8 values and scale of rows [heads, dim]."""
    x = np.asarray(x, F32)
    with np.errstate(all="ignore"):
        m = np.abs(x).max(-1)
        odd = ~np.isfinite(x).all(-1)
        live = ~odd & (m >= F32(2.0 ** -118))
        s = np.where(odd, F32(np.nan), np.where(live, m / F32(127), F32(0)))
        inv = np.where(live, F32(1) / s, F32(0))
        q = np.where(live[:, None], np.rint(x * inv[:, None]), 0)
    return q.astype(np.int8), s.astype(F32)


def same(a, b):
    a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
    if a.dtype == F32:
        return np.array_equal(a, b, equal_nan=True)
    return np.array_equal(a, b)


def rows_of(oracle, rng, n, heads, dim, dtype, scale=1.0):
    x = (rng.standard_normal((n, heads, dim)) * scale).astype(F32)
    bits = oracle.f32_to_bf16_bits(x)
    return (bits, oracle.bf16_bits_to_f32(bits)) if dtype == "bf16" else (x, x)


def narrow(oracle, x, dtype):
    return oracle.f32_to_bf16_bits(x) if dtype == "bf16" else x
