"""The operators between the q/k/v linears and the output projection, with the
state they carry from call to call, as measurable cases.

A case is a dict of plain values; `prepare` makes the inputs (and, with `own`,
the context, buffers and, where a step is replayed, its captured graph), `run`
is one pass, `exact` the operator's definition in float64.

Kinds
  write      rows of keys and values into the pages of a cache (bf16, or 8-bit
             values with a scale per token and head), and those rows read back
  read       whole prefixes read back from such a cache
  attention  a chunk of new rows per sequence over its pages (which hold the
             chunk's own keys too): row i of n, of a sequence of L keys, sees
             the keys 0 .. L - n + i
  delta      the gated delta rule over a chunk of rows per sequence, from a
             state [value heads, key dim, value dim] to the next

Without `own` everything is elementary torch in float32 on each sequence by
itself: rows gathered from the pages, the whole matrix of scores, and the
delta rule row after row.
"""
import math

import torch

own = False

EPS = 1e-6  # of the delta rule's norms
GOLDEN = 0.6180339887498949


def _case(kind, **kw):
    c = {"kind": kind, "dtype": "bf16", "graph": False, "sequences": 1, "spread": 0.0, "pad": 0}
    c.update(kw)
    return c


def _cache(kind, rows, context, **kw):
    return _case(kind, rows=rows, context=context,
                 **dict({"kv_heads": 4, "dim": 256, "page": 64, "format": "q8"}, **kw))


def _attention(rows, context, **kw):
    return _cache("attention", rows, context, **dict({"heads": 16, "format": "bf16"}, **kw))


def _delta(rows, **kw):
    return _case("delta", rows=rows, **dict({"key_heads": 16, "value_heads": 32, "key_dim": 128,
                                             "value_dim": 128, "fresh": False, "normalize": True},
                                            **kw))


def listed():
    return [
        # one decoded token's keys and values: latency
        dict(_cache("write", 1, 2047, graph=True), name="write_token_q8"),
        # a long prompt's
        dict(_cache("write", 4096, 4096), name="write_prompt_q8"),
        # ragged prefixes as f32 rows, from pages of 48 slots
        dict(_cache("read", 1531, 1531, sequences=5, spread=0.9, dtype="f32", kv_heads=8, dim=128,
                    page=48), name="read_prefixes_f32"),
        # one decoded token over a short context: latency
        dict(_attention(1, 2048, page=256, graph=True), name="attention_token_bf16"),
        # sequences decoding together, their contexts of all lengths
        dict(_attention(1, 8192, sequences=32, spread=0.9, format="q8", graph=True),
             name="attention_batch_q8"),
        # short odd chunks in f32 over small pages; sequences without rows, without
        # keys and with rows before the first key; rows behind the last sequence
        dict(_attention(61, 700, sequences=9, spread=1.0, dtype="f32", heads=12, kv_heads=3,
                        dim=64, page=20, pad=3), name="attention_ragged_f32"),
        # two prompts' next chunks over their long prefixes
        dict(_attention(512, 8192, sequences=2, spread=0.25, heads=32, kv_heads=8, dim=128,
                        format="q8"), name="attention_chunk_q8"),
        # a long prompt (the largest)
        dict(_attention(4096, 4096, page=256), name="attention_prompt_bf16"),
        # one decoded token: latency
        dict(_delta(1, graph=True), name="delta_token_bf16"),
        # sequences decoding together
        dict(_delta(1, sequences=32, graph=True), name="delta_batch_bf16"),
        # ragged prompts in one call, some without rows
        dict(_delta(333, sequences=6, spread=1.0, fresh=True, pad=5), name="delta_ragged_bf16"),
        # a long prompt
        dict(_delta(4096, fresh=True), name="delta_prompt_bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("write", "read", "attention", "attention", "attention", "delta", "delta"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    seqs = rng.choice((1, 1, _log_int(rng, 2, 32)))
    common = {"dtype": dtype, "sequences": seqs, "pad": rng.choice((0, 0, 7)),
              "spread": rng.choice((0.0, 0.5, 1.0)) if seqs > 1 else 0.0}
    if kind == "delta":
        kh, vh, kd, vd = rng.choice(((16, 32, 128, 128), (16, 32, 128, 128), (8, 8, 64, 64),
                                     (4, 12, 128, 64), (6, 6, 64, 160)))
        most = 512 if dtype == "f32" else 4096  # f32 rows are a short check's or a decode step's
        rows = rng.choice((1, _log_int(rng, 1, 16), _log_int(rng, 2, max(2, most // seqs))))
        return _delta(rows, key_heads=kh, value_heads=vh, key_dim=kd, value_dim=vd,
                      fresh=rng.random() < 0.5, normalize=rng.random() < 0.8,
                      graph=rows == 1, **common)
    common.update(page=rng.choice((16, 64, 256, _log_int(rng, 8, 200))),
                  format=rng.choice(("bf16", "q8")))
    if kind != "attention":
        hkv, d = rng.choice(((4, 256), (8, 128), (3, 64)))
        rows = _log_int(rng, 1, 4096 // seqs)
        return _cache(kind, rows, rows if kind == "read" else rows + _log_int(rng, 1, 2048),
                      kv_heads=hkv, dim=d, graph=rows == 1, **common)
    h, hkv, d = rng.choice(((16, 4, 256), (16, 4, 256), (32, 8, 128), (8, 8, 128), (12, 3, 64),
                            (24, 1, 64)))
    rows = rng.choice((1, 1, _log_int(rng, 2, 32), _log_int(rng, 16, max(16, 4096 // seqs))))
    # no more scores than the largest listed case has
    most = min(16384, 4096 * 2048 * 16 * 256 // (seqs * rows * h * d))
    return _attention(rows, max(rows, _log_int(rng, 16, max(16, most))), heads=h, kv_heads=hkv,
                      dim=d, graph=rows == 1, **common)


def _sequences(c):
    """(new rows, keys) of each sequence: the first has the case's, the others
    spread * that much less at most; with spread 1 one has no rows, one no
    keys, and one fewer keys than rows."""
    out = []
    for i in range(c["sequences"]):
        less = 1.0 - c["spread"] * (i * GOLDEN % 1.0)
        n = max(1, round(c["rows"] * less))
        length = n if c["kind"] == "read" else max(n, round(c.get("context", n) * less))
        if c["spread"] == 1.0:
            n = 0 if i == 2 else n
            length = {4: 0, 5: n // 2}.get(i, length)
        out.append((n, length))
    return out


# ------------------------------------------------------------- the inputs --

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 101)
    return g


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _cast(x, dtype):
    return x.to(torch.bfloat16) if dtype == "bf16" else x


def _q8(x):
    """int8 values and f32 scales of rows [..., dim]: d = max|x| / 127 and
    round(x / d), half to even, by the reciprocal."""
    d = x.abs().amax(-1, keepdim=True) / 127.0
    inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    return torch.round(x * inv).to(torch.int8), d.squeeze(-1)


class _Pages:
    """The batch and the cache's buffers, pages [pages, heads, slots, dim] in
    no order; slots that no sequence has hold whatever was there (here NaN)."""

    def __init__(self, c, g):
        self.sequences = _sequences(c)
        page, heads, dim = c["page"], c["kv_heads"], c["dim"]
        need = [-(-length // page) for _, length in self.sequences]
        self.count, self.width = sum(need) + 2, max(1, max(need))
        order = torch.randperm(self.count, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(need), self.width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, k in enumerate(need):
            self.table[i, :k] = order[at:at + k]
            at += k
        shape = (self.count, heads, page, dim)
        if c["format"] == "q8":
            self.k, self.v = (torch.full(shape, -128, dtype=torch.int8, device="cuda")
                              for _ in range(2))
            self.ks, self.vs = (torch.full(shape[:3], math.nan, device="cuda") for _ in range(2))
        else:
            self.k, self.v = (torch.full(shape, math.nan, dtype=torch.bfloat16, device="cuda")
                              for _ in range(2))
            self.ks = self.vs = None
        starts = [0]
        for n, _ in self.sequences:
            starts.append(starts[-1] + n)
        self.rows = starts[-1] + c["pad"]
        self.bounds = starts
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.lengths = torch.tensor([length for _, length in self.sequences], dtype=torch.int32,
                                    device="cuda")
        self.page = page

    def slots(self, i, lo, hi):
        """Pages and slots of the positions lo .. hi - 1 of sequence i."""
        p = torch.arange(lo, hi, device="cuda")
        return self.table[i][p // self.page].long(), p % self.page

    def put(self, i, lo, k, v):
        """Rows [n, heads, dim] f32 at the positions from lo."""
        page, slot = self.slots(i, lo, lo + k.shape[0])
        for rows, values, scales in ((k, self.k, self.ks), (v, self.v, self.vs)):
            if scales is None:
                values[page, :, slot] = rows.to(torch.bfloat16)
            else:
                values[page, :, slot], scales[page, :, slot] = _q8(rows)

    def get(self, i, lo, hi):
        """The values that the positions lo .. hi - 1 stand for, f32."""
        page, slot = self.slots(i, lo, hi)
        out = []
        for values, scales in ((self.k, self.ks), (self.v, self.vs)):
            rows = values[page, :, slot].float()
            out.append(rows if scales is None else rows * scales[page, :, slot][..., None])
        return out


def _inputs(c, seed):
    g, dt = _gen(seed), c["dtype"]
    d = {}
    if c["kind"] == "delta":
        ns = [n for n, _ in _sequences(c)]
        bounds = [0]
        for n in ns:
            bounds.append(bounds[-1] + n)
        rows, hk, hv, kd, vd = (bounds[-1] + c["pad"], c["key_heads"], c["value_heads"],
                                c["key_dim"], c["value_dim"])
        d["bounds"], d["rows"] = bounds, rows
        d["starts"] = torch.tensor(bounds, dtype=torch.int32, device="cuda")
        # one row of q, k and v side by side, as the linear in front leaves it
        # (rows without the norm stay near length 1 by themselves)
        near = 1.0 if c["normalize"] else kd ** -0.5
        q, k = _randn(g, rows, hk * kd, scale=near), _randn(g, rows, hk * kd, scale=near)
        d["qkv"] = _cast(torch.cat((q, k, _randn(g, rows, hv * vd)), 1), dt)
        d["decay"] = -0.5 * torch.rand(rows, hv, generator=g, device="cuda") ** 2 - 1e-3
        d["beta"] = torch.rand(rows, hv, generator=g, device="cuda")
        d["state"] = None if c["fresh"] else _randn(g, len(ns), hv, kd, vd, scale=0.3)
        return d
    d["pages"] = p = _Pages(c, g)
    heads, dim = c["kv_heads"], c["dim"]
    if c["kind"] == "write":
        d["k"], d["v"] = (_cast(_randn(g, p.rows, heads, dim), dt) for _ in range(2))
        return d
    for i, (_, length) in enumerate(p.sequences):
        p.put(i, 0, _randn(g, length, heads, dim), _randn(g, length, heads, dim))
    if c["kind"] == "attention":
        d["q"] = _cast(_randn(g, p.rows, c["heads"], dim, scale=2.0), dt)
    return d


def _split(c, d):
    """q, k [rows, key heads, key dim] and v [rows, value heads, value dim]
    of the rows of a delta case."""
    hk, kd = c["key_heads"], c["key_dim"]
    q, k, v = d["qkv"].split((hk * kd, hk * kd, c["value_heads"] * c["value_dim"]), 1)
    return (q.reshape(-1, hk, kd), k.reshape(-1, hk, kd),
            v.reshape(-1, c["value_heads"], c["value_dim"]))


# --------------------------------------------------------- the plain forms --

def _delta_rows(c, d, ftype):
    """The rows of a delta case padded to [sequences, longest, ...], the padding
    leaving the state alone: q, k (over their norms, q scaled, one per value
    head), v, exp(log decay), beta, the state, and where the rows are."""
    q, k, v = (x.to(ftype) for x in _split(c, d))
    if c["normalize"]:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + EPS)
    per = c["value_heads"] // c["key_heads"]
    q = (q * c["key_dim"] ** -0.5).repeat_interleave(per, 1)
    k = k.repeat_interleave(per, 1)
    ns = [b - a for a, b in zip(d["bounds"], d["bounds"][1:])]
    longest = max(ns)
    at = torch.zeros(len(ns), longest, dtype=torch.long, device="cuda")
    live = torch.zeros(len(ns), longest, dtype=torch.bool, device="cuda")
    for i, n in enumerate(ns):
        at[i, :n] = torch.arange(d["bounds"][i], d["bounds"][i] + n, device="cuda")
        live[i, :n] = True
    decay = torch.where(live[..., None], torch.exp(d["decay"].to(ftype))[at], 1.0)
    beta = torch.where(live[..., None], d["beta"].to(ftype)[at], 0.0)
    shape = (len(ns), c["value_heads"], c["key_dim"], c["value_dim"])
    state = (torch.zeros(shape, dtype=ftype, device="cuda") if d["state"] is None
             else d["state"].to(ftype))
    return q[at], k[at], v[at], decay, beta, state, at, live


def _plain(state):
    c, d = state.case, state.inputs
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    if c["kind"] == "delta":
        q, k, v, decay, beta, s, at, live = _delta_rows(c, d, torch.float32)
        o = torch.zeros_like(v)
        for t in range(q.shape[1]):
            s = s * decay[:, t, :, None, None]
            u = beta[:, t, :, None] * (v[:, t] - (s * k[:, t, :, :, None]).sum(2))
            s = s + k[:, t, :, :, None] * u[:, :, None, :]
            o[:, t] = (s * q[:, t, :, :, None]).sum(2)
        out = torch.zeros(d["rows"], c["value_heads"], c["value_dim"], dtype=dt, device="cuda")
        out[at[live]] = o[live].to(dt)
        return [out, s]
    p = d["pages"]
    if c["kind"] != "attention":
        k, v = (torch.zeros(p.rows, c["kv_heads"], c["dim"], dtype=dt, device="cuda")
                for _ in range(2))
        for i, (n, length) in enumerate(p.sequences):
            a, first = p.bounds[i], max(0, n - length)
            if first == n:
                continue
            if c["kind"] == "write":
                p.put(i, length - n + first, d["k"][a + first:a + n].float(),
                      d["v"][a + first:a + n].float())
            rows = p.get(i, length - n + first, length)
            k[a + first:a + n], v[a + first:a + n] = (r.to(dt) for r in rows)
        return [k, v]
    h, hkv, dim = c["heads"], c["kv_heads"], c["dim"]
    out = torch.zeros(p.rows, h, dim, dtype=dt, device="cuda")
    for i, (n, length) in enumerate(p.sequences):
        if n == 0 or length == 0:
            continue
        a = p.bounds[i]
        k, v = (x.transpose(0, 1).contiguous() for x in p.get(i, 0, length))
        q = d["q"][a:a + n].float().view(n, hkv, h // hkv, dim).transpose(0, 1).reshape(hkv, -1, dim)
        s = torch.bmm(q, k.transpose(1, 2).contiguous()) * dim ** -0.5
        hidden = (torch.arange(length, device="cuda")[None, :]
                  > (length - n + torch.arange(n, device="cuda"))[:, None])
        s = s.view(hkv, n, h // hkv, length).masked_fill_(hidden[:, None, :], -math.inf)
        top = s.amax(-1, keepdim=True)
        e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = e.sum(-1, keepdim=True)
        o = torch.bmm((e / torch.where(total == 0, 1.0, total)).view(hkv, -1, length), v)
        out[a:a + n] = o.view(hkv, n, h // hkv, dim).transpose(0, 1).reshape(n, h, dim).to(dt)
    return [out]


# ---------------------------------------------------------- the framework --

class _Buf:
    """A torch tensor as the front end takes buffers (by address)."""

    def __init__(self, tensor, offset=0):
        self.tensor, self.ptr = tensor, tensor.data_ptr() + offset * tensor.element_size()


class _State:
    """The inputs; with the framework also the context, buffers and captured
    pass."""

    stream = None  # the one stream that all passes are queued on

    def __init__(self, case, inputs):
        self.case, self.inputs, self.graph, self.keep, self.ctx = case, inputs, None, [], None

    def open(self):
        import llmcp_amd as q8
        if _State.stream is None:
            _State.stream = torch.cuda.Stream()
        self.q8, self.ctx = q8, q8.Context(0)
        q8.check(q8.lib().llmcp_q8_ctx_set_stream(self.ctx.handle, _State.stream.cuda_stream))
        return self.ctx

    def buf(self, tensor, offset=0):
        self.keep.append(_Buf(tensor, offset))
        return self.keep[-1]

    def out(self, *shape, dtype=None):
        """A buffer of zeros (rows that no sequence has stay so)."""
        dt = dtype or (torch.bfloat16 if self.case["dtype"] == "bf16" else torch.float32)
        return self.buf(torch.zeros(*shape, device="cuda", dtype=dt))

    def cache(self, p):
        c = self.case
        scales = (None, None) if p.ks is None else (self.buf(p.ks), self.buf(p.vs))
        cache = self.q8.KVCache(self.buf(p.k), self.buf(p.v), p.count, c["page"], c["kv_heads"],
                                c["dim"], key_scales=scales[0], value_scales=scales[1])
        batch = self.q8.KVBatch(self.buf(p.starts), self.buf(p.lengths), self.buf(p.table),
                                len(p.sequences), p.width)
        return cache, batch

    def __del__(self):
        try:
            if self.graph is not None:
                self.ctx.sync()
                self.ctx.graph_destroy(self.graph)
            if self.ctx is not None:
                self.ctx.close()
        except Exception:
            pass


def _framework(s):
    """The calls of one pass and its outputs."""
    c, d, dt = s.case, s.inputs, s.case["dtype"]
    ctx = s.open()
    if c["kind"] == "delta":
        hk, hv, kd, vd, rows = (c["key_heads"], c["value_heads"], c["key_dim"], c["value_dim"],
                                d["rows"])
        q, k, v = (s.buf(d["qkv"], at) for at in (0, hk * kd, 2 * hk * kd))
        wide = d["qkv"].shape[1]
        decay, beta, starts = s.buf(d["decay"]), s.buf(d["beta"]), s.buf(d["starts"])
        before = None if d["state"] is None else s.buf(d["state"])
        seqs = len(d["bounds"]) - 1
        after = s.out(seqs, hv, kd, vd, dtype=torch.float32)
        o = s.out(rows, hv, vd)

        def calls():
            ctx.delta_rule(q, k, v, decay, beta, o, rows, hk, hv, kd, vd, state=before,
                           new_state=after, row_starts=starts, sequences=seqs, scale=kd ** -0.5,
                           eps=EPS if c["normalize"] else None, strides=(wide, wide, wide),
                           dtype=dt)
        return calls, lambda: [o.tensor, after.tensor]
    p = d["pages"]
    cache, batch = s.cache(p)
    if c["kind"] == "attention":
        q, o = s.buf(d["q"]), s.out(p.rows, c["heads"], c["dim"])

        def calls():
            ctx.attention(q, cache, batch, o, p.rows, c["heads"], scale=c["dim"] ** -0.5, dtype=dt)
        return calls, lambda: [o.tensor]
    k, v = (s.out(p.rows, c["kv_heads"], c["dim"]) for _ in range(2))
    if c["kind"] == "write":
        new = s.buf(d["k"]), s.buf(d["v"])

        def calls():
            ctx.kv_write(new[0], new[1], cache, batch, p.rows, dtype=dt)
            ctx.kv_read(cache, batch, k, v, p.rows, dtype=dt)
    else:
        def calls():
            ctx.kv_read(cache, batch, k, v, p.rows, dtype=dt)
    return calls, lambda: [k.tensor, v.tensor]


def prepare(case, seed):
    s = _State(case, _inputs(case, seed))
    if own:
        s.calls, s.outputs = _framework(s)
        torch.cuda.synchronize()
        if case["graph"]:
            # once outside the capture: the workspace grows to this size
            s.calls()
            s.ctx.sync()
            s.ctx.graph_begin()
            s.calls()
            s.graph = s.ctx.graph_end()
    torch.cuda.synchronize()
    return s


def run(state):
    if not own:
        return _plain(state)
    if state.graph is not None:
        state.ctx.graph_launch(state.graph)
    else:
        state.calls()
    return state.outputs()


# ------------------------------------------------------------ the yardstick --

def work(case):
    c, e, seqs = case, 2 if case["dtype"] == "bf16" else 4, _sequences(case)
    rows = sum(n for n, _ in seqs)
    if c["kind"] == "delta":
        hk, hv, kd, vd = c["key_heads"], c["value_heads"], c["key_dim"], c["value_dim"]
        state = len(seqs) * hv * kd * vd * 4
        return {"bytes": rows * (e * (2 * hk * kd + 2 * hv * vd) + 8 * hv)
                + state * (1 if c["fresh"] else 2), "flops": 7 * rows * hv * kd * vd}
    hkv, dim = c["kv_heads"], c["dim"]
    token = 2 * hkv * (dim + 4 if c["format"] == "q8" else 2 * dim)  # a position's bytes
    held = sum(min(n, length) for n, length in seqs)
    if c["kind"] == "write":
        return {"bytes": held * (2 * token + 4 * hkv * dim * e), "flops": 10 * held * hkv * dim}
    if c["kind"] == "read":
        return {"bytes": held * (token + 2 * hkv * dim * e), "flops": 2 * held * hkv * dim}
    seen = keys = 0
    for n, length in seqs:
        live = min(n, length)
        keys += length if live else 0
        seen += live * length - live * (live - 1) // 2
    return {"bytes": keys * token + 2 * rows * c["heads"] * dim * e,
            "flops": 4 * seen * c["heads"] * dim}


def _kept64(x, c):
    """What a cache of the case's format keeps of rows [n, heads, dim]: its
    scale and steps are f32's by definition."""
    if c["format"] == "bf16":
        return x.to(torch.bfloat16).double()
    q, scale = _q8(x.float())
    return q.double() * scale.double()[..., None]


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["kind"] == "delta":
        q, k, v, decay, beta, s, at, live = _delta_rows(c, d, torch.float64)
        o = torch.zeros_like(v)
        for t in range(q.shape[1]):
            decayed = decay[:, t, :, None, None] * s
            seen = torch.matmul(k[:, t, :, None, :], decayed)[:, :, 0]
            s = decayed + k[:, t, :, :, None] * (beta[:, t, :, None] * (v[:, t] - seen))[:, :, None]
            o[:, t] = torch.matmul(q[:, t, :, None, :], s)[:, :, 0]
        out = torch.zeros(d["rows"], c["value_heads"], c["value_dim"], dtype=torch.float64,
                          device="cuda")
        out[at[live]] = o[live]
        return [out, s]
    p = d["pages"]
    if c["kind"] != "attention":
        k, v = (torch.zeros(p.rows, c["kv_heads"], c["dim"], dtype=torch.float64, device="cuda")
                for _ in range(2))
        for i, (n, length) in enumerate(p.sequences):
            a, first = p.bounds[i], max(0, n - length)
            if first == n:
                continue
            if c["kind"] == "write":
                k[a + first:a + n] = _kept64(d["k"][a + first:a + n], c)
                v[a + first:a + n] = _kept64(d["v"][a + first:a + n], c)
            else:
                page, slot = p.slots(i, length - n + first, length)
                for out, values, scales in ((k, p.k, p.ks), (v, p.v, p.vs)):
                    rows = values[page, :, slot].double()
                    out[a + first:a + n] = (rows if scales is None else
                                            rows * scales[page, :, slot].double()[..., None])
        return [k, v]
    out = torch.zeros(p.rows, c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    group = c["heads"] // c["kv_heads"]
    for i, (n, length) in enumerate(p.sequences):
        for h in range(c["kv_heads"] if n and length else 0):
            a = p.bounds[i]
            page, slot = p.slots(i, 0, length)
            k, v = p.k[page, h, slot].double(), p.v[page, h, slot].double()
            if p.ks is not None:
                k = k * p.ks[page, h, slot].double()[:, None]
                v = v * p.vs[page, h, slot].double()[:, None]
            position = length - n + torch.arange(n, device="cuda")
            sees = torch.arange(length, device="cuda")[None, :] <= position[:, None]
            for j in range(h * group, (h + 1) * group):
                s = d["q"][a:a + n, j].double() @ k.t() / math.sqrt(c["dim"])
                e = torch.where(sees, s, -1e300)
                e = torch.exp(e - e.amax(-1, keepdim=True)) * sees
                out[a:a + n, j] = (e @ v) / e.sum(-1, keepdim=True).clamp(min=1e-300)
    return [out]
