"""The operators of a mixture-of-experts block around the Q8_0 linears, as
measurable cases.

A case is a dict of plain values; `prepare` makes the inputs (and, with `own`,
the context, registered weights, buffers and, where a step is replayed, its
captured graph), `run` is one pass, `exact` the operator's definition in
float64.

Kinds
  norm    s = x + residual; y = RMSNorm(s) * w; y as Q8_1 (8-bit values with a
          scale per 32, returned as the values they stand for)
  route   the top_k of the router's logits per row and their softmax weights
  linear  each row through the experts its slots name (ragged groups)
  mlp     the SwiGLU MLPs of the experts each row is routed to, combined by
          the router's weights, with the residual's addition (bf16, the type
          of such a model's hidden state)

Without `own` everything is elementary torch: float32 products and sums
(float64 for the norm's sum, on which the border of a quantizer's step
hangs), experts batched by padding each to the longest.  Activations are
quantized to Q8_1 as the format defines it, and a bf16 result is rounded
where the graph of separate bf16 operators would round it.
"""
import math

import torch

own = False

EPS = 2.0 ** -20  # about 1e-6, the same number in f32 and f64
ACTIVATIONS = ("none", "silu", "sigmoid", "softplus")


def _case(kind, **kw):
    c = {"kind": kind, "dtype": "bf16", "graph": False}
    c.update(kw)
    return c


def _norm(m, h, **kw):
    return _case("norm", m=m, h=h, **dict({"zero_centered": True}, **kw))


def _route(m, e, k, **kw):
    return _case("route", m=m, e=e, k=k, **dict({"normalize": True, "masked": 0.0}, **kw))


def _linear(m, e, k, n, cols, **kw):
    return _case("linear", m=m, e=e, k=k, n=n, cols=cols,
                 **dict({"act": "none", "per_slot": False, "masked": 0.0, "skew": 0.0,
                         "platform": "aarch64"}, **kw))


def _mlp(m, e, k, h, f, **kw):
    return _case("mlp", m=m, e=e, k=k, h=h, f=f,
                 **dict({"residual": True, "masked": 0.0, "skew": 0.0, "platform": "aarch64"}, **kw))


def listed():
    return [
        # the norm in front of one token's experts: latency
        dict(_norm(1, 2560, graph=True), name="norm_token_bf16"),
        # a short prompt in f32, rows of 69 blocks
        dict(_norm(37, 2208, dtype="f32", zero_centered=False), name="norm_ragged_f32"),
        # a long prompt chunk's rows
        dict(_norm(4096, 2560), name="norm_prompt_bf16"),
        # one token's choice of experts
        dict(_route(1, 128, 8, dtype="f32", graph=True), name="route_token_f32"),
        # a long prompt chunk's, from bf16 logits (which tie)
        dict(_route(4096, 128, 8), name="route_prompt_bf16"),
        # odd sizes on the x86 platform's arithmetic: K of 69 blocks, ragged
        # tiles, an activation, every fifth slot without an expert
        dict(_linear(45, 20, 3, 1000, 2208, act="silu", masked=0.2, platform="x86"),
             name="experts_ragged_x86_bf16"),
        # rows that already belong to a slot each (a down projection), f32
        dict(_linear(160, 32, 4, 2560, 768, per_slot=True, dtype="f32"), name="experts_slots_f32"),
        # one token through its eight experts: the decode step
        dict(_mlp(1, 128, 8, 2560, 768, graph=True), name="mlp_token_bf16"),
        # a batch of sixteen sequences decoding together
        dict(_mlp(16, 128, 8, 2560, 768, graph=True), name="mlp_batch_m16_bf16"),
        # a prompt whose tokens prefer a few of the experts
        dict(_mlp(333, 128, 8, 2560, 768, skew=1.0), name="mlp_prompt_m333_bf16"),
        # a long prompt chunk (the largest)
        dict(_mlp(4096, 128, 8, 2560, 768), name="mlp_prompt_m4096_bf16"),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(("norm", "norm", "route", "linear", "linear", "linear", "mlp", "mlp", "mlp"))
    dtype = rng.choice(("f32", "bf16"))
    platform = rng.choice(("aarch64", "aarch64", "x86"))
    masked = rng.choice((0.0, 0.0, 0.1, 0.6))
    skew = rng.choice((0.0, 0.0, 1.0, 2.0))
    if kind == "norm":
        h = _log_int(rng, 64, 8192, 32)
        m = _log_int(rng, 1, min(4096, 4096 * 2560 // h))
        return _norm(m, h, dtype=dtype, zero_centered=rng.random() < 0.5, graph=m <= 16)
    if kind == "route":
        e = _log_int(rng, 16, 512)
        m, k = _log_int(rng, 1, 4096), rng.randint(1, 16)
        # (a single chosen expert's normalized weight would be 1 whatever the logits)
        return _route(m, e, k, dtype=dtype, masked=masked, normalize=k > 1 and rng.random() < 0.5,
                      graph=m <= 16)
    e = _log_int(rng, 4, 128)
    k = rng.randint(1, min(e, 8))
    if kind == "linear":
        m = 1 if rng.random() < 0.2 else _log_int(rng, 2, 512)
        return _linear(m, e, k, _log_int(rng, 64, 2560, 8), _log_int(rng, 64, 2560, 32),
                       act=rng.choice(ACTIVATIONS), per_slot=rng.random() < 0.4, dtype=dtype,
                       masked=masked, skew=skew, platform=platform, graph=m <= 16)
    m = 1 if rng.random() < 0.2 else _log_int(rng, 2, 4096)
    return _mlp(m, e, k, _log_int(rng, 256, 2560, 32), _log_int(rng, 64, 768, 32),
                residual=rng.random() < 0.7, masked=masked, skew=skew, platform=platform,
                graph=m <= 16)


# ------------------------------------------------------------- the inputs --

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 9973 + 29)
    return g


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * scale


def _cast(x, dtype):
    return x.to(torch.bfloat16) if dtype == "bf16" else x


def _weight(g, e, n, k):
    """e experts' N(0, 0.02) weights as Q8_0: int8 values [e, n, k/32, 32] and
    f16 scales [e, n, k/32] (max|w| / 127, rounding half away from zero)."""
    w = _randn(g, e, n, k, scale=0.02).view(e, n, k // 32, 32)
    scale = w.abs().amax(-1, keepdim=True) / 127.0
    r = w / scale
    q = torch.where(r < 0, -torch.floor(0.5 - r), torch.floor(0.5 + r)).to(torch.int8)
    return q, scale.squeeze(-1).to(torch.float16)


def _logits(c, g):
    """Router logits: `skew` prefers some experts, `masked` is the share of
    entries that are out of the choice."""
    l = _randn(g, c["m"], c["e"], scale=2.0)
    if c.get("skew"):
        l = l + c["skew"] * 2.0 * _randn(g, 1, c["e"])
    return l


def _routing(c, g):
    """int32 expert ids [m, k] (-1: a slot without an expert) and weights."""
    p, ids = torch.sort(_logits(c, g), dim=-1, descending=True)
    p, ids = torch.exp(p - p[:, :1])[:, :c["k"]], ids[:, :c["k"]].to(torch.int32)
    p = p / p.sum(-1, keepdim=True)
    if c["masked"]:
        out = torch.rand(ids.shape, generator=g, device="cuda") < c["masked"]
        out[0, 0] = False  # one slot at least has an expert
        ids, p = torch.where(out, -1, ids), torch.where(out, 0.0, p)
    return ids.contiguous(), p.contiguous()


def _inputs(c, seed):
    g, m, dt, kind = _gen(seed), c["m"], c["dtype"], c["kind"]
    d = {}
    if kind == "norm":
        d["x"] = _cast(_randn(g, m, c["h"]), dt)
        d["r"] = _cast(_randn(g, m, c["h"], scale=2.0), dt)
        d["w"] = _cast(_randn(g, c["h"], scale=0.1) + (0.0 if c["zero_centered"] else 1.0), dt)
    elif kind == "route":
        l = _logits(c, g)
        if c["masked"]:
            l = torch.where(torch.rand(l.shape, generator=g, device="cuda") < c["masked"],
                            -math.inf, l)
        d["logits"] = _cast(l, dt)
    elif kind == "linear":
        d["ids"], _ = _routing(c, g)
        d["x"] = _cast(_randn(g, m * c["k"] if c["per_slot"] else m, c["cols"]), dt)
        d["w"] = _weight(g, c["e"], c["n"], c["cols"])
    else:
        d["ids"], d["p"] = _routing(c, g)
        d["x"] = _cast(_randn(g, m, c["h"]), dt)
        d["r"] = _cast(_randn(g, m, c["h"]), dt) if c["residual"] else None
        d["gate"] = _weight(g, c["e"], c["f"], c["h"])
        d["up"] = _weight(g, c["e"], c["f"], c["h"])
        d["down"] = _weight(g, c["e"], c["h"], c["f"])
    return d


# --------------------------------------------------------- the plain forms --

def _q8_1(x):
    """Q8_1 of f32 rows, dequantized: per 32 values d = max|x| / 127 and
    round(x / d), half to even, by the reciprocal as the format has it."""
    v = x.view(x.shape[0], -1, 32)
    d = v.abs().amax(-1, keepdim=True) / 127.0
    inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    return (torch.round(v * inv) * d).view(x.shape)


def _act(v, name):
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    if name == "softplus":
        return torch.log(1.0 + torch.exp(v))
    return v


class _Groups:
    """The slots by expert: every expert's rows padded to the longest, or,
    with no more slots than experts, one group a slot."""

    def __init__(self, ids, experts):
        slots = ids.reshape(-1).long()
        self.live = slots >= 0
        self.slot_experts = slots.clamp(min=0)
        self.each = slots.numel() <= experts
        if not self.each:
            order = torch.argsort(torch.where(self.live, slots, experts), stable=True)
            counts = torch.bincount(slots[self.live], minlength=experts)
            start = torch.cumsum(counts, 0) - counts
            pad = int(counts.max())
            at = start[:, None] + torch.arange(pad, device=ids.device)
            self.has = torch.arange(pad, device=ids.device) < counts[:, None]
            self.rows = order[at.clamp(max=slots.numel() - 1)]

    def matmul(self, xs, qd):
        """Row i of xs [slots, K] times its expert's weight, f32; rows without
        an expert are zero."""
        q, d = qd
        if self.each:
            q, d = q[self.slot_experts], d[self.slot_experts]
        w = (q.float() * d.float()[..., None]).flatten(2).transpose(1, 2).contiguous()
        if self.each:
            return torch.bmm(xs[:, None, :], w)[:, 0] * self.live[:, None]
        y = torch.bmm(xs[self.rows], w)
        out = torch.zeros(xs.shape[0], w.shape[2], device=xs.device)
        out[self.rows[self.has]] = y[self.has]
        return out


def _plain(state):
    c, d = state.case, state.inputs
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    rnd = lambda v: v.to(dt).float()  # noqa: E731
    if c["kind"] == "norm":
        s = (d["x"].float() + d["r"].float()).to(dt)
        v = s.float()
        mean = v.double().square().sum(-1, keepdim=True) / c["h"]
        rstd = (1.0 / torch.sqrt(mean + EPS)).float()
        w = d["w"].float() + 1.0 if c["zero_centered"] else d["w"].float()
        y = (v * rstd * w).to(dt)
        return [s, y, _q8_1(y.float()).to(dt)]
    if c["kind"] == "route":
        l = d["logits"].float()
        e = torch.exp(l - l.amax(-1, keepdim=True))
        e = torch.where(l == -math.inf, 0.0, e)
        _, ids = torch.sort(l, dim=-1, descending=True, stable=True)
        ids = ids[:, :c["k"]]
        chosen = torch.gather(e, 1, ids)
        total = (chosen if c["normalize"] else e).sum(-1, keepdim=True)
        p = torch.where(chosen > 0, chosen / total, 0.0)
        return [torch.where(torch.gather(l, 1, ids) == -math.inf, -1, ids).to(torch.int32), p]
    g = _Groups(d["ids"], c["e"])
    x = _q8_1(d["x"].float())
    if x.shape[0] != g.live.numel():
        x = x.repeat_interleave(c["k"], 0)
    if c["kind"] == "linear":
        return [(_act(g.matmul(x, d["w"]), c["act"]) * g.live[:, None]).to(dt)]
    h = rnd(rnd(_act(g.matmul(x, d["gate"]), "silu")) * rnd(g.matmul(x, d["up"])))
    o = rnd(g.matmul(_q8_1(h), d["down"])).view(c["m"], c["k"], c["h"])
    y = (o * d["p"][..., None]).sum(1)
    return [(y + d["r"].float() if c["residual"] else y).to(dt)]


# ---------------------------------------------------------- the framework --

class _Buf:
    """A torch tensor as the front end takes buffers (by address)."""

    def __init__(self, tensor):
        self.tensor, self.ptr = tensor, tensor.data_ptr()


class _State:
    """The inputs; with the framework also the context, its weights, buffers
    and captured pass."""

    stream = None  # the one stream that all passes are queued on

    def __init__(self, case, inputs):
        self.case, self.inputs, self.graph, self.keep, self.ctx = case, inputs, None, [], None

    def open(self):
        import llmcp_amd as q8
        if _State.stream is None:
            _State.stream = torch.cuda.Stream()
        self.q8, self.ctx = q8, q8.Context(0)
        q8.check(q8.lib().llmcp_q8_ctx_set_stream(self.ctx.handle, _State.stream.cuda_stream))
        self.ctx.set_platform(self.case.get("platform", "aarch64"))
        return self.ctx

    def buf(self, tensor):
        self.keep.append(_Buf(tensor))
        return self.keep[-1]

    def out(self, *shape, dtype=None):
        dt = dtype or (torch.bfloat16 if self.case["dtype"] == "bf16" else torch.float32)
        return self.buf(torch.empty(*shape, device="cuda", dtype=dt))

    def experts(self, qd):
        """Registers a stack of experts, packed as the arena's q8_0_p4 records
        (4 scales, then 8 chunks of 4 rows x 4 values)."""
        q, d = qd
        e, n, b = d.shape
        rec = torch.empty(e * n // 4, b, 136, dtype=torch.uint8, device="cuda")
        rec[:, :, :8] = (d.view(e * n // 4, 4, b).transpose(1, 2).contiguous()
                         .view(torch.uint8))
        rec[:, :, 8:] = (q.view(e * n // 4, 4, b, 8, 4).permute(0, 2, 3, 1, 4)
                         .reshape(e * n // 4, b, 128).view(torch.uint8))
        torch.cuda.synchronize()
        return self.ctx.register_device_experts_p4(_Buf(rec), e, n, 32 * b)

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
    c, d, m, dt = s.case, s.inputs, s.case["m"], s.case["dtype"]
    ctx = s.open()
    if c["kind"] == "norm":
        h = c["h"]
        x, r, w = s.buf(d["x"]), s.buf(d["r"]), s.buf(d["w"])
        total, y = s.out(m, h), s.out(m, h)
        values, scales = s.out(m, h // 32, 32, dtype=torch.int8), s.out(m, h // 32, 1, dtype=torch.float32)
        wide = s.out(m, h // 32, 32)
        rows = s.q8.Q8Rows(values, scales, m, h)

        def calls():
            ctx.add_rmsnorm(x, r, w, total, m, h, normed=y, quantized=rows, eps=EPS,
                            zero_centered=c["zero_centered"], dtype=dt)

        def outputs():
            with torch.cuda.stream(_State.stream):
                torch.mul(values.tensor, scales.tensor, out=wide.tensor)
            return [total.tensor, y.tensor, wide.tensor.view(m, h)]
        return calls, outputs
    if c["kind"] == "route":
        logits = s.buf(d["logits"])
        ids, p = s.out(m, c["k"], dtype=torch.int32), s.out(m, c["k"], dtype=torch.float32)

        def calls():
            ctx.route(logits, m, c["e"], c["k"], ids, p, normalize=c["normalize"], dtype=dt)
        return calls, lambda: [ids.tensor, p.tensor]
    x, ids = s.buf(d["x"]), s.buf(d["ids"])
    if c["kind"] == "linear":
        w, y = s.experts(d["w"]), s.out(m * c["k"], c["n"])

        def calls():
            ctx.expert_linear(x, ids, m, c["k"], w, y, per_slot=c["per_slot"],
                              activation=c["act"], dtype=dt)
        return calls, lambda: [y.tensor]
    p, r = s.buf(d["p"]), s.buf(d["r"]) if c["residual"] else None
    gate, up, down = s.experts(d["gate"]), s.experts(d["up"]), s.experts(d["down"])
    y = s.out(m, c["h"])

    def calls():
        ctx.expert_mlp(x, ids, p, m, c["k"], gate, up, down, y, residual=r, dtype=dt)
    return calls, lambda: [y.tensor]


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
    c, m, e = case, case["m"], 2 if case["dtype"] == "bf16" else 4
    if c["kind"] == "norm":
        # x, residual and weight in; sum, normed rows, values and scales out
        return {"bytes": m * c["h"] * (4 * e + 1) + m * c["h"] // 8 + c["h"] * e,
                "flops": 10 * m * c["h"]}
    if c["kind"] == "route":
        return {"bytes": m * c["e"] * e + m * c["k"] * 8, "flops": 4 * m * c["e"]}
    # experts that m rows of k of e reach, evenly routed, each read once
    slots = max(1.0, m * c["k"] * (1.0 - c["masked"]))
    met = c["e"] * (1.0 - (1.0 - slots / m / c["e"]) ** m)
    q = lambda n, k: n * k * 34 / 32  # noqa: E731
    if c["kind"] == "linear":
        rows = m * c["k"] if c["per_slot"] else m
        return {"bytes": int(met * q(c["n"], c["cols"]) + rows * c["cols"] * e
                             + m * c["k"] * (c["n"] * e + 4)),
                "flops": int(2 * slots * c["n"] * c["cols"])}
    return {"bytes": int(3 * met * q(c["f"], c["h"]) + m * c["h"] * e * (3 if c["residual"] else 2)
                         + m * c["k"] * 8),
            "flops": int(6 * slots * c["f"] * c["h"])}


def _rnd64(v, dtype):
    """The stored value of a float64 result."""
    return (v.float().to(torch.bfloat16) if dtype == "bf16" else v.float()).double()


def _quantized64(v):
    """Q8_1 of stored rows: the format takes its scale and steps in f32."""
    x = v.float().reshape(v.shape[0], -1, 32)
    d = x.abs().amax(-1, keepdim=True) / 127.0
    inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    return (torch.round(x * inv).double() * d.double()).reshape(v.shape)


def _expert64(x, ids, qd):
    """x [slots, K] by the slots' experts, one expert after another."""
    q, d = qd
    y = torch.zeros(x.shape[0], q.shape[1], dtype=torch.float64, device=x.device)
    for e in range(q.shape[0]):
        at = (ids == e).nonzero()[:, 0]
        if at.numel():
            w = (q[e].double() * d[e].double()[..., None]).flatten(1)
            y[at] = x[at] @ w.t()
    return y


def exact(case, seed):
    c, dt, d = case, case["dtype"], _inputs(case, seed)
    if c["kind"] == "norm":
        s = _rnd64(d["x"].double() + d["r"].double(), dt)
        w = d["w"].double() + (1.0 if c["zero_centered"] else 0.0)
        rstd = 1.0 / torch.sqrt(s.square().mean(-1, keepdim=True) + EPS)
        # the quantizer takes the stored rows: rstd and both products in f32
        stored = _rnd64(_rnd64(_rnd64(s * _rnd64(rstd, "f32"), "f32") * _rnd64(w, "f32"), "f32"), dt)
        return [s, s * rstd * w, _quantized64(stored)]
    if c["kind"] == "route":
        l = d["logits"].double()
        top = l.amax(-1, keepdim=True)
        p = torch.where(l == -math.inf, 0.0, torch.exp(l - torch.where(top == -math.inf, 0.0, top)))
        chosen = torch.sort(l, dim=-1, descending=True, stable=True)[1][:, :c["k"]]
        best = p.gather(1, chosen)
        total = best.sum(-1, keepdim=True) if c["normalize"] else p.sum(-1, keepdim=True)
        return [None, best / torch.where(total == 0, 1.0, total)]
    ids = d["ids"].reshape(-1)
    x = _quantized64(d["x"].double())
    if x.shape[0] != ids.numel():
        x = x[torch.arange(ids.numel(), device=x.device) // c["k"]]
    live = (ids >= 0)[:, None]
    if c["kind"] == "linear":
        y = _expert64(x, ids, d["w"])
        if c["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif c["act"] == "sigmoid":
            y = torch.sigmoid(y)
        elif c["act"] == "softplus":
            y = torch.log1p(torch.exp(y))
        return [torch.where(live, y, 0.0)]
    gate = _expert64(x, ids, d["gate"])
    h = _rnd64(_rnd64(gate * torch.sigmoid(gate), dt) * _rnd64(_expert64(x, ids, d["up"]), dt), dt)
    o = _rnd64(_expert64(_quantized64(h), ids, d["down"]), dt).view(c["m"], c["k"], c["h"])
    y = torch.einsum("mkh,mk->mh", o, d["p"].double())
    return [y + d["r"].double() if c["residual"] else y]
