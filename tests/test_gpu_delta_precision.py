"""What the delta rule's kernels keep of their states and outputs, over hundreds of
rows whose carried state matters: root mean square errors next to those of the
same rule in float32, outputs of bf16 next to the magnitudes they are summed
from.  test_delta_bounds.py shows what the bounds catch."""
import numpy as np
import pytest

import delta_reference as ref

pytestmark = pytest.mark.gpu

F32 = np.float32


def call(q8, ctx, oracle, r, dtype, pieces):
    """(o, last state): the rows in `pieces` calls that hand the state on."""
    narrow = oracle.f32_to_bf16_bits if dtype == "bf16" else (lambda x: x)
    d = [ctx.to_device(narrow(x)) for x in (r.q, r.k, r.v)] + [ctx.to_device(x) for x in (r.decay, r.beta)]
    state = ctx.to_device(r.state[None])
    size = 2 if dtype == "bf16" else 4
    y = ctx.to_device(np.zeros((r.n, r.vh, r.vd), np.uint16 if dtype == "bf16" else F32))
    cuts = np.linspace(0, r.n, pieces + 1).astype(int)
    wide = [r.kh * r.kd * size, r.kh * r.kd * size, r.vh * r.vd * size, r.vh * 4, r.vh * 4]
    for a, b in zip(cuts, cuts[1:]):
        ctx.delta_rule(*(x.ptr + int(a) * w for x, w in zip(d, wide)), y.ptr + int(a) * r.vh * r.vd * size,
                       int(b - a), r.kh, r.vh, r.kd, r.vd, state=state, new_state=state, scale=r.scale,
                       eps=r.eps, dtype=dtype)
    got = ctx.to_host(y, (r.n, r.vh, r.vd), np.uint16 if dtype == "bf16" else F32)
    return (oracle.bf16_bits_to_f32(got) if dtype == "bf16" else got), ctx.to_host(state, r.state.shape, F32)


# chunks from 10 rows on of bf16, else row after row; several calls of each
FORMS = {"chunks": ("bf16", 1), "chunks, three calls": ("bf16", 3), "rows": ("bf16", 60), "f32": ("f32", 1)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("key_dim", [64, 128])
@pytest.mark.parametrize("kind", ref.Rows.KINDS)
def test_precision(q8, ctx, oracle, kind, key_dim, form):
    if ctx.platform != "aarch64":
        pytest.skip("the same kernels on either platform")
    dtype, pieces = FORMS[form]
    chunked = form.startswith("chunks")
    r = ref.Rows(np.random.default_rng(1), kind, key_dim)
    o, s, _, _ = ref.rows(*r.args(), np.float64)
    o32, s32, _, _ = ref.rows(*r.args(), F32)
    got, after = call(q8, ctx, oracle, r, dtype, pieces)
    # (a call's last chunk may be a short one: one more exponential per call)
    exps = r.exps(chunked) + (pieces if chunked and r.exps(True) else 0)
    worst = float(ref.share(after, s, s32, chunked, ref.largest_state(r.args()), exps).max())
    assert worst <= 1
    most = ref.magnitudes(*r.args())
    if dtype == "bf16":
        worst = float(ref.output_share(got, o, most).max())
    else:
        got, o, o32, most = (x.swapaxes(0, 1) for x in (got, o, o32, most))
        worst = float(ref.share(got, o, o32, chunked, ref.rms(most), exps).max())
    assert worst <= 1
