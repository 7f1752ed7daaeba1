"""The bounds of test_gpu_delta_precision.py let the chunks' formulas in float32 pass
and catch the mistakes they are there for (numpy only)."""
import numpy as np
import pytest

import delta_reference as ref

# the mistakes that each kind of rows has to show
STATE = {"long": ("state", "reset"), "keep": ("state", "reset", "s0", "u"),
         "reset": ("state", "reset", "u", "sums"), "cancel": ("state", "reset", "s0", "u")}
OUTPUT = {"long": ("state", "reset", "o s0"), "keep": ("state", "reset", "o s0", "o u", "o a"),
          "reset": ("state", "sums", "o s0", "o u", "o a"), "cancel": ("o s0", "o u", "o a")}


@pytest.mark.parametrize("key_dim", [64, 128])
@pytest.mark.parametrize("kind", ref.Rows.KINDS)
def test_bounds_catch_mistakes(kind, key_dim):
    r = ref.Rows(np.random.default_rng(1), kind, key_dim)
    args = r.args()
    o, s, _, _ = ref.rows(*args, np.float64)
    o32, s32, _, _ = ref.rows(*args, np.float32)
    most, carried = ref.magnitudes(*args), ref.largest_state(args)

    def shares(plant):
        oc, sc = ref.chunks(*args, plant=plant)
        return ref.share(sc, s, s32, True, carried, r.exps(True)).max(), ref.output_share(ref.bf16(oc), o, most).max()
    clean = shares(None)
    assert clean[0] < 0.7 and clean[1] < 0.95
    for plant in STATE[kind]:
        assert shares(plant)[0] > 1.4, plant
    for plant in OUTPUT[kind]:
        assert shares(plant)[1] > 1.4, plant
    # row after row: float32 is within, a state kept as bf16 is not
    assert ref.share(s32, s, s32, False, carried, r.exps(False)).max() <= 0.5
    assert ref.share(ref.bf16(s32), s, s32, False, carried, r.exps(False)).min() > 8


def test_magnitudes_bound_the_outputs():
    for kind in ref.Rows.KINDS:
        args = ref.Rows(np.random.default_rng(2), kind, 64).args()
        o, _, _, _ = ref.rows(*args, np.float64)
        assert (np.abs(o) <= ref.magnitudes(*args) * (1 + 1e-9)).all()
