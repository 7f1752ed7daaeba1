"""The silu of the experts' bf16 SwiGLU, over every float."""
import pytest

pytestmark = pytest.mark.gpu


def test_silu_rounds_alike_over_all_floats(ctx):
    """The f32 form's values that are taken, each by itself, and the whole
    function round to the bf16 of silu_f32; the exact form is left a small part of
    the range: 35 of 65536 places of a value's low half within |v| < 80, all of
    |v| >= 80 and NaN, and of |v| < 2^-100 but zero."""
    wrong, off, left = ctx.selftest_silu()
    assert wrong == 0
    assert off == 0
    exponents = 254 - (127 - 100) + 1  # of 255 that hold values, those from 2^-100 on
    near = 2 ** 32 * exponents // 256 * 35 // 65536
    outside = 2 * ((0x80000000 - 0x42A00000) + (0x0D800000 - 1))
    assert outside <= left <= outside + 2 * near
