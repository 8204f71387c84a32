"""The "ramp" blend of ``ops.rope_inv_freq`` against its definition, written out component by
component in Python floats: one rounding per operation on both sides, 1e-12 relative."""

import math

import pytest


def ramp(rotary_dim, base, factor, context, slow, fast):
    """Components up to the one that makes `fast` turns over the context are kept, those from
    the one that makes `slow` turns on are divided, linear in the index between; the two
    indices are rounded outwards and limited to 0 .. rotary_dim - 1."""
    def index_of(turns):
        return rotary_dim * math.log(context / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    lo = max(math.floor(index_of(fast)), 0)
    hi = min(math.ceil(index_of(slow)), rotary_dim - 1)
    out = []
    for i in range(rotary_dim // 2):
        f = base ** (-2.0 * i / rotary_dim)
        away = 0.0 if i <= lo else 1.0 if i >= hi else (i - lo) / (hi - lo)
        out.append(f * (1.0 - away) + f / factor * away)
    return out


@pytest.mark.parametrize("rotary_dim,base,factor,context,slow,fast", [
    (64, 10000.0, 4.0, 4096, 1.0, 32.0),       # both indices inside
    (128, 10000.0, 4.0, 131072, 1.0, 32.0),    # 45 and 70 of 64 components
    (64, 10000.0, 8.0, 65537, 1.0, 16.0),
    (128, 500000.0, 16.0, 8192, 1.0, 32.0),
    (20, 100.0, 3.0, 1 << 20, 2.0, 7.0),       # every component turns often: all kept
    (2, 10000.0, 4.0, 131072, 1.0, 32.0),
    (96, 10000.0, 40.0, 1 << 17, 0.5, 64.0),
])
def test_ramp(rotary_dim, base, factor, context, slow, fast):
    from evograd_b200 import ops

    got, mscale = ops.rope_inv_freq(rotary_dim, base, scaling="ramp", factor=factor, original_context=context,
                                    slow=slow, fast=fast)
    want = ramp(rotary_dim, base, factor, context, slow, fast)
    assert mscale == 0.1 * math.log(factor) + 1.0
    for i, (a, b) in enumerate(zip(got.tolist(), want)):
        assert math.isclose(a, b, rel_tol=1e-12), (i, a, b)


def test_ramp_beyond_the_last_component():
    """Base 10000 over 128 columns and a context of 131072: the last component makes 2.4 turns
    and lies at 18 / 25 of the ramp from index 45 to index 70."""
    from evograd_b200 import ops

    f = ops.rope_inv_freq(128, 10000.0, scaling="ramp", factor=4.0, original_context=131072, slow=1.0, fast=32.0)[0]
    plain = ops.rope_inv_freq(128, 10000.0)[0]
    assert 131072 * float(plain[-1]) / (2.0 * math.pi) > 2.4
    assert math.isclose(float(f[-1] / plain[-1]), 1.0 - 18.0 / 25.0 * 0.75, rel_tol=1e-12)
