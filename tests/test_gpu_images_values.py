"""Values that image calls meet at the ends of their ranges."""
import numpy as np
import pytest

import image_cases as ic

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [False, True])
def test_gates_far_below_zero(hm, bits):
    """silu(g) u for gates down to -104 with large u: e^g is down to the smallest f32 there, and the result is an ordinary number.

    In f32: e^-|g| and the quotient to 2 units of 2^-23 (of 2^-149 below 2^-126), two products and a sum to 2^-24 each: below 8 * 2^-23 of the result
    and 3 * 2^-149 |g u| together.  Then a rounding to bf16: 2^-8."""
    rng = np.random.default_rng(3)
    rows, K = 6, 420
    gate = np.concatenate([np.linspace(-104, -80, 300), np.linspace(-80, 100, 100), [0.0, -0.0, -87.3, -87.4, -88.0, -88.5, -88.7, -88.72, -88.73, -88.8, -103.9, 88.0, 88.8, 99.0, 1e-30, -1e-30, 1e-3, -1e-3, 30.0, -30.0]])
    g = np.tile(gate, (rows, 1))
    u = rng.standard_normal((rows, K)) * 2.0 ** np.array([0, 20, 60, 100, 110, -20])[:, None]
    x = np.concatenate([g, u], 1).astype(np.float32)
    if bits:
        x = ic.bf16_value(ic.bf16_bits(x))
    g, u = x[:, :K].astype(np.float64), x[:, K:].astype(np.float64)
    want = g / (1 + np.exp(-g)) * u
    got = hm.image_unpack(hm.image_pack(ic.bf16_bits(x) if bits else x, hm.DType.BF16, glu=True), hm.DType.BF16, K, rows)
    limit = (2.0**-8 + 8 * 2.0**-23) * np.abs(want) + 3 * 2.0**-149 * np.abs(g * u) * (1 + 2.0**-8) + 2.0**-134
    err = np.abs(got - want)
    assert (err <= limit).all(), (g[err > limit][:5], got[err > limit][:5], want[err > limit][:5])
