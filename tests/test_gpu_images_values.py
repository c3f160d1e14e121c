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


@pytest.mark.parametrize("M", [1, 4, 5, 8])
@pytest.mark.parametrize("K", [64, 896, 1500])
@pytest.mark.parametrize("bits,above", [(False, 20), (False, 27), (False, 40), (True, 20), (True, 30), (True, 36)])
def test_a_channel_that_stands_out(hm, bits, above, M, K):
    """One channel is 2^above times the others, and the weights there are zero: what the others give does not suffer.

    A row's largest value enters as 2^14 to 2^15.  bf16 rows: one f16 term, exact where a value is at least 2^-31 of the largest, else off by at most half an f16
    subnormal step, 2^-25 of 2^14: 2^-39 of it.  f32 rows: the second term is what the first leaves, 2^12 times, in f16: 2^-22 of a value, or 2^-25 of 2^26: 2^-51 of
    the largest.  Two MMAs per block of 32 values to 4 * 2^-23 of the sum of magnitudes; ceil(K / 32) blocks, the halves and at most eight parts are added to nearest,
    2^-24 each."""
    rng = np.random.default_rng(M + K + above)
    N = 130
    x = (rng.uniform(0.5, 1.0, (M, K)) * np.where(rng.random((M, K)) < 0.5, -1, 1)).astype(np.float32)
    x[:, 5] = 2.0**above
    if bits:
        x = ic.bf16_value(ic.bf16_bits(x))
    codes, scales = rng.integers(0, 16, (N, -(-K // 32) * 32), dtype=np.uint8), rng.integers(110, 125, (N, -(-K // 32)), dtype=np.uint8)
    codes[:, K:] = 0
    codes[:, 5] = 0
    w = ic.mx_values(codes, scales, K)
    wide = x.astype(np.float64)
    want, size = wide @ w.T, np.abs(wide) @ np.abs(w).T
    got = hm.gemv_mx4(ic.bf16_bits(x) if bits else x, ic.mx_image(codes, scales, K), N).astype(np.float64)
    units = 4 + (0 if bits else 2) + (-(-K // 32) + 2 + 8) / 2
    floor = 2.0**-39 * (above > 30) if bits else 2.0**-51
    limit = units * 2.0**-23 * size + floor * 2.0**above * np.abs(w).sum(1)
    assert (np.abs(got - want) <= limit).all(), float((np.abs(got - want) / limit).max())
