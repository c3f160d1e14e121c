"""Operand images on a B200: packing is compared bit for bit, products with 64-bit results of the same operands.

Tolerances of products, per element, with S = sum_k |x_k w_k|:
  * products of two 4-bit values, or of two bf16, are exact in f32; an MMA's sum and its addition to the accumulator each truncate by at
    most 2^-23 of a magnitude of at most S, and an accumulator takes at most 32 MMAs: 64 * 2^-23 S; accumulators and cluster parts (at most 70 + 16
    here) are added to nearest, 2^-24 S each: 43 * 2^-23 S.  Together below 128 * 2^-23 S.
  * few rows: x as two f16 terms, 2^-22 of a value and 2^-32 of the row's largest (bf16 rows: the latter only); two MMAs per block, 4 * 2^-23 S; blocks, halves and
    cluster parts (at most 280 + 16) added to nearest in f32, 2^-24 S each: below 160 * 2^-23 S.
  * a bf16 result: 2^-8 of the value more.
"""
import numpy as np
import pytest

import image_cases as ic
from conftest import record_error

pytestmark = pytest.mark.gpu

TYPES = {"mxfp4": 10, "bf16": 1}


def close(got, want, size, units, what):
    """|got - want| <= units * 2^-23 * size (+ 2^-8 |want| where got is bf16 bits)."""
    bits = got.dtype == np.uint16
    g = (ic.bf16_value(got) if bits else got).astype(np.float64)
    limit = units * 2.0**-23 * size + (2.0**-8 * np.abs(want) if bits else 0.0) + 1e-37
    err = np.abs(g - want)
    assert np.isfinite(g).all()
    worst = float((err / limit).max())
    record_error(what + (" bf16" if bits else ""), float(err.max()), float(np.abs(want).max() + 1e-30))
    assert worst <= 1.0, worst


@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (3, 31), (2, 33), (129, 256), (5, 257), (130, 896), (7, 1000), (33, 8960), (300, 40)])
@pytest.mark.parametrize("bits", [False, True])
def test_pack_mx_bit_for_bit(hm, rows, K, bits):
    rng = np.random.default_rng(rows * 1000 + K)
    x = ic.activations(rng, rows, K)
    x[0, : min(K, 40)] = 0.0  # a block of zeros
    x[rows - 1] *= np.float32(2.0**-130)  # below the scales' range, subnormal
    if bits:
        x = ic.bf16_value(ic.bf16_bits(x))
    codes, scales = ic.mx_quantise(x)
    image = hm.image_pack(ic.bf16_bits(x) if bits else x, hm.DType.MXFP4)
    np.testing.assert_array_equal(image, ic.mx_image(codes, scales, K))
    np.testing.assert_array_equal(hm.image_unpack(image, hm.DType.MXFP4, K, rows), ic.mx_values(codes, scales, K).astype(np.float32))
    np.testing.assert_array_equal(hm.image_unpack(image, hm.DType.MXFP4, K, rows, out_dtype=hm.DType.BF16), ic.bf16_bits(ic.mx_values(codes, scales, K)))


def test_pack_mx_ties_saturation_and_no_numbers(hm):
    # every tie and both sides of it, scaled so that the block's exponent is known (6 is its largest value)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    v = np.concatenate([[6.0], ties, np.nextafter(ties, np.float32(9)), np.nextafter(ties, np.float32(0)), -ties]).astype(np.float32)
    x = np.zeros((8, 32 * 3), np.float32)
    for r in range(8):
        x[r, : v.size] = v * np.float32(2.0 ** (r * 30 - 110))
    x[1, 32:40] = [7.99, -7.5, 4, 6.5, 5.5, -8e-3, 7, 0.1]  # beyond 6: saturated
    x[2, 40] = np.inf
    x[3, 33] = np.nan
    x[4, 64] = -np.inf
    x[5, 64:] = np.float32(3.4e38)
    x[6, 64:] = np.float32(1e-45)
    codes, scales = ic.mx_quantise(x)
    image = hm.image_pack(x, hm.DType.MXFP4)
    np.testing.assert_array_equal(image, ic.mx_image(codes, scales, x.shape[1]))
    got = hm.image_unpack(image, hm.DType.MXFP4, x.shape[1], 8)
    np.testing.assert_array_equal(got, ic.mx_values(codes, scales).astype(np.float32))
    assert np.isnan(got[2, 32:64]).all() and np.isnan(got[3, 32:64]).all() and np.isfinite(got[3, :32]).all()


@pytest.mark.parametrize("rows,K", [(1, 1), (3, 63), (129, 64), (5, 65), (40, 1001)])
def test_pack_bf16_is_the_tensor_core_layout(hm, rows, K):
    rng = np.random.default_rng(K)
    x = rng.standard_normal((rows, K)).astype(np.float32)
    image = hm.image_pack(x, hm.DType.BF16)
    np.testing.assert_array_equal(image.view(np.uint16), hm.pack_bf16_tc(ic.bf16_bits(x).T))
    np.testing.assert_array_equal(hm.image_unpack(image, hm.DType.BF16, K, rows), ic.bf16_value(ic.bf16_bits(x)))


@pytest.mark.parametrize("rows,K", [(1, 32), (130, 64), (3, 896)])
def test_gguf_blocks(hm, rows, K):
    rng = np.random.default_rng(rows + K)
    codes, scales = rng.integers(0, 16, (rows, K), dtype=np.uint8), rng.integers(0, 256, (rows, K // 32), dtype=np.uint8)
    image = hm.image_from_blocks(ic.gguf_blocks(codes, scales), K)
    np.testing.assert_array_equal(image, ic.mx_image(codes, scales, K))
    scales = np.minimum(scales, 250)  # values of f32
    image = hm.image_from_blocks(ic.gguf_blocks(codes, scales), K)
    np.testing.assert_array_equal(hm.image_unpack(image, hm.DType.MXFP4, K, rows), ic.mx_values(codes, scales).astype(np.float32))


def test_gated_pack(hm):
    rng = np.random.default_rng(4)
    for K in (64, 100):
        x = rng.standard_normal((9, 2 * K)).astype(np.float32) * 2
        g, u = x[:, :K].astype(np.float64), x[:, K:].astype(np.float64)
        want = g / (1 + np.exp(-g)) * u
        got = hm.image_unpack(hm.image_pack(x, hm.DType.BF16, glu=True), hm.DType.BF16, K, 9)
        # expf and the division: a few units of 2^-23; then a rounding to bf16
        assert (np.abs(got - want) <= (2.0**-8 + 8 * 2.0**-23) * np.abs(want)).all()
        # 4 bits: within half a step of the largest step (a value at a border may go either way)
        got = hm.image_unpack(hm.image_pack(x, hm.DType.MXFP4, glu=True), hm.DType.MXFP4, K, 9)
        pad = np.zeros((9, -K % 32 + K))
        pad[:, :K] = np.abs(want)
        top = np.repeat(pad.reshape(9, -1, 32).max(-1), 32, axis=1)[:, :K]
        # the largest value saturates by at most a quarter; all others are half a step off, at most a sixth of it where the step is 2 (values above 4)
        assert (np.abs(got - want) <= 0.2501 * top).all()


@pytest.mark.parametrize("dtype", ["mxfp4", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1, 32, 1), (1, 896, 130), (5, 64, 128), (16, 256, 127), (17, 288, 129), (64, 2240, 384), (127, 512, 64), (128, 96, 100), (129, 320, 256),
                                   (191, 160, 40), (192, 544, 200), (193, 1000, 300), (320, 1536, 1100), (385, 2400, 257), (1000, 896, 128), (64, 8960, 150)])
def test_products(hm, dtype, M, K, N):
    rng = np.random.default_rng(M * 7 + K * 3 + N)
    x, w = ic.activations(rng, M, K), (rng.standard_normal((N, K)) * 0.02).astype(np.float32)
    d = hm.DType(TYPES[dtype])
    xi, wi = hm.image_pack(x, d), hm.image_pack(w, d)
    xr, wr = ic.rounded(x, dtype), ic.rounded(w, dtype)
    want, size = xr @ wr.T, np.abs(xr) @ np.abs(wr).T
    got = hm.gemm_image(xi, wi, N, d, K, M)
    close(got, want, size, 128, "image product " + dtype)
    close(hm.gemm_image(xi, wi, N, d, K, M, y_dtype=hm.DType.BF16), want, size, 128, "image product " + dtype)
    np.testing.assert_array_equal(got, hm.gemm_image(xi, wi, N, d, K, M))


def test_product_of_no_numbers(hm):
    """A block without a number makes its row's results no numbers, and nobody else's."""
    rng = np.random.default_rng(11)
    x, w = rng.standard_normal((20, 512)).astype(np.float32), rng.standard_normal((140, 512)).astype(np.float32)
    x[3, 300], w[130, 5] = np.nan, np.inf
    got = hm.gemm_image(hm.image_pack(x, hm.DType.MXFP4), hm.image_pack(w, hm.DType.MXFP4), 140, hm.DType.MXFP4, 512, 20)
    bad = np.zeros((20, 140), bool)
    bad[3], bad[:, 130] = True, True
    np.testing.assert_array_equal(np.isnan(got), bad)
    got = hm.gemv_mx4(x[:8], hm.image_pack(w, hm.DType.MXFP4), 140)
    assert np.isnan(got[3]).all() and np.isnan(got[:, 130]).all() and np.isfinite(np.delete(np.delete(got, 3, 0), 130, 1)).all()


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 32, 1), (1, 896, 9728), (2, 64, 130), (3, 1000, 128), (4, 4864, 896), (5, 288, 129), (7, 1536, 20000), (8, 8960, 1536), (8, 32768, 140), (6, 1, 5), (1, 255, 40000)])
def test_few_rows(hm, bits, M, K, N):
    rng = np.random.default_rng(M + K * 3 + N)
    x = ic.activations(rng, M, K)
    x[M - 1] = np.where(np.arange(K) % 3 == 0, x[M - 1] * 1e-3, x[M - 1])
    if bits:
        x = ic.bf16_value(ic.bf16_bits(x))
    codes, scales = rng.integers(0, 16, (N, -(-K // 32) * 32), dtype=np.uint8), rng.integers(110, 125, (N, -(-K // 32)), dtype=np.uint8)
    codes[:, K:] = 0
    wi, w = ic.mx_image(codes, scales, K) if N < 2000 else hm.image_from_blocks(ic.gguf_blocks(codes, scales), codes.shape[1]), ic.mx_values(codes, scales, K)
    want, size = x.astype(np.float64) @ w.T, np.abs(x).astype(np.float64) @ np.abs(w).T
    size = size + 2.0**-32 * 2.0**23 / 160 * np.abs(x).max(1, keepdims=True) * np.abs(w).sum(1)
    arg = ic.bf16_bits(x) if bits else x
    got = hm.gemv_mx4(arg, wi, N)
    close(got, want, size, 160, "few rows x 4 bits")
    close(hm.gemv_mx4(arg, wi, N, y_dtype=hm.DType.BF16), want, size, 160, "few rows x 4 bits")
    np.testing.assert_array_equal(got, hm.gemv_mx4(arg, wi, N))


def test_few_rows_with_infinities(hm):
    x = np.ones((2, 64), np.float32)
    x[0, 10] = np.inf
    codes, scales = np.full((3, 64), 2, np.uint8), np.full((3, 2), 127, np.uint8)
    codes[1, 10], codes[2, 10] = 10, 0  # minus one, zero
    got = hm.gemv_mx4(x, ic.mx_image(codes, scales, 64), 3)
    assert got[0, 0] == np.inf and got[0, 1] == -np.inf and np.isnan(got[0, 2])
    np.testing.assert_array_equal(got[1], [64, 62, 63])


def test_few_rows_at_the_ends_of_the_scales(hm):
    """Scales 2^-127 (no normal f32), 2^-126 and 2^100, rows of 2^100 and 2^-90: results from 2^-217 (zero in f32) to beyond its largest."""
    rng = np.random.default_rng(21)
    K, N = 320, 12
    x = rng.standard_normal((4, K)).astype(np.float32)
    x[1] *= np.float32(2.0**100)
    x[2] *= np.float32(2.0**-90)
    x[3] = 0.0
    codes, scales = rng.integers(0, 16, (N, K), dtype=np.uint8), np.tile(np.array([0, 1, 127, 227], np.uint8)[:, None], (3, K // 32))
    w = ic.mx_values(codes, scales)
    got = hm.gemv_mx4(x, ic.mx_image(codes, scales, K), N).astype(np.float64)
    want, size = x.astype(np.float64) @ w.T, np.abs(x).astype(np.float64) @ np.abs(w).T
    beyond = np.abs(want) > 3.5e38
    assert beyond.any() and (got[beyond] == np.sign(want[beyond]) * np.inf).all()
    # the bound of the head of this file; sums of scaled rows below 2^-126 lose up to 2^-149 per addition, and the row's scale (2^-100 at least) is taken back: 2^-40 of
    # the largest x times the smallest w covers it; results below 2^-126 are rounded to 2^-149
    slack = 2.0**-40 * np.abs(x).max(1, keepdims=True).astype(np.float64) * 2.0**-127 * K + 2.0**-149
    limit = 160 * 2.0**-23 * size + 2.0**-32 * np.abs(x).max(1, keepdims=True) * np.abs(w).sum(1) + slack
    assert (np.abs(got - want)[~beyond] <= limit[~beyond]).all()
    assert (got[3] == 0).all()


@pytest.mark.parametrize("dtype", ["mxfp4", "bf16"])
def test_nobody_has_an_expert(hm, dtype):
    T, top, E, K, N = 9, 2, 4, 64, 40
    d, ids = hm.DType(TYPES[dtype]), np.full((T, top), -1, np.int32)
    ids[3, 0] = E  # one beyond the last
    plan = hm.expert_plan(ids, E)
    np.testing.assert_array_equal(plan, np.concatenate(ic.plan(np.where(ids < E, ids, -1), E)))
    x, w = np.ones((T, K), np.float32), np.ones((N, K), np.float32)
    images = np.concatenate([hm.image_pack(w, d)] * E)
    y = hm.expert_gemm(hm.image_pack(x, d, plan=plan, experts=E, top=top), images, plan, N, d, T * top, E, K, y=np.full((T * top, N), 5.0, np.float32))
    assert (y == 5.0).all()
    if dtype == "mxfp4":
        assert (hm.expert_gemv(x, images, ids, N, top, E, y=np.full((T * top, N), 5.0, np.float32)) == 5.0).all()
    np.testing.assert_array_equal(hm.expert_sum(y, ids, np.ones((T, top), np.float32), top, E, resid=np.full((T, N), 2.0, np.float32)), np.full((T, N), 2.0))


def routing(rng, tokens, top, experts, none):
    ids = np.stack([rng.permutation(experts + none)[:top] for _ in range(tokens)]) if tokens else np.zeros((0, top), int)
    return np.where(ids < experts, ids, -1).astype(np.int32)


@pytest.mark.parametrize("tokens,top,experts,none", [(0, 2, 8, 0), (1, 1, 1, 0), (1, 4, 16, 0), (5, 2, 8, 2), (64, 8, 32, 2), (517, 4, 16, 0), (300, 1, 1, 1), (129, 6, 1024, 0), (4000, 8, 64, 3)])
def test_plan(hm, tokens, top, experts, none):
    ids = routing(np.random.default_rng(tokens + experts), tokens, top, experts, none)
    got = hm.expert_plan(ids, experts)
    np.testing.assert_array_equal(got, np.concatenate(ic.plan(ids, experts)))
    if tokens > 3:  # ids that are no experts' at all
        ids[1, 0], ids[3, 0] = experts + 7, -2147483648
        np.testing.assert_array_equal(hm.expert_plan(ids, experts), np.concatenate(ic.plan(ids, experts)))


@pytest.mark.parametrize("dtype", ["mxfp4", "bf16"])
@pytest.mark.parametrize("tokens,top,experts,none,K,N", [(1, 1, 1, 0, 32, 1), (1, 4, 16, 0, 896, 130), (5, 2, 8, 2, 320, 128), (64, 8, 32, 2, 288, 200), (517, 4, 8, 0, 160, 129), (700, 1, 2, 1, 1000, 70)])
def test_grouped_products(hm, dtype, tokens, top, experts, none, K, N):
    rng = np.random.default_rng(tokens + K + N)
    ids = routing(rng, tokens, top, experts, none)
    if tokens == 700:
        ids[:690] = 1  # one expert has nearly all rows
    x, w = ic.activations(rng, tokens, K), (rng.standard_normal((experts, N, K)) * 0.02).astype(np.float32)
    d, pairs = hm.DType(TYPES[dtype]), tokens * top
    plan = hm.expert_plan(ids, experts)
    xi = hm.image_pack(x, d, plan=plan, experts=experts, top=top)
    wi = np.concatenate([hm.image_pack(w[e], d) for e in range(experts)])
    xr, wr, flat = ic.rounded(x, dtype), ic.rounded(w.reshape(-1, K), dtype).reshape(w.shape), ids.reshape(-1)
    real = flat >= 0
    want, size = np.zeros((pairs, N)), np.zeros((pairs, N))
    for p in np.flatnonzero(real):
        want[p], size[p] = wr[flat[p]] @ xr[p // top], np.abs(wr[flat[p]]) @ np.abs(xr[p // top])
    before = np.full((pairs, N), 7.0, np.float32)
    got = hm.expert_gemm(xi, wi, plan, N, d, pairs, experts, K, y=before.copy())
    close(got[real], want[real], size[real], 128, "grouped product " + dtype)
    assert (got[~real] == 7.0).all()
    close(hm.expert_gemm(xi, wi, plan, N, d, pairs, experts, K, y_dtype=hm.DType.BF16)[real], want[real], size[real], 128, "grouped product " + dtype)
    np.testing.assert_array_equal(got, hm.expert_gemm(xi, wi, plan, N, d, pairs, experts, K, y=before.copy()))


@pytest.mark.parametrize("tokens,top,experts,none,K,N", [(1, 4, 16, 0, 896, 390), (3, 2, 8, 2, 64, 130), (2, 8, 32, 0, 1536, 129), (9, 1, 3, 1, 1000, 40)])
def test_pairs_without_a_plan(hm, tokens, top, experts, none, K, N):
    rng = np.random.default_rng(tokens + K)
    ids = routing(rng, tokens, top, experts, none)
    x, w = ic.activations(rng, tokens, K), (rng.standard_normal((experts, N, K)) * 0.02).astype(np.float32)
    wi = np.concatenate([hm.image_pack(w[e], hm.DType.MXFP4) for e in range(experts)])
    wr, flat = ic.mx_round(w.reshape(-1, K)).reshape(w.shape), ids.reshape(-1)
    got = hm.expert_gemv(x, wi, ids, N, top, experts, y=np.full((tokens * top, N), 3.0, np.float32))
    for p, e in enumerate(flat):
        if e < 0:
            assert (got[p] == 3.0).all()
        else:
            xp = x[p // top].astype(np.float64)
            close(got[p], wr[e] @ xp, np.abs(wr[e]) @ np.abs(xp) + 2.0**-9 / 160 * np.abs(xp).max() * np.abs(wr[e]).sum(1), 160, "pairs x 4 bits")


@pytest.mark.parametrize("bits,out,W,resid", [(False, 0, 37, True), (True, 1, 1536, True), (False, 1, 896, False), (True, 0, 6, False)])
def test_weighted_sum(hm, bits, out, W, resid):
    rng = np.random.default_rng(W)
    tokens, top, experts = 21, 4, 9
    ids = routing(rng, tokens, top, experts, 2)
    rows, wt, x = rng.standard_normal((tokens * top, W)).astype(np.float32), rng.random((tokens, top)).astype(np.float32), rng.standard_normal((tokens, W)).astype(np.float32)
    rows[(ids < 0).reshape(-1)] = np.nan  # rows nobody wrote
    if bits:
        rows = ic.bf16_value(ic.bf16_bits(rows))
    got = hm.expert_sum(ic.bf16_bits(rows) if bits else rows, ids, wt, top, experts, resid=x if resid else None, y_dtype=hm.DType(out))
    terms = np.where(ids[..., None] >= 0, wt[..., None].astype(np.float64) * np.nan_to_num(rows.reshape(tokens, top, W).astype(np.float64)), 0.0)
    want = terms.sum(1) + (x if resid else 0.0)
    size = np.abs(terms).sum(1) + (np.abs(x) if resid else 0.0)
    close(got, want, size, 3, "weighted sum")  # five additions, 2^-24 each


@pytest.mark.parametrize("dtype", ["mxfp4", "bf16"])
@pytest.mark.parametrize("tokens", [3, 150])
def test_feed_forward_of_a_mixture(hm, dtype, tokens):
    """Router, plan, gate and up, gated activations, down, weighted sum: as they are used together.  Between the two products the activations are rounded, and a
    value next to a border may go either way: each stage is held to 64-bit results of its own input."""
    rng = np.random.default_rng(tokens)
    W, ff, experts, top = 320, 96, 8, 2
    y, x0, nw = rng.standard_normal((tokens, W)).astype(np.float32), rng.standard_normal((tokens, W)).astype(np.float32), np.ones(W, np.float32)
    router = ic.bf16_bits(rng.standard_normal((experts + 1, W)) * 0.1)
    x, ids, wts, _ = hm.post_norm_route(y, x0, nw, 0.25, 1e-6, router=router, correction=np.zeros(experts + 1, np.float32), experts=experts, top=top)
    assert (ids < 0).any() or tokens < 10
    gu, down = (rng.standard_normal((experts, 2 * ff, W)) * 0.05).astype(np.float32), (rng.standard_normal((experts, W, ff)) * 0.05).astype(np.float32)
    d, pairs, flat = hm.DType(TYPES[dtype]), tokens * top, ids.reshape(-1)
    images = lambda w: np.concatenate([hm.image_pack(w[e], d) for e in range(experts)])
    plan = hm.expert_plan(ids, experts)
    h = hm.expert_gemm(hm.image_pack(x, d, plan=plan, experts=experts, top=top), images(gu), plan, 2 * ff, d, pairs, experts, W)
    act = hm.image_pack(h, d, plan=plan, experts=experts, glu=True)
    rows = hm.expert_gemm(act, images(down), plan, W, d, pairs, experts, ff)
    out = hm.expert_sum(rows, ids, wts, top, experts, resid=x)
    xr, guw, dw = ic.rounded(x, dtype), ic.rounded(gu.reshape(-1, W), dtype).reshape(gu.shape), ic.rounded(down.reshape(-1, ff), dtype).reshape(down.shape)
    place, held = hm.expert_plan(ids, experts)[2 * experts + 1 : 2 * experts + 1 + pairs], hm.image_unpack(act, d, ff, hm.expert_plan_rows(pairs, experts)).astype(np.float64)
    for p, e in enumerate(flat):
        if e < 0:
            assert place[p] == -1
            continue
        close(h[p], guw[e] @ xr[p // top], np.abs(guw[e]) @ np.abs(xr[p // top]), 128, "feed-forward gate and up")
        a = held[place[p]]
        gate, up = h[p, :ff].astype(np.float64), h[p, ff:].astype(np.float64)
        exact = gate / (1 + np.exp(-gate)) * up
        top_of = np.repeat(np.abs(exact).reshape(-1, 32).max(-1), 32) if dtype == "mxfp4" else np.abs(exact)
        assert (np.abs(a - exact) <= (0.2501 if dtype == "mxfp4" else 2.0**-8 * 1.001) * top_of).all()
        close(rows[p], dw[e] @ a, np.abs(dw[e]) @ np.abs(a), 128, "feed-forward down")
    terms = np.where(ids[..., None] >= 0, wts[..., None].astype(np.float64) * rows.reshape(tokens, top, W), 0.0)
    close(out, x + terms.sum(1), np.abs(x) + np.abs(terms).sum(1), 3, "feed-forward sum")
