"""Forms of the image calls at sizes where a CTA or a warp has several pieces of work: products of many units, packs of three k-blocks per warp, gated rows of either type,
pairs with bf16 rows and results, sums of more tokens than a grid's second dimension, and a mixture with identity experts.

Images are compared bit for bit with the format restated over all rows at once; products with 64-bit results, to the tolerances derived in test_gpu_images.py."""
import numpy as np
import pytest

import image_cases as ic
from test_gpu_images import close, routing

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, BF16, MX = 0, 1, 10
TYPES = {F32: torch.float32, BF16: torch.bfloat16}
NAMES = {MX: "mxfp4", BF16: "bf16"}


def stream():
    return torch.cuda.current_stream().cuda_stream


def tiles(pieces, dtype):
    """[rows, k-blocks, 8, 16] bytes -> [blocks, k-blocks, 128 rows, 128] with the pieces of row r at piece ^ (r & 7)."""
    rows, kb = pieces.shape[:2]
    full = np.zeros((-(-rows // 128) * 128, kb, 8, 16), np.uint8)
    r = np.arange(rows)
    full[r[:, None], :, np.arange(8)[None] ^ (r[:, None] & 7)] = pieces.transpose(0, 2, 1, 3)
    return full.reshape(-1, 128, kb, 128).transpose(0, 2, 1, 3)


def image_restated(x, dtype):
    rows, K = x.shape
    if dtype == BF16:
        kb = -(-K // 64)
        v = np.zeros((rows, kb * 64), np.uint16)
        v[:, :K] = ic.bf16_bits(x)
        return np.ascontiguousarray(tiles(v.view(np.uint8).reshape(rows, kb, 8, 16), dtype)).reshape(-1)
    kb = -(-K // 256)
    codes, scales = ic.mx_quantise(x)
    c, s = np.zeros((rows, kb * 256), np.uint8), np.zeros((-(-rows // 128) * 128, kb, 8), np.uint8)
    c[:, : codes.shape[1]] = codes
    s[:rows].reshape(rows, -1)[:, : scales.shape[1]] = scales
    body = tiles((c[:, 0::2] | c[:, 1::2] << 4).reshape(rows, kb, 8, 16), dtype)
    # scale of row r, block b of a k-block: half b / 4, then r % 32, r / 32, b % 4
    head = s.reshape(-1, 4, 32, kb, 2, 4).transpose(0, 3, 4, 2, 1, 5)
    return np.concatenate([head.reshape(*head.shape[:2], 1024), body.reshape(*body.shape[:2], 16384)], -1).reshape(-1)


def test_the_restatement_over_all_rows():
    rng = np.random.default_rng(0)
    for rows, K in [(1, 1), (130, 300), (257, 512)]:
        x = ic.activations(rng, rows, K)
        np.testing.assert_array_equal(image_restated(x, MX), ic.mx_image(*ic.mx_quantise(x), K))


# ---- three k-blocks per warp (18944 k-blocks of rows and more) ------------------------------------


@pytest.mark.parametrize("dtype,rows,K", [(MX, 600, 8960), (MX, 2200, 2304), (MX, 2400, 2100), (MX, 1999, 2560), (BF16, 2200, 576), (BF16, 2000, 640), (BF16, 1800, 700), (BF16, 601, 2113)])
@pytest.mark.parametrize("bits", [False, True])
def test_pack_and_unpack_of_many_rows(hm, dtype, rows, K, bits):
    d = hm.DType(dtype)
    x = ic.activations(np.random.default_rng(rows + K), rows, K)
    x[5, 3], x[rows - 1, K - 1] = np.nan, np.inf
    if bits:
        x = ic.bf16_value(ic.bf16_bits(x))
    assert rows * -(-K // (256 if dtype == MX else 64)) >= 18944
    image = hm.image_pack(ic.bf16_bits(x) if bits else x, d)
    want = image_restated(x, dtype)
    if dtype == BF16:  # (which of its NaNs a bf16 is, nobody says)
        a, b = ic.bf16_value(image.view(np.uint16)), ic.bf16_value(want.view(np.uint16))
        np.testing.assert_array_equal(a, b)
    else:
        np.testing.assert_array_equal(image, want)
    values = ic.rounded(x, NAMES[dtype])
    np.testing.assert_array_equal(hm.image_unpack(image, d, K, rows), values.astype(np.float32))
    got = hm.image_unpack(image, d, K, rows, out_dtype=hm.DType.BF16)
    np.testing.assert_array_equal(ic.bf16_value(got), ic.bf16_value(ic.bf16_bits(values.astype(np.float32))))


@pytest.mark.parametrize("dtype,rows,K", [(MX, 6400, 520), (MX, 6400, 700), (BF16, 2200, 576), (BF16, 2200, 650)])
@pytest.mark.parametrize("xt", [F32, BF16])
def test_grouped_pack_of_many_rows_and_choices(hm, dtype, rows, K, xt):
    """40 choices of 64 experts: a row's places fill more than one warp's lanes, for each of a warp's k-blocks."""
    top, experts = 40, 64
    pairs, n = rows * top, hm.expert_plan_rows(rows * top, experts)
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(rows, K, generator=g, device="cuda").to(TYPES[xt])
    ids = torch.rand(rows, experts + 3, generator=g, device="cuda").argsort(1)[:, :top].to(torch.int32)
    ids[ids >= experts] = -1
    ids = ids.contiguous()
    plan = torch.empty(hm.expert_plan_ints(pairs, experts), dtype=torch.int32, device="cuda")
    hm.expert_plan((ids.data_ptr(), pairs), experts, plan=plan.data_ptr(), stream=stream())
    im = torch.zeros(hm.image_bytes(dtype, n, K), dtype=torch.uint8, device="cuda")
    hm.image_pack((x.data_ptr(), rows), dtype, K=K, x_dtype=xt, plan=plan.data_ptr(), pairs=pairs, experts=experts, top=top, image=im.data_ptr(), stream=stream())
    own = torch.zeros(hm.image_bytes(dtype, rows, K), dtype=torch.uint8, device="cuda")
    hm.image_pack((x.data_ptr(), rows), dtype, K=K, x_dtype=xt, image=own.data_ptr(), stream=stream())
    held, want = torch.empty(n, K, dtype=torch.bfloat16, device="cuda"), torch.empty(rows, K, dtype=torch.bfloat16, device="cuda")
    hm.image_unpack((im.data_ptr(), n), dtype, K=K, out=held.data_ptr(), out_dtype=BF16, stream=stream())
    hm.image_unpack((own.data_ptr(), rows), dtype, K=K, out=want.data_ptr(), out_dtype=BF16, stream=stream())
    first, count, place, row = ic.plan(ids.cpu().numpy(), experts)
    np.testing.assert_array_equal(plan.cpu().numpy(), np.concatenate([first, count, place, row]))
    at = torch.from_numpy(row).cuda().long()
    used = at >= 0
    assert torch.equal(held[used], want[at[used] // top])
    assert not held[~used].any()  # rows that no pair has are left as they were


# ---- gated rows ----------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [MX, BF16])
@pytest.mark.parametrize("rows,K", [(9, 63), (5, 101), (40, 64), (7, 1216), (2200, 2100), (300, 4500)])
def test_gated_rows_of_either_type(hm, dtype, rows, K):
    """bf16 rows give what f32 rows of the same values do, bit for bit; those are held to silu(g) u in 64 bits (tolerances: test_gated_pack)."""
    d = hm.DType(dtype)
    x = ic.bf16_value(ic.bf16_bits(ic.activations(np.random.default_rng(rows + K), rows, 2 * K)))
    from_f32 = hm.image_pack(x, d, glu=True)
    np.testing.assert_array_equal(from_f32, hm.image_pack(ic.bf16_bits(x), d, glu=True))
    got = hm.image_unpack(from_f32, d, K, rows)
    g, u = x[:, :K].astype(np.float64), x[:, K:].astype(np.float64)
    with np.errstate(over="ignore"):
        want = g / (1 + np.exp(-g)) * u
    if dtype == BF16:
        assert (np.abs(got - want) <= (2.0**-8 + 8 * 2.0**-23) * np.abs(want) + 2.0**-126).all()
    else:
        pad = np.zeros((rows, -(-K // 32) * 32))
        pad[:, :K] = np.abs(want)
        top = np.repeat(pad.reshape(rows, -1, 32).max(-1), 32, axis=1)[:, :K]
        assert (np.abs(got - want) <= 0.2501 * top + 2.0**-126).all()


@pytest.mark.parametrize("dtype", [MX, BF16])
@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("rows,K,ld,shift", [(50, 300, 600, 0), (50, 300, 617, 1), (33, 63, 130, 3), (2300, 2100, 4208, 0)])
def test_gated_rows_in_groups_and_apart(hm, dtype, xt, rows, K, ld, shift):
    """Strided, unaligned, and one pair per row in a plan: the bits of the plain rows."""
    experts = 5
    g = torch.Generator(device="cuda").manual_seed(rows + ld)
    flat = torch.randn(rows * ld + shift, generator=g, device="cuda").to(TYPES[xt])
    x = flat[shift:].view(rows, ld)
    dense = x[:, : 2 * K].contiguous()
    ids = torch.randint(-1, experts, (rows,), generator=g, device="cuda", dtype=torch.int32)
    plan = torch.empty(hm.expert_plan_ints(rows, experts), dtype=torch.int32, device="cuda")
    hm.expert_plan((ids.data_ptr(), rows), experts, plan=plan.data_ptr(), stream=stream())
    n = hm.expert_plan_rows(rows, experts)
    out = []
    for src, step, many in [(dense, 2 * K, rows), (x, ld, rows), (x, ld, n)]:
        im = torch.zeros(hm.image_bytes(dtype, many, K), dtype=torch.uint8, device="cuda")
        grouped = dict(plan=plan.data_ptr(), pairs=rows, experts=experts) if many == n else {}
        hm.image_pack((src.data_ptr(), rows), dtype, K=K, x_dtype=xt, ldx=step, glu=True, image=im.data_ptr(), stream=stream(), **grouped)
        out.append(torch.empty(many, K, device="cuda"))
        hm.image_unpack((im.data_ptr(), many), dtype, K=K, out=out[-1].data_ptr(), stream=stream())
    assert torch.equal(out[0], out[1])
    place = torch.from_numpy(ic.plan(ids.cpu().numpy(), experts)[2]).cuda().long()
    assert torch.equal(out[2][place[place >= 0]], out[0][place >= 0])


# ---- products of several units per CTA -----------------------------------------------------------


def wide_product(x, w):
    return (x @ w.T).cpu().numpy(), (x.abs() @ w.abs().T).cpu().numpy()


def cuda64(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


@pytest.mark.parametrize("dtype,K", [(MX, 1536), (MX, 2560), (BF16, 448), (BF16, 640), (MX, 33), (BF16, 1025)])
@pytest.mark.parametrize("M,N", [(1999, 4000), (2113, 4097)])
def test_products_of_many_units(hm, dtype, K, M, N):
    """352 and 396 units: two or three for a CTA, up to eight k-blocks (one accumulator each) and more, last units of 79 and of one row."""
    assert -(-M // 192) * -(-N // 128) > 2 * 148
    d, name = hm.DType(dtype), NAMES[dtype]
    rng = np.random.default_rng(M + K)
    x, w = ic.activations(rng, M, K), (rng.standard_normal((N, K)) * 0.02).astype(np.float32)
    xi, wi = hm.image_pack(x, d), hm.image_pack(w, d)
    want, size = wide_product(cuda64(ic.rounded(x, name)), cuda64(ic.rounded(w, name)))
    got = hm.gemm_image(xi, wi, N, d, K, M)
    close(got, want, size, 128, "image product of many units " + name)
    close(hm.gemm_image(xi, wi, N, d, K, M, y_dtype=hm.DType.BF16), want, size, 128, "image product of many units " + name)
    np.testing.assert_array_equal(got, hm.gemm_image(xi, wi, N, d, K, M))


@pytest.mark.parametrize("dtype,K", [(MX, 1536), (MX, 2560), (BF16, 448), (BF16, 640)])
def test_grouped_products_of_many_units(hm, dtype, K):
    """Groups of 1, 33, 65, 193, no, 700, 1200, 128 and 500 rows, some rows without an expert: 20 units times 18 tiles."""
    sizes, none, N = [1, 33, 65, 193, 0, 700, 1200, 128, 500], 40, 2300
    d, name, experts = hm.DType(dtype), NAMES[dtype], len(sizes)
    rng = np.random.default_rng(K)
    ids = rng.permutation(np.concatenate([np.full(n, e) for e, n in enumerate(sizes)] + [np.full(none, -1)])).astype(np.int32)
    pairs = ids.size
    x, w = ic.activations(rng, pairs, K), (rng.standard_normal((experts * N, K)) * 0.02).astype(np.float32)
    plan = hm.expert_plan(ids, experts)
    xi = hm.image_pack(x, d, plan=plan, experts=experts)
    wi = np.concatenate([hm.image_pack(w[e * N : (e + 1) * N], d) for e in range(experts)])
    xr, wr = cuda64(ic.rounded(x, name)), cuda64(ic.rounded(w, name))
    want, size = np.zeros((pairs, N)), np.zeros((pairs, N))
    for e in range(experts):
        mine = np.flatnonzero(ids == e)
        want[mine], size[mine] = wide_product(xr[torch.from_numpy(mine).cuda()], wr[e * N : (e + 1) * N])
    real = ids >= 0
    for out in (F32, BF16):
        before = np.full((pairs, N), 7.0, np.float32) if out == F32 else np.full((pairs, N), 0x40E0, np.uint16)
        got = hm.expert_gemm(xi, wi, plan, N, d, pairs, experts, K, y=before.copy(), y_dtype=hm.DType(out))
        close(got[real], want[real], size[real], 128, "grouped product of many units " + name)
        np.testing.assert_array_equal(got[~real], before[~real])


# ---- pairs, sums ---------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [False, True])
@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("tokens,top,experts,none,K,N", [(1, 4, 16, 0, 896, 390), (3, 2, 8, 2, 64, 130), (2, 8, 32, 0, 1536, 129), (9, 1, 3, 1, 1000, 40), (4, 6, 64, 2, 2016, 70)])
def test_pairs_of_either_type(hm, bits, out, tokens, top, experts, none, K, N):
    """Tolerances of the few rows; from strided rows into strided rows on the device too, where rows without an expert stay."""
    rng = np.random.default_rng(tokens + K + out)
    ids = routing(rng, tokens, top, experts, none)
    x = ic.activations(rng, tokens, K)
    if bits:
        x = ic.bf16_value(ic.bf16_bits(x))
    w = (rng.standard_normal((experts * N, K)) * 0.02).astype(np.float32)
    wi = np.concatenate([hm.image_pack(w[e * N : (e + 1) * N], hm.DType.MXFP4) for e in range(experts)])
    wr, flat, pairs = ic.mx_round(w).reshape(experts, N, K), ids.reshape(-1), tokens * top
    real = flat >= 0
    wide = np.repeat(x.astype(np.float64), top, 0)
    want = np.stack([wr[e] @ wide[p] if e >= 0 else np.zeros(N) for p, e in enumerate(flat)])
    size = np.stack([np.abs(wr[e]) @ np.abs(wide[p]) if e >= 0 else np.zeros(N) for p, e in enumerate(flat)])
    before = np.full((pairs, N), 3.0, np.float32) if out == F32 else np.full((pairs, N), 0x4040, np.uint16)
    got = hm.expert_gemv(ic.bf16_bits(x) if bits else x, wi, ids, N, top, experts, y=before.copy(), y_dtype=hm.DType(out))
    close(got[real], want[real], size[real], 160, "pairs x 4 bits")
    np.testing.assert_array_equal(got[~real], before[~real])
    ld, xt = K + 3, BF16 if bits else F32
    xd = torch.zeros(tokens * ld + 1, device="cuda", dtype=TYPES[xt])
    xd[1:].view(tokens, ld)[:, :K] = torch.from_numpy(x).cuda().to(TYPES[xt])
    y = torch.full((pairs, N + 5), 3.0, device="cuda", dtype=TYPES[out])
    wd, idd = torch.from_numpy(wi).cuda(), torch.from_numpy(ids).cuda()
    hm.expert_gemv((xd[1:].data_ptr(), tokens), wd.data_ptr(), idd.data_ptr(), N, top=top, experts=experts, K=K, x_dtype=xt, ldx=ld, y=y.data_ptr(), y_dtype=out, ldy=N + 5, stream=stream())
    h = y[:, :N].float().cpu().numpy()
    np.testing.assert_array_equal(h, got if out == F32 else ic.bf16_value(got))
    assert (y[:, N:] == 3.0).all()


@pytest.mark.parametrize("W", [24, 5])
@pytest.mark.parametrize("rows_t,out", [(F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
def test_sums_of_more_tokens_than_a_grid_has_rows(hm, W, rows_t, out):
    tokens, top, experts = 140001, 2, 7
    g = torch.Generator(device="cuda").manual_seed(W)
    rows = torch.randn(tokens * top, W, generator=g, device="cuda").to(TYPES[rows_t])
    ids = torch.randint(-1, experts, (tokens, top), generator=g, device="cuda", dtype=torch.int32)
    rows[ids.view(-1) < 0] = float("nan")
    wt, x = torch.rand(tokens, top, generator=g, device="cuda"), torch.randn(tokens, W, generator=g, device="cuda")
    y = x.clone() if out == F32 else torch.full((tokens, W), 9.0, device="cuda", dtype=TYPES[out])  # f32: in place
    hm.expert_sum((rows.data_ptr(), tokens), ids.data_ptr(), wt.data_ptr(), top=top, experts=experts, width=W, rows_dtype=rows_t, resid=y.data_ptr() if out == F32 else x.data_ptr(), y=y.data_ptr(), y_dtype=out, stream=stream())
    terms = torch.where(ids[..., None] >= 0, wt[..., None].double() * rows.double().nan_to_num().view(tokens, top, W), 0.0)
    want, size = terms.sum(1) + x.double(), terms.abs().sum(1) + x.double().abs()
    # two products and three sums, 2^-24 each
    close(y.cpu().numpy() if out == F32 else y.view(torch.int16).cpu().numpy().view(np.uint16), want.cpu().numpy(), size.cpu().numpy(), 3, "weighted sum of many tokens")


@pytest.mark.parametrize("dtype", [MX, BF16])
@pytest.mark.parametrize("tokens", [3, 150])
def test_a_mixture_with_identity_experts(hm, dtype, tokens):
    """Two layers' ends: the sum of the chosen experts without a residual, the identity experts' share and the norm from hm_post_norm_route.

    x + mult * n(z) * w with z = y + share * x, n(z) = z / sqrt(mean(z^2) + eps), from the rows as they came out.  In f32, with u = 2^-24: z is off by at most
    e = 6 u (sum of magnitudes); the mean of W squares by W u of itself, what z's error makes of it aside, the root by half of that; a few more roundings of the
    factor and the products: |error| <= |mult w| (e / r + |z| / r (W u / 2 + |e| / |z| over the row + 8 u)) + 2 u |result|."""
    rng = np.random.default_rng(tokens + dtype)
    W, ff, experts, identities, top = 320, 96, 6, 3, 3
    d, name = hm.DType(dtype), NAMES[dtype]
    f = lambda *n: rng.standard_normal(n).astype(np.float32)
    router = ic.bf16_bits(f(experts + identities, W) * 0.1)
    x, ids, wts, share = hm.post_norm_route(f(tokens, W), f(tokens, W), np.ones(W, np.float32), 0.25, 1e-6, router=router, correction=np.zeros(experts + identities, np.float32), experts=experts, top=top)
    assert (ids < 0).any() and (share > 0).any() and (ids >= 0).any()
    pairs = tokens * top
    image = lambda w: np.concatenate([hm.image_pack(w[e], d) for e in range(experts)])
    plan = hm.expert_plan(ids, experts)
    h = hm.expert_gemm(hm.image_pack(x, d, plan=plan, experts=experts, top=top), image(f(experts, 2 * ff, W) * 0.05), plan, 2 * ff, d, pairs, experts, W)
    rows = hm.expert_gemm(hm.image_pack(h, d, plan=plan, experts=experts, glu=True), image(f(experts, W, ff) * 0.05), plan, W, d, pairs, experts, ff)
    y = hm.expert_sum(rows, ids, wts, top, experts)
    nw, mult, eps = (1 + 0.1 * f(W)).astype(np.float32), 0.5, 1e-6
    got = hm.post_norm_route(y, x, nw, mult, eps, identity=share).astype(np.float64)
    terms = np.where(ids[..., None] >= 0, wts[..., None].astype(np.float64) * rows.reshape(tokens, top, W), 0.0)
    own = share[:, None].astype(np.float64) * x
    z, u = terms.sum(1) + own, 2.0**-24
    r = np.sqrt((z**2).mean(1, keepdims=True) + eps)
    want = x + mult * z / r * nw
    e = 6 * u * (np.abs(terms).sum(1) + np.abs(own))
    norm = lambda a: np.sqrt((a**2).sum(1, keepdims=True))
    limit = np.abs(mult * nw) * (e / r + np.abs(z) / r * (W * u / 2 + norm(e) / norm(z) + 8 * u)) + 2 * u * np.abs(want)
    assert (np.abs(got - want) <= limit).all(), float((np.abs(got - want) / limit).max())
    # the share of the identity experts is no rounding: without it the result is another
    without = x + mult * terms.sum(1) / np.sqrt((terms.sum(1) ** 2).mean(1, keepdims=True) + eps) * nw
    assert (np.abs(without - want) > limit).any(1).sum() >= (share > 0).sum() * 0.9
