"""Operand images and grouped products on device memory: strides, alignment, streams, graphs, long offsets, what is left as it was.
Values are compared with the host-mode calls (tests/test_gpu_images.py holds those to 64-bit results), bit for bit."""
import numpy as np
import pytest

import image_cases as ic

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, BF16, MX = 0, 1, 10
TYPES = {F32: torch.float32, BF16: torch.bfloat16}


def bits(t):
    """Rows as the host-mode calls take them: f32, or bf16 bit patterns."""
    t = t.detach().cpu().contiguous()
    return t.numpy() if t.dtype == torch.float32 else t.view(torch.int16).numpy().view(np.uint16)


def rows_of(seed, rows, K, dtype, ld=None, shift=0):
    """A device tensor of rows `ld` apart that starts `shift` elements into its allocation."""
    ld = ld or K
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat = torch.randn(rows * ld + shift + 8, generator=g, device="cuda").to(TYPES[dtype])
    return flat[shift : shift + rows * ld].view(rows, ld)[:, :K], flat


def image(hm, dtype, rows, K):
    return torch.full((hm.image_bytes(dtype, rows, K),), 0xEE, dtype=torch.uint8, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("dtype", [MX, BF16])
@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("rows,K,ld,shift", [(5, 300, 300, 0), (5, 300, 301, 0), (40, 256, 260, 1), (131, 70, 97, 3), (3, 1000, 1008, 2)])
def test_strided_and_unaligned_rows(hm, dtype, xt, rows, K, ld, shift):
    x, keep = rows_of(rows + ld, rows, K, xt, ld, shift)
    im = image(hm, dtype, rows, K)
    hm.image_pack((x.data_ptr(), rows), dtype, K=K, x_dtype=xt, ldx=ld, image=im.data_ptr(), stream=stream())
    host = hm.image_pack(bits(x), hm.DType(dtype))
    got = im.cpu().numpy().reshape(-1, hm.image_bytes(dtype, 1, 1))
    kb = got.shape[0] // ((rows + 127) // 128)
    # rows beyond the last are left as they were: their codes stay 0xEE (scales of all rows share 16-byte pieces and are looked at by the values below)
    off = 1024 if dtype == MX else 0
    for i in range(rows, (rows + 127) // 128 * 128):
        assert (got[i // 128 * kb : (i // 128 + 1) * kb, off + i % 128 * 128 : off + i % 128 * 128 + 128] == 0xEE).all()
    for out_t in (F32, BF16):
        y = torch.full((rows, ld + 5), 9.0, device="cuda", dtype=TYPES[out_t])
        hm.image_unpack((im.data_ptr(), rows), dtype, K=K, out=y.data_ptr(), out_dtype=out_t, ldo=ld + 5, stream=stream())
        np.testing.assert_array_equal(bits(y[:, :K]), hm.image_unpack(host, hm.DType(dtype), K, rows, out_dtype=hm.DType(out_t)))
        assert (y[:, K:] == 9.0).all()


@pytest.mark.parametrize("dtype,M,K,N", [(MX, 70, 320, 130), (BF16, 70, 320, 130), (MX, 5, 4096, 60), (MX, 400, 2304, 257)])
@pytest.mark.parametrize("out", [F32, BF16])
def test_products_into_strided_rows(hm, dtype, M, K, N, out):
    x, _ = rows_of(1, M, K, F32)
    w, _ = rows_of(2, N, K, BF16)
    xi, wi = image(hm, dtype, M, K), image(hm, dtype, N, K)
    hm.image_pack((x.data_ptr(), M), dtype, K=K, image=xi.data_ptr(), stream=stream())
    hm.image_pack((w.data_ptr(), N), dtype, K=K, x_dtype=BF16, image=wi.data_ptr(), stream=stream())
    want = hm.gemm_image(hm.image_pack(bits(x), hm.DType(dtype)), hm.image_pack(bits(w), hm.DType(dtype)), N, hm.DType(dtype), K, M, y_dtype=hm.DType(out))
    for ld, shift in [(N, 0), (N + 1, 0), (N + 3, 1), ((N + 15) // 8 * 8, 0)]:  # aligned rows, odd ones, a start off 16 bytes
        y = torch.full((M * ld + shift,), 9.0, device="cuda", dtype=TYPES[out])
        hm.gemm_image((xi.data_ptr(), M), wi.data_ptr(), N, dtype, K=K, y=y[shift:].data_ptr(), y_dtype=out, ldy=ld, stream=stream())
        got = y[shift:].view(M, ld)
        np.testing.assert_array_equal(bits(got[:, :N]), want)
        assert (got[:, N:] == 9.0).all() and (y[:shift] == 9.0).all()


def test_few_rows_strided(hm):
    M, K, N = 6, 1000, 390
    for xt in (F32, BF16):
        x, _ = rows_of(3, M, K, xt, 1003, 1)
        w, _ = rows_of(4, N, K, F32)
        wi = image(hm, MX, N, K)
        hm.image_pack((w.data_ptr(), N), MX, K=K, image=wi.data_ptr(), stream=stream())
        want = hm.gemv_mx4(bits(x), hm.image_pack(bits(w), hm.DType.MXFP4), N)
        y = torch.full((M, N + 3), 9.0, device="cuda")
        hm.gemv_mx4((x.data_ptr(), M), wi.data_ptr(), N, K=K, x_dtype=xt, ldx=1003, y=y.data_ptr(), ldy=N + 3, stream=stream())
        np.testing.assert_array_equal(bits(y[:, :N]), want)
        assert (y[:, N:] == 9.0).all()


def test_more_choices_than_lanes(hm):
    """Every row goes to 40 experts of 64."""
    rows, top, experts, K = 9, 40, 64, 96
    ids = np.stack([np.random.default_rng(r).permutation(experts + 3)[:top] for r in range(rows)]).astype(np.int32)
    ids[ids >= experts] = -1
    x, _ = rows_of(5, rows, K, F32)
    plan = hm.expert_plan(ids, experts)
    for dtype in (MX, BF16):
        im = hm.image_pack(bits(x), hm.DType(dtype), plan=plan, experts=experts, top=top)
        held = hm.image_unpack(im, hm.DType(dtype), K, hm.expert_plan_rows(rows * top, experts))
        own = hm.image_unpack(hm.image_pack(bits(x), hm.DType(dtype)), hm.DType(dtype), K, rows)
        place = ic.plan(ids, experts)[2]
        for p, at in enumerate(place):
            if at >= 0:
                np.testing.assert_array_equal(held[at], own[p // top])


def test_the_same_expert_twice(hm):
    """A token may choose an expert more than once: each choice is a pair of its own."""
    rng = np.random.default_rng(6)
    T, top, E, K, N = 70, 3, 4, 160, 70
    ids = rng.integers(-1, E, (T, top)).astype(np.int32)
    x, _ = rows_of(12, T, K, F32)
    w, _ = rows_of(13, E * N, K, F32)
    images = np.concatenate([hm.image_pack(bits(w[e * N : (e + 1) * N]), hm.DType.MXFP4) for e in range(E)])
    plan = hm.expert_plan(ids, E)
    np.testing.assert_array_equal(plan, np.concatenate(ic.plan(ids, E)))
    got = hm.expert_gemm(hm.image_pack(bits(x), hm.DType.MXFP4, plan=plan, experts=E, top=top), images, plan, N, hm.DType.MXFP4, T * top, E, K)
    few = hm.expert_gemv(ic.mx_round(bits(x)).astype(np.float32), images, ids, N, top, E)
    for p, e in enumerate(ids.reshape(-1)):
        want = hm.gemm_image(hm.image_pack(bits(x[p // top : p // top + 1]), hm.DType.MXFP4), images.reshape(E, -1)[e], N, hm.DType.MXFP4, K, 1)[0] if e >= 0 else np.zeros(N, np.float32)
        np.testing.assert_array_equal(got[p], want)  # products of 4-bit values and their sums over 160 of them are exact
        np.testing.assert_allclose(few[p], want, rtol=0, atol=1e-5 * float(np.abs(want).max() + 1))


def feed_forward(hm, s, st):
    """A mixture's feed-forward on the buffers of `s`."""
    pairs, E, top, W, ff, T = s["pairs"], s["E"], s["top"], s["W"], s["ff"], s["T"]
    hm.expert_plan((s["ids"].data_ptr(), pairs), E, plan=s["plan"].data_ptr(), stream=st)
    hm.image_pack((s["x"].data_ptr(), T), MX, K=W, plan=s["plan"].data_ptr(), pairs=pairs, experts=E, top=top, image=s["xi"].data_ptr(), stream=st)
    hm.expert_gemm(s["xi"].data_ptr(), s["gu"].data_ptr(), s["plan"].data_ptr(), 2 * ff, MX, pairs=pairs, experts=E, K=W, y=s["h"].data_ptr(), stream=st)
    hm.image_pack((s["h"].data_ptr(), pairs), MX, K=ff, plan=s["plan"].data_ptr(), pairs=pairs, experts=E, glu=True, image=s["hi"].data_ptr(), stream=st)
    hm.expert_gemm(s["hi"].data_ptr(), s["dn"].data_ptr(), s["plan"].data_ptr(), W, MX, pairs=pairs, experts=E, K=ff, y=s["rows"].data_ptr(), stream=st)
    hm.expert_sum((s["rows"].data_ptr(), T), s["ids"].data_ptr(), s["wt"].data_ptr(), top=top, experts=E, width=W, resid=s["x"].data_ptr(), y=s["y"].data_ptr(), stream=st)


def mixture(hm, seed, T, E=8, top=2, W=320, ff=96):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *n: torch.randn(*n, generator=g, device="cuda")
    pairs = T * top
    s = dict(T=T, E=E, top=top, W=W, ff=ff, pairs=pairs, x=r(T, W), wt=torch.rand(T, top, generator=g, device="cuda"))
    s["ids"] = torch.stack([torch.randperm(E + 1, generator=g, device="cuda")[:top] for _ in range(T)]).to(torch.int32)
    s["ids"][s["ids"] == E] = -1
    n = hm.expert_plan_rows(pairs, E)
    e = lambda *n, d=torch.float32: torch.zeros(*n, dtype=d, device="cuda")
    s |= dict(plan=e(hm.expert_plan_ints(pairs, E), d=torch.int32), xi=image(hm, MX, n, W), hi=image(hm, MX, n, ff), h=e(pairs, 2 * ff), rows=e(pairs, W), y=e(T, W))
    for name, N, K in (("gu", 2 * ff, W), ("dn", W, ff)):
        each = hm.image_bytes(MX, N, K)
        s[name] = torch.empty(E * each, dtype=torch.uint8, device="cuda")
        w = r(E * N, K) * 0.05
        for i in range(E):
            hm.image_pack((w[i * N :].data_ptr(), N), MX, K=K, image=s[name].data_ptr() + i * each, stream=stream())
        s["keep" + name] = w
    return s


def test_graph_replays_and_two_streams(hm):
    """Captured once, replayed on other inputs; two of them at a time on two streams, and eager calls between them."""
    a, b = mixture(hm, 1, 70), mixture(hm, 2, 33)
    feed_forward(hm, a, stream())
    feed_forward(hm, b, stream())
    torch.cuda.synchronize()
    want_a, want_b = a["y"].clone(), b["y"].clone()
    graphs = []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            feed_forward(hm, s, stream())
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        a["y"].zero_()
        b["y"].zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(a["y"], want_a) and torch.equal(b["y"], want_b)
    # the graph on inputs that it was not captured with: the same as eager calls
    a["x"].mul_(0.37)
    a["ids"].copy_(a["ids"].roll(1, 0))
    graphs[0].replay()
    torch.cuda.synchronize()
    got = a["y"].clone()
    a["y"].zero_()
    for st in streams:  # eager on two streams at once, on buffers of their own
        with torch.cuda.stream(st):
            feed_forward(hm, a if st is streams[0] else b, st.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(a["y"], got) and torch.equal(b["y"], want_b)
    hm.dev_sync()


def test_offsets_beyond_32_bits(hm):
    """Experts' images of more than 2^32 bytes, rows of y more than 2^32 bytes behind its start."""
    K, N, E = 8192, 120000, 10
    each = hm.image_bytes(MX, N, K)
    assert (E - 1) * each > 2**32
    w, _ = rows_of(7, 200, K, F32)
    images = torch.empty(E * each, dtype=torch.uint8, device="cuda")
    last = images[(E - 1) * each :]
    # the first 200 features of the last expert; the other features of it are zero
    last.zero_()
    hm.image_pack((w.data_ptr(), 200), MX, K=K, image=last.data_ptr(), stream=stream())
    x, _ = rows_of(8, 2, K, F32)
    want = hm.gemv_mx4(bits(x), hm.image_pack(bits(w), hm.DType.MXFP4), 200)
    ids = torch.tensor([E - 1, -1], dtype=torch.int32, device="cuda")
    y = torch.full((2, N), 5.0, device="cuda")
    hm.expert_gemv((x.data_ptr(), 2), images.data_ptr(), ids.data_ptr(), N, top=1, experts=E, K=K, y=y.data_ptr(), stream=stream())
    np.testing.assert_allclose(bits(y[:1, :200]), want[:1], rtol=0, atol=2e-6 * float(np.abs(want).max()))  # sums of other parts: K shared by other clusters
    assert (y[0, 200:] == 0).all() and (y[1] == 5.0).all()
    plan = torch.empty(hm.expert_plan_ints(2, E), dtype=torch.int32, device="cuda")
    xi = image(hm, MX, hm.expert_plan_rows(2, E), K)
    hm.expert_plan((ids.data_ptr(), 2), E, plan=plan.data_ptr(), stream=stream())
    hm.image_pack((x.data_ptr(), 2), MX, K=K, plan=plan.data_ptr(), pairs=2, experts=E, image=xi.data_ptr(), stream=stream())
    y.fill_(5.0)
    hm.expert_gemm(xi.data_ptr(), images.data_ptr(), plan.data_ptr(), N, MX, pairs=2, experts=E, K=K, y=y.data_ptr(), stream=stream())
    want = hm.gemm_image(hm.image_pack(bits(x[:1]), hm.DType.MXFP4), hm.image_pack(bits(w), hm.DType.MXFP4), 200, hm.DType.MXFP4, K, 1)
    np.testing.assert_allclose(bits(y[:1, :200]), want, rtol=0, atol=2e-6 * float(np.abs(want).max()))
    assert (y[0, 200:] == 0).all() and (y[1] == 5.0).all()
    del images, last
    ld = 600_000_000
    rows, cols = 5, 70
    xs, _ = rows_of(9, rows, 64, F32)
    ws, _ = rows_of(10, cols, 64, F32)
    xi, wi = image(hm, MX, rows, 64), image(hm, MX, cols, 64)
    hm.image_pack((xs.data_ptr(), rows), MX, K=64, image=xi.data_ptr(), stream=stream())
    hm.image_pack((ws.data_ptr(), cols), MX, K=64, image=wi.data_ptr(), stream=stream())
    big = torch.empty(4 * ld + cols, device="cuda")
    hm.gemm_image((xi.data_ptr(), rows), wi.data_ptr(), cols, MX, K=64, y=big.data_ptr(), ldy=ld, stream=stream())
    want = hm.gemm_image(hm.image_pack(bits(xs), hm.DType.MXFP4), hm.image_pack(bits(ws), hm.DType.MXFP4), cols, hm.DType.MXFP4, 64, rows)
    got = torch.stack([big[r * ld : r * ld + cols] for r in range(rows)])
    np.testing.assert_array_equal(bits(got), want)
    out = torch.empty(4 * ld + 64, device="cuda")
    hm.image_unpack((xi.data_ptr(), rows), MX, K=64, out=out.data_ptr(), ldo=ld, stream=stream())
    np.testing.assert_array_equal(bits(out[4 * ld : 4 * ld + 64]), ic.mx_round(bits(xs))[4].astype(np.float32))


def test_calls_refuse_what_does_not_fit(hm):
    x, _ = rows_of(1, 4, 64, F32)
    im = image(hm, MX, 4, 64)
    y = torch.zeros(4, 8, device="cuda")
    with pytest.raises(hm.HomuraError):
        hm.image_pack((x.data_ptr() + 2, 4), MX, K=64, image=im.data_ptr())  # rows off their type's alignment
    with pytest.raises(hm.HomuraError):
        hm.gemm_image((im.data_ptr() + 8, 4), im.data_ptr(), 4, MX, K=64, y=y.data_ptr())  # images start on 16 bytes
    with pytest.raises(hm.HomuraError):
        hm.gemv_mx4((x.data_ptr(), 9), im.data_ptr(), 4, K=64, y=y.data_ptr())
    with pytest.raises(hm.HomuraError):
        hm.image_pack(np.zeros((3, 64), np.float32), hm.DType.MXFP4, plan=np.zeros(5, np.int32), experts=4, top=2)
    with pytest.raises(hm.HomuraError):
        hm.gemm_image(np.zeros(5, np.uint8), np.zeros(5, np.uint8), 4, hm.DType.MXFP4, 64, 4)
