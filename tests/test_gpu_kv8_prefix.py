"""Attention over the 8-bit cache whose shared pages are taken on their own: every call here asks for work memory for their parts, so that a limit that is moved past these sizes fails them."""
import numpy as np
import pytest

import kv8_cases as kc
from conftest import record_error
from kv8_cases import Model, bf16_bits, bf16_value
from kv8_prefix_cases import OnDevice, check_rows, formula, on_their_own, prompt, refill, some
from test_gpu_rope import turned

pytestmark = pytest.mark.gpu


def attend(m, seq, pos, heads, bf16, rows, scale=None, q=None, seen=None, what="kv8 shared pages on their own"):
    """A call with host arrays, some rows of it checked."""
    scale = m.dim**-0.5 if scale is None else scale
    q = m.queries(len(seq), heads, bf16) if q is None else q
    assert on_their_own(m.cache, len(seq), heads, len(m.shared))
    out = m.cache.attend(q, seq, pos, heads, scale, shared=m.shared)
    record_error(f"{what} {'bf16' if bf16 else 'f32'}, of the bound", check_rows(m, out, q, seq, pos, heads, scale, rows, seen), 1.0)
    return q, out


def pointed(m, q, heads, size):
    """Queries with one element of one size in every head: what a key has there decides its score."""
    x = (bf16_value(q) if q.dtype == np.uint16 else q).reshape(len(q), heads, m.dim).copy()
    x[..., 0] = size
    x = x.reshape(len(q), -1)
    return bf16_bits(x) if q.dtype == np.uint16 else x


# ---- values of different sizes ------------------------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("factor", [24, 60])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (6, 2, 128)])
def test_values_that_a_row_does_not_see_leave_it_as_it_is(hm, heads, kv_heads, dim, factor, bf16):
    n = 1000
    m = prompt(hm, factor + dim, n, kv_heads, dim, dim)
    seq, pos = np.zeros(n, int), np.arange(n)
    q, clean = attend(m, seq, pos, heads, bf16, some(n, 1))
    m.v[0][900] *= np.float32(2.0**factor)
    refill(m)
    out = m.cache.attend(q, seq, pos, heads, dim**-0.5, shared=m.shared)
    np.testing.assert_array_equal(out[:900], clean[:900])
    check_rows(m, out, q, seq, pos, heads, dim**-0.5, [*some(n, 2), 899, 900, 901])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("dim,vdim", [(64, 64), (128, 128), (96, 40)])
def test_values_of_very_different_sizes(hm, dim, vdim, bf16):
    """Large values whose weights are next to nothing, and small ones that matter: a prompt's rows, and rows with a context of their own behind."""
    rng = np.random.default_rng(dim)
    heads, kvh, M, pages = 8, 2, 700, 10
    S = 64 * pages
    m = Model(hm, dim, kvh, dim, vdim, [S + 100, S, S + 3], n_shared=pages)
    for k, v in zip(m.k, m.v):
        k[:, :, 0] = 0
        v[::3] *= np.float32(2.0**-20)
    for t in (3, 200, 201, 450, 639):
        m.k[0][t, :, 0] = -40
        m.v[0][t] = m.rng.standard_normal((kvh, vdim)).astype(np.float32) * np.float32(2.0**20)
    refill(m)
    seq = rng.integers(0, 3, M)
    pos = np.where(rng.random(M) < 0.5, np.array(m.lens)[seq] - 1, rng.integers(-1, S, M))
    q = pointed(m, m.queries(M, heads, bf16), heads, 8.0 * (dim / 64) ** 0.5)
    attend(m, seq, pos, heads, bf16, some(M, 3, 40), q=q, what="kv8 values of different sizes")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.1, -1.0, 2.0])
def test_scales_of_either_sign(hm, scale, bf16):
    heads, M, pages = 8, 500, 13
    m = Model(hm, 3, 2, 64, 64, [64 * pages + 50, 64 * pages], n_shared=pages)
    seq, pos = np.arange(M) % 2, 64 * pages - 1 - np.arange(M) % 400
    pos[::5] = np.array(m.lens)[seq[::5]] - 1
    attend(m, seq, pos, heads, bf16, some(M, 4), scale=scale)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("small,large", [(-110, 112), (100, -95), (60, 40)])
def test_queries_and_keys_far_apart_in_size(hm, small, large, bf16):
    """Sizes whose products are ordinary scores: sums of digits times codes stay within f32 when a key's scale has joined them."""
    heads, M, pages = 8, 400, 16
    m = Model(hm, 6, 2, 64, 64, [64 * pages], n_shared=pages)
    m.k[0] *= np.float32(2.0**large)
    refill(m)
    q = (m.rng.standard_normal((M, heads * 64))).astype(np.float32) * np.float32(2.0**small)
    scale = 0.125 * 2.0 ** -(small + large)
    attend(m, np.zeros(M, int), 64 * pages - 1 - np.arange(M), heads, bf16, some(M, 8), scale=scale, q=bf16_bits(q) if bf16 else q, what="kv8 sizes far apart")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,pages,own", [(400, 16, 0), (400, 16, 200), (66, 130, 0), (66, 130, 100), (74, 84, 3000)])
@pytest.mark.parametrize("large", ["first", "middle", "last", "own"])
def test_weights_that_belong_to_values_of_nothing(hm, large, M, pages, own, bf16):
    """Some tokens have all of the weight and values of zero, others have next to no weight and values of 2^110: a sum is relative to a product, and both kinds count."""
    heads, S = 8, 64 * pages
    m = Model(hm, pages, 2, 64, 64, [S + own] * 2, n_shared=pages)
    for k, v in zip(m.k, m.v):
        k[:, :, 0], v[:] = 20, 0
        at = {"first": slice(0, 40), "middle": slice(S // 2, S // 2 + 150), "last": slice(S - 70, S), "own": slice(S, S + own)}[large]
        k[at, :, 0], v[at] = -10, m.rng.standard_normal(v[at].shape).astype(np.float32) * np.float32(2.0**110)
    refill(m)
    seq, pos = np.arange(M) % 2, S + own - 1 - np.arange(M) % 20
    q = (m.rng.standard_normal((M, heads * 64)) * 0.1).astype(np.float32)
    q = pointed(m, bf16_bits(q) if bf16 else q, heads, 8.0)
    attend(m, seq, pos, heads, bf16, some(M, 9, 6), q=q, what="kv8 weights of nothing")


@pytest.mark.parametrize("bf16,M,heads,dim,pages", [(False, 300, 8, 64, 256), (False, 2000, 8, 64, 256), (False, 1500, 6, 128, 200), (False, 260, 8, 96, 81), (True, 5000, 8, 64, 270), (True, 2600, 16, 128, 140)])
def test_values_of_one_sign(hm, bf16, M, heads, dim, pages):
    """Sums in tensor memory round towards zero at every step: long ones would lose all of that."""
    m = Model(hm, M, 2, dim, dim, [64 * pages, 64 * pages - 70], n_shared=pages)
    for v in m.v:
        v *= np.float32(0.1)
        v += 1
    refill(m)
    q = m.queries(M, heads, False) * np.float32(0.2)
    seq = np.arange(M) % 2
    pos = np.array(m.lens)[seq] - 1
    pos[3::4] -= 1000
    rows = np.array([0, 1, 3, M // 2, M - 2, M - 1])
    attend(m, seq, pos, heads, bf16, rows, q=bf16_bits(q) if bf16 else q, what="kv8 values of one sign")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size", [1e5, 1e6, 1e7, 1e8, 1e9, 1e12, 1e20])
@pytest.mark.parametrize("M,pages,sign", [(400, 16, 1), (66, 130, 1), (400, 16, -1), (2000, 40, 1)])
def test_scores_of_any_size(hm, M, pages, sign, size, bf16):
    """Where one token's score is far above all others, by more than the scores' own roundings, the result is that token's value."""
    heads, S = 8, 64 * pages
    m = Model(hm, pages, 2, 64, 64, [S], n_shared=pages)
    if sign < 0:  # all scores far below zero
        m.k[0][:, :, 0] = -30
    refill(m)
    q = m.queries(M, heads, bf16)
    q = pointed(m, q, heads, 8.0) if sign < 0 else q
    seq, pos = np.zeros(M, int), S - 1 - np.arange(M)
    assert on_their_own(m.cache, M, heads, pages)
    out = m.cache.attend(q, seq, pos, heads, size, shared=m.shared)
    x, o = (bf16_value(q), bf16_value(out)) if bf16 else (q, out)
    k, v = kc.held(m.k[0]).astype(np.float64), kc.held(m.v[0]).astype(np.float64)
    clear = 0
    for r in some(M, 10):
        for h in range(heads):
            s = k[: pos[r] + 1, h // 4] @ x[r].astype(np.float64).reshape(heads, 64)[h]
            terms = (np.abs(k[: pos[r] + 1, h // 4]) @ np.abs(x[r].astype(np.float64).reshape(heads, 64)[h])).max()
            first, second = s.argmax(), np.partition(s, -2)[-2]
            if s[first] - second < terms * 2.0**-14 + 40 / size:  # twice what a score may be off, and a weight of e^-40
                continue
            clear += 1
            got, want = o[r].reshape(heads, 64)[h], v[first, h // 4]
            assert (np.abs(got - want) <= np.abs(want) * (2.0**-7 if bf16 else 2.0**-17) + 1e-12).all(), (r, h)
    assert clear > 50


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("small", [-60, -80, -93, -99])
@pytest.mark.parametrize("M,pages,own", [(400, 16, 0), (66, 130, 100)])
def test_values_next_to_nothing(hm, M, pages, own, small, bf16):
    """The smallest values that the cache holds keep their weights' bits."""
    heads, S = 8, 64 * pages
    m = Model(hm, pages, 2, 64, 64, [S + own] * 2, n_shared=pages)
    for v in m.v:
        v[:] = m.rng.standard_normal(v.shape).astype(np.float32) * np.float32(2.0**small)
    refill(m)
    attend(m, np.arange(M) % 2, S + own - 1 - np.arange(M), heads, bf16, some(M, 11), what="kv8 smallest values")


# ---- what is not there, and what is not finite ----------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,pages,more", [(74, 84, 40), (74, 84, 90), (100, 66, 20), (100, 66, 90)])
def test_own_pages_that_are_not_there_behind_low_scores(hm, M, pages, more, bf16):
    """Rows whose own pages are all missing have the prefix's average, however low its scores are: items of a CTA as a whole, cut ones, and those of teams of warps."""
    heads, rng = 8, np.random.default_rng(more)
    S = 64 * pages
    m = Model(hm, M + more, 2, 64, 64, [S] * 4, n_shared=pages, max_pages=pages + more)
    for k in m.k:
        k[:, :, 0] = -20
    refill(m)
    seq, pos = np.arange(M) % 4, S + rng.integers(0, 64 * more, M)
    pos[::9] = S - 1 - np.arange(len(pos[::9]))
    q = (m.rng.standard_normal((M, heads * 64)) * 0.1).astype(np.float32)
    q = pointed(m, bf16_bits(q) if bf16 else q, heads, 60.0)
    _, out = attend(m, seq, pos, heads, bf16, some(M, 5), q=q, what="kv8 low scores")
    assert (out != 0).any(-1).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,pages,own", [(66, 130, 0), (66, 130, 70), (100, 200, 0), (1000, 9, 0)])
def test_queries_that_are_not_finite(hm, M, pages, own, bf16):
    """Their own head is NaN, whether a row has pages of its own or not, and whether the shared ones are left in one part or in several."""
    heads, S = 8, 64 * pages
    m = Model(hm, M, 2, 64, 64, [S + own] * 2, n_shared=pages, max_pages=pages + 2)
    seq, pos = np.arange(M) % 2, S + own - 1 - np.arange(M) % 300
    clean = OnDevice(m, heads, seq, pos, m.queries(M, heads, bf16), 0.125)
    clean.run()
    x = (bf16_value(clean.q) if bf16 else clean.q).copy().reshape(M, heads, 64)
    hit = [(1, 4), (M - 1, 0), (M // 2, 5)]
    for (r, h), bad in zip(hit, (np.nan, np.inf, -np.inf)):
        x[r, h, 7 * h] = bad
    x = x.reshape(M, -1)
    call = OnDevice(m, heads, seq, pos, bf16_bits(x) if bf16 else x, 0.125)
    call.run()
    if M == 66 and not bf16:
        assert call.parts() > 1
    a, b = call.rows().reshape(M, heads, 64), clean.rows().reshape(M, heads, 64)
    keep = np.ones((M, heads), bool)
    for r, h in hit:
        keep[r, h] = False
    f = bf16_value(a) if bf16 else a
    assert np.isnan(f[~keep]).all()
    np.testing.assert_array_equal(a[keep], b[keep])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,pages", [(66, 130), (300, 30)])
def test_vectors_that_are_not_finite(hm, M, pages, bf16):
    """All values that a row sees NaN, or one key, or one value: rows that see them are NaN, others as they were; also with scores that leave weights of nothing."""
    heads, S = 8, 64 * pages
    m = Model(hm, M, 2, 64, 64, [S] * 2, n_shared=pages)
    seq, pos = np.arange(M) % 2, 63 + np.arange(M) * (S - 64) // M
    q = m.queries(M, heads, bf16)
    clean = m.cache.attend(q, seq, pos, heads, 0.125, shared=m.shared)
    one = hm.KV8Cache(2, 64, 64, m.pool.ptr, m.n_pages, m.shared[None])
    flat = lambda x: np.ascontiguousarray(x.reshape(len(x), -1))
    for part, t in ((0, S // 2), (1, S // 2)):
        k, v = (x[t : t + 1].copy() for x in m.common)
        (v if part else k)[0, :, 9] = np.nan
        one.write(flat(k), flat(v), [0], [t])
        out = m.cache.attend(q, seq, pos, heads, 0.125, shared=m.shared)
        f = bf16_value(out) if bf16 else out
        assert np.isnan(f[pos >= t]).all()
        np.testing.assert_array_equal(out[pos < t], clean[pos < t])
        one.write(flat(m.common[0][t : t + 1]), flat(m.common[1][t : t + 1]), [0], [t])
    # every value NaN, scores far below and far above zero
    v = np.full_like(m.common[1], np.nan)
    one.write(flat(m.common[0]), flat(v), np.zeros(S), np.arange(S))
    for scale in (0.125, 30.0, -30.0):
        f = m.cache.attend(q, seq, pos, heads, scale, shared=m.shared)
        assert np.isnan(bf16_value(f) if bf16 else f).all()


# ---- rows at any place ------------------------------------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,pages", [(300, 22), (66, 110), (40, 180)])
@pytest.mark.parametrize("dim,vdim,offset,pad", [(64, 64, 1, 0), (64, 64, 2, 2), (128, 128, 4, 4), (33, 31, 1, 3), (32, 48, 8, 8), (20, 6, 3, 1)])
def test_strided_rows_at_any_address(hm, dim, vdim, offset, pad, M, pages, bf16):
    """Results stand where they belong and nowhere else; rows of no sequence are left, rows that see nothing are zeros; work memory ends where it says."""
    heads, kvh, S, rng = 6, 2, 64 * pages, np.random.default_rng(M + dim)
    m = Model(hm, dim, kvh, dim, vdim, [S + 100, S + 7, S], n_shared=pages)
    seq = rng.integers(0, 3, M)
    pos = np.where(rng.random(M) < 0.6, np.array(m.lens)[seq] - 1, rng.integers(0, S, M))
    seq[2::11], pos[3::13] = [-1, 3, 2**31 - 1, -(2**31)][M % 4], -1
    call = OnDevice(m, heads, seq, pos, m.queries(M, heads, bf16), 0.2, offset, pad)
    call.run()
    out = call.rows()
    call.parts()  # guard bytes
    gone = (seq < 0) | (seq >= 3)
    assert (out[gone] == 5).all() and (out[~gone & (pos < 0)] == 0).all()
    call.check(some(M, 6))


@pytest.mark.parametrize("bf16,heads", [(False, 1024), (True, 128)])
def test_the_most_rows(hm, bf16, heads):
    """8192 rows, the most of a call; f32 sums behind the parts, beyond 32 bits of work memory."""
    import torch

    M, kvh, dim, pages = 8192, 2, 64, 21
    m = Model(hm, 30, kvh, dim, dim, [64 * pages], n_shared=pages)
    seq, pos = np.zeros(M, int), 64 * pages - 1 - np.arange(M) % 700
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(M, heads * dim, generator=g, device="cuda").to(torch.bfloat16 if bf16 else torch.float32)
    q = q.view(torch.uint16).cpu().numpy() if bf16 else q.cpu().numpy()
    call = OnDevice(m, heads, seq, pos, q, 0.125)
    assert bf16 or call.size > 6 << 30
    call.run()
    torch.cuda.synchronize()
    o = call.ob.view(M, -1)
    at = some(M, 12, 6)
    check_rows(m, torch.stack([o[int(r)] for r in at]).cpu().numpy(), q[at], seq[at], pos[at], heads, 0.125, np.arange(len(at)))
    assert (call.work[-64:] == 255).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_shared_pages_behind_four_gigabytes(hm, bf16):
    kvh, dim, M, heads, n = 8, 128, 200, 16, 36000
    size = hm.kv8_pool_bytes(kvh, dim, dim, n)
    assert size > 4 << 30
    pool = hm.DeviceBuffer(size)
    shared = np.array([n - 1, 0, n // 2, n - 2, 35000, 1, 33333, 7], np.int32)
    cache = hm.KV8Cache(kvh, dim, dim, pool.ptr, n, shared[None])
    rng, S = np.random.default_rng(0), 64 * len(shared)
    k, v = (rng.standard_normal((S, kvh * dim)).astype(np.float32) for _ in range(2))
    cache.write(k, v, np.zeros(S), np.arange(S))
    x = rng.standard_normal((M, heads * dim)).astype(np.float32)
    q = bf16_bits(x) if bf16 else x
    x = bf16_value(q) if bf16 else x
    assert on_their_own(cache, M, heads, len(shared))
    pos = S - 1 - np.arange(M)
    out = cache.attend(q, np.zeros(M), pos, heads, dim**-0.5, shared=shared)
    o = bf16_value(out) if bf16 else out
    hk, hv = (kc.held(y.reshape(S, kvh, dim)).astype(np.float64) for y in (k, v))
    for r in some(M, 13, 5):
        want, tol = formula(x[r].astype(np.float64).reshape(heads, dim), hk[: pos[r] + 1], hv[: pos[r] + 1], dim**-0.5, bf16, pos[r] + 1)
        assert (np.abs(o[r].reshape(heads, dim) - want) <= tol).all(), r


# ---- streams and graphs ---------------------------------------------------------------------------------


def calls(hm):
    out = []
    for seed, M, heads, dim, lens, pages, bf16 in [(1, 300, 8, 64, (100, 0, 9), 22, False), (2, 66, 8, 128, (0, 0), 110, False), (3, 600, 6, 64, (64, 1), 12, True), (4, 70, 8, 128, (500, 20), 100, True), (5, 1000, 8, 64, (0,), 16, True)]:
        m = Model(hm, seed, 2, dim, dim, [64 * pages + n for n in lens], n_shared=pages)
        seq = np.arange(M) % len(lens)
        pos = np.array(m.lens)[seq] - 1 - (np.arange(M) % 3) * (np.arange(M) % 50)
        out.append(OnDevice(m, heads, seq, pos, m.queries(M, heads, bf16), dim**-0.5))
    return out


def test_calls_on_two_streams(hm):
    import torch

    streams, all_ = [torch.cuda.Stream(), torch.cuda.Stream()], calls(hm)
    for c in all_:
        c.run()
    torch.cuda.synchronize()
    first = [c.ob.clone() for c in all_]
    for c in all_:
        c.check(some(c.M, 7, 8))
        c.ob.fill_(5)
        c.work.fill_(255)
    torch.cuda.synchronize()
    for _ in range(5):
        for i, c in enumerate(all_):
            c.run(streams[i % 2])
    torch.cuda.synchronize()
    for c, o in zip(all_, first):  # no order of arrival changes a result
        assert torch.equal(c.ob, o)


def test_graphs_with_one_work_memory_and_positions_that_move(hm):
    """Captured calls, replayed one behind the other over the same work memory, with other queries and positions each time."""
    import torch

    all_ = calls(hm)
    work = torch.empty(max(c.size for c in all_), dtype=torch.uint8, device="cuda")
    graphs, stream = [], torch.cuda.Stream()
    for c in all_:
        c.run()
    torch.cuda.synchronize()
    for c in all_:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            c.run(stream, work)
        graphs.append(g)
    rng = np.random.default_rng(0)
    for turn in range(3):
        for c in all_:
            n = np.array(c.m.lens)[c.seq]
            c.pos = n - 1 - (rng.random(c.M) ** 4 * (n + 1)).astype(int)
            c.q = c.m.queries(c.M, c.heads, c.bf16)
            c.pd.copy_(torch.from_numpy(c.pos.astype(np.int32)))
            c.qd.copy_(torch.from_numpy(c.q))
        work.fill_(255)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for c in all_:
            c.check(some(c.M, turn, 6))


# ---- a run of the operators together --------------------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
def test_a_prompt_in_portions(hm, bf16):
    """Rotary positions, the write and the attention of two portions of a prompt, large enough for its pages to be taken on their own, captured once a portion; then a row behind them."""
    import torch

    heads, kvh, dim, n = 8, 2, 64, 1200
    t, dt, size, width = (torch.uint16, hm.DType.BF16, 2, (heads + 2 * kvh) * dim) if bf16 else (torch.float32, hm.DType.F32, 4, (heads + 2 * kvh) * dim)
    rng = np.random.default_rng(5)
    turns, mult = hm.rope_turns(1e6, dim, "bands", factor=4.0, original=256)
    pages = -(-(n + 1) // 64)
    table = rng.permutation(pages).reshape(1, pages).astype(np.int32)
    own = hm.KV8Cache(kvh, dim, dim, None, pages, table)
    td, turns_d = torch.from_numpy(table).cuda(), torch.from_numpy(turns).cuda()
    cache = hm.KV8Cache(kvh, dim, dim, own.c.pages, pages, (td.data_ptr(), 1, pages))
    stream = torch.cuda.Stream()
    x = rng.standard_normal((n + 1, width)).astype(np.float32)
    bits = bf16_bits(x) if bf16 else x
    x = bf16_value(bits) if bf16 else x
    y = turned(x[:, : (heads + kvh) * dim], heads + kvh, dim, turns, np.arange(n + 1), dim, False, mult)[0].reshape(n + 1, heads + kvh, dim).astype(np.float32)
    y = bf16_value(bf16_bits(y)) if bf16 else y
    k, v = kc.held(y[:, heads:]).astype(np.float64), kc.held(x[:, (heads + kvh) * dim :].reshape(n + 1, kvh, dim)).astype(np.float64)
    keep = []
    for first, M in ((0, 700), (700, 500), (1200, 1)):
        d, sd, pd = torch.from_numpy(bits[first : first + M]).cuda(), torch.zeros(M, dtype=torch.int32, device="cuda"), torch.arange(first, first + M, dtype=torch.int32, device="cuda")
        out = torch.zeros(M, heads * dim, dtype=t, device="cuda")
        work = torch.empty(cache.attend_bytes(M, heads, pages), dtype=torch.uint8, device="cuda")
        assert M == 1 or on_their_own(cache, M, heads, pages)
        torch.cuda.synchronize()
        g, at = torch.cuda.CUDAGraph(), d.data_ptr()
        with torch.cuda.graph(g, stream=stream):
            s = stream.cuda_stream
            hm.rope((at, M), heads + kvh, dim, turns_d.data_ptr(), pd.data_ptr(), magnitude=mult, dtype=dt, ldx=width, y=at, ldy=width, stream=s)
            cache.write((at + heads * dim * size, M), at + (heads + kvh) * dim * size, sd.data_ptr(), pd.data_ptr(), dtype=dt, ldk=width, ldv=width, stream=s)
            cache.attend((at, M), sd.data_ptr(), pd.data_ptr(), heads, dim**-0.5, shared=(td.data_ptr(), pages), dtype=dt, ldq=width, out=out.data_ptr(), work=work.data_ptr(), stream=s)
        g.replay()
        torch.cuda.synchronize()
        keep.append((g, d, sd, pd, work))
        o = out.cpu().numpy()
        o = bf16_value(o) if bf16 else o
        for r in some(M, first, 10) if M > 1 else [0]:
            p = first + r
            want, tol = formula(y[p, :heads].astype(np.float64), k[: p + 1], v[: p + 1], dim**-0.5, bf16, p + 1)
            _, (mag, terms, _, _) = kc.attention(y[p, :heads].astype(np.float64), k[: p + 1], v[: p + 1], dim**-0.5)
            # turned elements may fall on the other side of a rounding (bf16 rows: 2^-7 of a product), and codes too: a step, 1 / 127 of the largest, for every element of a key; a weight
            # is off by twice what its score is
            off = dim**-0.5 * np.abs(y[p, :heads]).sum(-1) * np.abs(k[: p + 1]).max() / 127 + terms * (2.0**-7 if bf16 else 2.0**-18)
            assert (np.abs(o[r].reshape(heads, dim) - want) <= tol + mag * np.expm1(2 * off)[:, None]).all(), p
