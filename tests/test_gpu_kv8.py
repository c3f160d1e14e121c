"""The 8-bit paged cache and attention over it, against the formulas in 64 bits."""
import numpy as np
import pytest

import kv8_cases as kc
from conftest import record_error
from kv8_cases import Model, bf16_bits, bf16_value

pytestmark = pytest.mark.gpu


# ---- the cache --------------------------------------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,kv_heads,dim,vdim", [(1, 1, 1, 1), (5, 2, 64, 64), (130, 1, 128, 128), (67, 3, 33, 80), (9, 8, 256, 7), (64, 2, 20, 255), (2, 1, 32, 30), (300, 2, 96, 64)])
def test_rows_come_back_as_the_formula_says(hm, M, kv_heads, dim, vdim, bf16):
    m = Model(hm, M + dim, kv_heads, dim, vdim, [0, 0], max_pages=1)
    pages = -(-M // 64) + 1
    pool = hm.DeviceBuffer(hm.kv8_pool_bytes(kv_heads, dim, vdim, 2 * pages))
    table = m.rng.permutation(2 * pages).reshape(2, pages)
    cache = hm.KV8Cache(kv_heads, dim, vdim, pool.ptr, 2 * pages, table)
    k, v = m.rows(M)
    k[0] *= 1e-20
    v[M // 2] *= 1e30
    seq, pos = m.rng.integers(0, 2, M), m.rng.permutation(64 * pages)[:M]
    if bf16:
        kb, vb = bf16_bits(k).reshape(M, -1), bf16_bits(v).reshape(M, -1)
        k, v = bf16_value(kb).reshape(k.shape), bf16_value(vb).reshape(v.shape)
        cache.write(kb, vb, seq, pos)
    else:
        cache.write(k.reshape(M, -1), v.reshape(M, -1), seq, pos)
    for got, x in zip(cache.read(seq, pos), (k, v)):
        np.testing.assert_array_equal(got.reshape(x.shape), kc.held(x))
    for got, x in zip(cache.read(seq, pos, dtype=hm.DType.BF16), (k, v)):
        np.testing.assert_array_equal(got.reshape(x.shape), bf16_bits(kc.held(x)))


def test_zeros_infinities_nan_and_the_smallest_values(hm):
    pool = hm.DeviceBuffer(hm.kv8_pool_bytes(1, 48, 48, 1))
    cache = hm.KV8Cache(1, 48, 48, pool.ptr, 1, [[0]])
    rng = np.random.default_rng(0)
    x = rng.standard_normal((9, 48)).astype(np.float32)
    x[0] = 0
    x[1, 3] = np.inf
    x[2, 47] = np.nan
    x[3] *= np.float32(2.0**-103) / np.abs(x[3]).max()
    x[4] *= np.float32(2.0**-100) / np.abs(x[4]).max()
    x[5] *= np.float32(3e38) / np.abs(x[5]).max()
    x[6, 1] = -np.inf
    x[7] = -0.0
    x[8] = np.float32(1e-45)
    cache.write(x, x[::-1].copy(), np.zeros(9), np.arange(9))
    k, v = cache.read(np.zeros(9), np.arange(9))
    np.testing.assert_array_equal(k, kc.held(x))
    np.testing.assert_array_equal(v, kc.held(x[::-1]))
    assert np.isnan(k[[1, 2, 6]]).all() and (k[[0, 3, 7, 8]] == 0).all() and (k[4] != 0).any()


def test_rows_without_a_place(hm):
    """Sequences, positions and pages out of range: nothing is written, and nothing is read."""
    n = 4
    pool = hm.DeviceBuffer(hm.kv8_pool_bytes(2, 64, 64, n))
    pool.upload(np.full(pool.nbytes, 7, np.uint8))
    before = pool.download(np.uint8, pool.nbytes)
    cache = hm.KV8Cache(2, 64, 64, pool.ptr, n, [[0, -1, n, 2**31 - 1], [-(2**31), 1, 2, 3]])
    seq = np.array([-1, 2, 0, 0, 0, 1, 1, 0, 0, -(2**31), 2**31 - 1])
    pos = np.array([0, 0, 64, 128, 192, 63, 256, -1, 2**31 - 1, 5, 5])
    x = np.ones((len(seq), 128), np.float32)
    cache.write(x, x, seq, pos)
    assert (pool.download(np.uint8, pool.nbytes) == before).all()
    k, v = cache.read(seq, pos)
    assert (k == 0).all() and (v == 0).all()  # the host form's arrays start with zeros


# ---- attention --------------------------------------------------------------------------------------


def attend(m, row_seq, row_pos, heads, bf16, scale=None, shared=False, seen=None, what="kv8 attention"):
    M = len(row_seq)
    scale = m.dim**-0.5 if scale is None else scale
    q = m.queries(M, heads, bf16)
    out = m.cache.attend(q, row_seq, row_pos, heads, scale, shared=m.shared if shared else None)
    worst = m.check(out, q, row_seq, row_pos, heads, scale, seen, shared)
    record_error(f"{what} {'bf16' if bf16 else 'f32'}, of the bound", worst, 1.0)
    return q, out


SIZES = [  # heads, kv_heads, dim, vdim
    (14, 2, 64, 64), (12, 2, 128, 128), (32, 4, 64, 64), (16, 8, 128, 128), (8, 8, 32, 32), (1, 1, 1, 1), (3, 1, 80, 48), (24, 2, 192, 128), (16, 1, 256, 256), (34, 2, 33, 255), (5, 5, 255, 31), (2, 1, 96, 96),
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,vdim", SIZES)
def test_uneven_contexts(hm, heads, kv_heads, dim, vdim, bf16):
    lens = [1, 64, 65, 0, 127, 200, 63, 2, 513]
    m = Model(hm, dim + vdim, kv_heads, dim, vdim, lens)
    attend(m, np.arange(len(lens)), np.array(lens) - 1, heads, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("length", [1, 31, 32, 33, 64, 300, 4097, 20000])
def test_one_row(hm, length, bf16):
    m = Model(hm, length, 2, 64, 64, [length])
    attend(m, [0], [length - 1], 14, bf16)


def test_many_rows_of_one_token_and_of_none(hm):
    lens = [1] * 300 + [0] * 300
    m = Model(hm, 1, 1, 32, 32, lens)
    attend(m, np.arange(600), np.array(lens) - 1, 2, False)


def test_rows_of_one_sequence_and_positions_inside_it(hm):
    """Rows in any order, some of one sequence, some at positions in front of its last."""
    m = Model(hm, 5, 2, 64, 64, [300, 100])
    attend(m, [0, 1, 0, 0, 1, 0], [299, 0, 17, 64, 99, 63], 8, False)


def test_positions_behind_the_table_mean_its_last(hm):
    m = Model(hm, 6, 1, 64, 64, [128, 128])
    q, out = attend(m, [0, 1, 0], [127, 127, 127], 4, False)
    np.testing.assert_array_equal(m.cache.attend(q, [0, 1, 0], [128, 2**31 - 1, 1000000], 4, 0.125), out)
    low = m.cache.attend(q, [0, 1, 0], [-1, -2, -(2**31)], 4, 0.125)
    assert (low == 0).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_pages_that_are_not_there(hm, bf16):
    m = Model(hm, 7, 2, 128, 64, [500, 200, 64])
    gone = {0: [1, 4], 1: [0], 2: [0]}
    for i, pages in gone.items():
        for p, bad in zip(pages, [-1, m.n_pages]):
            m.table[i, p] = bad
    m.cache = hm.KV8Cache(2, 128, 64, m.pool.ptr, m.n_pages, m.table)
    attend(m, [0, 1, 2, 0], [499, 199, 63, 100], 8, bf16, seen=lambda i: ~np.isin(np.arange(m.lens[i]) // 64, gone[i]))


def test_rows_of_no_sequence_stay_as_they_are(hm):
    import torch

    m = Model(hm, 8, 2, 64, 64, [70, 130])
    seq, pos = torch.tensor([-1, 0, 2, 1, -(2**31), 2**31 - 1], dtype=torch.int32).cuda(), torch.tensor([5, 69, 5, 129, 0, 0], dtype=torch.int32).cuda()
    q = torch.randn(6, 8 * 64, device="cuda")
    out = torch.full((6, 8 * 64 + 5), 7.0, device="cuda")
    table = torch.from_numpy(m.table).cuda()
    cache = hm.KV8Cache(2, 64, 64, m.pool.ptr, m.n_pages, (table.data_ptr(), 2, m.table.shape[1]))
    work = torch.empty(cache.attend_bytes(6, 8), dtype=torch.uint8, device="cuda")
    cache.attend((q.data_ptr(), 6), seq.data_ptr(), pos.data_ptr(), 8, 0.125, out=out.data_ptr(), ldo=8 * 64 + 5, work=work.data_ptr())
    torch.cuda.synchronize()
    o = out.cpu().numpy()
    assert (o[:, 512:] == 7).all() and (o[[0, 2, 4, 5]] == 7).all()
    m.check(o[:, :512], q.cpu().numpy(), [-1, 0, 2, 1, -1, -1], [5, 69, 5, 129, 0, 0], 8, 0.125)


@pytest.mark.parametrize("bf16", [False, True])
def test_nan_and_infinity_stay_where_they_are_seen(hm, bf16):
    """A vector with one is NaN as a whole; rows that do not see it are as without it."""
    m = Model(hm, 9, 1, 64, 64, [200, 200])
    seq, pos = np.array([0, 0, 1, 1, 0]), np.array([149, 150, 199, 30, 99])
    q, clean = attend(m, seq, pos, 4, bf16)
    bad = m.k[0][150].copy(), m.v[1][40].copy()
    bad[0][0, 5], bad[1][0, 60] = np.nan, np.inf
    m.cache.write(bad[0], m.v[0][150], [0], [150])
    m.cache.write(m.k[1][40], bad[1], [1], [40])
    out = m.cache.attend(q, seq, pos, 4, 0.125)
    f = bf16_value(out) if bf16 else out
    assert np.isnan(f[[1, 2]]).all()
    np.testing.assert_array_equal(out[[0, 3, 4]], clean[[0, 3, 4]])


@pytest.mark.parametrize("bf16", [False, True])
def test_large_and_small_scales(hm, bf16):
    """Values of very different sizes in one context, queries whose scores spread over hundreds, tokens of zeros."""
    m = Model(hm, 10, 2, 64, 64, [400])
    for i in range(400):
        m.v[0][i] *= np.float32(10.0 ** ((i * 7) % 13 - 6))
        if i % 11 == 0:
            m.k[0][i] = 0
        if i % 17 == 0:
            m.v[0][i] = 0
    m.fill()
    attend(m, [0, 0, 0], [399, 350, 10], 8, bf16, scale=3.0)
    attend(m, [0], [399], 8, bf16, scale=0.0)
    attend(m, [0], [399], 8, bf16, scale=-0.1)


# ---- shared pages -----------------------------------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,vdim", SIZES)
def test_a_shared_prefix(hm, heads, kv_heads, dim, vdim, bf16):
    S = 3 * 64
    lens = [S + 1, S, S + 64, S + 100, S + 400, S + 65]
    m = Model(hm, dim, kv_heads, dim, vdim, lens, n_shared=3)
    m.table[:, :3] = -1  # what the table says in their place is not looked at
    m.cache = hm.KV8Cache(kv_heads, dim, vdim, m.pool.ptr, m.n_pages, m.table)
    attend(m, np.arange(6), np.array(lens) - 1, heads, bf16, shared=True, what="kv8 shared prefix")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,pages", [(1, 1), (2, 40), (17, 7), (33, 2), (64, 20), (130, 1), (200, 9)])
def test_rows_behind_a_shared_prefix(hm, M, pages, bf16):
    """Own parts of no token, of one, of many; rows that end inside the prefix."""
    rng = np.random.default_rng(M)
    S = 64 * pages
    lens = [S + int(n) for n in rng.choice([0, 1, 5, 63, 64, 130], M)]
    m = Model(hm, M + pages, 2, 64, 64, lens, n_shared=pages)
    pos = np.array(lens) - 1
    pos[::7] = rng.integers(-1, S, len(pos[::7]))
    attend(m, np.arange(M), pos, 8, bf16, shared=True, what="kv8 shared prefix")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,first,rows", [(12, 2, 128, 0, 130), (12, 2, 128, 77, 64), (14, 2, 64, 1000, 100), (4, 1, 80, 63, 2), (16, 1, 256, 5, 40), (8, 8, 64, 640, 129)])
def test_a_portion_of_a_prompt(hm, heads, kv_heads, dim, first, rows, bf16):
    """All rows in one sequence whose pages are all shared: each sees the positions up to its own."""
    n = first + rows
    m = Model(hm, n, kv_heads, dim, dim, [n], n_shared=-(-n // 64))
    m.k[0], m.v[0] = m.common[0][:n], m.common[1][:n]
    m.lens = [n]
    attend(m, np.zeros(rows, int), first + np.arange(rows), heads, bf16, shared=True, what="kv8 prompt")


@pytest.mark.parametrize("bf16", [False, True])
def test_missing_pages_in_a_shared_prefix(hm, bf16):
    m = Model(hm, 11, 2, 64, 64, [64 * 5 + 30] * 20, n_shared=5)
    good, m.shared = m.shared, m.shared.copy()
    m.shared[[0, 3]] = [-1, m.n_pages]
    attend(m, np.arange(20), np.arange(20) * 17 + 10, 8, bf16, shared=True, seen=lambda i: ~np.isin(np.arange(m.lens[i]) // 64, [0, 3]))
    m.shared[:] = -1
    attend(m, np.arange(20), np.full(20, 300), 8, bf16, shared=True, seen=lambda i: np.arange(m.lens[i]) >= 320)


def test_shared_rows_of_no_sequence_and_nan_behind_a_row(hm):
    """Padded rows stay out; a NaN that only later rows of a prompt see leaves the earlier ones alone."""
    m = Model(hm, 12, 1, 64, 64, [200], n_shared=4)
    m.k[0], m.v[0] = m.common[0][:200], m.common[1][:200]
    q, clean = attend(m, np.zeros(200, int), np.arange(200), 4, False, shared=True)
    bad = m.v[0][150].copy()
    bad[0, 3] = np.inf
    m.cache.write(m.k[0][150], bad, [0], [150])
    out = m.cache.attend(q, np.zeros(200, int), np.arange(200), 4, 0.125, shared=m.shared)
    assert np.isnan(out[150:]).all() and np.isfinite(out[:150]).all()
    m.check(out[:150], q[:150], np.zeros(150, int), np.arange(150), 4, 0.125, shared=True)
    seq = np.where(np.arange(200) % 3 == 0, -1, 0)
    out = m.cache.attend(q[:150], seq[:150], np.arange(150), 4, 0.125, shared=m.shared)
    assert (out[0::3] == 0).all()
    m.check(out, q[:150], seq[:150], np.arange(150), 4, 0.125, shared=True)
