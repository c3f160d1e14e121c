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


def calls(hm):
    out = []
    for seed, M, heads, dim, lens, pages, bf16 in [(1, 300, 8, 64, (100, 0, 9), 22, False), (2, 66, 8, 128, (0, 0), 110, False), (3, 600, 6, 64, (64, 1), 12, True), (4, 70, 8, 128, (500, 20), 100, True), (5, 1000, 8, 64, (0,), 16, True)]:
        m = Model(hm, seed, 2, dim, dim, [64 * pages + n for n in lens], n_shared=pages)
        seq = np.arange(M) % len(lens)
        pos = np.array(m.lens)[seq] - 1 - (np.arange(M) % 3) * (np.arange(M) % 50)
        out.append(OnDevice(m, heads, seq, pos, m.queries(M, heads, bf16), dim**-0.5))
    return out
