"""The 8-bit cache and attention over it at the ends of what their arguments may be."""
import numpy as np
import pytest

import kv8_cases as kc
from kv8_cases import Model, bf16_bits, bf16_value

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("small,large", [(-110, 112), (-99, 101), (100, -95)])
@pytest.mark.parametrize("rows,width", [(3, 3), (200, 3), (3, 100)])
def test_queries_and_keys_far_apart_in_size(hm, rows, width, small, large, bf16):
    """Products of an ordinary size: items of a CTA, of teams of warps, and cut ones."""
    m = Model(hm, rows, 1, 64, 64, [150, 40], max_pages=width)
    for k in m.k:
        k *= np.float32(2.0**large)
    m.fill()
    heads, scale = 4, 0.125 * 2.0 ** -(small + large)
    x = m.rng.standard_normal((rows, heads * 64)).astype(np.float32) * np.float32(2.0**small)
    q = bf16_bits(x) if bf16 else x
    x = bf16_value(q) if bf16 else x
    seq = np.arange(rows) % 2
    pos = np.array(m.lens)[seq] - 1
    out = m.cache.attend(q, seq, pos, heads, scale)
    o = bf16_value(out) if bf16 else out
    for r in range(min(rows, 12)):
        k, v = (kc.held(y[seq[r]]).astype(np.float64) for y in (m.k, m.v))
        want, parts = kc.attention(x[r].astype(np.float64).reshape(heads, 64), k, v, scale)
        # beside the bound of ordinary queries: a query's elements have no step below 2^-127, and its factor, about 2^-127 too, none below 2^-149: 2^-20 of a score
        off = 2 * (scale * np.abs(k).sum(-1).max() * 2.0**-128 + parts[1] * 2.0**-20)[:, None]
        assert (np.abs(o[r].reshape(heads, 64) - want) <= kc.bound(want, parts, bf16) + parts[0] * off).all(), r


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("values_first", [False, True])
@pytest.mark.parametrize("on_device", [False, True])
def test_keys_and_values_read_into_one_buffer(hm, on_device, values_first, bf16):
    """Rows of keys beside rows of values: each call brings both, and leaves what stands between and the rows without a place."""
    import ctypes as C

    import torch

    kvh, dim, vdim, M = 2, 40, 24, 9
    m = Model(hm, 3, kvh, dim, vdim, [M])
    wk, wv, pad = kvh * dim, kvh * vdim, 3
    ld = wk + wv + pad
    seq, pos = np.zeros(M, np.int32), np.arange(M, dtype=np.int32)
    seq[4] = -1
    buf = torch.full((M, ld), 5, dtype=torch.uint16 if bf16 else torch.float32, device="cuda" if on_device else "cpu")
    k_at, v_at = (wv, 0) if values_first else (0, wk)
    at = lambda i: C.c_void_p(buf.data_ptr() + i * buf.element_size())
    host = lambda x: C.c_void_p(x.ctypes.data)
    rc = hm.load_library().hm_kv8_read(C.byref(m.cache.c), host(seq), host(pos), M, at(k_at), at(v_at), 1 if bf16 else 0, ld, ld, None)
    torch.cuda.synchronize()
    assert rc == 0
    got = buf.cpu().numpy()
    for i, w, x in ((k_at, wk, m.k[0]), (v_at, wv, m.v[0])):
        want = kc.held(x).reshape(M, w)
        want = bf16_bits(want) if bf16 else want
        want[4] = 5
        np.testing.assert_array_equal(got[:, i : i + w], want)
    assert (got[:, wk + wv :] == 5).all()


def test_places_beyond_32_bits(hm):
    """Arrays of 64 bits: sequences, positions and pages beyond 32 are nobody's, behind the table, or not there."""
    rng = np.random.default_rng(0)
    k, v, q = (rng.standard_normal((n, 64)).astype(np.float32) for n in (64, 64, 3))
    cache = hm.KV8Cache(1, 64, 64, None, 2, np.array([[0], [2**32 + 1]]))
    cache.write(k, v, np.zeros(64, np.int64), np.arange(64))
    cache.write(k[:4] + 1, v[:4], np.array([2**32, 0, 0, 1]), np.array([5, 2**32 + 6, -(2**32) + 7, 8]))  # none of them has a place
    got, _ = cache.read(np.zeros(64, np.int64), np.arange(64))
    np.testing.assert_array_equal(got, kc.held(k[:, None])[:, 0])
    assert (cache.read([2**32, 0, 1], [5, 2**32 + 6, 8])[0] == 0).all()
    out = cache.attend(q, np.array([0, 2**32, 1]), np.array([2**40, 63, 63]), 1, 0.125)
    np.testing.assert_array_equal(out[0], cache.attend(q[:1], [0], [63], 1, 0.125)[0])
    assert (out[1:] == 0).all()
    np.testing.assert_array_equal(cache.attend(q[:1], [0], [63], 1, 0.125, shared=np.array([2**32])), np.zeros((1, 64), np.float32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size", [1e6, 1e9, 1e20])
@pytest.mark.parametrize("rows,width", [(20, 8), (200, 8), (20, 100)])
def test_scores_of_any_size(hm, rows, width, size, bf16):
    """Where one token's score is far above all others, by more than the scores' own roundings, the result is that token's value."""
    heads, n = 8, 500
    m = Model(hm, rows, 2, 64, 64, [n], max_pages=width)
    q = m.queries(rows, heads, bf16)
    pos = n - 1 - np.arange(rows)
    out = m.cache.attend(q, np.zeros(rows), pos, heads, size)
    x, o = (bf16_value(q), bf16_value(out)) if bf16 else (q, out)
    k, v = kc.held(m.k[0]).astype(np.float64), kc.held(m.v[0]).astype(np.float64)
    clear = 0
    for r in range(0, rows, max(1, rows // 20)):
        for h in range(heads):
            y = x[r].astype(np.float64).reshape(heads, 64)[h]
            s, terms = k[: pos[r] + 1, h // 4] @ y, (np.abs(k[: pos[r] + 1, h // 4]) @ np.abs(y)).max()
            # twice what a score may be off (bf16 queries: half of 1 / 32639 of their largest element for each), and a weight of e^-40
            off = 2 * (terms * 2.0**-21 + (np.abs(y).max() * np.abs(k[: pos[r] + 1, h // 4]).sum(-1).max() * 2.0**-15.9 if bf16 else 0))
            if s.max() - np.partition(s, -2)[-2] < 2 * off + 40 / size:
                continue
            clear += 1
            want = v[s.argmax(), h // 4]
            # a weight has 31 bits (bf16 rows: 16) of the largest product
            assert (np.abs(o[r].reshape(heads, 64)[h] - want) <= np.abs(want) * (2.0**-8 + 2.0**-14 if bf16 else 2.0**-20)).all(), (r, h)
    assert clear > 50


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("small", [-60, -85, -95, -99])
@pytest.mark.parametrize("rows,width", [(20, 8), (200, 8), (20, 100)])
def test_values_next_to_nothing(hm, rows, width, small, bf16):
    """The smallest values that the cache holds keep their weights' bits."""
    heads, n = 8, 500
    m = Model(hm, rows, 2, 64, 64, [n], max_pages=width)
    m.v[0] = m.rng.standard_normal(m.v[0].shape).astype(np.float32) * np.float32(2.0**small)
    m.fill()
    q = m.queries(rows, heads, bf16)
    pos = n - 1 - np.arange(rows)
    out = m.cache.attend(q, np.zeros(rows), pos, heads, 0.125)
    assert m.check(out, q, np.zeros(rows, int), pos, heads, 0.125) <= 1


def test_calls_of_several_threads(hm):
    """Host calls of four threads at once: writes, reads and attention of caches of their own, with and without shared pages."""
    import threading

    def work(seed, said):
        try:
            bf16, M, pages = seed % 2 == 1, 300, 22
            m = Model(hm, seed, 2, 64, 64, [64 * pages + 40 * seed, 64 * pages], n_shared=pages)
            seq, pos = np.arange(M) % 2, 64 * pages - 1 - np.arange(M)
            pos[::2] = m.lens[0] - 1
            q = m.queries(M, 8, bf16)
            first = [m.cache.attend(q, seq, pos, 8, 0.125, shared=s) for s in (m.shared, None)]
            for _ in range(6):
                for s, want in zip((m.shared, None), first):
                    np.testing.assert_array_equal(m.cache.attend(q, seq, pos, 8, 0.125, shared=s), want)
                n = m.lens[0] - 64 * pages
                if n:
                    own = np.arange(64 * pages, m.lens[0])
                    m.cache.write(m.k[0][own].reshape(n, -1), m.v[0][own].reshape(n, -1), np.zeros(n), own)
                    np.testing.assert_array_equal(m.cache.read(np.zeros(n), own)[0].reshape(n, 2, 64), kc.held(m.k[0][own]))
            said[seed] = True
        except BaseException as e:  # told by the test's own thread
            said[seed] = e

    said = {}
    threads = [threading.Thread(target=work, args=(i, said)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert [said[i] for i in range(4)] == [True] * 4
