"""Calls of the rotary and 8-bit cache entry points that need no GPU: sizes, frequencies, refusals."""
import ctypes as C
import math

import numpy as np
import pytest

F32, BF16 = 0, 1
INV, UNS = 1, 5


def formula(theta, rot, kind, factor, a, b, original):
    out = []
    for i in range(rot // 2):
        f = theta ** (-2 * i / rot)
        wave = 2 * math.pi / f
        if kind == "linear":
            f /= factor
        elif kind == "bands":
            if wave > original / a:
                f /= factor
            elif wave >= original / b:
                s = (original / wave - a) / (b - a)
                f = (1 - s) * f / factor + s * f
        elif kind == "yarn":
            at = lambda times: rot * math.log(original / (times * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(at(b)), 0), min(math.ceil(at(a)), rot - 1)
            r = min(max((i - lo) / max(hi - lo, 0.001), 0), 1)
            f = f / factor * r + f * (1 - r)
        out.append(f / (2 * math.pi))
    return np.array(out)


@pytest.mark.parametrize("rot", [0, 2, 32, 64, 128, 1024])
@pytest.mark.parametrize("kind,a,b", [("plain", 1, 4), ("linear", 1, 4), ("bands", 1, 4), ("yarn", 1, 32), ("yarn", 1, 1.5)])
def test_frequencies(hm, rot, kind, a, b):
    for theta, original, factor in [(1e4, 4096, 4.0), (5e5, 8192, 8.0), (1e6, 32768, 1.5)]:
        names = dict(slow=a, fast=b) if kind == "yarn" else dict(low=a, high=b)
        got, mult = hm.rope_turns(theta, rot, kind, factor=factor, original=original, **names)
        assert len(got) == rot // 2
        np.testing.assert_allclose(got, formula(theta, rot, kind, factor, a, b, original), rtol=4e-15)
        assert mult == np.float32(0.1 * math.log(factor) + 1 if kind == "yarn" else 1)


def test_frequencies_that_are_refused(hm):
    lib = hm.load_library()
    t = np.zeros(64)
    call = lambda theta=1e4, rot=8, kind=0, factor=2.0, low=1.0, high=4.0, original=4096.0: lib.hm_rope_turns(theta, rot, kind, factor, low, high, original, t.ctypes.data_as(C.c_void_p), None)
    assert call() == 0
    for bad in [dict(theta=0.0), dict(theta=-1.0), dict(theta=math.nan), dict(theta=math.inf), dict(rot=-2), dict(rot=7), dict(rot=1026), dict(kind=1, factor=0.0), dict(kind=1, factor=math.nan), dict(kind=2, original=0.0),
                dict(kind=2, low=4.0), dict(kind=3, low=0.0), dict(kind=3, high=math.inf), dict(kind=3, theta=1.0)]:
        assert call(**bad) == INV, bad
    assert call(kind=4) == UNS and call(kind=-1) == UNS
    assert lib.hm_rope_turns(1e4, 8, 0, 1.0, 1.0, 4.0, 0.0, None, None) == INV
    with pytest.raises(hm.HomuraError):
        hm.rope_turns(1e4, 8, "other")


def test_pool_sizes(hm):
    assert hm.kv8_pool_bytes(2, 64, 64, 10) == 10 * 2 * 64 * (8 + 128)
    assert hm.kv8_pool_bytes(1, 1, 33, 1) == 64 * (8 + 32 + 64)
    assert hm.kv8_pool_bytes(1024, 256, 256, 2**31 - 1) == (2**31 - 1) * 1024 * 64 * 520
    for bad in [(0, 64, 64, 1), (1025, 64, 64, 1), (1, 0, 64, 1), (1, 257, 64, 1), (1, 64, 0, 1), (1, 64, 257, 1), (1, 64, 64, 0), (-1, 64, 64, 1), (1, 64, 64, -5)]:
        assert hm.kv8_pool_bytes(*bad) == 0
        with pytest.raises(hm.HomuraError):
            hm.KV8Cache(*bad[:3], 16, bad[3], [[0]])


@pytest.fixture
def memory():
    raw = np.zeros((1 << 16) + 16, np.uint8)
    return raw[-raw.ctypes.data % 16 :]


def at(memory, offset=0):
    return C.c_void_p(memory.ctypes.data + offset)


def test_rope_refusals(hm, memory):
    lib, p = hm.load_library(), at(memory)
    ok = dict(x=p, dtype=F32, ldx=128, M=4, heads=2, dim=64, rot=64, neighbours=0, pos=at(memory, 8192), turns=at(memory, 8448), mult=1.0, y=at(memory, 16384), ldy=128)
    call = lambda **kw: lib.hm_rope(*{**ok, **kw}.values(), None)
    for bad in [dict(x=None), dict(y=None), dict(pos=None), dict(turns=None), dict(M=-1), dict(heads=0), dict(heads=65537, ldx=2**30, ldy=2**30), dict(dim=0), dict(dim=1025), dict(rot=-2), dict(rot=66), dict(rot=3), dict(ldx=127), dict(ldy=127),
                dict(ldx=2**62), dict(x=at(memory, 2)), dict(y=at(memory, 16386)), dict(pos=at(memory, 8193)), dict(turns=at(memory, 8452)),
                dict(y=p, ldy=256), dict(y=at(memory, 4)), dict(y=at(memory, 4 * 128 * 4 - 4)), dict(x=at(memory, 256), y=p, ldx=256, ldy=256)]:
        assert call(**bad) == INV, bad
    assert call(dtype=2) == UNS and call(dtype=3) == UNS
    assert call(M=0) == 0
    if not hm.device_count():
        for fine in [dict(), dict(y=p), dict(rot=0, turns=None), dict(y=at(memory, 4 * 128 * 4)), dict(y=at(memory, 512), ldx=256, ldy=256), dict(dtype=BF16, x=at(memory, 2))]:
            assert call(**fine) == hm.HM_ERR_CUDA, fine


def cache(hm, memory, **kw):
    return hm.HmKv8(**{**dict(pages=memory.ctypes.data, page_table=memory.ctypes.data + 4096, n_pages=4, n_seq=2, max_pages=2, kv_heads=2, dim=64, vdim=32), **kw})


BAD_CACHES = [dict(pages=None), dict(page_table=None), dict(n_pages=0), dict(n_pages=-1), dict(n_seq=0), dict(max_pages=0), dict(max_pages=2**24 + 1), dict(kv_heads=0), dict(kv_heads=1025), dict(dim=0), dict(dim=257), dict(vdim=0), dict(vdim=257)]


def test_cache_row_refusals(hm, memory):
    lib, p = hm.load_library(), at(memory, 8192)
    ok = dict(k=p, v=at(memory, 16384), dtype=F32, ldk=128, ldv=64, seq=at(memory, 32768), pos=at(memory, 36864), M=3)

    def calls(c, **kw):
        a = {**ok, **kw}
        ref = C.byref(c) if c is not None else None
        w = lib.hm_kv8_write(ref, a["k"], a["v"], a["dtype"], a["ldk"], a["ldv"], a["seq"], a["pos"], a["M"], None)
        r = lib.hm_kv8_read(ref, a["seq"], a["pos"], a["M"], a["k"], a["v"], a["dtype"], a["ldk"], a["ldv"], None)
        assert w == r
        return w

    good = cache(hm, memory)
    assert calls(None) == INV
    for bad in BAD_CACHES + [dict(pages=memory.ctypes.data + 8), dict(page_table=memory.ctypes.data + 2)]:
        assert calls(cache(hm, memory, **bad)) == INV, bad
    for bad in [dict(k=None), dict(v=None), dict(seq=None), dict(pos=None), dict(M=-1), dict(M=2**30), dict(ldk=127), dict(ldv=63), dict(ldk=2**61), dict(k=at(memory, 8194)), dict(v=at(memory, 16385)), dict(seq=at(memory, 32770)), dict(pos=at(memory, 36865))]:
        assert calls(good, **bad) == INV, bad
    assert calls(good, dtype=2) == UNS and calls(good, dtype=3) == UNS
    assert calls(good, M=0) == 0
    if not hm.device_count():
        assert calls(good) == hm.HM_ERR_CUDA


def test_attention_refusals(hm, memory):
    lib = hm.load_library()
    ok = dict(q=at(memory, 8192), dtype=F32, ldq=256, seq=at(memory, 32768), pos=at(memory, 36864), M=3, heads=4, scale=0.125, shared=None, n_shared=0, out=at(memory, 16384), ldo=128, work=None)
    call = lambda c, **kw: lib.hm_kv8_attn(C.byref(c) if c is not None else None, *{**ok, **kw}.values(), None)
    good = cache(hm, memory)
    assert call(None) == INV
    for bad in BAD_CACHES + [dict(pages=memory.ctypes.data + 8), dict(page_table=memory.ctypes.data + 2)]:
        assert call(cache(hm, memory, **bad)) == INV, bad
    for bad in [dict(q=None), dict(out=None), dict(seq=None), dict(pos=None), dict(M=-1), dict(M=8193), dict(heads=0), dict(heads=3), dict(heads=4098, ldq=2**20, ldo=2**20), dict(scale=math.nan), dict(scale=math.inf), dict(n_shared=-1), dict(n_shared=1),
                dict(n_shared=3, shared=at(memory, 40960)), dict(ldq=255), dict(ldo=127), dict(ldq=2**61), dict(q=at(memory, 8193)), dict(out=at(memory, 16386)), dict(shared=at(memory, 40961), n_shared=1), dict(work=at(memory, 49160)),
                dict(out=at(memory, 8192)), dict(out=at(memory, 8192 + 3 * 256 * 4 - 4))]:
        assert call(good, **bad) == INV, bad
    assert call(good, dtype=2) == UNS
    assert call(good, M=0) == 0
    # results beside the queries in one row: not an overlap
    beside = dict(ldq=384, ldo=384, out=at(memory, 8192 + 1024))
    if not hm.device_count():
        for fine in [dict(), beside, dict(n_shared=2, shared=at(memory, 40960))]:
            assert call(good, **fine) == hm.HM_ERR_CUDA, fine
    assert call(good, **{**beside, "ldo": 385}) == INV
    assert call(good, **{**beside, "out": at(memory, 8192 + 1020)}) == INV


def test_work_memory(hm, memory):
    c = cache(hm, memory)
    lib = hm.load_library()
    size = lambda M, heads, n: lib.hm_kv8_attn_bytes(C.byref(c), M, heads, n)
    assert size(1, 4, 0) > 0 and size(8192, 4096, 2) > 0
    assert lib.hm_kv8_attn_bytes(None, 1, 4, 0) == 0
    for bad in [(-1, 4, 0), (8193, 4, 0), (1, 3, 0), (1, 0, 0), (1, 4, 3), (1, 4, -1)]:
        assert size(*bad) == 0


def test_python_forms_refuse_what_does_not_fit(hm):
    with pytest.raises(hm.HomuraError):
        hm.rope(np.zeros((2, 10), np.float32), 1, 8, np.zeros(4), [0, 1])
    with pytest.raises(hm.HomuraError):
        hm.rope(np.zeros((2, 8), np.float32), 1, 8, np.zeros(3), [0, 1])
    with pytest.raises(hm.HomuraError):
        hm.rope(np.zeros((2, 8), np.float32), 1, 8, np.zeros(4), [0])
    c = hm.KV8Cache(2, 64, 32, 16, 4, [[0, 1]])
    rows = lambda *s: np.zeros(s, np.float32)
    for call in [lambda: c.write(rows(2, 128), rows(2, 64), [0], [0]), lambda: c.write(rows(2, 128), rows(1, 64), [0, 0], [0, 1]), lambda: c.write(rows(2, 127), rows(2, 64), [0, 0], [0, 1]), lambda: c.write(rows(2, 128), rows(2, 64).astype(np.uint16), [0, 0], [0, 1]),
                 lambda: c.read([0, 0], [0]), lambda: c.attend(rows(2, 255), [0, 0], [0, 1], 4, 1.0), lambda: c.attend(rows(2, 256), [0], [0, 1], 4, 1.0)]:
        with pytest.raises(hm.HomuraError):
            call()


def test_attention_over_tables_too_wide(hm, memory):
    """Rows times the table's width times heads has a limit, as the pieces of all items are counted."""
    lib = hm.load_library()
    size = lambda max_pages, M, heads: lib.hm_kv8_attn_bytes(C.byref(cache(hm, memory, max_pages=max_pages)), M, heads, 0)
    assert size(2**24, 32, 128) > 0 and size(2**24, 33, 128) == 0
    assert size(2**24, 1, 4096) > 0 and size(2**24, 2, 4096) == 0
