"""Rows of the 8-bit cache's host forms and refusals that need no GPU."""
import ctypes as C

import numpy as np
import pytest

INV = 1


def test_keys_and_values_that_overlap_are_not_read(hm):
    raw = np.zeros(1 << 16, np.uint8)
    base = raw.ctypes.data + -raw.ctypes.data % 16
    c = hm.HmKv8(base, base + 4096, 4, 2, 2, 2, 64, 32)  # keys 128 wide, values 64
    lib = hm.load_library()
    read = lambda k, v, ldk, ldv, M=3: lib.hm_kv8_read(C.byref(c), C.c_void_p(base + 32768), C.c_void_p(base + 36864), M, C.c_void_p(k), C.c_void_p(v), 0, ldk, ldv, None)
    at = base + 8192
    for k, v, ldk, ldv in [(at, at, 192, 192), (at, at + 508, 192, 192), (at + 4, at, 192, 192), (at, at + 256, 128, 64), (at, at + 3 * 512 - 4, 128, 64), (at, at + 512, 192, 193)]:
        assert read(k, v, ldk, ldv) == INV, (k - at, v - at, ldk, ldv)
    if not hm.device_count():
        for k, v, ldk, ldv in [(at, at + 512, 192, 192), (at + 256, at, 192, 192), (at, at + 3 * 512, 128, 64)]:
            assert read(k, v, ldk, ldv) == hm.HM_ERR_CUDA, (k - at, v - at, ldk, ldv)
    assert read(at, at, 192, 192, M=0) == 0


FAR = [2**31, 2**32, 2**32 + 1, 2**40 + 3, -(2**31) - 1, -(2**32), -(2**32) + 1]


@pytest.mark.parametrize("kind", [np.int64, np.float64, object])
def test_pages_beyond_32_bits_are_no_pages(hm, kind):
    table = np.array([[0, *FAR, 3], [1, *FAR[::-1], -1]], dtype=kind)
    c = hm.KV8Cache(2, 64, 32, 16, 4, table).c
    held = np.ctypeslib.as_array(C.cast(c.page_table, C.POINTER(C.c_int32)), (2, table.shape[1]))
    near = np.array([[x < 2**31 and x >= -(2**31) for x in row] for row in table.tolist()])
    assert (held[near] == table[near].astype(np.int64)).all()
    assert ((held[~near] < 0) | (held[~near] >= 4)).all()
    table[:] = 2  # the cache has a copy
    assert held[0, 0] == 0
    assert hm.KV8Cache(1, 64, 32, 16, 4, np.array([[3, 2**40]], np.uint64)).c.max_pages == 2


def test_rotary_positions_beyond_32_bits_are_refused(hm):
    x = np.zeros((2, 8), np.float32)
    for far in FAR + [np.nan]:
        with pytest.raises(hm.HomuraError) as e:
            hm.rope(x, 1, 8, np.zeros(4), [0, far])
        assert e.value.status == INV
