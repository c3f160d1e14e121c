"""Calls of the image entry points that cannot be answered, refused on the host before a device is asked."""
import ctypes as C

import numpy as np
import pytest

F32, BF16, MX = 0, 1, 10


@pytest.fixture
def memory():
    raw = np.zeros((1 << 16) + 16, np.uint8)
    return raw[-raw.ctypes.data % 16 :]


def at(memory, offset=0):
    return C.c_void_p(memory.ctypes.data + offset)


def test_bf16_sums_over_the_residual(hm, memory):
    """A bf16 row takes half the room of its f32 residual: written over it, a token's results would land in residuals that other tokens still read."""
    lib = hm.load_library()
    T, W, p = 4, 8, at(memory)
    rows, ids, weights = at(memory, 4096), at(memory, 8192), at(memory, 12288)
    call = lambda resid, y, dtype: lib.hm_expert_sum(rows, F32, ids, weights, T, 1, 4, W, resid, y, dtype, None)
    for y in [p, at(memory, 4 * W * T - 2), at(memory, 64)]:
        assert call(p, y, BF16) == hm.HM_ERR_INVALID
    assert call(at(memory, 2 * W * T - 4), p, BF16) == hm.HM_ERR_INVALID
    if not hm.device_count():
        assert call(p, p, F32) == hm.HM_ERR_CUDA  # y may be resid
        assert call(p, at(memory, 4 * W * T), BF16) == hm.HM_ERR_CUDA
        assert call(at(memory, 2 * W * T), p, BF16) == hm.HM_ERR_CUDA
        assert call(None, p, BF16) == hm.HM_ERR_CUDA


def test_rows_too_far_apart_to_count(hm, memory):
    """Rows so far apart that their bytes do not fit 64 bits: the room of host rows was the remainder."""
    lib, INV, p = hm.load_library(), hm.HM_ERR_INVALID, at(memory)
    for ld in [2**64 - 64, 2**62, 2**60]:
        assert lib.hm_image_pack(p, F32, 5, 32, ld, 0, MX, p, None) == INV
        assert lib.hm_image_unpack(p, MX, 5, 32, p, F32, ld, None) == INV
        assert lib.hm_gemv_mx4(p, F32, ld, p, 5, 32, 8, p, F32, 8, None) == INV
        assert lib.hm_gemv_mx4(p, F32, 32, p, 5, 32, 8, p, F32, ld, None) == INV
        assert lib.hm_expert_pack(p, F32, 32, ld, 0, p, 4, 4, 2, MX, p, None) == INV
        assert lib.hm_expert_gemv(p, F32, ld, p, p, 4, 1, 4, 32, 8, p, F32, 8, None) == INV
        assert lib.hm_expert_gemv(p, F32, 32, p, p, 4, 1, 4, 32, 8, p, F32, ld, None) == INV
    if not hm.device_count():
        assert lib.hm_image_pack(p, F32, 1, 32, 2**40, 0, MX, p, None) == hm.HM_ERR_CUDA


def test_sums_of_rows_as_wide_as_int_goes(hm, memory):
    """The number of blocks over a row of nearly 2^31 values was counted in an int that does not hold it."""
    lib, p = hm.load_library(), at(memory)
    for W in [2**31 - 1, 2**31 - 255]:
        assert lib.hm_expert_sum(p, F32, p, p, 1, 1, 4, W, None, p, F32, None) == hm.HM_ERR_INVALID
    if not hm.device_count():
        assert lib.hm_expert_sum(p, F32, p, p, 1, 1, 4, 2**31 - 256, None, p, F32, None) == hm.HM_ERR_CUDA
