"""Operand images and grouped products without a GPU: sizes, refusals, and the numpy restatement the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import image_cases as ic


def refused(hm, status, rc):
    assert rc == status, (rc, hm.load_library().hm_last_error_global())
    assert hm.load_library().hm_last_error_global()


def test_sizes(hm):
    assert hm.image_bytes(hm.DType.MXFP4, 1, 1) == 17408 and hm.image_bytes(hm.DType.MXFP4, 129, 257) == 4 * 17408
    assert hm.image_bytes(hm.DType.BF16, 128, 64) == 16384 == 2 * hm.load_library().hm_tc_packed_elems(64, 128)
    assert hm.image_bytes(hm.DType.BF16, 129, 65) == 4 * 16384
    for dtype, rows, K in [(0, 1, 1), (3, 1, 1), (10, 0, 1), (10, 1, 0), (10, -1, 5)]:
        assert hm.image_bytes(dtype, rows, K) == 0
    assert hm.image_bytes(hm.DType.MXFP4, 2**31 - 300, 8192) == (2**31 // 128 - 2) * 32 * 17408  # beyond 32 bits
    assert hm.image_bytes(hm.DType.MXFP4, 2**31 - 1, 32) == 0 and hm.image_bytes(hm.DType.BF16, 1, 2**23 + 1) == 0  # more than a call takes
    for pairs, experts in [(0, 1), (1, 4), (5, 3), (1000, 16), (128 * 9, 8)]:
        first, count, place, row = ic.plan(np.arange(pairs) % experts, experts)
        assert hm.expert_plan_rows(pairs, experts) == row.size and row.size >= first[-1] * 128
        assert hm.expert_plan_ints(pairs, experts) == first.size + count.size + place.size + row.size
    assert hm.expert_plan_ints(5, 0) == 0 and hm.expert_plan_ints(-1, 4) == 0 and hm.expert_plan_ints(5, 1025) == 0


def test_refusals(hm):
    lib, INV, UNS = hm.load_library(), hm.HM_ERR_INVALID, hm.HM_ERR_UNSUPPORTED
    raw = np.zeros(1 << 16, np.uint8)
    raw = raw[-raw.ctypes.data % 16 :]
    p, odd = C.c_void_p(raw.ctypes.data), C.c_void_p(raw.ctypes.data + 1)
    half = C.c_void_p(raw.ctypes.data + 8)
    F32, BF16, MX, Q8 = 0, 1, 10, 3
    refused(hm, INV, lib.hm_image_pack(None, F32, 1, 32, 32, 0, MX, p, None))
    refused(hm, INV, lib.hm_image_pack(p, F32, -1, 32, 32, 0, MX, p, None))
    refused(hm, INV, lib.hm_image_pack(p, F32, 1, 0, 32, 0, MX, p, None))
    refused(hm, INV, lib.hm_image_pack(p, F32, 1, 32, 31, 0, MX, p, None))
    refused(hm, INV, lib.hm_image_pack(p, F32, 1, 32, 63, 1, MX, p, None))  # gate and up are 2 K values
    refused(hm, UNS, lib.hm_image_pack(p, Q8, 1, 32, 32, 0, MX, p, None))
    refused(hm, UNS, lib.hm_image_pack(p, F32, 1, 32, 32, 0, F32, p, None))
    refused(hm, INV, lib.hm_image_pack(odd, BF16, 1, 32, 32, 0, MX, p, None))
    refused(hm, INV, lib.hm_image_pack(p, F32, 1, 32, 32, 0, MX, half, None))
    refused(hm, INV, lib.hm_image_unpack(p, MX, 1, 32, p, F32, 31, None))
    refused(hm, UNS, lib.hm_image_unpack(p, Q8, 1, 32, p, F32, 32, None))
    refused(hm, INV, lib.hm_image_from_blocks(p, 1, 48, p, None))
    refused(hm, INV, lib.hm_gemm_image(p, p, MX, 1, 32, 0, p, F32, 8, None))
    refused(hm, INV, lib.hm_gemm_image(p, p, MX, 1, 32, 8, p, F32, 7, None))
    refused(hm, UNS, lib.hm_gemm_image(p, p, F32, 1, 32, 8, p, F32, 8, None))
    refused(hm, UNS, lib.hm_gemm_image(p, p, MX, 1, 32, 8, p, 2, 8, None))
    refused(hm, INV, lib.hm_gemm_image(half, p, MX, 1, 32, 8, p, F32, 8, None))
    refused(hm, INV, lib.hm_image_pack(p, F32, 2**31 - 1, 32, 32, 0, MX, p, None))
    refused(hm, INV, lib.hm_image_pack(p, F32, 1, 2**23 + 1, 2**24, 0, MX, p, None))
    refused(hm, INV, lib.hm_gemm_image(p, p, MX, 2**31 - 1, 32, 8, p, F32, 8, None))
    refused(hm, INV, lib.hm_gemm_image(p, p, MX, 1, 32, 8, p, F32, 2**30 + 1, None))
    refused(hm, INV, lib.hm_gemv_mx4(p, F32, 32, p, 9, 32, 8, p, F32, 8, None))
    refused(hm, UNS, lib.hm_gemv_mx4(p, F32, 32769, p, 1, 32769, 8, p, F32, 8, None))
    refused(hm, INV, lib.hm_expert_plan(p, 4, 1025, p, None))
    refused(hm, INV, lib.hm_expert_plan(None, 4, 8, p, None))
    refused(hm, INV, lib.hm_expert_pack(p, F32, 32, 32, 0, p, 5, 4, 2, MX, p, None))  # pairs are a multiple of the choices
    refused(hm, UNS, lib.hm_expert_pack(p, F32, 32, 32, 0, p, 4, 4, 2, Q8, p, None))
    refused(hm, INV, lib.hm_expert_gemm(p, p, MX, None, 4, 4, 32, 8, p, F32, 8, None))
    refused(hm, INV, lib.hm_expert_gemm(p, p, MX, p, 4, 0, 32, 8, p, F32, 8, None))
    refused(hm, INV, lib.hm_expert_gemv(p, F32, 32, p, p, 65536, 1, 4, 32, 8, p, F32, 8, None))
    refused(hm, INV, lib.hm_expert_sum(p, F32, p, p, 1, 0, 4, 8, None, p, F32, None))
    refused(hm, UNS, lib.hm_expert_sum(p, Q8, p, p, 1, 1, 4, 8, None, p, F32, None))


def test_nothing_to_do_is_no_error(hm):
    lib = hm.load_library()
    raw = np.zeros(4096, np.uint8)
    p = C.c_void_p(raw.ctypes.data + -raw.ctypes.data % 16)
    assert lib.hm_image_pack(p, 0, 0, 32, 32, 0, 10, p, None) == 0
    assert lib.hm_image_unpack(p, 10, 0, 32, p, 0, 32, None) == 0
    assert lib.hm_gemm_image(p, p, 10, 0, 32, 8, p, 0, 8, None) == 0
    assert lib.hm_gemv_mx4(p, 0, 32, p, 0, 32, 8, p, 0, 8, None) == 0
    assert lib.hm_expert_gemm(p, p, 10, p, 0, 4, 32, 8, p, 0, 8, None) == 0
    assert lib.hm_expert_sum(p, 0, p, p, 0, 1, 4, 8, None, p, 0, None) == 0


def test_no_device_is_an_error(hm):
    if hm.device_count():
        pytest.skip("a device is there")
    with pytest.raises(hm.HomuraError) as e:
        hm.image_pack(np.zeros((1, 32), np.float32), hm.DType.MXFP4)
    assert e.value.status == hm.HM_ERR_CUDA


def test_restatement_of_the_format():
    """Every value of the grid stands for itself, at both ends of the scales; halfway values go to the even code."""
    for s in (0, 1, 127, 252):
        x = (np.concatenate([ic.GRID, -ic.GRID]) * 2.0 ** (s - 127)).astype(np.float32)[None]
        codes, scales = ic.mx_quantise(x)
        np.testing.assert_array_equal(codes[0, :16], np.arange(16))
        assert scales[0, 0] == s
        np.testing.assert_array_equal(ic.mx_values(codes, scales, 16)[0], x[0].astype(np.float64))
    half = (ic.GRID[:-1] + ic.GRID[1:]) / 2
    codes, _ = ic.mx_quantise(np.concatenate([[6.0], half]).astype(np.float32)[None])
    np.testing.assert_array_equal(codes[0, 1:8], [0, 2, 2, 4, 4, 6, 6])
