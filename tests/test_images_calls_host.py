"""Arguments of the host-mode image calls that do not fit are refused before the library (or a device) is asked: without a device a call that
is let through ends in HM_ERR_CUDA."""
import numpy as np
import pytest

MX, BF16, F32 = 10, 1, 0
T, TOP, E, K, N = 3, 2, 4, 64, 40
PAIRS = T * TOP


def invalid(hm, call):
    with pytest.raises(hm.HomuraError) as e:
        call()
    assert e.value.status == hm.HM_ERR_INVALID, e.value


def let_through(hm, call):
    if hm.device_count():
        return call()
    with pytest.raises(hm.HomuraError) as e:
        call()
    assert e.value.status == hm.HM_ERR_CUDA, e.value


def grouped(hm, **more):
    plan = np.zeros(hm.expert_plan_ints(PAIRS, E), np.int32)
    image = np.zeros(hm.image_bytes(MX, hm.expert_plan_rows(PAIRS, E), K), np.uint8)
    weights = np.zeros(E * hm.image_bytes(MX, N, K), np.uint8)
    return lambda: hm.expert_gemm(image, weights, more.pop("plan", plan), N, hm.DType.MXFP4, PAIRS, E, K, **more)


def pairs(hm, **more):
    weights = np.zeros(E * hm.image_bytes(MX, N, K), np.uint8)
    return lambda: hm.expert_gemv(np.zeros((T, K), np.float32), weights, np.full((T, TOP), -1, np.int32), N, TOP, E, **more)


@pytest.mark.parametrize("call", [grouped, pairs])
def test_rows_to_be_written_over_have_the_results_type_and_shape(hm, call):
    for y in [np.full((PAIRS, N), 7.0), np.zeros((PAIRS, N), np.float16), np.zeros((PAIRS, N), ">f4"), np.zeros((PAIRS, N), np.uint16), np.zeros((PAIRS - 1, N), np.float32), np.zeros((PAIRS, N - 1), np.float32), np.zeros(PAIRS * N, np.float32),
              np.zeros((T, TOP, N), np.float32), [[0.0] * N] * PAIRS]:
        invalid(hm, call(hm, y=y))
    for y in [np.zeros((PAIRS, N), np.float32), np.zeros((PAIRS, N), np.int16), np.zeros((PAIRS, N // 2), np.uint16)]:
        invalid(hm, call(hm, y=y, y_dtype=hm.DType.BF16))
    fixed = np.zeros((PAIRS, N), np.float32)
    fixed.flags.writeable = False
    invalid(hm, call(hm, y=fixed))
    let_through(hm, call(hm))
    let_through(hm, call(hm, y=np.zeros((PAIRS, N), np.float32)))
    let_through(hm, call(hm, y=np.zeros((PAIRS, N), np.uint16), y_dtype=hm.DType.BF16))


@pytest.mark.parametrize("name", ["expert_gemm", "expert_gemv"])
@pytest.mark.parametrize("y", [np.full((PAIRS, N), 7.0, np.float32), np.full((N, PAIRS), 7.0, np.float32).T, np.full((PAIRS, 2 * N), 7.0, np.float32)[:, ::2]], ids=["rows", "columns", "strided"])
def test_the_callers_rows_are_what_is_written_and_returned(hm, monkeypatch, name, y):
    """A stand-in for the library's call writes row 1 of what it is given."""
    import ctypes as C

    real, before = hm.load_library(), y.copy()

    class Library:
        def __getattr__(self, at):
            if at != "hm_" + name:
                return getattr(real, at)

            def call(*args):
                rows = np.ctypeslib.as_array(C.cast(args[-4], C.POINTER(C.c_float)), (PAIRS, N))
                np.testing.assert_array_equal(rows, before)
                rows[1] = 1.5
                return 0

            return call

    monkeypatch.setattr(hm, "load_library", Library)
    got = {"expert_gemm": grouped, "expert_gemv": pairs}[name](hm, y=y)()
    assert got is y
    want = before.copy()
    want[1] = 1.5
    np.testing.assert_array_equal(y, want)
    y[...] = 7.0


def test_a_plan_of_other_pairs_or_experts(hm):
    for words in [0, 3, hm.expert_plan_ints(PAIRS, E) - 1, hm.expert_plan_ints(PAIRS, E) + 1, hm.expert_plan_ints(PAIRS + 1, E), hm.expert_plan_ints(PAIRS, E + 1)]:
        invalid(hm, grouped(hm, plan=np.zeros(words, np.int32)))
    let_through(hm, grouped(hm))


def test_rows_that_do_not_come_out_even(hm):
    invalid(hm, lambda: hm.image_pack(np.zeros((3, 65), np.float32), hm.DType.MXFP4, glu=True))  # gate and up: half of 65
    let_through(hm, lambda: hm.image_pack(np.zeros((3, 64), np.float32), hm.DType.MXFP4, glu=True))
    for blocks, width in [(np.zeros((3, 1, 17), np.uint8), 64), (np.zeros(3 * 17 + 1, np.uint8), 32), (np.zeros((2, 4, 17), np.uint8), 64), (np.zeros((2, 34), np.uint8), 32), (np.zeros((2, 34), np.uint8), 48), (np.zeros(0, np.uint8), 32)]:
        invalid(hm, lambda: hm.image_from_blocks(blocks, width))
    for blocks, width in [(np.zeros((3, 2, 17), np.uint8), 64), (np.zeros((2, 34), np.uint8), 64), (np.zeros(3 * 17, np.uint8), 32)]:
        let_through(hm, lambda: hm.image_from_blocks(blocks, width))


def test_a_width_that_is_not_the_rows(hm):
    """Host rows say their width themselves; a K beside them has to be the same."""
    w = np.zeros(E * hm.image_bytes(MX, N, 32), np.uint8)
    x, ids = np.zeros((T, K), np.float32), np.zeros((T, TOP), np.int32)
    invalid(hm, lambda: hm.image_pack(x, hm.DType.MXFP4, K=32))
    invalid(hm, lambda: hm.image_pack(x, hm.DType.MXFP4, K=64, glu=True))
    invalid(hm, lambda: hm.gemv_mx4(x, w[: hm.image_bytes(MX, N, 32)], N, K=32))
    invalid(hm, lambda: hm.expert_gemv(x, w, ids, N, TOP, E, K=32))
    let_through(hm, lambda: hm.image_pack(x, hm.DType.MXFP4, K=64))
    let_through(hm, lambda: hm.image_pack(x, hm.DType.MXFP4, K=32, glu=True))
    let_through(hm, lambda: hm.gemv_mx4(x, w[: hm.image_bytes(MX, N, 32)], N, K=64))


def test_ids_beyond_32_bits_are_nobodys(hm, monkeypatch):
    """An id that is no expert's stays one: 2^32 + 1 is not expert 1.  A stand-in for the library keeps the ids it is given."""
    import ctypes as C

    real, seen = hm.load_library(), {}

    class Library:
        def __getattr__(self, at):
            if not at.startswith("hm_expert_") or at.startswith("hm_expert_plan_"):
                return getattr(real, at)

            def call(*args):
                where = {"hm_expert_plan": 0, "hm_expert_gemv": 4, "hm_expert_sum": 2}[at]
                seen[at] = np.ctypeslib.as_array(C.cast(args[where], C.POINTER(C.c_int32)), (PAIRS,)).tolist()
                return 0

            return call

    monkeypatch.setattr(hm, "load_library", Library)
    weights = np.zeros(E * hm.image_bytes(MX, N, K), np.uint8)
    for ids, want in [(np.array([0, 2**32 + 1, -(2**32), 3, 2**31, 7]), [0, -1, -1, 3, -1, 7]), (np.array([1, 2**63, 2**32, 0, 2, 3], np.uint64), [1, -1, -1, 0, 2, 3]), ([[0, 1], [2, 3], [-1, 2**40]], [0, 1, 2, 3, -1, -1]),
                      (np.array([0, 1, -1, -(2**31), 2**31 - 1, 2], np.int32), [0, 1, -1, -(2**31), 2**31 - 1, 2])]:
        hm.expert_plan(ids, E)
        hm.expert_gemv(np.zeros((T, K), np.float32), weights, ids, N, TOP, E)
        hm.expert_sum(np.zeros((PAIRS, N), np.float32), ids, np.zeros((T, TOP), np.float32), TOP, E)
        assert seen == {"hm_expert_plan": want, "hm_expert_gemv": want, "hm_expert_sum": want}
