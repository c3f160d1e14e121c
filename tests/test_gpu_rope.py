"""Rotary positions against the formula in 64 bits."""
import numpy as np
import pytest

from conftest import record_error
from image_cases import bf16_bits, bf16_value

pytestmark = pytest.mark.gpu


def turned(x, heads, dim, turns, pos, rot, neighbours, mult):
    y = np.asarray(x, np.float64).reshape(len(x), heads, dim).copy()
    size = np.abs(y)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if neighbours else (slice(0, rot // 2), slice(rot // 2, rot))
    t = np.asarray(turns, np.longdouble)[None] * np.asarray(pos, np.longdouble)[:, None]
    angle = np.asarray(2 * np.pi * (t - np.rint(t)), np.float64)[:, None]
    u, w = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = mult * (u * np.cos(angle) - w * np.sin(angle)), mult * (u * np.sin(angle) + w * np.cos(angle))
    both = mult * (np.abs(u) + np.abs(w))
    size[..., a] = size[..., b] = both
    return y.reshape(len(x), -1), size.reshape(len(x), -1)


def check(got, x, want, size, bf16, rot_only=None):
    """Sine and cosine: 1.5 units of 2^-23 and the angle's rounding (2^-25); the factor, two products and their sum: 2^-24 each: within 2^-21 of the pair's magnitudes."""
    err = np.abs((bf16_value(got) if bf16 else got) - want)
    tol = size * 2.0**-21 + (np.abs(want) * 2.0**-8 if bf16 else 0)
    assert (err <= tol).all(), float((err / np.maximum(tol, 1e-300)).max())
    record_error(f"rope {'bf16' if bf16 else 'f32'}", float(err.max()), float(np.abs(want).max()))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("M,heads,dim,rot", [(1, 16, 64, 64), (5, 3, 64, 32), (33, 2, 128, 128), (2, 1, 2, 2), (7, 4, 80, 20), (3, 5, 33, 6), (4, 1, 256, 256), (2, 2, 1024, 1024), (9, 40, 96, 48), (3, 2, 16, 0), (1, 1, 1, 0), (300, 2, 64, 62)])
def test_rows_against_the_formula(hm, M, heads, dim, rot, neighbours, bf16):
    rng = np.random.default_rng(M + dim)
    x = rng.standard_normal((M, heads * dim)).astype(np.float32)
    xb = bf16_bits(x)
    if bf16:
        x = bf16_value(xb)
    pos = rng.integers(0, 200000, M)
    turns, mult = hm.rope_turns(1e6, rot, "yarn", factor=4, original=4096) if rot else (np.zeros(0), 1.0)
    got = hm.rope(xb if bf16 else x, heads, dim, turns, pos, rot=rot, neighbours=neighbours, magnitude=mult)
    want, size = turned(x, heads, dim, turns, pos, rot, neighbours, mult)
    check(got, x, want, size, bf16)
    rest = (bf16_value(got) if bf16 else got).reshape(M, heads, dim)[..., rot:]
    np.testing.assert_array_equal(rest, x.reshape(M, heads, dim)[..., rot:])


def test_far_and_negative_positions(hm):
    """The angle of a far position keeps its bits: products in 64 bits hold turns * 2^31 to 2^-22 of a turn at the fastest pair."""
    rng = np.random.default_rng(1)
    pos = np.array([0, 1, -1, 2**20, -(2**20) + 1, 2**24 + 1, 10**7])
    x = rng.standard_normal((len(pos), 128)).astype(np.float32)
    turns, _ = hm.rope_turns(1e4, 128)
    got = hm.rope(x, 1, 128, turns, pos)
    want, size = turned(x, 1, 128, turns, pos, 128, False, 1.0)
    check(got, x, want, size, False)
    back = hm.rope(got, 1, 128, turns, -pos)
    assert np.abs(back - x).max() <= 2.0**-20 * 2 * np.abs(x).max()
    edge = np.array([2**31 - 1, -(2**31)])
    assert np.isfinite(hm.rope(x[:2], 1, 128, turns, edge)).all()


def test_quarter_turns_are_exact(hm):
    x = np.array([[1.0, 0.0, 3.0, -2.0]], np.float32)
    for n, (c, s) in enumerate([(1, 0), (0, 1), (-1, 0), (0, -1)]):
        got = hm.rope(np.repeat(x, 2, 0), 1, 4, np.array([0.25, 0.25]), [n, n - 400])
        want = np.array([c * 1 - s * 3, s * 2, 3 * c + s, -2 * c], np.float32)
        np.testing.assert_array_equal(got, np.repeat(want[None], 2, 0))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("offset,ldx,ldy", [(0, 512, 256), (1, 515, 257), (3, 300, 300), (8, 264, 512)])
def test_strided_rows_at_any_address_and_in_place(hm, offset, ldx, ldy, bf16):
    import torch

    t = torch.bfloat16 if bf16 else torch.float32
    M, heads, dim = 9, 4, 64
    g = torch.Generator().manual_seed(offset)
    x = torch.randn(M * ldx + 16, generator=g).to(t).cuda()
    y = torch.full((M * ldy + 16,), 7.0, dtype=t).cuda()
    turns, _ = hm.rope_turns(1e4, 32)
    tt, pos = torch.from_numpy(turns).cuda(), torch.arange(5, 5 + M, dtype=torch.int32).cuda()
    size = x.element_size()
    call = lambda src, dst, ls, ld: hm.rope((src.data_ptr() + offset * size, M), heads, dim, tt.data_ptr(), pos.data_ptr(), rot=32, dtype=hm.DType.BF16 if bf16 else hm.DType.F32, ldx=ls, y=dst.data_ptr() + offset * size, ldy=ld)
    keep = x.clone()
    call(x, y, ldx, ldy)
    torch.cuda.synchronize()
    assert torch.equal(x, keep)
    rows = lambda b, ld: np.stack([b.float().cpu().numpy()[offset + m * ld : offset + m * ld + heads * dim] for m in range(M)])
    want, mag = turned(rows(x, ldx), heads, dim, turns, np.arange(5, 5 + M), 32, False, 1.0)
    err, tol = np.abs(rows(y, ldy) - want), mag * 2.0**-21 + (np.abs(want) * 2.0**-8 if bf16 else 0)
    assert (err <= tol).all()
    touched = torch.zeros(y.numel(), dtype=torch.bool)
    for m in range(M):
        touched[offset + m * ldy : offset + m * ldy + heads * dim] = True
    assert (y.cpu()[~touched] == 7).all()
    call(x, x, ldx, ldx)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(rows(x, ldx), rows(y, ldy))
    outside = torch.ones(x.numel(), dtype=torch.bool)
    for m in range(M):
        outside[offset + m * ldx : offset + m * ldx + heads * dim] = False
    assert torch.equal(x.cpu()[outside], keep.cpu()[outside])
