"""4-bit microscaled floats, images and grouped rows restated in numpy (64 bits), for the tests of the image entry points."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def bf16_value(bits):
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def mx_quantise(x):
    """[rows, K] -> (codes [rows, K32] of 0 .. 15, scale bytes [rows, K32 / 32]) with K32 = K rounded up to 32."""
    x = np.asarray(x, np.float32)
    rows, K = x.shape
    full = np.zeros((rows, -(-K // 32) * 32), np.float32)
    full[:, :K] = x
    b = full.reshape(rows, -1, 32).astype(np.float64)
    bad = ~np.isfinite(b).all(-1)
    top = np.where(bad, 0, np.abs(np.where(np.isfinite(b), b, 0)).max(-1))
    e = np.maximum(np.where(top > 0, np.frexp(top)[1] - 1, -1000) - 2, -127)
    mag = np.where(np.isfinite(b), np.abs(b), 0) / np.exp2(e.astype(np.float64))[..., None]
    # nearest code, ties to the even one: distances in 64 bits are exact
    d = np.abs(mag[..., None] - GRID)
    best = d.min(-1, keepdims=True)
    even_first = np.where(d == best, np.arange(8) % 2, 2)  # among the nearest: an even code
    code = even_first.argmin(-1)
    code = np.where(mag >= 6, 7, code)
    code = np.where(np.signbit(b), code + 8, code)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(rows, -1).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def mx_values(codes, scales, K=None):
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    out = (v.reshape(*scales.shape, 32) * s[..., None]).reshape(codes.shape)
    return out[:, :K]


def mx_round(x):
    return mx_values(*mx_quantise(x), K=np.asarray(x).shape[1])


def gguf_blocks(codes, scales):
    c = codes.reshape(*scales.shape, 32)
    return np.concatenate([scales[..., None], c[..., :16] | (c[..., 16:] << 4)], -1).astype(np.uint8)


def mx_image(codes, scales, K):
    """The image's bytes (rows beyond the last: zero)."""
    rows = codes.shape[0]
    kb = -(-K // 256)
    out = np.zeros((-(-rows // 128), kb, 17408), np.uint8)
    c = np.zeros((rows, kb * 256), np.uint8)
    c[:, : codes.shape[1]] = codes
    s = np.zeros((rows, kb * 8), np.uint8)
    s[:, : scales.shape[1]] = scales
    packed = (c[:, 0::2] | (c[:, 1::2] << 4)).reshape(rows, kb, 8, 16)
    for r in range(rows):
        b, i = divmod(r, 128)
        for p in range(8):
            at = 1024 + i * 128 + ((p ^ (i & 7)) << 4)
            out[b, :, at : at + 16] = packed[r, :, p]
            out[b, :, (p >> 2) * 512 + (i & 31) * 16 + (i >> 5) * 4 + (p & 3)] = s[r].reshape(kb, 8)[:, p]
    return out.reshape(-1)


def rounded(x, dtype):
    """Rows as an image of the type ("mxfp4" or "bf16") holds them, in 64 bits."""
    return mx_round(x) if dtype == "mxfp4" else bf16_value(bf16_bits(np.asarray(x, np.float32))).astype(np.float64)


def plan(ids, experts):
    """(first, count, place, row) as the library lays them out."""
    ids = np.asarray(ids).reshape(-1)
    pairs = ids.size
    rows = (pairs // 128 + min(pairs, experts)) * 128
    first, count, place, row = np.zeros(experts + 1, np.int32), np.zeros(experts, np.int32), np.full(pairs, -1, np.int32), np.full(rows, -1, np.int32)
    for e in range(experts):
        mine = np.flatnonzero(ids == e)
        count[e] = mine.size
        first[e + 1] = first[e] + -(-mine.size // 128)
        place[mine] = first[e] * 128 + np.arange(mine.size)
        row[first[e] * 128 : first[e] * 128 + mine.size] = mine
    return first, count, place, row


def activations(rng, rows, K):
    x = rng.standard_normal((rows, K)) * np.exp(rng.standard_normal((rows, 1)))
    return (x * np.where(rng.random((1, K)) < 0.02, 12.0, 1.0)).astype(np.float32)
