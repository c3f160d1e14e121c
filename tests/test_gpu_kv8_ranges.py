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
