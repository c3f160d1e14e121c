"""The 8-bit cache and attention over it restated in numpy (64 bits), and the bounds that results are held to."""
import numpy as np

from image_cases import bf16_bits, bf16_value  # noqa: F401

PAGE = 64


def block_bytes(dim, vdim):
    up = lambda d: -(-d // 32) * 32
    return PAGE * (8 + up(dim) + up(vdim))


def quantise(x):
    """[..., dim] f32 -> (codes, scales [..., 1]); every step is an f32 operation."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        m = np.abs(x).max(-1, keepdims=True)
        bad = ~np.isfinite(x).all(-1, keepdims=True)
        some = ~bad & (m >= np.float32(2.0**-100))
        up = np.float32(127) * (np.float32(1) / np.where(some, m, np.float32(1)))
        codes = np.where(some, np.rint(np.where(some, x, 0) * up), 0).astype(np.int32)
        scales = np.where(bad, np.float32(np.nan), np.where(some, m * (np.float32(1) / np.float32(127)), np.float32(0))).astype(np.float32)
    return codes, scales


def held(x):
    """What the cache holds of rows [..., dim], as f32."""
    codes, scales = quantise(x)
    return codes.astype(np.float32) * scales


def attention(q, ks, vs, scale):
    """q [heads, dim], ks [tokens, kv_heads, dim], vs [tokens, kv_heads, vdim] (f64) -> out [heads, vdim], and what the bound is made of: the sum of weighted magnitudes
    [heads, vdim], the largest sum of magnitudes of a score's terms [heads], the largest sum of a score's terms with the queries' largest
    element in every place [heads], the weighted largest magnitudes of the values [heads]."""
    H, G = q.shape[0], ks.shape[1]
    if ks.shape[0] == 0:
        z = np.zeros((H, vs.shape[2]))
        return z, (z, np.zeros(H), np.zeros(H), np.zeros(H))
    group = H // G
    out, mag, terms, full, wide = [], [], [], [], []
    for h in range(H):
        k, v = ks[:, h // group], vs[:, h // group]
        s = scale * (k @ q[h])
        p = np.exp(s - s.max())
        p /= p.sum()
        out.append(p @ v)
        mag.append(p @ np.abs(v))
        terms.append(abs(scale) * (np.abs(k) @ np.abs(q[h])).max())
        full.append(abs(scale) * np.abs(q[h]).max() * np.abs(k).sum(-1).max())
        wide.append((p * np.abs(v).max(-1)).sum())
    return np.array(out), (np.array(mag), np.array(terms), np.array(full), np.array(wide))


def bound(out, parts, bf16, prefix=None):
    """Scores: sums of digits times codes are exact; a query's element is off by half of the last digit's step, 2^-30 (bf16 rows: 1 / 32639 / 2) of its largest one, the
    digits' sums and the factors are f32: together 2^-21 of the terms' magnitudes.  A weight is off by twice what its score is (itself and the sum it is divided by), and by half a
    step of its digits: 2^-31 (bf16 rows: 2^-16) of the largest weight times value among 32 tokens, so that these 32 are off by at most 2^-26 (2^-11) of the sum of their
    weights times their largest values.  The exponential and f32 sums over at most a few hundred parts: 2^-18.  bf16 results are rounded (2^-8)."""
    mag, terms, full, wide = parts
    e = 2 * (terms * 2.0**-21 + full * (2.0**-15.9 if bf16 else 2.0**-30))[..., None] + 2.0**-18
    tol = mag * e + wide[..., None] * (2.0**-11 if bf16 else 2.0**-26) + 1e-37
    if prefix:
        # Shared pages on their own: (tokens, largest value that any row sees).  Scores: products exact but for the f16 terms of a query (2^-22 of a value, bf16 rows exactly; no step
        # below 2^-38 of the row's largest), a chain of at most 16 truncating sums of 2^-23: 2^-18.9.  A weight has one f16 term in bf16 rows (2^-11) or two (2^-22), and no step
        # below 2^-24: half of it is 2^-28 of the weight 1 of the reference times the largest value, to each token's share.
        n, largest = prefix
        e = 2 * (terms * 2.0**-18.9 + full * 2.0**-38)[..., None] + 2.0**-18
        tol = tol + mag * e + n * 2.0**-28 * largest + (mag * 2.0**-11 if bf16 else 0)
    return tol + np.abs(out) * 2.0**-8 if bf16 else tol


class Model:
    """A cache filled with rows, and the same rows in numpy."""

    def __init__(self, hm, seed, kv_heads, dim, vdim, lens, n_shared=0, spare=2, max_pages=None, poison=True):
        self.hm, self.rng = hm, np.random.default_rng(seed)
        self.kv_heads, self.dim, self.vdim, self.n_shared, self.lens = kv_heads, dim, vdim, n_shared, list(lens)
        need = [max(0, -(-n // PAGE) - n_shared) for n in lens]
        self.n_pages = n_shared + sum(need) + spare
        order = self.rng.permutation(self.n_pages).astype(np.int32)
        self.shared = order[:n_shared].copy()
        width = max_pages or max(1, n_shared + max(need + [0]))
        self.table = np.full((len(lens), width), -1, np.int32)
        at = n_shared
        for i, n in enumerate(need):
            self.table[i, :n_shared] = self.shared
            self.table[i, n_shared : n_shared + n] = order[at : at + n]
            at += n
        self.pool = hm.DeviceBuffer(hm.kv8_pool_bytes(kv_heads, dim, vdim, self.n_pages))
        if poison:
            self.pool.upload(np.full(self.pool.nbytes, 255, np.uint8))
        self.cache = hm.KV8Cache(kv_heads, dim, vdim, self.pool.ptr, self.n_pages, self.table)
        S = n_shared * PAGE
        self.k, self.v = [], []
        common = self.rows(S)
        for i, n in enumerate(lens):
            k, v = self.rows(max(0, n - S))
            self.k.append(np.concatenate([common[0], k])[:n] if n_shared else k)
            self.v.append(np.concatenate([common[1], v])[:n] if n_shared else v)
        self.common = common
        self.fill()

    def rows(self, n):
        k = self.rng.standard_normal((n, self.kv_heads, self.dim)).astype(np.float32)
        v = self.rng.standard_normal((n, self.kv_heads, self.vdim)).astype(np.float32)
        k *= np.where(self.rng.random((1, self.kv_heads, self.dim)) < 0.03, 4, 1).astype(np.float32)
        v[::5] *= 0.125
        return k, v

    def fill(self):
        if self.n_shared:
            n = self.n_shared * PAGE
            table = self.hm.KV8Cache(self.kv_heads, self.dim, self.vdim, self.pool.ptr, self.n_pages, self.shared[None])
            table.write(self.common[0].reshape(n, -1), self.common[1].reshape(n, -1), np.zeros(n), np.arange(n))
        for i, (k, v) in enumerate(zip(self.k, self.v)):
            first = min(self.n_shared * PAGE, len(k))
            if len(k) > first:
                self.cache.write(k[first:].reshape(len(k) - first, -1), v[first:].reshape(len(k) - first, -1), np.full(len(k) - first, i), np.arange(first, len(k)))

    def queries(self, M, heads, bf16):
        q = (self.rng.standard_normal((M, heads * self.dim)) * np.exp(0.5 * self.rng.standard_normal((M, 1)))).astype(np.float32)
        return bf16_bits(q) if bf16 else q

    def check(self, out, q, row_seq, row_pos, heads, scale, seen=None, shared=False):
        """Every row of out against the formula; rows of other sequences are not looked at.  seen(i): positions of sequence i that have a place."""
        bf16 = out.dtype == np.uint16
        o, x = (bf16_value(out), bf16_value(q)) if bf16 else (out, q)
        worst = 0.0
        finite = lambda x: np.where(np.isfinite(x), x, 0)
        prefix = (self.n_shared * PAGE, max([float(np.abs(finite(held(x))).max()) for x in [*self.v, self.common[1]] if x.size] + [0.0])) if shared else None
        for m, (i, p) in enumerate(zip(row_seq, row_pos)):
            if not 0 <= i < len(self.lens):
                continue
            at = np.arange(min(p + 1, len(self.k[i])))
            if seen is not None:
                at = at[seen(i)[: len(at)]]
            k, v = held(self.k[i])[at].astype(np.float64), held(self.v[i])[at].astype(np.float64)
            want, parts = attention(x[m].astype(np.float64).reshape(heads, self.dim), k, v, scale)
            err, tol = np.abs(o[m].reshape(heads, self.vdim) - want), bound(want, parts, bf16, prefix)
            assert (err <= tol).all(), (m, i, p, float((err / tol).max()), float(err.max()))
            worst = max(worst, float((err / tol).max()))
        return worst
