"""Calls of attention over the 8-bit cache whose shared pages are taken on their own, and the bounds that their results are held to: those follow what a row sees, not what others see."""
import numpy as np

import kv8_cases as kc
from kv8_cases import Model, bf16_bits, bf16_value


def on_their_own(cache, M, heads, pages):
    """Whether such a call has parts of the shared pages in its work memory."""
    return cache.attend_bytes(M, heads, pages) > cache.attend_bytes(M, heads)


def formula(q, k, v, scale, bf16, tokens):
    """out [heads, vdim] of q [heads, dim] over k, v [n, kv_heads, .] (f64), `tokens` of which are shared ones, and how far a result may be off.

    To the bound of pages that are not shared:  scores of shared ones have a query's f16 terms (2^-22 of a value, bf16 rows exactly; no step below 2^-38 of the row's largest) and a chain of at
    most 16 truncating sums of 2^-23: 2^-18.9 of the terms' magnitudes.  A weight times its value's scale has two f16 terms (2^-22 of itself) or, in bf16 rows, one (2^-11), and no
    step below 2^-24; what it is relative to is no more than 2^-7 times the largest of these products that the row sees, so that half a step is 2^-32 of that product (times 127, of the largest
    weight times the largest element of its value), or of 2^-100 of the largest weight where all products are below.  2^-31.5: the reference's logarithm is approximate.  The products
    are summed in chunks of 64 (bf16 rows: 512) steps that round towards zero, 2^-23 each: 2^-17 (2^-14)."""
    want, parts = kc.attention(q, k, v, scale)
    tol = kc.bound(want, parts, bf16)
    if tokens == 0 or len(k) == 0:
        return want, tol
    mag, terms, full, _ = parts
    group = q.shape[0] // k.shape[1]
    peak = np.zeros(q.shape[0])
    for h in range(q.shape[0]):
        s = scale * (k[:, h // group] @ q[h])
        p = np.exp(s - s.max())
        peak[h] = (p / p.sum() * np.abs(v[:, h // group]).max(-1)).max()
    e = 2 * (terms * 2.0**-18.9 + full * 2.0**-38)[:, None] + 2.0**-18
    e = e + (2.0**-14 if bf16 else 2.0**-17)
    return want, tol + mag * e + (tokens * (2.0**-31.5 * peak + 2.0**-125))[:, None] + (mag * 2.0**-11 if bf16 else 0)


def check_rows(m, out, q, seq, pos, heads, scale, rows, seen=None):
    """Some rows of a call over a Model's shared pages against the formula."""
    bf16 = out.dtype == np.uint16
    o, x = (bf16_value(out), bf16_value(q)) if bf16 else (out, q)
    known, worst = {}, 0.0
    for r in rows:
        i, p = int(seq[r]), int(pos[r])
        if not 0 <= i < len(m.lens):
            continue
        if i not in known:
            known[i] = tuple(kc.held(y).astype(np.float64) for y in (m.k[i], m.v[i]))
        at = np.arange(max(0, min(p + 1, len(m.k[i]))))
        if seen is not None:
            at = at[seen(i)[: len(at)]]
        want, tol = formula(x[r].astype(np.float64).reshape(heads, m.dim), known[i][0][at], known[i][1][at], scale, bf16, int((at < m.n_shared * 64).sum()))
        err = np.abs(o[r].reshape(heads, m.vdim) - want)
        assert (err <= tol).all(), (r, i, p, float(np.nanmax(err / tol)), float(np.nanmax(err)))
        worst = max(worst, float((err / tol).max()))
    return worst


def prompt(hm, seed, n, kv_heads, dim, vdim):
    """A Model of one sequence whose pages are all shared."""
    m = Model(hm, seed, kv_heads, dim, vdim, [n], n_shared=-(-n // 64))
    m.k[0], m.v[0], m.lens = m.common[0][:n].copy(), m.common[1][:n].copy(), [n]
    return m


def refill(m):
    """Writes a Model's rows again where they were changed; the shared ones are those of its longest sequence."""
    i = int(np.argmax([len(k) for k in m.k]))
    n = min(m.n_shared * 64, len(m.k[i]))
    m.common[0][:n], m.common[1][:n] = m.k[i][:n], m.v[i][:n]
    for j in range(len(m.k)):
        s = min(n, len(m.k[j]))
        m.k[j][:s], m.v[j][:s] = m.common[0][:s], m.common[1][:s]
    m.fill()


class OnDevice:
    """A call with everything on the device: rows `pad` elements further apart than they have to be, at an address `offset` elements behind an aligned one, work memory full of ones with guard bytes behind it."""

    def __init__(self, m, heads, seq, pos, q, scale, offset=0, pad=0, width=None):
        import torch

        hm, self.m, self.heads, self.scale, self.offset, self.M = m.hm, m, heads, scale, offset, len(seq)
        self.seq, self.pos, self.q, self.bf16 = np.asarray(seq), np.asarray(pos), q, q.dtype == np.uint16
        up = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()
        self.sd, self.pd, self.table, self.shared = up(seq), up(pos), up(m.table), up(m.shared)
        t = torch.uint16 if self.bf16 else torch.float32
        self.ldq, self.ldo = heads * m.dim + pad, heads * m.vdim + pad
        self.qb, self.ob = (torch.full((offset + self.M * ld,), 5, dtype=t, device="cuda") for ld in (self.ldq, self.ldo))
        self.qd = self.qb[offset:].view(self.M, self.ldq)[:, : heads * m.dim]
        self.qd.copy_(torch.from_numpy(q))
        self.cache = hm.KV8Cache(m.kv_heads, m.dim, m.vdim, m.pool.ptr, m.n_pages, (self.table.data_ptr(), *m.table.shape))
        self.pages = len(m.shared)
        self.line, self.size = self.cache.attend_bytes(self.M, heads), self.cache.attend_bytes(self.M, heads, self.pages)
        assert self.size > self.line, "the shared pages of this call are not taken on their own"
        self.work = torch.full((self.size + 64,), 255, dtype=torch.uint8, device="cuda")

    def run(self, stream=None, work=None):
        at = lambda b: b.data_ptr() + self.offset * b.element_size()
        hm = self.m.hm
        self.cache.attend((at(self.qb), self.M), self.sd.data_ptr(), self.pd.data_ptr(), self.heads, self.scale, shared=(self.shared.data_ptr(), self.pages), dtype=hm.DType.BF16 if self.bf16 else hm.DType.F32,
                          ldq=self.ldq, out=at(self.ob), ldo=self.ldo, work=(self.work if work is None else work).data_ptr(), stream=None if stream is None else stream.cuda_stream)

    def parts(self):
        """How many parts of the shared pages a call whose CTAs have few blocks has left in the work memory that was full of ones."""
        x = self.work.cpu().numpy()
        step = self.M * self.heads * ((self.m.vdim + 31) // 32 * 32 + 4) * 4
        assert (x[self.size :] == 255).all()
        return sum(bool((x[self.line + i * step : self.line + (i + 1) * step] != 255).any()) for i in range((self.size - self.line) // step))

    def rows(self):
        """The results; what stands between and in front of them is as it was."""
        o = self.ob.cpu().numpy()
        r = o[self.offset :].reshape(self.M, self.ldo)
        w = self.heads * self.m.vdim
        assert (o[: self.offset] == 5).all() and (r[:, w:] == 5).all()
        return np.ascontiguousarray(r[:, :w])

    def check(self, rows, seen=None):
        return check_rows(self.m, self.rows(), self.q, self.seq, self.pos, self.heads, self.scale, rows, seen)


def some(M, seed, n=20):
    return np.unique(np.concatenate([np.arange(3), M - 1 - np.arange(3), np.random.default_rng(seed).integers(0, M, n)]))
