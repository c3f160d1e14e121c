"""Attention over the 8-bit cache where its work is shared out in other ways: contexts that several CTAs share, rows behind long prefixes, calls on several streams, in graphs, with
strides, and together with rotary positions and the writes in front of it."""
import numpy as np
import pytest

import kv8_cases as kc
from kv8_cases import Model, bf16_bits, bf16_value
from test_gpu_kv8 import SIZES, attend
from test_gpu_rope import check as check_turned, turned

pytestmark = pytest.mark.gpu


# ---- contexts that are cut ----------------------------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,vdim", SIZES)
def test_contexts_in_a_wide_table(hm, heads, kv_heads, dim, vdim, bf16):
    """A table that has room for long contexts: items may be cut anywhere."""
    lens = [1, 64, 2100, 65, 0, 127, 200, 63, 2, 513]
    m = Model(hm, dim + vdim, kv_heads, dim, vdim, lens, max_pages=70)
    attend(m, np.arange(len(lens)), np.array(lens) - 1, heads, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,longest", [(37, 900), (150, 700), (700, 400), (1300, 100)])
def test_short_and_long_rows_side_by_side(hm, rows, longest, bf16):
    """Some items are a warp's own, others the line's; rows of four sequences, some without a context, some of no sequence."""
    m = Model(hm, rows, 2, 64, 64, [longest, 300, 33, 1], max_pages=80)
    rng = np.random.default_rng(rows)
    seq = rng.integers(0, 4, rows)
    pos = (rng.random(rows) ** 2 * np.array(m.lens)[seq]).astype(int) - (rng.random(rows) < 0.1)
    seq[5::17] = -1
    attend(m, seq, pos, 6, bf16)


def test_more_rows_than_threads(hm):
    """Several rows to a thread where the rows' lengths are added up; most have nothing, so that the cuts fall far apart."""
    m = Model(hm, 3, 1, 32, 32, [1500, 40], max_pages=30)
    seq, pos = np.zeros(5000, int), np.full(5000, -1)
    for i, p in [(0, 700), (1, 0), (388, 1499), (389, 640), (2000, 31), (2001, 32), (4999, 1400)]:
        pos[i] = p
    seq[4000:4100], pos[4000:4100] = 1, np.arange(100) % 40
    q, out = attend(m, seq, pos, 2, False)
    assert (out[pos < 0] == 0).all()


@pytest.mark.parametrize("lens", [[640] * 200, [385, 384, 383] * 60, [416] + [32] * 299, [32] * 299 + [2048], [0] * 200 + [3000]])
def test_equal_lengths_and_lengths_at_the_limits(hm, lens):
    m = Model(hm, 4, 1, 32, 64, lens, max_pages=70)
    attend(m, np.arange(len(lens)), np.array(lens) - 1, 3, True)


# ---- shared pages ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,pages,dim,vdim", [(3, 120, 64, 64), (5, 201, 128, 128), (97, 31, 64, 64), (97, 31, 128, 128), (97, 1, 128, 40), (300, 3, 96, 64), (300, 17, 33, 128), (65, 64, 128, 32)])
def test_long_prefixes_and_many_rows(hm, M, pages, dim, vdim, bf16):
    """One tile of pairs and several, an odd number of them, splits that are left to be joined with the rows' own pages; rows that end inside the prefix and rows of no sequence."""
    rng = np.random.default_rng(M + pages)
    S = 64 * pages
    lens = [S + int(n) for n in rng.choice([0, 1, 40, 64, 500], M)]
    m = Model(hm, M + dim, 2, dim, vdim, lens, n_shared=pages)
    seq, pos = np.arange(M), np.array(lens) - 1
    pos[1::5] = rng.integers(-1, S, len(pos[1::5]))
    seq[2::11] = -1
    attend(m, seq, pos, 8, bf16, shared=True, what="kv8 shared prefix")


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("pages,width", [(4, 4), (130, 130), (4, 90)])
def test_rows_that_have_nothing_but_the_prefix(hm, pages, width, bf16):
    """They are written as others are: zeros where a row sees nothing, nothing where it has no sequence."""
    import torch

    M, heads = 40, 8
    m = Model(hm, pages, 2, 64, 64, [64 * pages] * 3, n_shared=pages, max_pages=width)
    seq, pos = np.arange(M) % 3, np.arange(M) * 64 * pages // M
    seq[::7], pos[3::7] = 3, -1
    q = m.queries(M, heads, bf16)
    qd, sd, pd, table, shared = (torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (q, seq.astype(np.int32), pos.astype(np.int32), m.table, m.shared))
    out = torch.full((M, heads * 64), 9, dtype=torch.uint16 if bf16 else torch.float32, device="cuda")
    cache = hm.KV8Cache(2, 64, 64, m.pool.ptr, m.n_pages, (table.data_ptr(), 3, width))
    work = torch.empty(cache.attend_bytes(M, heads, pages), dtype=torch.uint8, device="cuda")
    cache.attend((qd.data_ptr(), M), sd.data_ptr(), pd.data_ptr(), heads, 0.125, shared=(shared.data_ptr(), pages), dtype=hm.DType.BF16 if bf16 else hm.DType.F32, out=out.data_ptr(), work=work.data_ptr())
    torch.cuda.synchronize()
    o = out.cpu().numpy()
    assert (o[::7] == 9).all() and (o[(seq < 3) & (pos < 0)] == 0).all()
    m.check(o, q, np.where(seq < 3, seq, -1), pos, heads, 0.125, shared=True)


# ---- rows and pools at any place --------------------------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("dim,vdim,offset,pad", [(64, 64, 1, 0), (64, 64, 2, 2), (128, 128, 4, 4), (33, 31, 1, 3), (32, 48, 8, 8), (20, 6, 3, 1)])
def test_strided_rows_at_any_address(hm, dim, vdim, offset, pad, bf16):
    import torch

    M, heads, kvh, pages = 45, 6, 2, 3
    m = Model(hm, dim, kvh, dim, vdim, [64 * pages + 100, 64 * pages + 7], n_shared=pages)
    t, dt = (torch.uint16, hm.DType.BF16) if bf16 else (torch.float32, hm.DType.F32)
    seq, pos = np.arange(M) % 2, np.arange(M) * 4 + 1
    pos = np.minimum(pos, np.array(m.lens)[seq] - 1)
    sd, pd, table, shared = (torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda() for x in (seq, pos, m.table, m.shared))

    def put(x):
        width = x.shape[1] + pad
        buf = torch.full((offset + M * width,), 5, dtype=t, device="cuda")
        buf[offset:].view(M, width)[:, : x.shape[1]] = torch.from_numpy(x).cuda()
        return buf, width

    at = lambda b: b.data_ptr() + offset * b.element_size()
    q = m.queries(M, heads, bf16)
    (qb, ldq), (ob, ldo) = put(q), put(np.zeros((M, heads * vdim), q.dtype))
    cache = hm.KV8Cache(kvh, dim, vdim, m.pool.ptr, m.n_pages, (table.data_ptr(), *m.table.shape))
    for n in (0, pages):
        work = torch.full((cache.attend_bytes(M, heads, n) + 64,), 3, dtype=torch.uint8, device="cuda")
        ob[:] = 5
        cache.attend((at(qb), M), sd.data_ptr(), pd.data_ptr(), heads, 0.2, shared=(shared.data_ptr(), n), dtype=dt, ldq=ldq, out=at(ob), ldo=ldo, work=work.data_ptr())
        torch.cuda.synchronize()
        o = ob.cpu().numpy()
        rows = o[offset:].reshape(M, ldo)
        assert (o[:offset] == 5).all() and (rows[:, heads * vdim :] == 5).all() and (work[-64:] == 3).all()
        m.check(np.ascontiguousarray(rows[:, : heads * vdim]), q, seq, pos, heads, 0.2, shared=n > 0)
    # the cache's rows
    k, v = m.rows(M)
    k, v = k.reshape(M, -1), v.reshape(M, -1)
    k, v = (bf16_bits(k), bf16_bits(v)) if bf16 else (k, v)
    (kb, ldk), (vb, ldv) = put(k), put(v)
    own = hm.KV8Cache(kvh, dim, vdim, None, 1, [[0]])
    places = torch.arange(M, dtype=torch.int32, device="cuda")
    zeros = torch.zeros(M, dtype=torch.int32, device="cuda")
    own.write((at(kb), M), at(vb), zeros.data_ptr(), places.data_ptr(), dtype=dt, ldk=ldk, ldv=ldv)
    own.read((zeros.data_ptr(), M), places.data_ptr(), at(kb), at(vb), dtype=dt, ldk=ldk, ldv=ldv)
    torch.cuda.synchronize()
    for buf, x, d, ld in ((kb, k, dim, ldk), (vb, v, vdim, ldv)):
        want = kc.held((bf16_value(x) if bf16 else x).reshape(M, kvh, d)).reshape(M, -1)
        rows = buf.cpu().numpy()[offset:].reshape(M, ld)
        np.testing.assert_array_equal(rows[:, : kvh * d], bf16_bits(want) if bf16 else want)
        assert (rows[:, kvh * d :] == 5).all()


def test_pages_behind_four_gigabytes(hm):
    kvh, dim, n = 8, 256, 20000
    size = hm.kv8_pool_bytes(kvh, dim, dim, n)
    assert size > 4 << 30
    pool = hm.DeviceBuffer(size)
    cache = hm.KV8Cache(kvh, dim, dim, pool.ptr, n, [[0, n - 1, n // 2, n - 2]])
    rng = np.random.default_rng(0)
    k, v = (rng.standard_normal((256, kvh * dim)).astype(np.float32) for _ in range(2))
    cache.write(k, v, np.zeros(256), np.arange(256))
    for got, x in zip(cache.read(np.zeros(256), np.arange(256)), (k, v)):
        np.testing.assert_array_equal(got.reshape(-1, kvh, dim), kc.held(x.reshape(-1, kvh, dim)))
    q = rng.standard_normal((20, kvh * dim)).astype(np.float32)
    out = cache.attend(q, np.zeros(20), np.arange(20) + 230, kvh, dim**-0.5)
    for i in range(20):
        hk, hv = (kc.held(x.reshape(-1, kvh, dim))[: 231 + i].astype(np.float64) for x in (k, v))
        want, parts = kc.attention(q[i].astype(np.float64).reshape(kvh, dim), hk, hv, dim**-0.5)
        assert (np.abs(out[i].reshape(kvh, dim) - want) <= kc.bound(want, parts, False)).all()


def test_one_page_in_several_places(hm):
    """Sequences may share pages, and a table may name one twice."""
    cache = hm.KV8Cache(1, 64, 64, None, 3, [[0, 1, 0], [0, 2, 2]])
    rng = np.random.default_rng(1)
    k, v = (rng.standard_normal((192, 64)).astype(np.float32) for _ in range(2))
    cache.write(k, v, np.repeat([0, 0, 1], 64), np.concatenate([np.arange(128), 64 + np.arange(64)]))
    cache.write(k[5:6].repeat(2, 0), v[5:6].repeat(2, 0), [0, 0], [5, 133])  # one place twice, with one value
    q = rng.standard_normal((2, 128)).astype(np.float32)
    out = cache.attend(q, [0, 1], [191, 191], 2, 0.125)
    for i, at in enumerate(([0, 1, 0], [0, 2, 2])):
        hk, hv = (np.concatenate([kc.held(x.reshape(192, 1, 64))[64 * p : 64 * p + 64] for p in at]).astype(np.float64) for x in (k, v))
        want, parts = kc.attention(q[i].astype(np.float64).reshape(2, 64), hk, hv, 0.125)
        assert (np.abs(out[i].reshape(2, 64) - want) <= kc.bound(want, parts, False)).all()


# ---- streams and graphs -------------------------------------------------------------------------------


class Call:
    """An attention call with everything on the device."""

    def __init__(self, hm, seed, M, heads, kvh, dim, lens, n_shared, max_pages=None):
        import torch

        self.m = m = Model(hm, seed, kvh, dim, dim, lens, n_shared=n_shared, max_pages=max_pages)
        self.M, self.heads = M, heads
        self.seq = np.arange(M) % len(lens)
        self.pos = np.array(lens)[self.seq] - 1
        self.q = m.queries(M, heads, False)
        up = lambda x, t=np.int32: torch.from_numpy(np.ascontiguousarray(x, t)).cuda()
        self.sd, self.pd, self.table, self.shared, self.qd = up(self.seq), up(self.pos), up(m.table), up(m.shared), up(self.q, np.float32)
        self.out = torch.zeros(M, heads * dim, device="cuda")
        self.cache = hm.KV8Cache(kvh, dim, dim, m.pool.ptr, m.n_pages, (self.table.data_ptr(), *m.table.shape))
        self.work = torch.empty(self.cache.attend_bytes(M, heads, n_shared), dtype=torch.uint8, device="cuda")

    def run(self, stream=None, work=None):
        c = self
        c.cache.attend((c.qd.data_ptr(), c.M), c.sd.data_ptr(), c.pd.data_ptr(), c.heads, c.m.dim**-0.5, shared=(c.shared.data_ptr(), c.m.n_shared), out=c.out.data_ptr(), work=(c.work if work is None else work).data_ptr(),
                       stream=None if stream is None else stream.cuda_stream)

    def check(self):
        self.m.check(self.out.cpu().numpy(), self.q, self.seq, self.pos, self.heads, self.m.dim**-0.5, shared=self.m.n_shared > 0)


def calls(hm):
    return [Call(hm, 1, 60, 8, 2, 64, [700, 30, 1000], 0), Call(hm, 2, 50, 8, 2, 128, [64 * 9 + 100, 64 * 9 + 1], 9), Call(hm, 3, 2, 14, 2, 64, [64, 100], 0), Call(hm, 4, 4, 16, 2, 64, [64 * 140 + 5], 140)]


def test_calls_on_two_streams(hm):
    import torch

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    all_ = calls(hm)
    for c in all_:
        c.run()
    torch.cuda.synchronize()
    first = [c.out.clone() for c in all_]
    for c in all_:
        c.check()
        c.out.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for i, c in enumerate(all_):
            c.run(streams[i % 2])
    torch.cuda.synchronize()
    for c, o in zip(all_, first):  # no order of arrival changes a result
        assert torch.equal(c.out, o)


def test_graphs_with_one_work_memory_and_positions_that_move(hm):
    """Two captured calls, replayed one behind the other over the same work memory, with other queries, positions and cached rows each time."""
    import torch

    all_ = calls(hm)
    work = torch.empty(max(c.work.numel() for c in all_), dtype=torch.uint8, device="cuda")
    for c in all_:
        c.run()
    torch.cuda.synchronize()
    graphs, stream = [], torch.cuda.Stream()
    for c in all_:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            c.run(stream, work)
        graphs.append(g)
    rng = np.random.default_rng(0)
    for turn in range(3):
        for c in all_:
            c.pos = np.array([int(rng.integers(-1, n)) for n in np.array(c.m.lens)[c.seq]])
            c.q = c.m.queries(c.M, c.heads, False)
            c.pd.copy_(torch.from_numpy(c.pos.astype(np.int32)))
            c.qd.copy_(torch.from_numpy(c.q))
            work.fill_(255)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for c in all_:
            c.check()


@pytest.mark.parametrize("bf16", [False, True])
def test_a_serving_step(hm, bf16):
    """Rotary positions over queries and keys side by side, the write and the attention behind them, on a stream of their own: a prompt in portions, then single tokens; captured once and
    replayed for every token."""
    import torch

    B, heads, kvh, dim = 5, 8, 2, 64
    t, dt = (torch.uint16, hm.DType.BF16) if bf16 else (torch.float32, hm.DType.F32)
    rng = np.random.default_rng(2)
    prompt, steps, width = 150, 4, (heads + 2 * kvh) * dim
    turns, mult = hm.rope_turns(1e6, dim, "yarn", factor=4.0, original=64)
    pages = -(-(prompt + steps) // 64)
    table = rng.permutation(B * pages).reshape(B, pages).astype(np.int32)
    cache = hm.KV8Cache(kvh, dim, dim, None, B * pages, table)
    td, turns_d = torch.from_numpy(table).cuda(), torch.from_numpy(turns).cuda()
    on_device = hm.KV8Cache(kvh, dim, dim, cache.c.pages, B * pages, (td.data_ptr(), B, pages))
    size = 2 if bf16 else 4
    stream = torch.cuda.Stream()

    def step(rows, seq, pos, out, work, shared=None):
        M, at, s = rows.shape[0], rows.data_ptr(), stream.cuda_stream
        hm.rope((at, M), heads + kvh, dim, turns_d.data_ptr(), pos.data_ptr(), magnitude=mult, dtype=dt, ldx=width, y=at, ldy=width, stream=s)
        on_device.write((at + heads * dim * size, M), at + (heads + kvh) * dim * size, seq.data_ptr(), pos.data_ptr(), dtype=dt, ldk=width, ldv=width, stream=s)
        on_device.attend((at, M), seq.data_ptr(), pos.data_ptr(), heads, dim**-0.5, shared=shared, dtype=dt, ldq=width, out=out.data_ptr(), work=work.data_ptr(), stream=s)

    ks, vs = [[] for _ in range(B)], [[] for _ in range(B)]

    def check(x, seq, pos, out, shared=0):
        """x: the rows as they came; the rows' turned queries and the cached rows follow from the formulas, in the types of the calls."""
        M = len(x)
        y = turned(x[:, : (heads + kvh) * dim], heads + kvh, dim, turns, pos, dim, False, mult)[0].reshape(M, heads + kvh, dim).astype(np.float32)
        y = bf16_value(bf16_bits(y)) if bf16 else y
        for r in range(M):
            ks[seq[r]].append(y[r, heads:])
            vs[seq[r]].append(x[r, (heads + kvh) * dim :].reshape(kvh, dim))
        for r in range(M):
            k, v = (kc.held(np.array(z[seq[r]][: pos[r] + 1], np.float32)).astype(np.float64) for z in (ks, vs))
            want, parts = kc.attention(y[r, :heads].astype(np.float64), k, v, dim**-0.5)
            mag, terms, _, _ = parts
            tol = kc.bound(want, parts, bf16, (shared * 64, float(np.abs(v).max())) if shared else None)
            # turned elements may fall on the other side of a rounding (bf16 rows: 2^-7 of a product), and codes too: a step, 1 / 127 of the largest, for every element of a key; a
            # weight is off by twice what its score is
            off = dim**-0.5 * np.abs(y[r, :heads]).sum(-1) * np.abs(k).max() / 127 + terms * (2.0**-7 if bf16 else 2.0**-18)
            tol = tol + mag * np.expm1(2 * off)[:, None]
            assert (np.abs(out[r].reshape(heads, dim) - want) <= tol).all(), r

    up = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    rows_of = lambda n: rng.standard_normal((n, width)).astype(np.float32)
    for b in range(B):  # prompts in portions of 100 and 50 rows, over the sequence's whole table
        for first, n in ((0, 100), (100, 50)):
            x = rows_of(n)
            bits = bf16_bits(x) if bf16 else x
            x = bf16_value(bits) if bf16 else x
            d, seq, pos = torch.from_numpy(bits).cuda(), np.full(n, b), first + np.arange(n)
            out = torch.zeros(n, heads * dim, dtype=t, device="cuda")
            work = torch.empty(on_device.attend_bytes(n, heads, pages), dtype=torch.uint8, device="cuda")
            sd, pd = up(seq), up(pos)
            torch.cuda.synchronize()
            step(d, sd, pd, out, work, (td.data_ptr() + 4 * b * pages, pages))
            torch.cuda.synchronize()
            o = out.cpu().numpy()
            check(x, seq, pos, bf16_value(o) if bf16 else o, pages)
    x = rows_of(B)
    d, sd, pd = torch.zeros(B, width, dtype=t, device="cuda"), up(np.arange(B)), up(np.full(B, -1))
    out = torch.zeros(B, heads * dim, dtype=t, device="cuda")
    work = torch.empty(on_device.attend_bytes(B, heads), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        step(d, sd, pd, out, work)
    for i in range(steps):
        x = rows_of(B)
        bits = bf16_bits(x) if bf16 else x
        x = bf16_value(bits) if bf16 else x
        pos = np.full(B, prompt + i)
        d.copy_(torch.from_numpy(bits))
        pd.copy_(torch.from_numpy(pos.astype(np.int32)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        o = out.cpu().numpy()
        check(x, np.arange(B), pos, bf16_value(o) if bf16 else o)


def test_no_rows(hm):
    cache = hm.KV8Cache(1, 64, 64, None, 1, [[0]])
    none = np.zeros((0, 64), np.float32)
    cache.write(none, none, [], [])
    assert cache.attend(none, [], [], 1, 1.0).shape == (0, 64)
    assert hm.rope(none, 1, 64, np.zeros(32), []).shape == (0, 64)


# ---- rotary positions: several rows to a block --------------------------------------------------------


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("M,heads,dim,rot,neighbours", [(20000, 1, 32, 32, False), (5000, 2, 64, 64, True), (1201, 3, 128, 64, False), (9473, 1, 20, 10, True), (2400, 1, 7, 6, False), (1300, 2, 16, 0, False)])
def test_many_rows_of_few_heads(hm, M, heads, dim, rot, neighbours, bf16):
    rng = np.random.default_rng(M)
    x = rng.standard_normal((M, heads * dim)).astype(np.float32)
    bits = bf16_bits(x) if bf16 else x
    x = bf16_value(bits) if bf16 else x
    turns, _ = hm.rope_turns(1e4, rot) if rot else (np.zeros(0), 1.0)
    pos = rng.integers(-1000, 1 << 20, M)
    got = hm.rope(bits, heads, dim, turns, pos, rot=rot, neighbours=neighbours)
    check_turned(got, x, *turned(x, heads, dim, turns, pos, rot, neighbours, 1.0), bf16)
    got = bf16_value(got) if bf16 else got
    if rot < dim:
        np.testing.assert_array_equal(got.reshape(M, heads, dim)[..., rot:], x.reshape(M, heads, dim)[..., rot:])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,pages,dim,width", [(5, 0, 64, 4), (5, 0, 64, 90), (300, 0, 32, 90), (60, 3, 64, 9), (60, 3, 128, 9), (40, 3, 64, 3)])
def test_queries_that_are_not_finite(hm, rows, pages, dim, width, bf16):
    """A query with a NaN or an infinity makes its own head's result NaN, and no other's."""
    m = Model(hm, rows + dim, 2, dim, dim, [64 * pages + (150 if width > pages else 0)] * 2, n_shared=pages, max_pages=width)
    seq, pos = np.arange(rows) % 2, np.full(rows, m.lens[0] - 1) - np.arange(rows) % 70
    q, clean = attend(m, seq, pos, 6, bf16, shared=pages > 0)
    bad = (bf16_value(q) if bf16 else q).copy().reshape(rows, 6, dim)
    bad[1, 4, 3], bad[rows - 1, 0, 0], bad[rows // 2, 5, dim - 1] = np.nan, np.inf, -np.inf
    bad = bad.reshape(rows, -1)
    out = m.cache.attend(bf16_bits(bad) if bf16 else bad, seq, pos, 6, dim**-0.5, shared=m.shared if pages else None)
    hit = np.zeros((rows, 6), bool)
    hit[[1, rows - 1, rows // 2], [4, 0, 5]] = True
    f = (bf16_value(out) if bf16 else out).reshape(rows, 6, dim)
    assert np.isnan(f[hit]).all()
    np.testing.assert_array_equal(out.reshape(rows, 6, dim)[~hit], clean.reshape(rows, 6, dim)[~hit])


@pytest.mark.parametrize("heads,kv_heads,dim,pages", [(256, 256, 8, 2), (1024, 2, 16, 2), (130, 1, 64, 5), (9, 1, 64, 2)])
def test_many_heads(hm, heads, kv_heads, dim, pages):
    m = Model(hm, heads, kv_heads, dim, dim, [64 * pages + 70, 64 * pages + 3], n_shared=pages)
    for shared in (False, True):
        attend(m, [0, 1, 0], [64 * pages + 69, 64 * pages + 2, 100], heads, False, shared=shared)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("own", [0, 130])
@pytest.mark.parametrize("heads,kv_heads,dim,vdim,pages", [(h, k, d, v, 5) for h, k, d, v in SIZES if max(d, v) <= 128] + [(8, 2, 64, 64, 130), (34, 2, 33, 100, 1), (6, 1, 128, 128, 64), (16, 8, 128, 128, 33)])
def test_prefixes_of_enough_rows(hm, heads, kv_heads, dim, vdim, pages, own, bf16):
    """As many rows as it takes for the shared pages to be taken on their own, and some beside: rows inside the prefix, at its end, behind it, of no sequence."""
    items = kv_heads * -(-heads // kv_heads // 8)
    M = min(8192, -(-32768 // (items * 2 * pages)) + 3)
    rng = np.random.default_rng(heads + dim + pages)
    S = 64 * pages
    m = Model(hm, heads + dim, kv_heads, dim, vdim, [S + own, S + own // 2, S], n_shared=pages)
    seq = rng.integers(0, 3, M)
    pos = np.where(rng.random(M) < 0.5, np.array(m.lens)[seq] - 1, rng.integers(-1, S, M))
    seq[1::9] = -1
    q = m.queries(M, heads, bf16)
    out = m.cache.attend(q, seq, pos, heads, dim**-0.5, shared=m.shared)
    at = np.unique(np.concatenate([np.arange(4), M - 1 - np.arange(4), rng.integers(0, M, 24)]))
    m.check(out[at], q[at], seq[at], pos[at], heads, dim**-0.5, shared=True)
    np.testing.assert_array_equal(out, m.cache.attend(q, seq, pos, heads, dim**-0.5, shared=m.shared))


@pytest.mark.parametrize("bf16", [False, True])
def test_missing_pages_and_bad_vectors_in_a_prefix_of_many_rows(hm, bf16):
    M, heads, pages = 1000, 8, 9
    m = Model(hm, 20, 2, 64, 64, [64 * pages + 30] * 2, n_shared=pages)
    m.shared = m.shared.copy()
    m.shared[[0, 5]] = [-1, m.n_pages]
    seq, pos = np.arange(M) % 2, np.arange(M) * 7 % (64 * pages + 30)
    q = m.queries(M, heads, bf16)
    out = m.cache.attend(q, seq, pos, heads, 0.125, shared=m.shared)
    at = np.arange(0, M, 29)
    m.check(out[at], q[at], seq[at], pos[at], heads, 0.125, shared=True, seen=lambda i: ~np.isin(np.arange(m.lens[i]) // 64, [0, 5]))
    one = hm.KV8Cache(2, 64, 64, m.pool.ptr, m.n_pages, m.shared[None])
    bad = m.common[1][200].copy()
    bad[0, 3] = np.inf
    one.write(m.common[0][200][None].reshape(1, -1), bad.reshape(1, -1), [0], [200])  # of the first key/value head alone
    f = m.cache.attend(q, seq, pos, heads, 0.125, shared=m.shared).reshape(M, heads, 64)
    assert np.isnan((bf16_value(f) if bf16 else f)[pos >= 200][:, :4]).all()
    np.testing.assert_array_equal(f[pos < 200], out.reshape(M, heads, 64)[pos < 200])
    np.testing.assert_array_equal(f[:, 4:], out.reshape(M, heads, 64)[:, 4:])
    queries = (bf16_value(q) if bf16 else q).copy()
    queries[10, 64 * 5 + 1] = np.nan
    g = m.cache.attend(bf16_bits(queries) if bf16 else queries, seq, pos, heads, 0.125, shared=m.shared).reshape(M, heads, 64)
    assert np.isnan((bf16_value(g) if bf16 else g)[10, 5]).all()
    keep = np.ones((M, heads), bool)
    keep[10, 5] = False
    np.testing.assert_array_equal(g[keep], f[keep])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,width,heads,kv_heads,dim", [(75, 48, 8, 2, 64), (100, 48, 12, 2, 128), (220, 40, 8, 2, 32), (400, 20, 4, 2, 64), (150, 3, 16, 2, 256), (1000, 20, 16, 2, 64), (160, 48, 6, 1, 192)])
def test_teams_of_warps(hm, rows, width, heads, kv_heads, dim, bf16):
    """More items than SMs in tables that leave none for the line: teams of one to four warps, some with fewer pieces than warps, several items to a team."""
    n = 64 * width
    m = Model(hm, rows + dim, kv_heads, dim, dim, [n, n // 2 + 5], max_pages=width)
    rng = np.random.default_rng(rows)
    seq = rng.integers(0, 2, rows)
    pos = (rng.random(rows) ** 3 * np.array(m.lens)[seq]).astype(int) - (rng.random(rows) < 0.05)
    seq[3::13] = -1
    q = m.queries(rows, heads, bf16)
    out = m.cache.attend(q, seq, pos, heads, dim**-0.5)
    at = np.unique(np.concatenate([np.arange(5), rng.integers(0, rows, 50), np.argsort(pos)[-3:]]))
    m.check(out[at], q[at], seq[at], pos[at], heads, dim**-0.5)
    assert (out[(seq >= 0) & (pos < 0)] == 0).all()
    np.testing.assert_array_equal(out, m.cache.attend(q, seq, pos, heads, dim**-0.5))
