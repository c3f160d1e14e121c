"""Rotary positions, a paged cache in 8 bits, and attention over it, for timing and for comparing with their plain forms.

Kinds of cases:

* ``rope``    rows of heads turned by their positions: either layout of the pairs, part of the head, scaled frequencies.
* ``cache``   keys and values of rows quantised into their pages, and read back from there.
* ``attend``  rows (tokens being decoded) over the contexts of their sequences.
* ``shared``  the same where all sequences begin with the same pages (a system prompt); with ``chunk`` the rows are a portion of
  a prompt, which follow one another in one sequence.

A key or value of a head has one scale: with m the largest magnitude, codes rint(x * (127 / m)) and the scale m / 127, all in f32; zeros where m is below
2^-100.  A page holds 64 tokens.  A row at position p sees the positions 0 .. p; at position -1 it sees none, and its result is zero.  Head counts and sizes
are those of the bench's and the sweeps' architectures.
"""
from __future__ import annotations

import math

import torch

own = False

F32, BF16 = 0, 1  # the library's type numbers
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
PAGE = 64
TINY = 2.0**-100

SCALINGS = {
    "plain": {},
    "linear": {"kind": "linear", "factor": 4.0},
    "bands": {"kind": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
    "yarn": {"kind": "yarn", "factor": 4.0, "fast": 32.0, "slow": 1.0, "original": 32768},
}


def listed():
    return [
        # one token's queries and keys of the 0.5 B stack: the smallest call
        {"name": "rope-token", "kind": "rope", "rows": 1, "heads": 16, "dim": 64, "rot": 64, "beside": 2, "neighbours": False, "scaling": "plain", "theta": 1e6, "far": 32768, "type": "f32"},
        # a batch, adjacent pairs in the first half of the head, frequencies scaled by bands
        {"name": "rope-batch", "kind": "rope", "rows": 64, "heads": 36, "dim": 64, "rot": 32, "beside": 4, "neighbours": True, "scaling": "bands", "theta": 5e5, "far": 131072, "type": "f32"},
        # a long prompt of the 1.5 B stack, queries and keys inside the rows of the projection
        {"name": "rope-prompt", "kind": "rope", "rows": 8191, "heads": 14, "dim": 128, "rot": 128, "beside": 2, "neighbours": False, "scaling": "yarn", "theta": 1e6, "far": 131072, "type": "bf16"},
        # the newest tokens of 64 sequences
        {"name": "cache-batch", "kind": "cache", "rows": 64, "seqs": 64, "kv_heads": 2, "dim": 128, "vdim": 128, "far": 4096, "type": "f32"},
        # a prompt's tokens
        {"name": "cache-prompt", "kind": "cache", "rows": 8191, "seqs": 1, "kv_heads": 8, "dim": 128, "vdim": 128, "far": 8191, "type": "bf16"},
        # one token of a short conversation, 0.5 B stack
        {"name": "attend-token", "kind": "attend", "rows": 1, "heads": 14, "kv_heads": 2, "dim": 64, "vdim": 64, "shared": 0, "low": 77, "high": 77, "type": "f32"},
        # a batch of uneven conversations
        {"name": "attend-batch", "kind": "attend", "rows": 64, "heads": 16, "kv_heads": 8, "dim": 128, "vdim": 128, "shared": 0, "low": 500, "high": 8000, "type": "bf16"},
        # a few long documents, 1.5 B stack
        {"name": "attend-long", "kind": "attend", "rows": 3, "heads": 12, "kv_heads": 2, "dim": 128, "vdim": 128, "shared": 0, "low": 20000, "high": 32768, "type": "f32"},
        # a few conversations behind one system prompt
        {"name": "shared-few", "kind": "shared", "rows": 7, "heads": 32, "kv_heads": 4, "dim": 64, "vdim": 64, "shared": 2048, "low": 1, "high": 300, "type": "f32"},
        # a batch behind one long instruction with examples
        {"name": "shared-batch", "kind": "shared", "rows": 64, "heads": 16, "kv_heads": 8, "dim": 128, "vdim": 128, "shared": 16384, "low": 1, "high": 500, "type": "bf16"},
        # many samples of one document: the most operations
        {"name": "shared-many", "kind": "shared", "rows": 256, "heads": 32, "kv_heads": 4, "dim": 64, "vdim": 64, "shared": 16384, "low": 0, "high": 200, "type": "bf16"},
        # a portion of a long prompt, 1.5 B stack
        {"name": "shared-chunk", "kind": "shared", "rows": 1021, "heads": 12, "kv_heads": 2, "dim": 128, "vdim": 128, "shared": 0, "chunk": 5000, "low": 0, "high": 0, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "cache", "cache", "attend", "attend", "attend", "shared", "shared", "shared"])
    t = rng.choice(["f32", "bf16"])
    if kind == "rope":
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        heads = rng.randrange(1, 41)
        return {"kind": kind, "rows": _log(rng, 1, min(8192, 14000000 // (heads * dim))), "heads": heads, "dim": dim, "rot": rng.choice([dim, dim, dim // 2, 2 * rng.randrange(1, dim // 2 + 1)]), "beside": rng.choice([0, 0, 1, 8]),
                "neighbours": rng.random() < 0.5, "scaling": rng.choice(sorted(SCALINGS)), "theta": rng.choice([1e4, 5e5, 1e6]), "far": _log(rng, 1, 1000000), "type": t}
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    vdim = rng.choice([dim, dim, dim, 64, 128, rng.randrange(1, 257)])
    kv_heads = rng.choice([1, 2, 4, 8])
    if kind == "cache":
        rows = _log(rng, 1, min(8192, 16000000 // (kv_heads * (dim + vdim))))
        return {"kind": kind, "rows": rows, "seqs": rng.randrange(1, min(rows, 64) + 1), "kv_heads": kv_heads, "dim": dim, "vdim": vdim, "far": rows + _log(rng, 1, 4000), "type": t}
    heads = kv_heads * rng.choice([1, 2, 4, 6, 7, 8, 8, 12])
    c = {"kind": kind, "rows": 1, "heads": heads, "kv_heads": kv_heads, "dim": dim, "vdim": vdim, "shared": 0, "low": 0, "high": 0, "type": t}
    if kind == "attend":
        high = _log(rng, 1, 32768)
        c["rows"] = _log(rng, 1, max(1, min(128, 120000000 // (high * kv_heads * (dim + vdim)))))
        c["low"], c["high"] = rng.choice([0, 1, high // 8, high]), high
        return c
    if rng.random() < 0.3:
        chunk = _log(rng, 1, 8192)
        c["rows"] = _log(rng, 1, max(1, min(2048, 16000000000 // (2 * (chunk + 1024) * heads * (dim + vdim)))))
        c["chunk"] = chunk
        return c
    c["shared"] = PAGE * _log(rng, 1, 256)
    c["rows"] = _log(rng, 1, max(1, min(256, 16000000000 // (2 * c["shared"] * heads * (dim + vdim)))))
    c["high"] = _log(rng, 1, 1000)
    c["low"] = rng.choice([0, 1, c["high"]])
    return c


# ---- inputs ------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows(g, n, heads, dim, t, channels=True):
    """Rows [n, heads, dim]: tokens of different sizes, a few channels that stand out."""
    x = torch.randn(n, heads, dim, generator=g, device="cuda")
    x *= torch.exp(0.3 * torch.randn(n, 1, 1, generator=g, device="cuda"))
    if channels:
        x *= torch.where(torch.rand(1, heads, dim, generator=g, device="cuda") < 0.02, 4.0, 1.0)
    return x.to(TYPES[t])


def turns_of(rot, theta, scaling):
    """Turns per position of every pair [rot / 2] (f64), and what the rotated elements are multiplied with."""
    s = SCALINGS[scaling]
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    mult = 1.0
    if scaling == "linear":
        f = [x / s["factor"] for x in f]
    elif scaling == "bands":
        out = []
        for x in f:
            waves = s["original"] * x / (2.0 * math.pi)  # how often the pair turns within the original length
            keep = min(max((waves - s["low"]) / (s["high"] - s["low"]), 0.0), 1.0)
            out.append(x * ((1.0 - keep) / s["factor"] + keep))
        f = out
    elif scaling == "yarn":
        at = lambda beta: rot * math.log(s["original"] / (2.0 * math.pi * beta)) / (2.0 * math.log(theta))
        lo, hi = max(math.floor(at(s["fast"])), 0), min(math.ceil(at(s["slow"])), rot - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(rot // 2)]
        f = [x * (r / s["factor"] + 1.0 - r) for x, r in zip(f, ramp)]
        mult = 0.1 * math.log(s["factor"]) + 1.0
    return torch.tensor([x / (2.0 * math.pi) for x in f], dtype=torch.float64), mult


def _rope_inputs(case, seed):
    g, rows = _gen(seed), case["rows"]
    x = _rows(g, rows, case["heads"] + case["beside"], case["dim"], case["type"]).view(rows, -1)
    first = int(torch.randint(0, max(1, case["far"] - rows + 1), (1,), generator=g, device="cuda"))
    pos = torch.randint(0, case["far"], (rows,), generator=g, device="cuda") if rows <= 64 else first + torch.arange(rows, device="cuda")
    return x, pos.to(torch.int32)


def _places(g, case):
    """Rows' sequences and positions, every sequence's length, the page table and the number of pages."""
    rows = case["rows"]
    if case["kind"] == "cache":
        seqs = case["seqs"]
        if seqs == rows:  # newest tokens
            seq, pos = torch.arange(rows, device="cuda"), torch.randint(0, case["far"], (rows,), generator=g, device="cuda")
        else:  # portions of prompts
            each = -(-rows // seqs)
            seq, pos = torch.arange(rows, device="cuda") // each, torch.arange(rows, device="cuda") % each + (case["far"] - rows) // 2
        lens = [case["far"]] * seqs
    elif "chunk" in case:
        seq, pos, lens = torch.zeros(rows, dtype=torch.int64, device="cuda"), case["chunk"] + torch.arange(rows, device="cuda"), [case["chunk"] + rows]
    else:
        # lengths between low and high tokens behind the shared ones, spread over their logarithm; the longest is there
        low, high = case["low"], case["high"]
        u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        length = torch.exp(math.log(low + 1) + u * (math.log(high + 1) - math.log(low + 1))) - 1
        length = length.round().long().clamp(low, high)
        length[rows // 2] = high
        seq, pos = torch.arange(rows, device="cuda"), case["shared"] + length - 1
        lens = (case["shared"] + length).tolist()
    shared = case.get("shared", 0) // PAGE
    need = [max(0, -(-n // PAGE) - shared) for n in lens]
    n_pages = shared + sum(need) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(1, shared + max(need)), dtype=torch.int32, device="cuda")
    table[:, :shared] = order[:shared]
    at = shared
    for i, n in enumerate(need):
        table[i, shared : shared + n] = order[at : at + n]
        at += n
    return seq.to(torch.int32), pos.to(torch.int32), lens, table, n_pages


def _context(lens, shared):
    """(sequence, position) of every cached token: the shared ones once, as the first sequence's."""
    seq = [torch.zeros(shared, dtype=torch.int64, device="cuda")] + [torch.full((max(0, n - shared),), i, dtype=torch.int64, device="cuda") for i, n in enumerate(lens)]
    pos = [torch.arange(shared, device="cuda")] + [torch.arange(shared, max(n, shared), device="cuda") for n in lens]
    return torch.cat(seq), torch.cat(pos)


def _cache_inputs(case, seed):
    """What the cache cases and the attention cases have before the library or the plain form sees it."""
    g = _gen(seed)
    seq, pos, lens, table, n_pages = _places(g, case)
    s = {"case": case, "seq": seq, "pos": pos, "table": table, "n_pages": n_pages}
    if case["kind"] == "cache":
        s["new"] = (seq.long(), pos.long())
    else:
        s["q"] = _rows(g, case["rows"], case["heads"], case["dim"], case["type"], channels=False)
        s["new"] = _context(lens, case["shared"])
    n = s["new"][0].numel()
    s["k"] = _rows(g, n, case["kv_heads"], case["dim"], case["type"])
    s["v"] = _rows(g, n, case["kv_heads"], case["vdim"], case["type"])
    if case["kind"] != "cache" and n:
        s["v"][::5] *= 0.125  # tokens that matter little, the first among them
    return s


def prepare(case, seed):
    if case["kind"] == "rope":
        x, pos = _rope_inputs(case, seed)
        s = {"case": case, "x": x, "pos": pos}
        if own:
            import homura_b200 as hm

            turns, s["mult"] = hm.rope_turns(case["theta"], case["rot"], **SCALINGS[case["scaling"]])
            s["turns"] = torch.from_numpy(turns).cuda()
            s["y"] = torch.empty(case["rows"], case["heads"] * case["dim"], dtype=x.dtype, device="cuda")
        else:
            turns, s["mult"] = turns_of(case["rot"], case["theta"], case["scaling"])
            s["turns"] = turns.cuda()
        return s
    s = _cache_inputs(case, seed)
    if own:
        _lay_out(s)
    else:
        shape = (s["n_pages"] * PAGE, case["kv_heads"])
        s["codes"] = [torch.zeros(*shape, case[d], dtype=torch.int8, device="cuda") for d in ("dim", "vdim")]
        s["scales"] = [torch.zeros(*shape, device="cuda") for _ in range(2)]
        if case["kind"] != "cache":
            _plain_write(s)
    if case["kind"] != "cache":
        del s["k"], s["v"], s["new"]
    return s


# ---- plain forms ---------------------------------------------------------------------------------


def _plain_rope(s):
    c, x = s["case"], s["x"]
    rows, heads, dim, rot = c["rows"], c["heads"], c["dim"], c["rot"]
    x = x[:, : heads * dim].float().view(rows, heads, dim)
    angle = 2.0 * math.pi * torch.remainder(s["pos"].double()[:, None] * s["turns"], 1.0)  # far positions: 64 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    turned, rest = x[..., :rot], x[..., rot:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if c["neighbours"] else (turned[..., : rot // 2], turned[..., rot // 2 :])
    na, nb = (a * cos - b * sin) * s["mult"], (a * sin + b * cos) * s["mult"]
    turned = torch.stack([na, nb], -1).flatten(-2) if c["neighbours"] else torch.cat([na, nb], -1)
    return torch.cat([turned, rest], -1).view(rows, heads * dim).to(s["x"].dtype)


def _quantised(x):
    """Codes (int8) and scales [..., 1] of rows [..., dim]."""
    x = x.float()
    m = x.abs().amax(-1, keepdim=True)
    some = m >= TINY
    safe = torch.where(some, m, 1.0)
    codes = torch.where(some, torch.round(x * (127.0 / safe)), 0.0)
    return codes.to(torch.int8), torch.where(some, m / 127.0, 0.0)


def _plain_slots(s, seq, pos):
    return s["table"][seq, pos // PAGE].long() * PAGE + pos % PAGE


def _plain_write(s):
    slots = _plain_slots(s, *s["new"])
    for i, x in enumerate((s["k"], s["v"])):
        codes, scales = _quantised(x)
        s["codes"][i].index_copy_(0, slots, codes)
        s["scales"][i].index_copy_(0, slots, scales[..., 0])


def _plain_cache(s):
    _plain_write(s)
    slots = _plain_slots(s, *s["new"])
    return [(s["codes"][i][slots].float() * s["scales"][i][slots][..., None]).to(x.dtype) for i, x in enumerate((s["k"], s["v"]))]


def _part(q, k, v, seen):
    """Maximum, sum and weighted values of a part of the softmax: q [b, pairs, dim], k and v [b, tokens, .], seen [b or 1, pairs, tokens]."""
    score = torch.bmm(q, k.transpose(1, 2)).masked_fill_(~seen, -math.inf)
    m = score.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(score - m)
    return m, p.sum(-1, keepdim=True), torch.bmm(p, v)


def _plain_attend(s):
    c, pos = s["case"], s["pos"].long()
    M, H, G, D, E = c["rows"], c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    group = H // G
    q = s["q"].float().view(M, G, group, D) * (1.0 / math.sqrt(D))
    values = lambda i, slots: s["codes"][i][slots].float() * s["scales"][i][slots][..., None]  # [..., tokens, G, dim]
    parts = []
    common = (c["chunk"] + M) if "chunk" in c else c["shared"]
    if common:
        at = torch.arange(common, device="cuda")
        slots = _plain_slots(s, 0, at)
        k, v = values(0, slots).transpose(0, 1), values(1, slots).transpose(0, 1)  # [G, tokens, dim]
        seen = (at[None] <= pos[:, None]).repeat_interleave(group, 0)[None]  # [1, M * group, tokens]
        parts.append([x.view(G, M, group, -1).transpose(0, 1) for x in _part(q.transpose(0, 1).reshape(G, M * group, D), k, v, seen)])
    most = s["table"].shape[1] * PAGE
    if most > common and "chunk" not in c:
        at = torch.arange(common, most, device="cuda")
        slots = _plain_slots(s, s["seq"].long()[:, None], at[None])
        k, v = values(0, slots).transpose(1, 2).reshape(M * G, -1, D), values(1, slots).transpose(1, 2).reshape(M * G, -1, E)
        seen = (at[None] <= pos[:, None]).repeat_interleave(G, 0)[:, None]
        parts.append([x.view(M, G, group, -1) for x in _part(q.reshape(M * G, group, D), k, v, seen)])
    top = torch.stack([m for m, _, _ in parts]).amax(0)
    total = sum(l * torch.exp(m - top) for m, l, _ in parts)
    out = sum(o * torch.exp(m - top) for m, _, o in parts) / total.clamp_min(1e-30)
    return out.reshape(M, H * E).to(s["q"].dtype)


# ---- the library's calls -------------------------------------------------------------------------


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _lay_out(s):
    """What a program keeps between calls: the cache and buffers.  Attention cases have their contexts written."""
    import homura_b200 as hm

    c, dev, t = s["case"], s["k"].device, TYPES[s["case"]["type"]]
    s["pool"] = torch.empty(hm.kv8_pool_bytes(c["kv_heads"], c["dim"], c["vdim"], s["n_pages"]), dtype=torch.uint8, device=dev)
    s["cache"] = hm.KV8Cache(c["kv_heads"], c["dim"], c["vdim"], s["pool"].data_ptr(), s["n_pages"], (s["table"].data_ptr(), *s["table"].shape))
    s["xt"] = F32 if c["type"] == "f32" else BF16
    if c["kind"] == "cache":
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        return
    seq, pos = (x.to(torch.int32).contiguous() for x in s["new"])
    s["cache"].write((s["k"].data_ptr(), pos.numel()), s["v"].data_ptr(), seq.data_ptr(), pos.data_ptr(), dtype=s["xt"], stream=_stream())
    torch.cuda.synchronize()  # seq and pos are let go
    s["out"] = torch.empty(c["rows"], c["heads"] * c["vdim"], dtype=t, device=dev)
    s["n_shared"] = -(-(c["chunk"] + c["rows"]) // PAGE) if "chunk" in c else c["shared"] // PAGE
    s["work"] = torch.empty(max(16, s["cache"].attend_bytes(c["rows"], c["heads"], s["n_shared"])), dtype=torch.uint8, device=dev)


def _own(s):
    import homura_b200 as hm

    c, st = s["case"], _stream()
    if c["kind"] == "rope":
        hm.rope((s["x"].data_ptr(), c["rows"]), c["heads"], c["dim"], s["turns"].data_ptr(), s["pos"].data_ptr(), rot=c["rot"], neighbours=c["neighbours"], magnitude=s["mult"],
                dtype=F32 if c["type"] == "f32" else BF16, ldx=s["x"].shape[1], y=s["y"].data_ptr(), stream=st)
        return s["y"]
    seq, pos, rows = s["seq"].data_ptr(), s["pos"].data_ptr(), c["rows"]
    if c["kind"] == "cache":
        s["cache"].write((s["k"].data_ptr(), rows), s["v"].data_ptr(), seq, pos, dtype=s["xt"], stream=st)
        s["cache"].read((seq, rows), pos, s["k_out"].data_ptr(), s["v_out"].data_ptr(), dtype=s["xt"], stream=st)
        return [s["k_out"], s["v_out"]]
    s["cache"].attend((s["q"].data_ptr(), rows), seq, pos, c["heads"], 1.0 / math.sqrt(c["dim"]), shared=(s["table"].data_ptr(), s["n_shared"]), dtype=s["xt"], out=s["out"].data_ptr(), work=s["work"].data_ptr(), stream=st)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    return _plain_rope(state) if kind == "rope" else _plain_cache(state) if kind == "cache" else _plain_attend(state)


# ---- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    c = case
    size, rows = {"f32": 4, "bf16": 2}[c["type"]], c["rows"]
    if c["kind"] == "rope":
        return {"bytes": int(rows * (c["heads"] * c["dim"] * 2 * size + 4) + 4 * c["rot"]), "flops": rows * c["heads"] * c["rot"] * 3}
    token = c["kv_heads"] * (c["dim"] + c["vdim"] + 8)  # codes and scales
    if c["kind"] == "cache":
        return {"bytes": int(rows * (c["kv_heads"] * (c["dim"] + c["vdim"]) * 2 * size + 2 * token + 8)), "flops": rows * c["kv_heads"] * (c["dim"] + c["vdim"]) * 4}
    if "chunk" in c:
        tokens, seen = c["chunk"] + rows, rows * (c["chunk"] + (rows + 1) / 2)
    else:
        # mean of the lengths, which are spread over their logarithm
        lo, hi = c["low"] + 1, c["high"] + 1
        mean = (hi - lo) / math.log(hi / lo) - 1 if hi > lo else c["low"]
        tokens, seen = c["shared"] + rows * mean, rows * (c["shared"] + mean)
    return {"bytes": int(tokens * token + rows * (c["heads"] * (c["dim"] + c["vdim"]) * size + 8)), "flops": int(2 * seen * c["heads"] * (c["dim"] + c["vdim"]))}


# ---- the definition in 64 bits -----------------------------------------------------------------------


def _exact_turns(case):
    """Radians per position, each pair on its own."""
    rot, theta, kind = case["rot"], case["theta"], case["scaling"]
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    f = torch.exp(-i / rot * math.log(theta))
    s = SCALINGS[kind]
    if kind == "linear":
        return f / s["factor"], 1.0
    if kind == "bands":
        wave = 2 * math.pi / f
        middle = (s["original"] / wave - s["low"]) / (s["high"] - s["low"])
        mixed = (1 - middle) * f / s["factor"] + middle * f
        return torch.where(wave > s["original"] / s["low"], f / s["factor"], torch.where(wave < s["original"] / s["high"], f, mixed)), 1.0
    if kind == "yarn":
        bound = [rot * math.log(s["original"] / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (s["fast"], s["slow"])]
        lo, hi = max(math.floor(bound[0]), 0), min(math.ceil(bound[1]), rot - 1)
        r = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / (hi - lo if hi > lo else 0.001)).clamp(0, 1)
        return f / s["factor"] * r + f * (1 - r), 1 + 0.1 * math.log(s["factor"])
    return f, 1.0


def _exact_rope(case, seed):
    x, pos = _rope_inputs(case, seed)
    rows, heads, dim, rot = case["rows"], case["heads"], case["dim"], case["rot"]
    f, mult = _exact_turns(case)
    angle = pos.double()[:, None] * f.cuda()
    z = torch.polar(torch.full_like(angle, mult), angle)[:, None, :]
    y = x[:, : heads * dim].double().reshape(rows, heads, dim).clone()
    if case["neighbours"]:
        w = torch.view_as_complex(y[..., :rot].reshape(rows, heads, rot // 2, 2).contiguous()) * z
        y[..., :rot] = torch.view_as_real(w).reshape(rows, heads, rot)
    else:
        w = torch.complex(y[..., : rot // 2].contiguous(), y[..., rot // 2 : rot].contiguous()) * z
        y[..., : rot // 2], y[..., rot // 2 : rot] = w.real, w.imag
    return y.reshape(rows, heads * dim)


def _exact_values(x):
    """What the cache holds of rows [..., dim]: the roundings of the definition are to f32, the rest is in 64 bits."""
    x = x.double()
    m = x.abs().max(-1, keepdim=True).values
    none = m < TINY
    up = (127.0 / m.masked_fill(none, 1.0)).float().double()
    codes = torch.round((x * up).float().double())
    return (codes * (m / 127.0).float().double()).masked_fill(none, 0.0)


def exact(case, seed):
    if case["kind"] == "rope":
        return _exact_rope(case, seed)
    s = _cache_inputs(case, seed)
    if case["kind"] == "cache":
        return [_exact_values(s["k"]), _exact_values(s["v"])]
    M, H, G = case["rows"], case["heads"], case["kv_heads"]
    q = s["q"].double().view(M, G, H // G, -1) / math.sqrt(case["dim"])
    # the context's tokens in the order they were made: the shared ones, then every sequence's own
    shared, pos = case["shared"], s["pos"].tolist()
    own_tokens = torch.bincount(s["new"][0][shared:], minlength=s["table"].shape[0]).tolist()
    first = [shared]
    for n in own_tokens:
        first.append(first[-1] + n)
    kp, vp = _exact_values(s["k"][:shared]), _exact_values(s["v"][:shared])
    out = torch.zeros(M, G, H // G, case["vdim"], dtype=torch.float64, device="cuda")
    ko = vo = None
    for m in range(M):
        if pos[m] < 0:
            continue
        i = int(s["seq"][m]) if "chunk" not in case else 0
        if "chunk" not in case or ko is None:
            ko, vo = _exact_values(s["k"][first[i] : first[i + 1]]), _exact_values(s["v"][first[i] : first[i + 1]])
        k, v = torch.cat([kp, ko])[: pos[m] + 1], torch.cat([vp, vo])[: pos[m] + 1]
        weight = torch.softmax(torch.einsum("ghd,tgd->ght", q[m], k), -1)
        out[m] = torch.einsum("ght,tgd->ghd", weight, v)
    return out.view(M, -1)
