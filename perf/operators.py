"""Operators on 4-bit microscaled floats and on products grouped by expert, for timing and for comparing with their plain forms.

Kinds of cases:

* ``quantise``   rows to the 4-bit image and back to the values it stands for.
* ``rows``       few rows as they are times 4-bit weights (decoding).
* ``pairs``      the same where every (token, chosen expert) pair has its own weights (decoding with a mixture).
* ``product``    many rows, rounded to the weights' type, times the weights: 4-bit on both sides, or bf16.
* ``experts``    the same grouped by expert: the plan from the router's ids, the rows gathered, one product over ragged groups.
* ``ffn``        a mixture's feed-forward as it is used: plan, gate and up, gated activations, down, weighted sum.

A block of 32 values along a row has the scale 2^(floor(log2 max|x|) - 2) and codes of 1 + 2 + 1 bits (sign, exponent, mantissa): values 0, 0.5, 1,
1.5, 2, 3, 4 and 6 times the scale, to nearest, ties to the even code, saturated at 6.  Weights come as GGUF blocks of 17 bytes: the scale's exponent
+ 127, then 16 bytes with the codes of values i (low) and i + 16 (high).  Widths and experts are those of the bench's 0.5 B and 1.5 B architectures.
"""
from __future__ import annotations

import math

import torch

own = False

F32, BF16, MXFP4 = 0, 1, 10  # the library's type numbers
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # a decoded token's row on its way into a 4-bit product: the smallest call
        {"name": "quantise-token", "kind": "quantise", "rows": 1, "K": 896, "type": "f32"},
        # the activations of a prompt in front of the down projection
        {"name": "quantise-prompt", "kind": "quantise", "rows": 1999, "K": 8960, "type": "bf16"},
        # one token, gate and up of the 0.5 B stack
        {"name": "token-gate-up", "kind": "rows", "rows": 1, "K": 896, "N": 9728, "type": "f32"},
        # seven sequences at the LM head of the 1.5 B stack: the most bytes
        {"name": "rows-head", "kind": "rows", "rows": 7, "K": 1536, "N": 151936, "type": "bf16"},
        # one token's chosen experts, gate and up
        {"name": "pairs-token", "kind": "pairs", "rows": 1, "top": 4, "experts": 16, "K": 896, "N": 1920, "type": "f32"},
        # a batch of 64 sequences, down projection of the 1.5 B stack
        {"name": "product-64", "kind": "product", "format": "mxfp4", "rows": 64, "K": 8960, "N": 1536, "type": "f32", "out": "f32"},
        # a prompt, gate and up of the 1.5 B stack: the most operations
        {"name": "product-prompt", "kind": "product", "format": "mxfp4", "rows": 1999, "K": 1536, "N": 17920, "type": "bf16", "out": "bf16"},
        # a batch of 64 sequences, mixture of 32 experts, gate and up (16 rows per expert)
        {"name": "experts-64", "kind": "experts", "format": "mxfp4", "rows": 64, "top": 8, "experts": 32, "none": 2, "K": 1536, "N": 2240, "type": "f32", "out": "f32"},
        # a prompt through the same kind of mixture, uneven groups of some 500 rows
        {"name": "experts-prompt", "kind": "experts", "format": "mxfp4", "rows": 2048, "top": 8, "experts": 32, "none": 0, "K": 1536, "N": 1920, "type": "bf16", "out": "bf16"},
        # bf16 experts of the 0.5 B mixture, a prompt of odd length
        {"name": "experts-bf16", "kind": "experts", "format": "bf16", "rows": 1021, "top": 4, "experts": 16, "none": 0, "K": 896, "N": 2432, "type": "bf16", "out": "bf16"},
        # whole feed-forwards: a few sequences, and a prompt
        {"name": "ffn-few", "kind": "ffn", "format": "mxfp4", "rows": 5, "top": 4, "experts": 16, "none": 0, "K": 896, "ff": 1216},
        {"name": "ffn-prompt", "kind": "ffn", "format": "mxfp4", "rows": 517, "top": 8, "experts": 32, "none": 2, "K": 1536, "ff": 1120},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _blocks(rng, lo, hi):
    return 32 * _log(rng, lo, hi)


def draw(rng):
    kind = rng.choice(["quantise", "quantise", "rows", "rows", "pairs", "product", "product", "experts", "experts", "experts", "ffn"])
    t = rng.choice(["f32", "bf16"])
    if kind == "quantise":
        K = _log(rng, 1, 18000)
        return {"kind": kind, "rows": _log(rng, 1, min(4000, 17000000 // K)), "K": K, "type": t}
    if kind == "rows":
        K = _blocks(rng, 1, 280)
        return {"kind": kind, "rows": rng.randrange(1, 9), "K": K, "N": _log(rng, 1, min(152000, 230000000 // K)), "type": t}
    if kind == "pairs":
        top, experts = rng.choice([(1, 8), (2, 8), (4, 16), (8, 32), (6, 64)])
        return {"kind": kind, "rows": rng.randrange(1, 5), "top": top, "experts": experts, "K": _blocks(rng, 2, 64), "N": _log(rng, 30, 3000), "type": t}
    fmt = rng.choice(["mxfp4", "mxfp4", "bf16"])
    if kind == "product":
        K, rows = _blocks(rng, 1, 280), _log(rng, 1, 4000)
        return {"kind": kind, "format": fmt, "rows": rows, "K": K, "N": _log(rng, 1, min(18000, 50000000000 // (K * rows), 120000000 // K)), "type": t, "out": rng.choice(["f32", "bf16"])}
    top, experts = rng.choice([(1, 8), (2, 8), (4, 16), (8, 32), (6, 64)])
    rows = _log(rng, 1, 2000)
    none = rng.choice([0, 0, 2])
    if kind == "experts":
        K = _blocks(rng, 2, 64)
        return {"kind": kind, "format": fmt, "rows": rows, "top": top, "experts": experts, "none": none, "K": K, "N": _log(rng, 30, min(3000, 40000000000 // (rows * top * K), 100000000 // (experts * K))), "type": t,
                "out": rng.choice(["f32", "bf16"])}
    return {"kind": kind, "format": "mxfp4", "rows": min(rows, 600), "top": top, "experts": experts, "none": none, "K": _blocks(rng, 2, 48), "ff": _blocks(rng, 1, 38)}


# ---- inputs ------------------------------------------------------------------------------------


def _activations(g, rows, K, t):
    """Rows of different sizes, a few channels that stand out."""
    x = torch.randn(rows, K, generator=g, device="cuda")
    x *= torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))
    x *= torch.where(torch.rand(1, K, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return x.to(TYPES[t])


def _gguf_weights(g, n, K):
    """Weights of about N(0, 0.02) as blocks [n, K / 32, 17] bytes."""
    w = torch.randn(n, K // 32, 32, generator=g, device="cuda") * 0.02
    values, exponent = _quantised(w)
    scaled = values * _power(-exponent)
    codes = (torch.searchsorted(torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda"), scaled.abs().contiguous()) + 8 * (scaled < 0)).to(torch.uint8)
    return torch.cat([(exponent + 127).to(torch.uint8), codes[..., :16] | (codes[..., 16:] << 4)], -1).contiguous()


def _weights(g, case, n, K):
    return _gguf_weights(g, n, K) if case["format"] == "mxfp4" else (torch.randn(n, K, generator=g, device="cuda") * 0.02).to(torch.bfloat16)


def _routing(g, case):
    """Ids of the chosen experts (-1: none) and their weights; some experts are chosen more often."""
    n = case["experts"] + case.get("none", 0)
    score = torch.randn(case["rows"], n, generator=g, device="cuda") + torch.randn(1, n, generator=g, device="cuda") * 0.5
    top = torch.topk(torch.softmax(score, -1), case["top"], dim=-1)
    ids = torch.where(top.indices < case["experts"], top.indices, -1).to(torch.int32)
    return ids.contiguous(), top.values.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, s = case["kind"], {"case": case}
    s["x"] = _activations(g, case["rows"], case["K"], case.get("type", "f32"))
    if kind == "rows":
        s["w"] = _gguf_weights(g, case["N"], case["K"])
    elif kind == "pairs":
        s["w"] = _gguf_weights(g, case["experts"] * case["N"], case["K"])
    elif kind == "product":
        s["w"] = _weights(g, case, case["N"], case["K"])
    elif kind == "experts":
        s["w"] = _weights(g, case, case["experts"] * case["N"], case["K"])
    elif kind == "ffn":
        s["w"] = _weights(g, case, case["experts"] * 2 * case["ff"], case["K"])
        s["w2"] = _weights(g, case, case["experts"] * case["K"], case["ff"])
    if "experts" in case:
        s["ids"], s["weights"] = _routing(g, case)
        # rows of the fullest expert: room of the plain form's groups
        s["most"] = int(torch.bincount((s["ids"].view(-1) + 1).long(), minlength=case["experts"] + 1)[1:].max())
    if own:
        _lay_out(s)
    return s


# ---- plain forms ---------------------------------------------------------------------------------


def _power(e):
    """2^e, e from -126 to 127, from its bits (pow() may be off by a bit)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantised(x):
    """Values and scale exponents of blocks [..., 32]."""
    x = x.float()
    exponent = (torch.frexp(x.abs().amax(-1, keepdim=True)).exponent - 3).clamp_min(-127)
    v = x * _power(-exponent)
    step = 0.5 * (1.0 + (v.abs() >= 2) + 2.0 * (v.abs() >= 4))
    return (torch.round(v / step) * step).clamp(-6.0, 6.0) * 0.5 * _power(exponent + 1), exponent


def _round_rows(x, fmt):
    """Rows [rows, K] rounded to the format, as f32."""
    if fmt == "bf16":
        return x.to(torch.bfloat16).float()
    K = x.shape[-1]
    pad = torch.nn.functional.pad(x.float(), (0, -K % 32))
    return _quantised(pad.view(*x.shape[:-1], -1, 32))[0].view(*x.shape[:-1], -1)[..., :K]


def _values(w):
    """Weights [n, K] as f32, from GGUF blocks or bf16."""
    if w.dtype == torch.bfloat16:
        return w.float()
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=w.device)
    codes = torch.cat([w[..., 1:] & 15, w[..., 1:] >> 4], -1)
    return (table[codes.int()] * 0.5 * _power(w[..., :1].int() - 126)).view(w.shape[0], -1)


def _grouped(x, w, ids, most):
    """[pairs, N]: row p of x times the weights [E, N, K] of expert ids[p]; zeros where there is none."""
    E = w.shape[0]
    order = torch.argsort(torch.where(ids < 0, E, ids), stable=True)
    sorted_ids = ids[order].long()
    count = torch.zeros(E + 1, dtype=torch.int64, device=x.device).index_add_(0, (ids + 1).long(), torch.ones_like(ids, dtype=torch.int64))
    first = torch.cumsum(count, 0) - count  # by id + 1: those without an expert stand last in `order`
    place = torch.arange(ids.numel(), device=x.device) - (first[sorted_ids + 1] - count[0])
    room = torch.zeros(E, max(most, 1), x.shape[1], device=x.device)
    real = sorted_ids >= 0
    e, at = torch.where(real, sorted_ids, 0), torch.where(real, place, 0)
    room.index_put_((e, at), torch.where(real[:, None], x[order], 0.0), accumulate=True)
    y = torch.bmm(room, w.transpose(1, 2))
    out = torch.empty(ids.numel(), w.shape[1], device=x.device)
    out[order] = torch.where(real[:, None], y[e, at], 0.0)
    return out


def _plain(s):
    c, x = s["case"], s["x"]
    kind = c["kind"]
    if kind == "quantise":
        return _round_rows(x, "mxfp4")
    if kind == "rows":
        return x.float() @ _values(s["w"]).T
    if kind == "product":
        return (_round_rows(x, c["format"]) @ _values(s["w"]).T).to(TYPES[c["out"]])
    ids = s["ids"].view(-1)
    if kind == "pairs":
        return _grouped(x.float().repeat_interleave(c["top"], 0), _values(s["w"]).view(c["experts"], c["N"], c["K"]), ids, s["most"])
    rows = _round_rows(x, c["format"]).repeat_interleave(c["top"], 0)
    if kind == "experts":
        return _grouped(rows, _values(s["w"]).view(c["experts"], c["N"], c["K"]), ids, s["most"]).to(TYPES[c["out"]])
    h = _grouped(rows, _values(s["w"]).view(c["experts"], 2 * c["ff"], c["K"]), ids, s["most"])
    gate, up = h[:, : c["ff"]], h[:, c["ff"] :]
    act = _round_rows(gate / (1.0 + torch.exp(-gate)) * up, c["format"])
    y = _grouped(act, _values(s["w2"]).view(c["experts"], c["K"], c["ff"]), ids, s["most"]).view(c["rows"], c["top"], c["K"])
    return (x + (y * s["weights"][..., None]).sum(1)).to(torch.bfloat16)


# ---- the library's calls -------------------------------------------------------------------------


def _lay_out(s):
    """What a program keeps between calls: weight images, and buffers."""
    import homura_b200 as hm

    c, dev = s["case"], s["x"].device
    kind, rows, K = c["kind"], c["rows"], c["K"]
    s["xt"] = F32 if s["x"].dtype == torch.float32 else BF16
    fmt = BF16 if c.get("format") == "bf16" else MXFP4

    def image(rows, K, fmt=fmt):
        return torch.empty(hm.image_bytes(fmt, rows, K), dtype=torch.uint8, device=dev)

    def weight_images(w, n, K):  # one image per n rows, back to back
        each = hm.image_bytes(fmt, n, K)
        to = torch.empty(w.shape[0] // n * each, dtype=torch.uint8, device=dev)
        step = w[0].numel() * w.element_size() * n
        for i in range(w.shape[0] // n):
            if fmt == MXFP4:
                hm.image_from_blocks((w.data_ptr() + i * step, n), K=K, image=to.data_ptr() + i * each, stream=_stream())
            else:
                hm.image_pack((w.data_ptr() + i * step, n), BF16, K=K, x_dtype=BF16, image=to.data_ptr() + i * each, stream=_stream())
        return to

    if kind == "quantise":
        s["image"], s["y"] = image(rows, K), torch.empty(rows, K, device=dev)
        return
    n = 2 * c["ff"] if kind == "ffn" else c["N"]
    s["wi"] = weight_images(s["w"], n, K)
    if kind in ("rows", "product"):
        s["y"] = torch.empty(rows, n, device=dev, dtype=TYPES[c.get("out", "f32")])
    else:
        s["y"] = torch.zeros(rows * c["top"], n, device=dev, dtype=TYPES[c.get("out", "f32")])
    if kind == "product":
        s["image"] = image(rows, K)
    if kind in ("experts", "ffn"):
        pairs = rows * c["top"]
        s["plan"] = torch.empty(hm.expert_plan_ints(pairs, c["experts"]), dtype=torch.int32, device=dev)
        s["plan_rows"] = hm.expert_plan_rows(pairs, c["experts"])
        s["image"] = image(s["plan_rows"], K)
    if kind == "ffn":
        s["w2i"] = weight_images(s["w2"], K, c["ff"])
        s["image2"] = image(s["plan_rows"], c["ff"])
        s["down"] = torch.empty(rows * c["top"], K, device=dev)
        s["out"] = torch.empty(rows, K, device=dev, dtype=torch.bfloat16)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own(s):
    import homura_b200 as hm

    c, st = s["case"], _stream()
    kind, rows, K = c["kind"], c["rows"], c["K"]
    x = (s["x"].data_ptr(), rows)
    if kind == "quantise":
        hm.image_pack(x, MXFP4, K=K, x_dtype=s["xt"], image=s["image"].data_ptr(), stream=st)
        hm.image_unpack((s["image"].data_ptr(), rows), MXFP4, K=K, out=s["y"].data_ptr(), stream=st)
        return s["y"]
    if kind == "rows":
        hm.gemv_mx4(x, s["wi"].data_ptr(), c["N"], K=K, x_dtype=s["xt"], y=s["y"].data_ptr(), stream=st)
        return s["y"]
    if kind == "pairs":
        hm.expert_gemv(x, s["wi"].data_ptr(), s["ids"].data_ptr(), c["N"], top=c["top"], experts=c["experts"], K=K, x_dtype=s["xt"], y=s["y"].data_ptr(), stream=st)
        return s["y"]
    fmt = BF16 if c["format"] == "bf16" else MXFP4
    if kind == "product":
        hm.image_pack(x, fmt, K=K, x_dtype=s["xt"], image=s["image"].data_ptr(), stream=st)
        hm.gemm_image((s["image"].data_ptr(), rows), s["wi"].data_ptr(), c["N"], fmt, K=K, y=s["y"].data_ptr(), y_dtype=F32 if c["out"] == "f32" else BF16, stream=st)
        return s["y"]
    pairs, plan = rows * c["top"], s["plan"].data_ptr()
    hm.expert_plan((s["ids"].data_ptr(), pairs), c["experts"], plan=plan, stream=st)
    hm.image_pack(x, fmt, K=K, x_dtype=s["xt"], plan=plan, pairs=pairs, experts=c["experts"], top=c["top"], image=s["image"].data_ptr(), stream=st)
    if kind == "experts":
        hm.expert_gemm(s["image"].data_ptr(), s["wi"].data_ptr(), plan, c["N"], fmt, pairs=pairs, experts=c["experts"], K=K, y=s["y"].data_ptr(), y_dtype=F32 if c["out"] == "f32" else BF16, stream=st)
        return s["y"]
    ff = c["ff"]
    hm.expert_gemm(s["image"].data_ptr(), s["wi"].data_ptr(), plan, 2 * ff, fmt, pairs=pairs, experts=c["experts"], K=K, y=s["y"].data_ptr(), stream=st)
    hm.image_pack((s["y"].data_ptr(), pairs), fmt, K=ff, plan=plan, pairs=pairs, experts=c["experts"], glu=True, image=s["image2"].data_ptr(), stream=st)
    hm.expert_gemm(s["image2"].data_ptr(), s["w2i"].data_ptr(), plan, K, fmt, pairs=pairs, experts=c["experts"], K=ff, y=s["down"].data_ptr(), stream=st)
    hm.expert_sum((s["down"].data_ptr(), rows), s["ids"].data_ptr(), s["weights"].data_ptr(), top=c["top"], experts=c["experts"], width=K, resid=s["x"].data_ptr(), y=s["out"].data_ptr(), y_dtype=BF16, stream=st)
    return s["out"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    c, size = case, {"f32": 4, "bf16": 2, "mxfp4": 17 / 32}
    kind, rows, K = c["kind"], c["rows"], c["K"]
    x = rows * K * size[c.get("type", "f32")]
    if kind == "quantise":
        return {"bytes": int(x + rows * K * 4), "flops": rows * K}
    if kind == "rows":
        return {"bytes": int(x + c["N"] * K * 17 / 32 + rows * c["N"] * 4), "flops": 2 * rows * c["N"] * K}
    if kind == "product":
        return {"bytes": int(x + c["N"] * K * size[c["format"]] + rows * c["N"] * size[c["out"]]), "flops": 2 * rows * c["N"] * K}
    pairs = rows * c["top"]
    used = c["experts"] * (1 - (1 - c["top"] / (c["experts"] + c.get("none", 0))) ** rows)  # experts that some token has chosen, about
    n = 2 * c["ff"] if kind == "ffn" else c["N"]
    w = used * n * K * size[c.get("format", "mxfp4")]
    if kind in ("pairs", "experts"):
        return {"bytes": int(x + pairs * 4 + w + pairs * n * size[c.get("out", "f32")]), "flops": 2 * pairs * n * K}
    return {"bytes": int(x + pairs * 8 + 1.5 * w + rows * K * 2), "flops": 6 * pairs * c["ff"] * K}


# ---- the definition in 64 bits -----------------------------------------------------------------------


def _two_to(n):
    """2^n in 64 bits for whole numbers n."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _exact_rows(x, fmt):
    """Rows [rows, K] (f64) rounded to the format, in 64 bits."""
    if fmt == "bf16":
        return x.float().bfloat16().double()
    rows, K = x.shape
    full = torch.zeros(rows, (K + 31) // 32 * 32, dtype=torch.float64, device=x.device)
    full[:, :K] = x
    blocks = full.view(rows, -1, 32)
    largest = blocks.abs().max(-1, keepdim=True).values
    e = torch.where(largest > 0, torch.floor(torch.log2(largest.clamp_min(1e-300))), torch.zeros_like(largest))
    e = e + (_two_to(e + 1) <= largest).double() - (_two_to(e) > largest).double()  # where the logarithm was rounded over a power of two
    scale = _two_to((e - 2).clamp_min(-127))
    a = blocks.abs() / scale
    m = 0.5 * ((a > 0.25).double() + (a >= 0.75).double() + (a > 1.25).double() + (a >= 1.75).double()) + (a > 2.5).double() + (a >= 3.5).double() + 2.0 * (a > 5.0).double()
    return (m * scale * torch.sign(blocks)).view(rows, -1)[:, :K]


def _exact_weights(w):
    if w.dtype == torch.bfloat16:
        return w.double()
    low, high = w[..., 1:] & 15, w[..., 1:] >> 4
    code = torch.stack([low, high], -2).reshape(*w.shape[:-1], 32).long()
    e, m = (code >> 1) & 3, code & 1
    magnitude = torch.where(e > 0, _two_to(e - 1) * (1 + 0.5 * m.double()), 0.5 * m.double())
    return (torch.where(code >= 8, -magnitude, magnitude) * _two_to(w[..., :1].long() - 127)).reshape(w.shape[0], -1)


def _exact_experts(x, w, ids):
    out = torch.zeros(ids.numel(), w.shape[1], dtype=torch.float64, device=x.device)
    for e in range(w.shape[0]):
        at = (ids == e).nonzero().view(-1)
        out[at] = x[at] @ w[e].T
    return out


def exact(case, seed):
    s = prepare(case, seed)
    c, x = case, s["x"].double()
    kind, K = c["kind"], c["K"]
    if kind == "quantise":
        return _exact_rows(x, "mxfp4")
    w = _exact_weights(s["w"])
    if kind == "rows":
        return x @ w.T
    if kind == "product":
        return _exact_rows(x, c["format"]) @ w.T
    ids, E = s["ids"].view(-1), c["experts"]
    if kind == "pairs":
        return _exact_experts(x.repeat_interleave(c["top"], 0), w.view(E, -1, K), ids)
    first = _exact_experts(_exact_rows(x, c["format"]).repeat_interleave(c["top"], 0), w.view(E, -1, K), ids)
    if kind == "experts":
        return first
    gate, up = first.chunk(2, dim=1)
    act = _exact_rows(torch.sigmoid(gate) * gate * up, c["format"])
    second = _exact_experts(act, _exact_weights(s["w2"]).view(E, K, -1), ids)
    return x + torch.einsum("tjk,tj->tk", second.view(c["rows"], c["top"], K), s["weights"].double())
