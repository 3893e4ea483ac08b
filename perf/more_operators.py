"""The operators of serving in 4 bits (microscaled floating point), as a list of cases to time.

The format: 32 consecutive values of a row share a scale 2^e (a byte, e + 127; 255: not a number), and each is a code of
4 bits: sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Two codes a byte, the first in the low half.  A row of n values is n / 2
bytes of codes and n / 32 of scales.

quantize: rows are quantised and read back.  matmul: rows times weights in 4 bits, the rows in 16 bits or in 4 as well.
append: new tokens' q and k are rotated (and normalised) and k, v stored into pages in 4 bits.  attn: the new tokens of every
sequence attend over such pages.  Shapes are the framework's own (hidden 1024 and 3584, 8 query and 2 KV heads of 256, 64 rotary
dimensions, vocabulary 248320) and generic ones.

With `own` false `run` is the plain form in elementary torch operations; with `own` true it calls spock_amd.ops.
`exact` restates the definitions in float64.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # the rows of a small decoding batch before a product: nothing but latency
        {"name": "quantize_rows_16", "op": "quantize", "dtype": "f16", "rows": 16, "dim": 1024},
        # a model's largest matrix, laid out once when it is loaded
        {"name": "quantize_lm_head", "op": "quantize", "dtype": "bf16", "rows": 248320, "dim": 1024},
        # one decoded token against the vocabulary: the weights are read once
        {"name": "matmul_lm_head_1", "op": "matmul", "dtype": "f16", "rows": 1, "out": 248320, "dim": 1024, "bits": 16, "residual": False},
        # a decoding batch through a projection that adds to the residual stream
        {"name": "matmul_down_17", "op": "matmul", "dtype": "bf16", "rows": 17, "out": 1024, "dim": 3584, "bits": 16, "residual": True},
        # a prompt of odd length through a wide projection, activations kept in 16 bits
        {"name": "matmul_prompt_2001", "op": "matmul", "dtype": "bf16", "rows": 2001, "out": 14336, "dim": 4096, "bits": 16, "residual": False},
        # a prefill batch with activations in 4 bits too
        {"name": "matmul_both_8192", "op": "matmul", "dtype": "bf16", "rows": 8192, "out": 8192, "dim": 8192, "bits": 4, "residual": False},
        # one new token of 64 young sequences, the framework's heads
        {"name": "append_decode_64", "op": "append", "dtype": "f16", "heads": 8, "kv": 2, "dim": 256, "rot": 64, "axes": 3,
         "pairing": "halves", "norm": True, "page": 16, "seqs": 64, "new": 1, "lo": 1, "hi": 33},
        # a server's prefill batch of ragged prompts, full-width rotation
        {"name": "append_prompts_32k", "op": "append", "dtype": "bf16", "heads": 16, "kv": 4, "dim": 128, "rot": 128, "axes": 1,
         "pairing": "halves", "norm": False, "page": 64, "lens": "8192:8192,8191:12000,16385:16385"},
        # one decoded token at an ordinary context
        {"name": "attn_decode_1500", "op": "attn", "dtype": "f16", "heads": 8, "kv": 2, "dim": 256, "page": 16,
         "lens": "1:1500", "window": 0, "gate": True},
        # one decode step of a serving batch, ragged contexts: the cache is read once
        {"name": "attn_decode_64seqs", "op": "attn", "dtype": "bf16", "heads": 32, "kv": 8, "dim": 128, "page": 32,
         "seqs": 64, "new": 1, "lo": 300, "hi": 16000, "window": 0, "gate": False},
        # eight drafted tokens and the last one accepted, of 16 sequences
        {"name": "attn_drafts_16x9", "op": "attn", "dtype": "bf16", "heads": 8, "kv": 2, "dim": 256, "page": 16,
         "seqs": 16, "new": 9, "lo": 1000, "hi": 9000, "window": 0, "gate": False},
        # a chunk of a long prompt over what is in the cache already
        {"name": "attn_chunk_2048", "op": "attn", "dtype": "f16", "heads": 8, "kv": 2, "dim": 256, "page": 16,
         "lens": "2048:16384", "window": 0, "gate": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "append", "attn", "attn"])
    if op == "quantize":
        dim = 32 * _log_int(rng, 1, 512)
        return {"op": op, "dtype": rng.choice(["f16", "bf16", "f32"]), "dim": dim, "rows": _log_int(rng, 1, 60_000_000 // dim)}
    if op == "matmul":
        dim, out = 32 * _log_int(rng, 2, 512), _log_int(rng, 16, 32768)
        rows = min(_log_int(rng, 1, 8192), 500_000_000_000 // (dim * out))
        return {"op": op, "dtype": rng.choice(["f16", "bf16"]), "rows": rows, "out": out, "dim": dim,
                "bits": rng.choice([16, 16, 4]), "residual": rng.random() < 0.4}
    heads, kv, dim = rng.choice([(8, 2, 256), (8, 2, 256), (16, 4, 128), (32, 8, 128), (8, 1, 128), (4, 4, 128), (12, 3, 64), (7, 1, 64)])
    case = {"op": op, "dtype": rng.choice(["f16", "bf16"]), "heads": heads, "kv": kv, "dim": dim,
            "page": rng.choice([8, 16, 16, 20, 32, 64, 256])}
    if op == "append":
        lens, room = [], 2_000_000 // (heads * dim) * 10
        for _ in range(rng.choice([1, 1, 2, 5, 20])):
            n = min(_log_int(rng, 1, 8000), room)
            if n < 1:
                break
            room -= n
            lens.append("%d:%d" % (n, n + rng.choice([0, _log_int(rng, 1, 1000)])))
        rot = rng.choice([r for r in (32, 64, 96, 128, 256) if r <= dim])
        return {**case, "rot": rot, "axes": rng.choice([1, 1, 2, 3]), "pairing": rng.choice(["halves", "halves", "adjacent"]),
                "norm": rng.random() < 0.5, "lens": ",".join(lens)}
    form = rng.choice(["decode", "drafts", "chunk"])
    case.update(window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]), gate=rng.random() < 0.3)
    if form == "chunk":
        lens = []
        for _ in range(rng.choice([1, 1, 2, 4])):
            n = _log_int(rng, 10, 2000)
            lens.append("%d:%d" % (n, n + rng.choice([0, _log_int(rng, 1, 6000)])))
        return {**case, "lens": ",".join(lens)}
    seqs, lo = _log_int(rng, 1, 64), _log_int(rng, 1, 4000)
    hi = lo + _log_int(rng, 1, 60_000 // seqs + 2000)
    return {**case, "seqs": seqs, "new": 1 if form == "decode" else rng.randint(2, 9), "lo": lo, "hi": hi}


# ---- inputs -------------------------------------------------------------------------------------------------


def _lens(case):
    """[(new tokens, context after them)] of every sequence."""
    if "lens" in case:
        return [tuple(int(x) for x in s.split(":")) for s in case["lens"].split(",")]
    at = [(0.5 + 0.6180339887498949 * s) % 1.0 for s in range(case["seqs"])]
    return [(case["new"], max(case["new"], case["lo"] + int((case["hi"] - case["lo"]) * f))) for f in at]


class _Rand:
    """Random values on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda") * std

    def rows(self, rows, dim):
        """Activations: some channels are much larger than others, in all rows."""
        return self.normal(rows, dim) * torch.exp(self.normal(dim, std=0.7))

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")

    def bytes(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.uint8)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_paged(case, seed):
    """The pool ([page][head][token] in memory; some pages are other sequences'), the sequences' pages in random order, and
    the step's tokens."""
    r, lens, dtype = _Rand(seed), _lens(case), DTYPES[case["dtype"]]
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    need = [-(-ctx // page) for _, ctx in lens]
    pages = sum(need) + 7
    order = r.perm(pages).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    first = 0
    for s, n in enumerate(need):
        table[s, :n] = order[first:first + n]
        first += n
    tokens = sum(n for n, _ in lens)
    state = {"case": dict(case), "table": table, "cu": _i32(np.concatenate([[0], np.cumsum([n for n, _ in lens])]).tolist()),
             "context": _i32([ctx for _, ctx in lens]), "max_new": max(n for n, _ in lens), "max_context": max(c for _, c in lens)}
    if case["op"] == "attn":
        state["k_cache"], state["v_cache"] = (_plain_quantize(r.normal(pages, kv, page, dim)) for _ in range(2))
        # normalised queries, sharpened as a trained layer's are: some keys weigh much more than others
        state["q"] = r.normal(tokens, heads, dim, std=2.0).to(dtype)
        state["gate"] = r.normal(tokens, heads, dim).to(dtype) if case["gate"] else None
        return state
    # what earlier steps left in the pages
    state["k_cache"], state["v_cache"] = ((r.bytes(0, 256, pages, kv, page, dim // 2), r.bytes(122, 128, pages, kv, page, dim // 32))
                                          for _ in range(2))
    state["q"], state["k"], state["v"] = (r.normal(tokens, h, dim).to(dtype) for h in (heads, kv, kv))
    state["qw"], state["kw"] = ((r.normal(dim, std=0.2).to(dtype) for _ in range(2)) if case["norm"] else (None, None))
    # positions: text advances all axes together; inside an image time stands still while height and width run over a grid
    t = torch.cat([torch.arange(c - n, c, device="cuda") for n, c in lens])
    image = (t // 256) % 2 == 1 if case["axes"] > 1 else torch.zeros_like(t, dtype=torch.bool)
    axes = [torch.where(image, t // 256 * 256, t), torch.where(image, t // 256 * 256 + t % 256 // 16, t),
            torch.where(image, t // 256 * 256 + t % 16, t)]
    state["positions"] = torch.stack(axes[:case["axes"]]).to(torch.int32).contiguous()
    pairs = case["rot"] // 2
    state["pair_axis"] = [i % case["axes"] for i in range(pairs)]
    rows = -(-max(c for _, c in lens) // 256) * 256
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * \
        1e7 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    state["rope"] = torch.stack([angle.cos(), angle.sin()], -1).reshape(rows, case["rot"]).float().contiguous()
    return state


def prepare(case, seed):
    if case["op"] in ("append", "attn"):
        return _prepare_paged(case, seed)
    r, dtype = _Rand(seed), DTYPES[case["dtype"]]
    x = r.rows(case["rows"], case["dim"]).to(dtype)
    if case["op"] == "quantize":
        return {"case": dict(case), "x": x}
    return {"case": dict(case), "x": x if case["bits"] == 16 else _plain_quantize(x),
            "w": _plain_quantize(r.normal(case["out"], case["dim"], std=0.02)),
            "residual": r.normal(case["rows"], case["out"]).to(dtype) if case["residual"] else None}


# ---- one pass -----------------------------------------------------------------------------------------------


def _plain_quantize(x):
    """(codes, scales) of x [..., n]: exact for 16 and 32 bits (a scale is a power of two), and in 64 for values in 64."""
    wide = x.dtype is torch.float64
    y = (x if wide else x.float()).unflatten(-1, (-1, 32))
    most = y.abs().amax(-1)
    fine = torch.isfinite(most)
    power = (torch.frexp(torch.where(fine, most, torch.ones_like(most)))[1] - 3).clamp(min=-127)
    power = torch.where(most == 0, torch.full_like(power, -127), power).to(torch.int64 if wide else torch.int32)
    # 2^-power from its bits (power is at most 125)
    scale = ((1023 - power) << 52).view(torch.float64) if wide else ((127 - power) << 23).view(torch.float32)
    t = y.abs() * scale[..., None]
    code = torch.zeros(t.shape, dtype=torch.uint8, device=t.device)
    for edge, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (t >= edge) if up else (t > edge)
    code += torch.signbit(y) * torch.full((), 8, dtype=torch.uint8, device=t.device)
    code = torch.where(fine[..., None], code, torch.zeros_like(code)).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.where(fine, power + 127, 255).to(torch.uint8)


def _plain_values(m):
    """The float32 values of (codes, scales)."""
    codes, scales = m
    grid = torch.tensor(GRID, dtype=torch.float32, device=codes.device)
    grid = torch.cat([grid, -grid])
    value = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).flatten(-2)
    # 2^(byte - 127) from its bits; byte 0 is 2^-127 and 255 is no number
    bits = scales.int() << 23
    scale = torch.where(bits == 0, 1 << 22, bits).view(torch.float32)
    scale = torch.where(scales == 255, torch.full_like(scale, math.nan), scale)
    return (value.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _plain_matmul(s):
    x = s["x"].float() if s["case"]["bits"] == 16 else _plain_values(s["x"])
    y = torch.matmul(x, _plain_values(s["w"]).T)
    if s["residual"] is not None:
        y += s["residual"].float()
    return y.to(DTYPES[s["case"]["dtype"]])


def _plain_turn(x, weight, c, sn, pairing):
    """Per-head RMSNorm (1 + weight) where there is one, then the rotation of the first dimensions."""
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + weight)
    rot = 2 * c.shape[-1]
    part, rest = x[..., :rot], x[..., rot:]
    x1, x2 = (part[..., :rot // 2], part[..., rot // 2:]) if pairing == "halves" else (part[..., 0::2], part[..., 1::2])
    y1, y2 = x1 * c - x2 * sn, x2 * c + x1 * sn
    turned = torch.cat([y1, y2], -1) if pairing == "halves" else torch.stack([y1, y2], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_append(s):
    """The keys in 64 bits: a value next to a border between two codes hangs on it."""
    case, pairs = s["case"], s["case"]["rot"] // 2
    axis = torch.tensor(s["pair_axis"], device="cuda")
    pos = s["positions"].long()[axis]                                     # [pairs][T]
    cs = s["rope"].view(-1, pairs, 2)[pos, torch.arange(pairs, device="cuda")[:, None]].transpose(0, 1)[:, None]
    c, sn = cs[..., 0], cs[..., 1]
    weights = [None if w is None else w.float() for w in (s["qw"], s["kw"])]
    q = _plain_turn(s["q"].float(), weights[0], c, sn, case["pairing"]).to(s["q"].dtype)
    k = _plain_turn(s["k"].double(), None if weights[1] is None else weights[1].double(), c.double(), sn.double(), case["pairing"])
    cu, t = s["cu"].long(), torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    at = s["context"].long()[seq] - cu[seq + 1] + t
    page, off = s["table"].long()[seq, at // case["page"]], at % case["page"]
    for cache, rows in ((s["k_cache"], k), (s["v_cache"], s["v"])):
        for pool, part in zip(cache, _plain_quantize(rows)):
            pool.transpose(1, 2)[page, off] = part
    return {"q": q, "k_cache": _plain_values(s["k_cache"]).to(q.dtype), "v_cache": _plain_values(s["v_cache"]).to(q.dtype)}


def _plain_attn(s):
    """All sequences as one padded batch: [S][kv][new * group][D] against [S][kv][context][D]."""
    case, cu, ctx = s["case"], s["cu"].long(), s["context"].long()
    heads, kv, dim, new, top = case["heads"], case["kv"], case["dim"], s["max_new"], s["max_context"]
    group, seqs = heads // kv, ctx.numel()
    n = cu[1:] - cu[:-1]
    i = torch.arange(new, device="cuda")
    row = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)              # [S][new], clamped rows are dropped below
    q = s["q"].float()[row].view(seqs, new, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv, new * group, dim)
    j = torch.arange(top, device="cuda")
    k, v = (_plain_values([x[s["table"].long()].transpose(1, 2).flatten(2, 3)[:, :, :top] for x in cache])
            for cache in (s["k_cache"], s["v_cache"]))
    pos = (ctx - n)[:, None] + i                                          # [S][new]
    seen = (j <= pos[..., None]) & (j < ctx[:, None, None])
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(seqs, 1, new, group, top).reshape(seqs, 1, new * group, top)
    score = torch.matmul(q * dim ** -0.5, k.transpose(2, 3).contiguous()).masked_fill_(~seen, -math.inf)
    most = score.amax(-1, keepdim=True)
    most = torch.where(seen.any(-1, keepdim=True), most, torch.zeros_like(most))
    weight = score.sub_(most).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v.contiguous()) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (most + torch.log(total))[..., 0]
    out = out.view(seqs, kv, new, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, new, heads, dim)
    lse = lse.view(seqs, kv, new, group).permute(0, 2, 1, 3).reshape(seqs, new, heads)
    keep = i < n[:, None]
    out, lse = out[keep], lse[keep]
    if s["gate"] is not None:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _own(s):
    from spock_amd import ops
    case = s["case"]
    if case["op"] == "quantize":
        return ops.mx4_dequantize(ops.mx4_quantize(s["x"]), s["x"].dtype)
    if case["op"] == "matmul":
        x = s["x"] if case["bits"] == 16 else ops.Mx4(*s["x"])
        return ops.mx4_matmul(x, ops.Mx4(*s["w"]), residual=s["residual"], dtype=DTYPES[case["dtype"]])
    # the operators take [page][token][head] with any strides
    k_cache, v_cache = (ops.Mx4(*[x.transpose(1, 2) for x in s[name]]) for name in ("k_cache", "v_cache"))
    if case["op"] == "append":
        q = ops.mrope_append_mx4(s["q"], s["k"], s["v"], s["positions"], s["rope"], s["pair_axis"], k_cache, v_cache,
                                 s["table"], s["cu"], s["context"], q_norm_weight=s["qw"], k_norm_weight=s["kw"], eps=EPS,
                                 pairing=case["pairing"])
        return {"q": q, "k_cache": ops.mx4_dequantize(ops.Mx4(*s["k_cache"]), q.dtype),
                "v_cache": ops.mx4_dequantize(ops.Mx4(*s["v_cache"]), q.dtype)}
    out, lse = ops.paged_attention_mx4(s["q"], k_cache, v_cache, s["table"], s["cu"], s["context"], s["max_new"],
                                       s["max_context"], window=case["window"], gate=s["gate"], return_lse=True)
    return {"out": out, "lse": lse}


def run(state):
    if own:
        return _own(state)
    if state["case"]["op"] == "quantize":
        return _plain_values(_plain_quantize(state["x"])).to(state["x"].dtype)
    return {"matmul": _plain_matmul, "append": _plain_append, "attn": _plain_attn}[state["case"]["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------


def _exact_values(codes, scales):
    """Float64 values, by the bits of a code: sign, two of exponent, one of mantissa."""
    c = torch.stack([codes % 16, codes // 16], -1).flatten(-2).double()
    sign = 1 - 2 * (c >= 8).double()
    c = c % 8
    e, m = torch.floor(c / 2), c % 2
    value = sign * torch.where(e == 0, m / 2, (1 + m / 2) * torch.pow(2.0, e - 1))
    return value * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)


def _exact_round(x):
    """x in float64 to the nearest representable value of its block."""
    y = x.unflatten(-1, (-1, 32))
    most = y.abs().amax(-1, keepdim=True)
    scale = torch.pow(2.0, (torch.floor(torch.log2(most.clamp(min=1e-300))) - 2).clamp(min=-127))
    t = (y / scale).abs()
    # the spacing of the grid is 0.5 below 2, 1 up to 4, 2 up to 6; torch.round takes ties to even, as a code's last bit is
    step = torch.where(t < 2, 0.5, torch.where(t < 4, 1.0, 2.0))
    return (torch.sign(y) * (torch.round(t / step) * step).clamp(max=6.0) * scale).flatten(-2)


def _exact_append(s):
    case, cu, ctx, table = s["case"], s["cu"].tolist(), s["context"].tolist(), s["table"].long()
    rope, half, page = s["rope"].double(), case["rot"] // 2, case["page"]
    result = {"q": torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"),
              "k_cache": _exact_values(*s["k_cache"]), "v_cache": _exact_values(*s["v_cache"])}

    def turn(x, w, lo, hi):
        y = x[lo:hi].double()
        if w is not None:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / y.shape[-1] + EPS) * (w.double() + 1)
        z = y.clone()
        for i in range(half):
            a, b = (i, i + half) if case["pairing"] == "halves" else (2 * i, 2 * i + 1)
            r = rope[s["positions"][s["pair_axis"][i], lo:hi].long()]
            c, n = r[:, 2 * i, None], r[:, 2 * i + 1, None]
            z[..., a], z[..., b] = y[..., a] * c - y[..., b] * n, y[..., b] * c + y[..., a] * n
        return z

    for b in range(len(ctx)):
        lo, hi = cu[b], cu[b + 1]
        at = torch.arange(ctx[b] - (hi - lo), ctx[b], device="cuda")
        pages = table[b, at // page]
        result["q"][lo:hi] = turn(s["q"], s["qw"], lo, hi)
        result["k_cache"].transpose(1, 2)[pages, at % page] = _exact_round(turn(s["k"], s["kw"], lo, hi))
        result["v_cache"].transpose(1, 2)[pages, at % page] = _exact_round(s["v"][lo:hi].double())
    return result


def _exact_attn(s):
    case, cu, ctx, table = s["case"], s["cu"].tolist(), s["context"].tolist(), s["table"].long()
    group, dim = case["heads"] // case["kv"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, length in enumerate(ctx):
        lo, hi = cu[b], cu[b + 1]
        keys, vals = (_exact_values(*[x[table[b]].transpose(0, 1).flatten(1, 2)[:, :length] for x in s[name]])
                      for name in ("k_cache", "v_cache"))
        j = torch.arange(length, device="cuda")
        for h in range(case["heads"]):
            k, v = keys[h // group], vals[h // group]
            for at in range(lo, hi, 1024):
                to = min(hi, at + 1024)
                pos = torch.arange(length - hi + at, length - hi + to, device="cuda")[:, None]
                hidden = (j > pos) | ((j <= pos - case["window"]) if case["window"] else (j < 0))
                x = (s["q"][at:to, h].double() @ k.T) / math.sqrt(dim)
                x[hidden] = -math.inf
                lse[at:to, h] = torch.logsumexp(x, -1)
                y = torch.exp(x - lse[at:to, h, None]) @ v
                out[at:to, h] = torch.where((~hidden).any(-1, keepdim=True), y, 0.0)
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return torch.cat([_exact_round(x.double()) for x in s["x"].split(16384)])
    if case["op"] == "matmul":
        w = _exact_values(*s["w"])
        y = (s["x"].double() if case["bits"] == 16 else _exact_values(*s["x"])) @ w.T
        return y if s["residual"] is None else y + s["residual"].double()
    return _exact_append(s) if case["op"] == "append" else _exact_attn(s)


# ---- what a pass cannot do without --------------------------------------------------------------------------


def work(case):
    size = {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "quantize":  # and the values read back
        n = case["rows"] * case["dim"]
        return {"bytes": 2 * n * size + 2 * (n // 2 + n // 32), "flops": 4 * n}
    if case["op"] == "matmul":
        m, n, k = case["rows"], case["out"], case["dim"]
        four = lambda rows: rows * (k // 2 + k // 32)  # noqa: E731
        return {"bytes": four(n) + (2 * m * k if case["bits"] == 16 else four(m)) + 2 * m * n * (2 if case["residual"] else 1),
                "flops": 2 * m * n * k}
    lens, heads, kv, dim = _lens(case), case["heads"], case["kv"], case["dim"]
    tokens = sum(n for n, _ in lens)
    row = dim // 2 + dim // 32
    if case["op"] == "append":  # and the pools' values read back
        pool = (sum(-(-c // case["page"]) for _, c in lens) + 7) * case["page"] * kv
        rows = min(tokens, max(c for _, c in lens))
        return {"bytes": 2 * tokens * (2 * heads + 2 * kv) * dim + 2 * tokens * kv * row + 2 * pool * (row + 2 * dim)
                + 4 * rows * case["rot"] + 4 * tokens * case["axes"],
                "flops": 3 * tokens * (heads + kv) * case["rot"] + (4 * tokens * (heads + kv) * dim if case["norm"] else 0)}
    window = case["window"]
    keys = pairs = 0
    for n, ctx in lens:
        keys += min(ctx, window + n - 1) if window else ctx
        pairs += sum(min(ctx - n + i + 1, window) if window else ctx - n + i + 1 for i in range(n))
    io = tokens * heads * dim * 2 * (3 if case["gate"] else 2) + tokens * heads * 4
    return {"bytes": io + 2 * keys * kv * row, "flops": 4 * dim * heads * pairs}
