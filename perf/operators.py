"""The operators of a serving step over a paged cache, as a list of cases to time.

One step of a server: the new tokens' q and k are rotated by positions with several axes and k, v stored into the pages
(mrope), the chunk of new tokens of every sequence attends over its pages (attn), and drafted tokens are accepted or
replaced by the target's distribution (verify).  Shapes are the framework's own (8 query and 2 KV heads of 256, 64
rotary dimensions, vocabulary 248320) and generic ones.

With `own` false `run` is the plain form in elementary torch operations; with `own` true it calls spock_amd.ops.
`exact` restates the definitions in float64, sequence by sequence.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one token of one sequence: nothing but latency
        {"name": "mrope_decode_1", "op": "mrope", "dtype": "f16", "heads": 8, "kv": 2, "dim": 256, "rot": 64, "axes": 3,
         "layout": "interleaved", "pairing": "halves", "norm": True, "page": 16, "lens": "1:1500"},
        # a prompt with an image in it, in two sequences of odd lengths, the framework's heads
        {"name": "mrope_prompt_2001", "op": "mrope", "dtype": "f16", "heads": 8, "kv": 2, "dim": 256, "rot": 64, "axes": 3,
         "layout": "interleaved", "pairing": "halves", "norm": True, "page": 16, "lens": "1501:1501,500:2777"},
        # a server's whole prefill batch, full-width rotation over blocks of axes
        {"name": "mrope_batch_32k", "op": "mrope", "dtype": "bf16", "heads": 16, "kv": 4, "dim": 128, "rot": 128, "axes": 3,
         "layout": "blocks", "pairing": "halves", "norm": False, "page": 64, "lens": "8192:8192,8191:12000,16385:16385"},
        # one decoded token at an ordinary context
        {"name": "attn_decode_1500", "op": "attn", "dtype": "f16", "heads": 8, "kv": 2, "dim": 256, "page": 16,
         "lens": "1:1500", "window": 0, "gate": True},
        # one decode step of a serving batch, ragged contexts: the cache is read once
        {"name": "attn_decode_64seqs", "op": "attn", "dtype": "f16", "heads": 8, "kv": 2, "dim": 256, "page": 16,
         "seqs": 64, "new": 1, "lo": 300, "hi": 16000, "window": 0, "gate": True},
        # one token at the end of a very long context: few rows, so the keys are what is split
        {"name": "attn_decode_long", "op": "attn", "dtype": "bf16", "heads": 32, "kv": 8, "dim": 128, "page": 32,
         "lens": "1:130001", "window": 0, "gate": False},
        # eight drafted tokens and the last one accepted, of 16 sequences
        {"name": "attn_drafts_16x9", "op": "attn", "dtype": "bf16", "heads": 8, "kv": 2, "dim": 256, "page": 16,
         "seqs": 16, "new": 9, "lo": 1000, "hi": 9000, "window": 0, "gate": False},
        # a chunk of a long prompt over what is in the cache already
        {"name": "attn_chunk_2048", "op": "attn", "dtype": "f16", "heads": 8, "kv": 2, "dim": 256, "page": 16,
         "lens": "2048:16384", "window": 0, "gate": True},
        # whole prompts of ragged lengths with decoding sequences among them
        {"name": "attn_prompts_ragged", "op": "attn", "dtype": "bf16", "heads": 16, "kv": 4, "dim": 128, "page": 64,
         "lens": "4001:4001,1061:1061,2504:3007,61:5000,1:2222,1:777", "window": 0, "gate": False},
        # four drafted tokens of one sequence
        {"name": "verify_1x4", "op": "verify", "kind": "logits", "dtype": "f16", "vocab": 248320, "seqs": 1, "drafts": 4,
         "ragged": False, "temp": 1.0, "greedy": 0.0, "draft": True},
        # a serving batch, ragged numbers of drafts, some sequences greedy
        {"name": "verify_64x5", "op": "verify", "kind": "logits", "dtype": "f16", "vocab": 248320, "seqs": 64, "drafts": 5,
         "ragged": True, "temp": 0.8, "greedy": 0.25, "draft": True},
        # probabilities that a sampler made, in float32, odd vocabulary, a drafter without probabilities of its own
        {"name": "verify_probs_f32", "op": "verify", "kind": "probs", "dtype": "f32", "vocab": 100003, "seqs": 48,
         "drafts": 3, "ragged": True, "temp": 1.0, "greedy": 0.0, "draft": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mrope", "attn", "attn", "attn", "verify"])
    if op == "verify":
        logits = rng.random() < 0.7
        seqs, drafts = _log_int(rng, 1, 64), rng.randint(1, 8)
        vocab = _log_int(rng, 1000, 248320)
        dtype = rng.choice(["f16", "bf16", "f32"] if logits else ["f32"])
        while seqs > 1 and seqs * (drafts + 1) * vocab * (4 if dtype == "f32" else 2) > 90_000_000:
            seqs -= 1
        return {"op": op, "kind": "logits" if logits else "probs", "dtype": dtype, "vocab": vocab, "seqs": seqs,
                "drafts": drafts, "ragged": rng.random() < 0.5, "temp": round(rng.uniform(0.3, 1.5), 2) if logits else 1.0,
                "greedy": rng.choice([0.0, 0.3, 1.0]) if logits else 0.0, "draft": rng.random() < 0.7}
    heads, kv, dim = rng.choice([(8, 2, 256), (8, 2, 256), (16, 4, 128), (32, 8, 128), (8, 1, 128), (4, 4, 128), (12, 3, 64), (7, 1, 64)])
    case = {"op": op, "dtype": rng.choice(["f16", "bf16"]), "heads": heads, "kv": kv, "dim": dim,
            "page": rng.choice([8, 16, 16, 20, 32, 64, 256])}
    if op == "mrope":
        lens, room = [], 2_000_000 // (heads * dim) * 10
        for _ in range(rng.choice([1, 1, 2, 5, 20])):
            n = _log_int(rng, 1, 8000)
            n = min(n, room)
            if n < 1:
                break
            room -= n
            lens.append("%d:%d" % (n, n + rng.choice([0, _log_int(rng, 1, 4000)])))
        rot = rng.choice([r for r in (32, 64, 96, 128, 256) if r <= dim])
        return {**case, "rot": rot, "axes": rng.choice([1, 2, 3, 3, 4]), "layout": rng.choice(["interleaved", "blocks"]),
                "pairing": rng.choice(["halves", "halves", "adjacent"]), "norm": rng.random() < 0.5, "lens": ",".join(lens)}
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


def _rows(case):
    """Rows of logits of every sequence: one more than its drafts."""
    drafts = case["drafts"]
    if not case["ragged"]:
        return [drafts + 1] * case["seqs"]
    return [1 + int((drafts + 1) * ((0.4 + 0.6180339887498949 * s) % 1.0)) for s in range(case["seqs"])]


class _Rand:
    """Random values on the GPU from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda") * std

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda")

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_paged(case, seed):
    """The pool (some pages are other sequences'), the sequences' pages in random order, and the step's tokens."""
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
    state = {"case": dict(case), "table": table, "k_cache": r.normal(pages, page, kv, dim).to(dtype),
             "v_cache": r.normal(pages, page, kv, dim).to(dtype),
             "cu": _i32(np.concatenate([[0], np.cumsum([n for n, _ in lens])]).tolist()),
             "context": _i32([ctx for _, ctx in lens]), "max_new": max(n for n, _ in lens), "max_context": max(c for _, c in lens)}
    if case["op"] == "attn":
        # normalised queries, sharpened as a trained layer's are: some keys weigh much more than others
        state["q"] = r.normal(tokens, heads, dim, std=2.0).to(dtype)
        state["gate"] = r.normal(tokens, heads, dim).to(dtype) if case["gate"] else None
        return state
    state["q"], state["k"], state["v"] = (r.normal(tokens, h, dim).to(dtype) for h in (heads, kv, kv))
    state["qw"], state["kw"] = ((r.normal(dim, std=0.2).to(dtype) for _ in range(2)) if case["norm"] else (None, None))
    # positions: text advances all axes together; inside an image time stands still while height and width run over a grid
    rows = -(-max(c for _, c in lens) // 256) * 256
    t = torch.cat([torch.arange(c - n, c, device="cuda") for n, c in lens])
    image = (t // 256) % 2 == 1
    axes = [torch.where(image, t // 256 * 256, t), torch.where(image, t // 256 * 256 + t % 256 // 16, t),
            torch.where(image, t // 256 * 256 + t % 16, t), t // 2]
    state["positions"] = torch.stack(axes[:case["axes"]]).to(torch.int32).contiguous()
    pairs = case["rot"] // 2
    state["pair_axis"] = [i % case["axes"] if case["layout"] == "interleaved" else i * case["axes"] // pairs for i in range(pairs)]
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * \
        1e7 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    state["rope"] = torch.stack([angle.cos(), angle.sin()], -1).reshape(rows, case["rot"]).float().contiguous()
    return state


def _prepare_verify(case, seed):
    """Rows of the step's logits: the drafter's are the target's with noise, and its tokens are drawn from its own
    distribution, so that most drafts are accepted and some are not."""
    r, dtype, vocab = _Rand(seed), DTYPES[case["dtype"]], case["vocab"]
    rows = _rows(case)
    total, cu = sum(rows), np.concatenate([[0], np.cumsum(rows)])
    target = r.normal(total, vocab, std=2.5)
    target[:, :64] += 6.0 * r.uniform(total, 64)
    draft = (target + r.normal(total, vocab, std=0.5)).to(dtype)
    target = target.to(dtype)
    greedy = [s < case["greedy"] * case["seqs"] for s in range(case["seqs"])]
    temp = torch.tensor([0.0 if x else case["temp"] for x in greedy], dtype=torch.float32, device="cuda")
    row_temp = torch.repeat_interleave(temp, _i32(rows).long()).clamp(min=1e-3)[:, None]
    noise = -torch.log(-torch.log(r.uniform(total, vocab).clamp(1e-12, 1 - 1e-7)))
    drawn = (draft.float() / row_temp + noise).argmax(-1)
    tokens = torch.cat([drawn.new_zeros(1), drawn[:-1]]).to(torch.int32)  # the token drawn after row t is the input of row t + 1
    if case["kind"] == "probs":
        target, draft = (torch.softmax(x.float(), -1).to(dtype) for x in (target, draft))
    return {"case": dict(case), "target": target, "draft": draft if case["draft"] else None, "tokens": tokens, "cu": _i32(cu.tolist()),
            "temp": temp if case["kind"] == "logits" else None, "u_accept": r.uniform(total), "u_sample": r.uniform(case["seqs"]),
            "context": _i32([1000 + 17 * s for s in range(case["seqs"])])}


def prepare(case, seed):
    return _prepare_verify(case, seed) if case["op"] == "verify" else _prepare_paged(case, seed)


# ---- one pass -----------------------------------------------------------------------------------------------


def _slots(s):
    """Sequence and cache slot of every token of the step."""
    cu, t = s["cu"].long(), torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    at = s["context"].long()[seq] - cu[seq + 1] + t
    page = s["case"]["page"]
    return s["table"].long()[seq, at // page], at % page


def _plain_rotate(x, weight, c, sn, pairing):
    """Per-head RMSNorm (1 + weight) where there is one, then the rotation of the first dimensions."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + weight.float())
    rot = 2 * c.shape[-1]
    part, rest = x[..., :rot], x[..., rot:]
    x1, x2 = (part[..., :rot // 2], part[..., rot // 2:]) if pairing == "halves" else (part[..., 0::2], part[..., 1::2])
    y1, y2 = x1 * c - x2 * sn, x2 * c + x1 * sn
    turned = torch.cat([y1, y2], -1) if pairing == "halves" else torch.stack([y1, y2], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_mrope(s):
    case, pairs = s["case"], s["case"]["rot"] // 2
    axis = torch.tensor(s["pair_axis"], device="cuda")
    pos = s["positions"].long()[axis]                                     # [pairs][T]
    cs = s["rope"].view(-1, pairs, 2)[pos, torch.arange(pairs, device="cuda")[:, None]].transpose(0, 1)[:, None]
    c, sn = cs[..., 0], cs[..., 1]
    q = _plain_rotate(s["q"], s["qw"], c, sn, case["pairing"]).to(s["q"].dtype)
    page, off = _slots(s)
    s["k_cache"][page, off] = _plain_rotate(s["k"], s["kw"], c, sn, case["pairing"]).to(s["k"].dtype)
    s["v_cache"][page, off] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


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
    k, v = (c[s["table"].long()].flatten(1, 2)[:, :top].permute(0, 2, 1, 3).float() for c in (s["k_cache"], s["v_cache"]))
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


def _plain_verify(s):
    """In 64 bits: the accepted length and the drawn token hang on comparisons."""
    case, cu, tokens = s["case"], s["cu"].long(), s["tokens"].long()
    seqs, total, vocab = case["seqs"], tokens.numel(), case["vocab"]
    t = torch.arange(total, device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    last = cu[1:][seq] - 1
    ids = torch.arange(vocab, device="cuda")
    logits = case["kind"] == "logits"
    hot = s["temp"].double() if logits else torch.ones(seqs, dtype=torch.float64, device="cuda")
    greedy = hot <= 0
    hot = torch.where(greedy, torch.ones_like(hot), hot)[seq][:, None]

    def probs(x):
        if not logits:
            return x.double()
        x = x.double() / hot
        e = torch.exp(x - x.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)

    p = probs(s["target"])
    follow = tokens[(t + 1).clamp(max=total - 1)]
    p_d = p[t, follow]
    if s["draft"] is None:
        q, q_d = None, torch.ones_like(p_d)
    else:
        q = probs(s["draft"])
        q_d = q[t, follow]
    best = torch.where(s["target"] == s["target"].amax(-1, keepdim=True), ids, vocab).amin(-1)
    yes = torch.where(greedy[seq], best == follow, s["u_accept"].double() * q_d < p_d) & (t < last)
    refused = torch.where(yes, total, t)
    stop = torch.full((seqs,), total, device="cuda").scatter_reduce(0, seq, refused, "amin")   # row that emits the new token
    accepted = stop - cu[:-1]
    at_end = stop == cu[1:] - 1
    base = p[stop]
    if q is None:
        rest = torch.where(ids == follow[stop][:, None], torch.zeros_like(base), base)
    else:
        rest = (base - q[stop]).clamp(min=0)
    rest = torch.where(at_end[:, None], base, rest)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, base)
    run_sum = rest.cumsum(-1)
    drawn = (run_sum <= s["u_sample"].double()[:, None] * run_sum[:, -1:]).sum(-1)
    drawn = torch.minimum(drawn, torch.where(rest > 0, ids, -1).amax(-1))
    drawn = torch.where(greedy, best[stop], drawn)
    out = torch.where(t < stop[seq], follow, torch.where(t == stop[seq], drawn[seq], -1))
    logp = torch.where(out >= 0, torch.log(p[t, out.clamp(min=0)]), 0.0)
    context = s["context"].long() - (cu[1:] - 1 - stop)
    return {"tokens": out.to(torch.int32), "accepted": accepted.to(torch.int32), "logprobs": logp.float(),
            "context": context.to(torch.int32)}


def _own(s):
    from spock_amd import ops
    case = s["case"]
    if case["op"] == "mrope":
        q = ops.mrope_append(s["q"], s["k"], s["v"], s["positions"], s["rope"], s["pair_axis"], s["k_cache"], s["v_cache"],
                             s["table"], s["cu"], s["context"], q_norm_weight=s["qw"], k_norm_weight=s["kw"], eps=EPS,
                             pairing=case["pairing"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "attn":
        out, lse = ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["context"], s["max_new"],
                                       s["max_context"], window=case["window"], gate=s["gate"], return_lse=True)
        return {"out": out, "lse": lse}
    tokens, accepted, logprobs, context = ops.verify_drafts(s["target"], s["tokens"], s["cu"], s["u_accept"], s["u_sample"],
                                                            draft=s["draft"], kind=case["kind"], temperature=s["temp"],
                                                            context_lens=s["context"])
    return {"tokens": tokens, "accepted": accepted, "logprobs": logprobs, "context": context}


def run(state):
    if own:
        return _own(state)
    return {"mrope": _plain_mrope, "attn": _plain_attn, "verify": _plain_verify}[state["case"]["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------


def _exact_mrope(s):
    case, cu, ctx, table = s["case"], s["cu"].tolist(), s["context"].tolist(), s["table"].long()
    rope, half, page = s["rope"].double(), case["rot"] // 2, case["page"]
    result = {"q": torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"),
              "k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}

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
        where = (table[b, at // page], at % page)
        result["q"][lo:hi] = turn(s["q"], s["qw"], lo, hi)
        result["k_cache"][where] = turn(s["k"], s["kw"], lo, hi)
        result["v_cache"][where] = s["v"][lo:hi].double()
    return result


def _exact_attn(s):
    case, cu, ctx, table = s["case"], s["cu"].tolist(), s["context"].tolist(), s["table"].long()
    group, dim = case["heads"] // case["kv"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, length in enumerate(ctx):
        lo, hi = cu[b], cu[b + 1]
        keys = s["k_cache"][table[b]].flatten(0, 1)[:length]
        vals = s["v_cache"][table[b]].flatten(0, 1)[:length]
        j = torch.arange(length, device="cuda")
        for h in range(case["heads"]):
            k, v = keys[:, h // group].double(), vals[:, h // group].double()
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


def _exact_verify(s):
    case, cu, tokens = s["case"], s["cu"].tolist(), s["tokens"].tolist()
    logp = torch.zeros(len(tokens), dtype=torch.float64, device="cuda")

    def dist(x, hot):
        return x.double() if case["kind"] == "probs" else torch.log_softmax(x.double() / hot, -1).exp()

    for b in range(case["seqs"]):
        hot = float(s["temp"][b]) if s["temp"] is not None else 1.0
        greedy, hot = hot <= 0, hot if hot > 0 else 1.0
        for t in range(cu[b], cu[b + 1]):
            p = dist(s["target"][t], hot)
            top = int((s["target"][t] == s["target"][t].max()).nonzero()[0])
            d = tokens[t + 1] if t + 1 < cu[b + 1] else -1
            q = None if d < 0 or s["draft"] is None else dist(s["draft"][t], hot)
            ratio = 0.0 if d < 0 else float(p[d]) / (1.0 if q is None else float(q[d]))
            if d >= 0 and (d == top if greedy else float(s["u_accept"][t]) < ratio):
                logp[t] = torch.log(p[d])
                continue
            w = p.clone()
            if d >= 0 and q is not None:
                w = torch.relu(p - q)
            elif d >= 0:
                w[d] = 0.0
            if not float(w.sum()) > 0:
                w = p
            c = torch.cumsum(w, 0)
            x = top if greedy else int((c > float(s["u_sample"][b]) * float(c[-1])).nonzero()[0])
            logp[t] = torch.log(p[x])
            break
    return {"tokens": None, "accepted": None, "logprobs": logp, "context": None}


def exact(case, seed):
    s = prepare(case, seed)
    return {"mrope": _exact_mrope, "attn": _exact_attn, "verify": _exact_verify}[case["op"]](s)


# ---- what a pass cannot do without --------------------------------------------------------------------------


def work(case):
    if case["op"] == "verify":
        rows = sum(_rows(case))
        size, vocab, seqs = {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]], case["vocab"], case["seqs"]
        sides = 2 if case["draft"] else 1
        if case["kind"] == "probs":  # single probabilities, and the one row that a token is drawn from
            return {"bytes": sides * (seqs * vocab * size + rows * 4) + rows * 16, "flops": 3 * seqs * vocab}
        return {"bytes": (sides * rows - (sides - 1) * seqs) * vocab * size + rows * 16, "flops": 4 * sides * rows * vocab}
    lens, heads, kv, dim = _lens(case), case["heads"], case["kv"], case["dim"]
    tokens = sum(n for n, _ in lens)
    if case["op"] == "mrope":
        elements = tokens * (heads + 2 * kv) * dim
        rows = min(tokens, max(c for _, c in lens))
        return {"bytes": 2 * 2 * elements + 4 * rows * case["rot"] + 4 * tokens * case["axes"],
                "flops": 3 * tokens * (heads + kv) * case["rot"] + (4 * tokens * (heads + kv) * dim if case["norm"] else 0)}
    window = case["window"]
    keys = pairs = 0
    for n, ctx in lens:
        keys += min(ctx, window + n - 1) if window else ctx
        full = [min(ctx - n + i + 1, window) if window else ctx - n + i + 1 for i in range(n)]
        pairs += sum(full)
    io = tokens * heads * dim * 2 * (3 if case["gate"] else 2) + tokens * heads * 4
    return {"bytes": io + keys * kv * dim * 2 * 2, "flops": 4 * dim * heads * pairs}
