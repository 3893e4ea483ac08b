"""The paged serving step in 64 bits on the CPU (torch float64), sequence by
sequence from the definitions, and the bounds that a 16-bit result computed in
fp32 keeps."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # relative error of one rounding


def spans(cu, ctx, total, room):
    """(first, n, ctx) per sequence, brought into the buffers as the header states."""
    out = []
    for s in range(len(ctx)):
        a = min(max(cu[s], 0), total)
        b = max(a, min(cu[s + 1], total))
        out.append((a, b - a, min(max(ctx[s], 0), room)))
    return out


def slots(table, s, lo, hi, page_size, num_pages):
    """(position, page, offset) of positions lo .. hi-1 that have a page."""
    for p in range(lo, hi):
        page = int(table[s][p // page_size])
        if 0 <= page < num_pages:
            yield p, page, p % page_size


def mrope_append(q, k, v, positions, rope, pair_axis, k_cache, v_cache, table, cu, ctx, qw=None, kw=None, eps=1e-6,
                 pairing="halves"):
    """(q_out, k_cache, v_cache) in float64; rows of no sequence are NaN in q_out."""
    pages, page_size = k_cache.shape[:2]
    rot = 2 * len(pair_axis)
    kc, vc = k_cache.double().clone(), v_cache.double().clone()
    qo = torch.full(q.shape, math.nan, dtype=torch.float64)

    def turn(x, w, t):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1 + w.double())
        y = x.clone()
        for i, axis in enumerate(pair_axis):
            row = min(max(int(positions[axis][t]), 0), rope.shape[0] - 1)
            c, s = float(rope[row][2 * i]), float(rope[row][2 * i + 1])
            a, b = (i, i + rot // 2) if pairing == "halves" else (2 * i, 2 * i + 1)
            y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        return y

    for s, (first, n, length) in enumerate(spans(cu, ctx, q.shape[0], table.shape[1] * page_size)):
        for t in range(first, first + n):
            qo[t] = turn(q[t], qw, t)
            p = length - n + t - first
            for _, page, off in slots(table, s, p, p + 1, page_size, pages) if p >= 0 else ():
                kc[page, off] = turn(k[t], kw, t)
                vc[page, off] = v[t].double()
    return qo, kc, vc


def attention(q, k_cache, v_cache, table, cu, ctx, scale=None, window=0, gate=None):
    """(out, lse, size): size is what the bound of an element scales with, softmax . |V| and its spread over the
    keys' scores; rows of no sequence are NaN."""
    pages, page_size, kv, dim = k_cache.shape
    heads = q.shape[1]
    group = heads // kv
    scale = scale or 1.0 / math.sqrt(dim)
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    lse = torch.full(q.shape[:2], math.nan, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    half = HALF[q.dtype]
    for s, (first, n, length) in enumerate(spans(cu, ctx, q.shape[0], table.shape[1] * page_size)):
        where = list(slots(table, s, 0, length, page_size, pages))
        pos = torch.tensor([w[0] for w in where], dtype=torch.long)
        K = torch.stack([k_cache[w[1], w[2]] for w in where]).double() if where else None
        V = torch.stack([v_cache[w[1], w[2]] for w in where]).double() if where else None
        for i in range(n):
            p = length - n + i
            see = (pos <= p) & (pos > p - window if window else pos >= 0)
            t = first + i
            if not where or not bool(see.any()):
                out[t], lse[t] = 0.0, -math.inf
                continue
            for h in range(heads):
                kk, vv, qq = K[see][:, h // group], V[see][:, h // group], q[t, h].double()
                x = kk @ qq * scale
                lse[t, h] = torch.logsumexp(x, 0)
                w = torch.exp(x - lse[t, h])
                out[t, h] = w @ vv
                # relative error of a weight: the score's dim products summed in fp32 and its scaling, exp2, and
                # the same in the running sum, which adds one rounding per key
                ds = (dim + 4) * 2.0 ** -24 * float((kk.abs() @ qq.abs() * scale).max()) + 8 * 2.0 ** -24
                rel = half + 2 * ds + 2 * len(kk) * 2.0 ** -24
                # and weights below 2^-21 of the largest lose bits in fp16: at most 2^-32 each; an element of the
                # result has only its own column's values in it, finite or not
                bound[t, h] = rel * (w @ vv.abs()) + len(kk) * 2.0 ** -32 * vv.abs().amax(0)
    if gate is not None:
        g = torch.sigmoid(gate.double())
        out, bound = out * g, bound * g + 2.0 ** -20 * out.abs()
    return out, lse, bound * 1.0 + half * out.abs() * (1 + half)
