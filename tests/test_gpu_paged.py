"""GPU parity of the paged serving step (spk_mrope_append, spk_paged_attention)
against the definitions in 64 bits (paged_ref.py).

Bars, from the arithmetic: a 16-bit result of the rotation is one rounding
(2^-11 fp16, 2^-8 bf16, relative) plus 40 fp32 roundings of the terms it is
made of (16 fused squares and their tree, 1/sqrt, three products, two fused
sums: under 40 x 2^-24 of |x1| + |x2|).  Attention: paged_ref.attention's
bound, one rounding of the weights and one of the result, plus the fp32 error
of dim-long scores and key-long sums."""
import math

import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _tables(lens, page_size, seed, spare=3, pages_of=None):
    """cu, ctx, table (random pages of a pool with some spare) as host lists / int32 tensor, and the pool's pages."""
    rng = np.random.default_rng(seed)
    need = [max(1, -(-c // page_size)) for _, c in lens]
    pages = sum(need) + spare
    order, at = rng.permutation(pages), 0
    table = torch.full((len(lens), max(need) + 1), pages + 7, dtype=torch.int32)
    for s, n in enumerate(need):
        table[s, :n] = torch.from_numpy(order[at:at + n].astype(np.int32))
        at += n
    cu = [0] + np.cumsum([n for n, _ in lens]).tolist()
    return cu, [c for _, c in lens], table, pages


def _normal(gen, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _attend(dev, q, kc, vc, table, cu, ctx, max_q=None, max_c=None, out=None, **kw):
    from spock_amd import ops
    n = max([b - a for a, b in zip(cu, cu[1:])] + [0])
    gate = kw.pop("gate", None)
    r = ops.paged_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), _i32(cu, dev), _i32(ctx, dev),
                            n if max_q is None else max_q, max(ctx) if max_c is None else max_c, return_lse=True,
                            gate=None if gate is None else gate.to(dev), out=out, **kw)
    torch.cuda.synchronize()
    return r[0].cpu(), r[1].cpu()


def _check(out, lse, ref, rows=None):
    want, wlse, bound = ref
    rows = torch.arange(want.shape[0]) if rows is None else rows
    have, want, bound = out.double()[rows], want[rows], bound[rows]
    off = (have - want).abs()
    assert bool((torch.isnan(have) == torch.isnan(want)).all())
    ok = (off <= bound + 2.0 ** -26) | torch.isnan(want) | (have == want)
    assert bool(ok.all()), (float((off / (bound + 1e-30))[~ok].max()), torch.nonzero(~ok)[:4].tolist())
    a, b = lse.double()[rows], wlse[rows]
    same = (a == b) | (torch.isnan(a) & torch.isnan(b))
    assert bool((same | ((a - b).abs() <= 2.0 ** -18 * (1 + b.abs()))).all()), float((a - b)[~same].abs().max())


HEADS = [(8, 2, 256), (4, 4, 128), (12, 3, 64), (7, 1, 64), (6, 1, 128), (1, 1, 256), (40, 2, 64)]
# one token; the smallest lengths and page ends; drafts; no new tokens, no context, more new tokens than positions;
# a chunk over a context that ends inside a page
LENS = [[(1, 1)], [(1, 15), (1, 16), (1, 17), (1, 33), (1, 128), (1, 129), (1, 700)], [(5, 5), (9, 300), (4, 131), (2, 40)],
        [(0, 10), (3, 0), (4, 2), (1, 50), (0, 0), (2, 2)], [(67, 131), (33, 33)], [(130, 391)]]


@pytest.mark.parametrize("lens", LENS, ids=lambda v: "+".join("%d:%d" % x for x in v))
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention(dev, dtype, heads, kv, dim, lens):
    print(f"[paged attention {dtype} {heads}/{kv}x{dim} {lens}]", flush=True)
    gen = torch.Generator().manual_seed(heads * 1000 + dim + len(lens))
    page = [16, 20, 1, 64][(heads + dim // 64 + len(lens)) % 4]
    cu, ctx, table, pages = _tables(lens, page, heads + dim)
    kc, vc = (_normal(gen, pages, page, kv, dim, dtype=DT[dtype]) for _ in range(2))
    q = _normal(gen, cu[-1], heads, dim, dtype=DT[dtype], std=2.0)
    gate = _normal(gen, cu[-1], heads, dim, dtype=DT[dtype]) if len(lens) % 2 else None
    window = 0 if len(lens) != 3 else 24
    ref = R.attention(q, kc, vc, table, cu, ctx, window=window, gate=gate)
    _check(*_attend(dev, q, kc, vc, table, cu, ctx, window=window, gate=gate), ref)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 100, 5000])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_windows(dev, dtype, window):
    lens = [(1, 300), (40, 300), (70, 70), (3, 2)]
    print(f"[paged attention window {window} {dtype}]", flush=True)
    gen = torch.Generator().manual_seed(window)
    cu, ctx, table, pages = _tables(lens, 16, window)
    kc, vc = (_normal(gen, pages, 16, 2, 128, dtype=DT[dtype]) for _ in range(2))
    q = _normal(gen, cu[-1], 8, 128, dtype=DT[dtype], std=2.0)
    ref = R.attention(q, kc, vc, table, cu, ctx, window=window)
    _check(*_attend(dev, q, kc, vc, table, cu, ctx, window=window), ref)


def _hide_nonfinite(t, table, ctx, page, value):
    """Every slot that no sequence holds becomes `value`."""
    seen = torch.zeros(t.shape[:2], dtype=torch.bool)
    for s, n in enumerate(ctx):
        for _, pg, off in R.slots(table, s, 0, n, page, t.shape[0]):
            seen[pg, off] = True
    t[~seen] = value


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens", [[(1, 37), (1, 300), (1, 5)], [(9, 300), (6, 6), (20, 45)], [(150, 200)]], ids=str)
@pytest.mark.parametrize("dtype,dim", [("f16", 256), ("bf16", 128), ("f16", 64)])
def test_what_a_row_does_not_see_cannot_reach_it(dev, dtype, dim, lens, value):
    """NaN and infinities in slots without a token, and in keys and values of tokens after a row or before its window:
    the rows that do not see them are as without them, those that do are as the formula says."""
    print(f"[paged attention unseen {value} {dtype} {dim} {lens}]", flush=True)
    gen = torch.Generator().manual_seed(dim)
    page = 16
    cu, ctx, table, pages = _tables(lens, page, dim)
    kc, vc = (_normal(gen, pages, page, 2, dim, dtype=DT[dtype]) for _ in range(2))
    q = _normal(gen, cu[-1], 8, dim, dtype=DT[dtype])
    for t in (kc, vc):
        _hide_nonfinite(t, table, ctx, page, value)
    _check(*_attend(dev, q, kc, vc, table, cu, ctx), R.attention(q, kc, vc, table, cu, ctx))
    # in the last sequence: the last token's value (only its own row sees it), one value early in the context seen by
    # rows with a window alone, one element only
    s = len(lens) - 1
    n, c = lens[s]
    for window in (0, 3):
        kk, vv = kc.clone(), vc.clone()
        pg, off = int(table[s][(c - 1) // page]), (c - 1) % page
        vv[pg, off, 1, 5] = value
        if window:
            pg, off = int(table[s][(c - n) // page]), (c - n) % page
            vv[pg, off, :, 3::7] = value
            if value != value:
                pg, off = int(table[s][0]), 0
                kk[pg, off] = value
        _check(*_attend(dev, q, kk, vv, table, cu, ctx, window=window), R.attention(q, kk, vv, table, cu, ctx, window=window))


def test_scores_of_infinity(dev):
    """A score of -inf weighs nothing; one of +inf or NaN makes its row NaN; scores all -inf leave zeros."""
    gen = torch.Generator().manual_seed(4)
    cu, ctx, table, pages = _tables([(1, 40)], 16, 4)
    kc, vc = (_normal(gen, pages, 16, 1, 64, dtype=torch.bfloat16) for _ in range(2))
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16)
    big = torch.full((64,), 3e38, dtype=torch.bfloat16)
    pg, off = int(table[0][1]), 3
    kc[pg, off, 0] = -big          # q . k = -inf
    ref = R.attention(q, kc.clone().index_put((torch.tensor([pg]), torch.tensor([off])), torch.full((1, 1, 64), -1e30, dtype=torch.bfloat16)),
                      vc, table, cu, ctx)
    out, lse = _attend(dev, q, kc, vc, table, cu, ctx)
    assert bool(((out.double() - ref[0]).abs() <= R.HALF[torch.bfloat16] * 8 * (1 + ref[0].abs())).all())
    kc[pg, off, 0] = big           # +inf
    out, lse = _attend(dev, q, kc, vc, table, cu, ctx)
    assert bool(torch.isnan(out).all())
    kc[:] = -big
    out, lse = _attend(dev, q, kc, vc, table, cu, ctx)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("n,ctx", [(1, 400), (5, 400), (80, 400)])
def test_bad_pages_and_lengths(dev, n, ctx):
    """Page ids outside the pool, contexts past the table, offsets past the rows: masked, and nothing outside written."""
    gen = torch.Generator().manual_seed(n)
    lens = [(n, ctx), (n, ctx)]
    cu, cl, table, pages = _tables(lens, 16, n)
    kc, vc = (_normal(gen, pages, 16, 2, 128, dtype=torch.float16) for _ in range(2))
    q = _normal(gen, cu[-1], 4, 128, dtype=torch.float16)
    table[0, 3], table[0, 7], table[1, 0], table[1, 24] = -1, pages, -2 ** 31, 2 ** 31 - 1
    _check(*_attend(dev, q, kc, vc, table, cu, cl), R.attention(q, kc, vc, table, cu, cl))
    table[1, :] = pages + 3        # no page at all
    _check(*_attend(dev, q, kc, vc, table, cu, cl), R.attention(q, kc, vc, table, cu, cl))
    cl2 = [10 ** 9, 400]
    _check(*_attend(dev, q, kc, vc, table, cu, cl2, max_c=400), R.attention(q, kc, vc, table, cu, cl2))
    cu2 = [0, n, 10 ** 6]
    _check(*_attend(dev, q, kc, vc, table, cu2, cl, max_q=n), R.attention(q, kc, vc, table, cu2, cl))


@pytest.mark.parametrize("max_c", [1, 100, 1000, 50000])
def test_context_bound_does_not_change_the_result(dev, max_c):
    gen = torch.Generator().manual_seed(9)
    lens = [(1, 1000), (4, 333), (2, 64)]
    cu, ctx, table, pages = _tables(lens, 16, 9)
    kc, vc = (_normal(gen, pages, 16, 2, 256, dtype=torch.float16) for _ in range(2))
    q = _normal(gen, cu[-1], 8, 256, dtype=torch.float16)
    _check(*_attend(dev, q, kc, vc, table, cu, ctx, max_c=max_c), R.attention(q, kc, vc, table, cu, ctx))


def test_rows_behind_the_last_sequence_stay(dev):
    gen = torch.Generator().manual_seed(3)
    lens = [(3, 200), (1, 90)]
    cu, ctx, table, pages = _tables(lens, 16, 3)
    kc, vc = (_normal(gen, pages, 16, 2, 128, dtype=torch.bfloat16) for _ in range(2))
    q = _normal(gen, 9, 4, 128, dtype=torch.bfloat16)
    from spock_amd import ops
    for max_c in (200, 20000):
        out = torch.full((9, 4, 128), 7.5, dtype=torch.bfloat16, device=dev)
        lse = torch.full((9, 4), 7.5, device=dev)
        ops.paged_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), _i32(cu, dev), _i32(ctx, dev), 3, max_c, out=out, lse=lse)
        torch.cuda.synchronize()
        ref = R.attention(q, kc, vc, table, cu, ctx)
        _check(out.cpu(), lse.cpu(), ref, rows=torch.arange(4))
        assert bool((out[4:] == 7.5).all()) and bool((lse[4:] == 7.5).all())


def test_layouts_and_scale(dev):
    """Queries and gates inside a projection's rows, a [page][head][token] pool, the session's [pos][K | V] rows as
    one page, outputs with strides, a scale of the caller's."""
    from spock_amd import ops
    gen = torch.Generator().manual_seed(8)
    lens = [(6, 70), (2, 33)]
    cu, ctx, table, pages = _tables(lens, 16, 8)
    kc, vc = (_normal(gen, pages, 16, 2, 256, dtype=torch.float16) for _ in range(2))
    qg = _normal(gen, cu[-1], 8, 512, dtype=torch.float16)
    q, gate = qg[..., :256], qg[..., 256:]
    ref = R.attention(q, kc, vc, table, cu, ctx, scale=0.11, gate=gate)
    dqg = qg.to(dev)
    hk, hv = (t.permute(0, 2, 1, 3).contiguous().to(dev).permute(0, 2, 1, 3) for t in (kc, vc))
    wide = torch.zeros(cu[-1], 8, 264, dtype=torch.float16, device=dev)
    out, lse = ops.paged_attention(dqg[..., :256], hk, hv, table.to(dev), _i32(cu, dev), _i32(ctx, dev), 6, 70, scale=0.11,
                                   gate=dqg[..., 256:], out=wide[..., :256], return_lse=True)
    torch.cuda.synchronize()
    _check(out.cpu(), lse.cpu(), ref)
    assert bool((wide[..., 256:] == 0).all())
    rows = _normal(gen, 100, 1024, dtype=torch.float16)
    drows = rows.to(dev)
    k1, v1 = (t.view(1, 100, 2, 256) for t in (rows[:, :512], rows[:, 512:]))
    one = torch.zeros(1, 1, dtype=torch.int32)
    ref = R.attention(q[:3], k1, v1, one, [0, 3], [91])
    out, lse = ops.paged_attention(dqg[:3, :, :256], drows[:, :512].unflatten(1, (2, 256))[None],
                                   drows[:, 512:].unflatten(1, (2, 256))[None], one.to(dev), _i32([0, 3], dev), _i32([91], dev),
                                   3, 91, return_lse=True)
    torch.cuda.synchronize()
    _check(out.cpu(), lse.cpu(), ref)


def test_offsets_past_32_bits(dev):
    """A pool of more than 2^32 elements: the last pages are read and written at their own place."""
    from spock_amd import ops
    page, kv, dim = 64, 4, 256
    pages = 2 ** 32 // (page * kv * dim) + 40
    kc = torch.zeros(pages, page, kv, dim, dtype=torch.float16, device=dev)
    vc = torch.zeros_like(kc)
    gen = torch.Generator().manual_seed(1)
    small = [_normal(gen, 3, page, kv, dim, dtype=torch.float16) for _ in range(2)]
    where = [pages - 1, pages - 20, 5]
    for i, p in enumerate(where):
        kc[p], vc[p] = small[0][i].to(dev), small[1][i].to(dev)
    table = torch.tensor([where], dtype=torch.int32)
    q = _normal(gen, 2, 8, dim, dtype=torch.float16)
    ref = R.attention(q, *small, torch.tensor([[0, 1, 2]]), [0, 2], [150])
    out, lse = ops.paged_attention(q.to(dev), kc, vc, table.to(dev), _i32([0, 2], dev), _i32([150], dev), 2, 150, return_lse=True)
    torch.cuda.synchronize()
    _check(out.cpu(), lse.cpu(), ref)
    x = _normal(gen, 2, kv, dim, dtype=torch.float16).to(dev)
    rope = torch.tensor([[1.0, 0.0] * 16], device=dev)
    table = torch.tensor([[5, pages - 1]], dtype=torch.int32, device=dev)
    ops.mrope_append(q.to(dev), x, x, torch.zeros(1, 2, dtype=torch.int32, device=dev), rope, [0] * 16, kc, vc, table,
                     _i32([0, 2], dev), _i32([65], dev))
    torch.cuda.synchronize()
    assert torch.equal(kc[5, 63], x[0]) and torch.equal(vc[pages - 1, 0], x[1]) and torch.equal(kc[pages - 1, 0], x[1])
    del kc, vc
    torch.cuda.empty_cache()


def _mrope_inputs(dtype, heads, kv, dim, rot, axes, lens, page, seed, norm):
    gen = torch.Generator().manual_seed(seed)
    cu, ctx, table, pages = _tables(lens, page, seed)
    T = cu[-1]
    q, k, v = (_normal(gen, T, h, dim, dtype=DT[dtype]) for h in (heads, kv, kv))
    kc, vc = (_normal(gen, pages, page, kv, dim, dtype=DT[dtype]) for _ in range(2))
    w = [_normal(gen, dim, dtype=DT[dtype], std=0.3) if norm else None for _ in range(2)]
    rows = 500
    pos = torch.randint(0, rows, (axes, T), generator=gen, dtype=torch.int32)
    angle = torch.arange(rows)[:, None].double() * 1e4 ** (-torch.arange(rot // 2).double() / (rot // 2))
    rope = torch.stack([angle.cos(), angle.sin()], -1).reshape(rows, rot).float()
    return q, k, v, pos, rope, kc, vc, table, cu, ctx, w


def _mrope_bound(x, w, want, rot, pairing, dtype):
    """40 fp32 roundings of |x1| + |x2| and one of the result."""
    x = x.double().abs()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (1 + w.double()).abs()
    y = x.clone()
    if pairing == "halves":
        s = x[..., :rot // 2] + x[..., rot // 2:rot]
        y[..., :rot // 2] = y[..., rot // 2:rot] = s
    else:
        s = x[..., 0:rot:2] + x[..., 1:rot:2]
        y[..., 0:rot:2] = y[..., 1:rot:2] = s
    return want.abs() * R.HALF[dtype] + y * 40 * 2.0 ** -24 + 2.0 ** -25


@pytest.mark.parametrize("heads,kv,dim,rot", [(8, 2, 256, 64), (3, 3, 128, 128), (12, 3, 64, 48), (5, 1, 256, 256), (2, 1, 64, 16)])
@pytest.mark.parametrize("pairing", ["halves", "adjacent"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_mrope_append(dev, dtype, pairing, heads, kv, dim, rot):
    from spock_amd import ops
    print(f"[mrope {dtype} {pairing} {heads}/{kv}x{dim} rot {rot}]", flush=True)
    for axes, norm, page, lens in ((1, False, 16, [(1, 1)]), (3, True, 20, [(5, 37), (1, 20), (0, 4), (3, 2), (18, 18)]), (4, True, 1, [(70, 70)]),
                                   (2, False, 64, [(1, 60 + i) for i in range(67)])):
        q, k, v, pos, rope, kc, vc, table, cu, ctx, (qw, kw) = _mrope_inputs(dtype, heads, kv, dim, rot, axes, lens, page, dim + axes, norm)
        axis = [i % axes if norm else i * axes // (rot // 2) for i in range(rot // 2)]
        want = R.mrope_append(q, k, v, pos, rope, axis, kc, vc, table, cu, ctx, qw, kw, pairing=pairing)
        dk, dv = kc.to(dev), vc.to(dev)
        to = lambda t: None if t is None else t.to(dev)
        out = ops.mrope_append(to(q), to(k), to(v), to(pos), to(rope), axis, dk, dv, to(table), _i32(cu, dev), _i32(ctx, dev),
                               q_norm_weight=to(qw), k_norm_weight=to(kw), pairing=pairing)
        torch.cuda.synchronize()
        assert bool(((out.cpu().double() - want[0]).abs() <= _mrope_bound(q, qw, want[0], rot, pairing, q.dtype)).all())
        assert torch.equal(dv.cpu().double(), want[2])
        # bound of the keys: through the same call of the reference with |k|'s bound at the stored slots
        wrote = (want[1] != kc.double()).flatten(2).any(-1) | (want[2] != vc.double()).flatten(2).any(-1)
        off = (dk.cpu().double() - want[1]).abs()
        assert bool((off[~wrote] == 0).all())
        size = _mrope_bound(k, kw, torch.zeros_like(k.double()), rot, pairing, q.dtype).amax(0)
        assert bool((off <= want[1].abs() * R.HALF[q.dtype] + size).all())


def test_mrope_bad_pages_positions_and_padding(dev):
    """Tokens without a page are rotated and not stored; positions outside the table take its ends; rows behind the
    last sequence, the other slots and the rest of a wide row stay as they were; q may be rotated in place."""
    from spock_amd import ops
    lens = [(6, 40), (4, 4), (3, 1)]
    q, k, v, pos, rope, kc, vc, table, cu, ctx, _ = _mrope_inputs("f16", 4, 2, 128, 64, 3, lens, 16, 5, False)
    T = cu[-1]
    pad = 5
    q, k, v = (torch.cat([t, torch.full((pad, *t.shape[1:]), 3.0, dtype=t.dtype)]) for t in (q, k, v))
    pos = torch.cat([pos, torch.full((3, pad), -9, dtype=torch.int32)], 1)
    pos[0, 0], pos[1, 1], pos[2, 2] = -5, 10 ** 9, -2 ** 31
    table[0, 2], table[1, 0] = kc.shape[0], -1
    axis = [i % 3 for i in range(32)]
    want = R.mrope_append(q, k, v, pos, rope, axis, kc, vc, table, cu, ctx)
    wide = torch.zeros(T + pad, 4, 136, dtype=torch.float16)
    wide[..., :128], wide[..., 128:] = q, 9.0
    dw, dk, dv = wide.to(dev), kc.to(dev), vc.to(dev)
    dq = dw[..., :128]
    out = ops.mrope_append(dq, k.to(dev), v.to(dev), pos.to(dev), rope.to(dev), axis, dk, dv, table.to(dev), _i32(cu, dev), _i32(ctx, dev), out=dq)
    torch.cuda.synchronize()
    assert out.data_ptr() == dq.data_ptr()
    got = dw.cpu()
    bound = _mrope_bound(q, None, want[0].nan_to_num(), 64, "halves", q.dtype)
    assert bool(((got[:T, :, :128].double() - want[0][:T]).abs() <= bound[:T]).all())
    assert bool((got[T:, :, :128] == 3.0).all()) and bool((got[..., 128:] == 9.0).all())
    assert torch.equal(dv.cpu().double(), want[2])
    assert bool(((dk.cpu().double() - want[1]).abs() <= 2.0 ** -10 * (1 + want[1].abs()) * (want[1] != kc.double())).all())


def test_step_as_it_is_used_and_replayed(dev):
    """Rotation, store and attention of a decode step on another stream, then captured once and replayed while the
    lengths, pages, positions and inputs in their buffers change: every replay as the eager calls."""
    from spock_amd import ops
    gen = torch.Generator().manual_seed(11)
    S, page, heads, kv, dim = 3, 16, 8, 2, 256
    pages, cols = 40, 12
    kc, vc = (_normal(gen, pages, page, kv, dim, dtype=torch.float16) for _ in range(2))
    angle = torch.arange(400)[:, None].double() * 1e4 ** (-torch.arange(32).double() / 32)
    rope = torch.stack([angle.cos(), angle.sin()], -1).reshape(400, 64).float().to(dev)
    axis = [i % 3 for i in range(32)]
    buf = {"q": torch.zeros(S, heads, dim, dtype=torch.float16, device=dev), "k": torch.zeros(S, kv, dim, dtype=torch.float16, device=dev),
           "v": torch.zeros(S, kv, dim, dtype=torch.float16, device=dev), "pos": torch.zeros(3, S, dtype=torch.int32, device=dev),
           "table": torch.zeros(S, cols, dtype=torch.int32, device=dev), "ctx": torch.ones(S, dtype=torch.int32, device=dev),
           "cu": _i32([0, 1, 2, 3], dev), "kc": kc.to(dev), "vc": vc.to(dev)}
    need = ops.paged_attention_workspace_bytes(S, heads, kv, dim, page, cols, S, 1, cols * page)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    out = torch.zeros(S, heads, dim, dtype=torch.float16, device=dev)
    lse = torch.zeros(S, heads, device=dev)

    def step():
        q = ops.mrope_append(buf["q"], buf["k"], buf["v"], buf["pos"], rope, axis, buf["kc"], buf["vc"], buf["table"], buf["cu"], buf["ctx"])
        ops.paged_attention(q, buf["kc"], buf["vc"], buf["table"], buf["cu"], buf["ctx"], 1, cols * page, out=out, lse=lse, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    rng = np.random.default_rng(2)
    for replay in range(5):
        ctx = [int(x) for x in rng.integers(1, cols * page, S)]
        order = rng.permutation(pages)[:S * cols].reshape(S, cols).astype(np.int32)
        fresh = {n: _normal(gen, *buf[n].shape, dtype=torch.float16) for n in ("q", "k", "v")}
        pos = torch.randint(0, 400, (3, S), generator=gen, dtype=torch.int32)
        for n, t in fresh.items():
            buf[n].copy_(t)
        buf["pos"].copy_(pos)
        buf["ctx"].copy_(torch.tensor(ctx, dtype=torch.int32))
        buf["table"].copy_(torch.from_numpy(order))
        before = buf["kc"].cpu(), buf["vc"].cpu()
        graph.replay()
        torch.cuda.synchronize()
        got = out.cpu(), lse.cpu()
        rq, rk, rv = R.mrope_append(fresh["q"], fresh["k"], fresh["v"], pos, rope.cpu(), axis, *before, torch.from_numpy(order), [0, 1, 2, 3], ctx)
        assert torch.equal(buf["vc"].cpu().double(), rv)
        assert bool(((buf["kc"].cpu().double() - rk).abs() <= 2.0 ** -11 * rk.abs() + 2.0 ** -20).all())
        step()  # the program's own eager work between replays
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), got[0]) and torch.equal(lse.cpu(), got[1])
        q16 = ops.mrope_append(buf["q"], buf["k"], buf["v"], buf["pos"], rope, axis, buf["kc"], buf["vc"], buf["table"], buf["cu"], buf["ctx"])
        _check(*got, R.attention(q16.cpu(), buf["kc"].cpu(), buf["vc"].cpu(), torch.from_numpy(order), [0, 1, 2, 3], ctx))


def test_argument_checks(dev):
    from spock_amd import _lib, ops
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=dev)
    c = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device=dev)
    t, cu, ctx = torch.zeros(1, 4, dtype=torch.int32, device=dev), _i32([0, 2], dev), _i32([5], dev)
    good = dict(q=q, k_cache=c, v_cache=c, block_table=t, cu_seqlens=cu, context_lens=ctx, max_query_len=2, max_context_len=64)
    ops.paged_attention(**good)
    for over in (dict(q=q.float()), dict(q=q[0]), dict(k_cache=c.bfloat16()), dict(v_cache=c[:2]), dict(block_table=t.long()),
                 dict(cu_seqlens=cu[:1]), dict(context_lens=ctx.cpu()), dict(v_cache=c.transpose(1, 2).contiguous().transpose(1, 2)),
                 dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(gate=q[:1]), dict(out=q.bfloat16()), dict(q=q[:, :3]),
                 dict(max_query_len=-1), dict(lse=torch.zeros(2, 5, device=dev)), dict(block_table=torch.zeros(4, 8, dtype=torch.int32, device=dev)[:1, ::2])):
        with pytest.raises(_lib.SpockError):
            ops.paged_attention(**{**good, **over})
    k = torch.zeros(2, 2, 64, dtype=torch.float16, device=dev)
    pos, rope = torch.zeros(3, 2, dtype=torch.int32, device=dev), torch.zeros(9, 32, device=dev)
    good = dict(q=q, k=k, v=k, positions=pos, rope=rope, pair_axis=[0] * 16, k_cache=c, v_cache=c, block_table=t, cu_seqlens=cu, context_lens=ctx)
    ops.mrope_append(**good)
    for over in (dict(k=k[:1]), dict(v=q), dict(positions=pos.long()), dict(positions=pos[:, :1]), dict(rope=rope[:, :30]), dict(rope=rope.half()),
                 dict(pair_axis=[0] * 15 + [3]), dict(pair_axis=[0] * 15 + [-1]), dict(pair_axis=16), dict(pairing="other"), dict(out=q[:1]),
                 dict(q_norm_weight=torch.zeros(32, dtype=torch.float16, device=dev)), dict(k_norm_weight=torch.zeros(64, device=dev)),
                 dict(pair_axis=[0] * 12, rope=rope[:, :24].contiguous())):
        with pytest.raises(_lib.SpockError):
            ops.mrope_append(**{**good, **over})
    torch.cuda.synchronize()
