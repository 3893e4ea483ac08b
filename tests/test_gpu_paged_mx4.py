"""GPU parity of the paged serving step in 4 bits (spk_mrope_append_mx4, spk_paged_attention_mx4) against the
definitions in 64 bits (mx4_ref.py, paged_ref.py).

Bars: what is stored is exact (the keys are computed in 64 bits before their one rounding), the rotated queries are
spk_mrope_append's bit for bit.  Attention: paged_ref.attention's bound over the values that the pages hold, which
counts one rounding of the weights and one of the result."""
import math

import numpy as np
import pytest
import torch

import mx4_ref as M
import paged_ref as R
from test_gpu_paged import HEADS, LENS, _i32, _normal, _tables

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
ORDERS = {"heads": (0, 2, 1, 3), "tokens": (0, 1, 2, 3), "pages inside": (2, 1, 0, 3)}


def _pool(gen, pages, page, kv, dim, spread=0.5):
    """(codes, scales) of a pool [pages][page][kv][dim] on the CPU."""
    x = torch.randn(pages, page, kv, dim, generator=gen) * torch.exp(spread * torch.randn(pages, page, kv, 1, generator=gen))
    return M.quantize(x)


def _on(dev, m, order="heads"):
    """An Mx4 on the device whose memory has that order of [page][token][head]."""
    from spock_amd import ops
    back = [ORDERS[order].index(i) for i in range(4)]
    return ops.Mx4(*(t.permute(ORDERS[order]).contiguous().to(dev).permute(back) for t in m))


def _attend(dev, q, k, v, table, cu, ctx, max_q=None, max_c=None, order="heads", gate=None, **kw):
    from spock_amd import ops
    n = max([b - a for a, b in zip(cu, cu[1:])] + [0])
    r = ops.paged_attention_mx4(q.to(dev), _on(dev, k, order), _on(dev, v, order), table.to(dev), _i32(cu, dev), _i32(ctx, dev),
                                n if max_q is None else max_q, max(ctx) if max_c is None else max_c, return_lse=True,
                                gate=None if gate is None else gate.to(dev), **kw)
    torch.cuda.synchronize()
    return r[0].cpu(), r[1].cpu()


def _check(out, lse, ref, rows=None):
    """Within the bound, plus half of fp16's smallest step (2^-24): many of a 4-bit column's values are 0, so that a result
    may be the sum of the lightest keys' alone and lie where that step is the rounding (9.3e-8 has 6.0e-8 and 1.2e-7 beside
    it: 2.6e-8 off, 2^-25 = 3.0e-8 at most)."""
    want, wlse, bound = ref
    rows = torch.arange(want.shape[0]) if rows is None else rows
    have, want, bound = out.double()[rows], want[rows], bound[rows]
    floor = 2.0 ** -25 if out.dtype is torch.float16 else 2.0 ** -126
    assert bool((torch.isnan(have) == torch.isnan(want)).all())
    off = (have - want).abs()
    ok = (off <= bound + floor) | torch.isnan(want) | (have == want)
    assert bool(ok.all()), (float((off / (bound + floor))[~ok].max()), torch.nonzero(~ok)[:4].tolist())
    a, b = lse.double()[rows], wlse[rows]
    same = (a == b) | (torch.isnan(a) & torch.isnan(b))
    assert bool((same | ((a - b).abs() <= 2.0 ** -18 * (1 + b.abs()))).all()), float((a - b)[~same].abs().max())


def _reference(q, k, v, table, cu, ctx, **kw):
    return R.attention(q, M.cached(*k, q.dtype), M.cached(*v, q.dtype), table, cu, ctx, **kw)


@pytest.mark.parametrize("lens", LENS, ids=lambda v: "+".join("%d:%d" % x for x in v))
@pytest.mark.parametrize("heads,kv,dim", HEADS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention(dev, dtype, heads, kv, dim, lens):
    print(f"[mx4 attention {dtype} {heads}/{kv}x{dim} {lens}]", flush=True)
    gen = torch.Generator().manual_seed(heads * 1000 + dim + len(lens))
    page = [16, 20, 1, 64][(heads + dim // 64 + len(lens)) % 4]
    cu, ctx, table, pages = _tables(lens, page, heads + dim)
    k, v = (_pool(gen, pages, page, kv, dim) for _ in range(2))
    q = _normal(gen, cu[-1], heads, dim, dtype=DT[dtype], std=2.0)
    gate = _normal(gen, cu[-1], heads, dim, dtype=DT[dtype]) if len(lens) % 2 else None
    window = 0 if len(lens) != 3 else 24
    order = list(ORDERS)[(heads + len(lens)) % 3]
    ref = _reference(q, k, v, table, cu, ctx, window=window, gate=gate)
    _check(*_attend(dev, q, k, v, table, cu, ctx, window=window, gate=gate, order=order), ref)


# rows on either side of where a sequence has many: 128, 256 and 512 for heads of 64, 128 and 256
@pytest.mark.parametrize("lens", [[(64, 200), (65, 200)], [(128, 300), (1, 40), (129, 140)], [(256, 300)], [(257, 300), (256, 256), (3, 9)]], ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (2, 1, 128), (4, 2, 256)])
def test_attention_where_rows_become_many(dev, heads, kv, dim, lens):
    print(f"[mx4 attention many {heads}/{kv}x{dim} {lens}]", flush=True)
    gen = torch.Generator().manual_seed(dim + len(lens))
    cu, ctx, table, pages = _tables(lens, 16, dim)
    k, v = (_pool(gen, pages, 16, kv, dim) for _ in range(2))
    q = _normal(gen, cu[-1], heads, dim, dtype=torch.bfloat16, std=2.0)
    _check(*_attend(dev, q, k, v, table, cu, ctx), _reference(q, k, v, table, cu, ctx))


# pieces of 16 rows, and tiles of 256 of sequences of many rows
@pytest.mark.parametrize("lens", [[(1, 400), (9, 90)], [(290, 310), (5, 40)]], ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (2, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_weights_keep_their_bits(dev, dtype, heads, kv, dim, lens):
    """A weight enters the product with V in two parts, each half a step off at most: what is lost of it is the square of one
    rounding, which shows where values of both signs cancel.  paged_ref's bound with that in the place of one rounding of
    softmax . |V|, which is the same attention over |V|."""
    print(f"[mx4 attention weights {dtype} {heads}/{kv}x{dim} {lens}]", flush=True)
    t, gen = DT[dtype], torch.Generator().manual_seed(dim + len(lens))
    cu, ctx, table, pages = _tables(lens, 16, dim)
    k, v = (_pool(gen, pages, 16, kv, dim) for _ in range(2))
    q = _normal(gen, cu[-1], heads, dim, dtype=t, std=2.0)
    want, lse, bound = _reference(q, k, v, table, cu, ctx)
    size = _reference(q, k, (v[0] & 0x77, v[1]), table, cu, ctx)[0]
    half = R.HALF[t]
    bound -= (half - half * half) * size
    _check(*_attend(dev, q, k, v, table, cu, ctx), (want, lse, bound))


@pytest.mark.parametrize("lens", [[(1, 400), (9, 90)], [(290, 310), (5, 40)]], ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (2, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_weights_keep_their_bits_of_exact_scores(dev, dtype, heads, kv, dim, lens):
    """As above where the scores leave no room for one rounding in fp16 either: a query has one element, so that a product
    with a key is exact.  Left of a weight's error are, in 2^-24, the scale's own (4 of the score's size), the sum
    with the maximum (2 of it, and 7 for fp16's shift) and exp2 (8): 8 of the scores' size and 16, and as much in the sum."""
    print(f"[mx4 attention exact scores {dtype} {heads}/{kv}x{dim} {lens}]", flush=True)
    t, gen = DT[dtype], torch.Generator().manual_seed(3 * dim + len(lens))
    cu, ctx, table, pages = _tables(lens, 16, dim)
    k, v = (_pool(gen, pages, 16, kv, dim) for _ in range(2))
    q = torch.zeros(cu[-1], heads, dim).scatter_(2, torch.randint(0, dim, (cu[-1], heads, 1), generator=gen), 16.0 if dim == 64 else 32.0).to(t)
    want, lse, _ = _reference(q, k, v, table, cu, ctx)
    size = _reference(q, k, (v[0] & 0x77, v[1]), table, cu, ctx)[0]
    half, most = R.HALF[t], float(M.values(*k).abs().max()) * 32 / math.sqrt(dim)
    rel = half * half + 2 * (8 * most + 16) * 2.0 ** -24 + 2 * max(ctx) * 2.0 ** -24
    assert rel < half / 4
    bound = rel * size + max(ctx) * 2.0 ** -32 * float(M.values(*v).abs().max()) + half * want.abs() * (1 + half)
    _check(*_attend(dev, q, k, v, table, cu, ctx), (want, lse, bound))


@pytest.mark.parametrize("window", [1, 2, 31, 32, 100, 5000])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_windows(dev, dtype, window):
    lens = [(1, 300), (40, 300), (70, 70), (3, 2)]
    print(f"[mx4 attention window {window} {dtype}]", flush=True)
    gen = torch.Generator().manual_seed(window)
    cu, ctx, table, pages = _tables(lens, 16, window)
    k, v = (_pool(gen, pages, 16, 2, 128) for _ in range(2))
    q = _normal(gen, cu[-1], 8, 128, dtype=DT[dtype], std=2.0)
    _check(*_attend(dev, q, k, v, table, cu, ctx, window=window), _reference(q, k, v, table, cu, ctx, window=window))


@pytest.mark.parametrize("lens", [[(1, 300), (1, 1), (0, 5), (7, 90)], [(150, 200)], [(300, 350)]], ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (8, 1, 128), (6, 3, 256)])
def test_scales_at_odd_bytes(dev, heads, kv, dim, lens):
    """Pools whose rows of scales begin at odd addresses and lie odd numbers of bytes apart."""
    from spock_amd import ops
    print(f"[mx4 odd scales {heads}/{kv}x{dim} {lens}]", flush=True)
    gen = torch.Generator().manual_seed(dim)
    cu, ctx, table, pages = _tables(lens, 16, dim)
    k, v = (_pool(gen, pages, 16, kv, dim) for _ in range(2))
    q = _normal(gen, cu[-1], heads, dim, dtype=torch.bfloat16, std=2.0)

    def odd(m):
        n = dim // 32
        return ops.Mx4(m[0].to(dev), torch.nn.functional.pad(m[1], (1, 2 - n % 2)).to(dev)[..., 1:1 + n])

    assert odd(k).scales.stride(2) % 2 == 1 and odd(k).scales.data_ptr() % 2 == 1
    out, lse = ops.paged_attention_mx4(q.to(dev), odd(k), odd(v), table.to(dev), _i32(cu, dev), _i32(ctx, dev),
                                       max(n for n, _ in lens), max(ctx), return_lse=True)
    rows = [r for r in range(cu[-1])]
    _check(out.cpu(), lse.cpu(), _reference(q, k, v, table, cu, ctx), torch.tensor(rows))


@pytest.mark.parametrize("lens", [[(1, 500), (1, 90)], [(150, 520), (1, 33)], [(300, 520), (1, 33)]], ids=str)
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (4, 2, 256)])
def test_pages_far_apart(dev, heads, kv, dim, lens):
    """Pages 2^27 bytes apart, more than 2^32 in all: stored and read as in a compact pool, bit for bit."""
    from spock_amd import ops
    print(f"[mx4 far pages {heads}/{kv}x{dim} {lens}]", flush=True)
    gen = torch.Generator().manual_seed(dim)
    cu, ctx, table, pages = _tables(lens, 16, dim)
    assert pages > 33

    def far(t):
        inner = t[0].contiguous().stride()
        hold = torch.empty(pages * 2 ** 27, dtype=torch.uint8, device=dev).as_strided(t.shape, (2 ** 27, *inner))
        return hold.copy_(t)

    k, v = (_on(dev, _pool(gen, pages, 16, kv, dim), "tokens") for _ in range(2))
    fk, fv = (ops.Mx4(*map(far, m)) for m in (k, v))
    q, nk, nv = (_normal(gen, cu[-1], n, dim, dtype=torch.float16).to(dev) for n in (heads, kv, kv))
    table, cu_d, ctx_d = table.to(dev), _i32(cu, dev), _i32(ctx, dev)
    positions = torch.arange(cu[-1], dtype=torch.int32, device=dev)[None]
    angle = torch.rand(cu[-1], dim // 2, generator=gen) * 6
    rope = torch.stack([angle.cos(), angle.sin()], -1).flatten(1).to(dev)
    outs = []
    for ck, cv in ((k, v), (fk, fv)):
        turned = ops.mrope_append_mx4(q, nk, nv, positions, rope, [0] * (dim // 2), ck, cv, table, cu_d, ctx_d)
        outs.append(ops.paged_attention_mx4(turned, ck, cv, table, cu_d, ctx_d, max(n for n, _ in lens), max(ctx)))
    assert torch.equal(*outs)
    for near, there in zip((*k, *v), (*fk, *fv)):
        assert torch.equal(near, there)


@pytest.mark.parametrize("byte", [255, 254, 141])
@pytest.mark.parametrize("lens", [[(1, 37), (1, 300), (1, 5)], [(9, 300), (6, 6), (20, 45)], [(150, 200)], [(530, 560)]], ids=str)
@pytest.mark.parametrize("dtype,dim", [("f16", 256), ("bf16", 128), ("f16", 64)])
def test_what_a_row_does_not_see_cannot_reach_it(dev, dtype, dim, lens, byte):
    """Blocks that are no numbers, or larger than the type, in slots without a token, and in keys and values of tokens after
    a row or before its window."""
    print(f"[mx4 attention unseen {byte} {dtype} {dim} {lens}]", flush=True)
    gen = torch.Generator().manual_seed(dim)
    page = 16
    cu, ctx, table, pages = _tables(lens, page, dim)
    k, v = (_pool(gen, pages, page, 2, dim) for _ in range(2))
    q = _normal(gen, cu[-1], 8, dim, dtype=DT[dtype])
    held = torch.zeros(pages, page, dtype=torch.bool)
    for s, n in enumerate(ctx):
        for _, pg, off in R.slots(table, s, 0, n, page, pages):
            held[pg, off] = True
    for _, scales in (k, v):
        scales[~held] = byte
    _check(*_attend(dev, q, k, v, table, cu, ctx), _reference(q, k, v, table, cu, ctx))
    if byte == 141 and dtype == "bf16":
        return  # a number there, of weight 2^14: the sums' bars do not hold for it
    s = len(lens) - 1
    n, c = lens[s]
    for window in (0, 3):
        kk, vv = ([t.clone() for t in m] for m in (k, v))
        pg, off = int(table[s][(c - 1) // page]), (c - 1) % page
        vv[1][pg, off, 1, 1] = byte
        if window:
            pg, off = int(table[s][(c - n) // page]), (c - n) % page
            vv[1][pg, off, :, 0] = byte
            kk[1][pg, off, 0, -1] = byte
        _check(*_attend(dev, q, kk, vv, table, cu, ctx, window=window), _reference(q, kk, vv, table, cu, ctx, window=window))


@pytest.mark.parametrize("lens", [[(1, 300)], [(9, 300), (2, 70)], [(150, 200), (1, 90)], [(530, 560), (1, 90)]], ids=str)
def test_bad_pages_and_bounds(dev, lens):
    """Pages outside the pool stand for no page; lengths beyond the table and bounds that are too low or too high change
    nothing but the rounding."""
    gen = torch.Generator().manual_seed(len(lens))
    cu, ctx, table, pages = _tables(lens, 16, 3)
    k, v = (_pool(gen, pages, 16, 2, 128) for _ in range(2))
    q = _normal(gen, cu[-1], 8, 128, dtype=torch.bfloat16)
    table[0, 1], table[-1, 0] = -1, pages
    ref = _reference(q, k, v, table, cu, ctx)
    for max_q, max_c in ((None, None), (1, 16), (0, 0), (5000, 100000)):
        print(f"[mx4 attention bounds {lens} {max_q} {max_c}]", flush=True)
        _check(*_attend(dev, q, k, v, table, cu, ctx, max_q=max_q, max_c=max_c), ref)
    table[:] = -5
    out, lse = _attend(dev, q, k, v, table, cu, ctx)
    assert not out.any() and bool((lse == -math.inf).all())


def test_rows_behind_the_last_sequence_and_workspaces(dev):
    from spock_amd import ops
    gen = torch.Generator().manual_seed(8)
    lens = [(1, 700), (5, 1200), (1, 0)]
    cu, ctx, table, pages = _tables(lens, 16, 8)
    k, v = (_pool(gen, pages, 16, 2, 128) for _ in range(2))
    q = _normal(gen, cu[-1] + 3, 8, 128, dtype=torch.float16)
    kd, vd = _on(dev, k), _on(dev, v)
    args = (q.to(dev), kd, vd, table.to(dev), _i32(cu, dev), _i32(ctx, dev), 5, 1200)
    out = torch.full_like(args[0], 7.0)
    lse = torch.full((cu[-1] + 3, 8), 7.0, device=dev)
    need = ops.paged_attention_mx4_workspace_bytes(cu[-1] + 3, 8, 2, 128, 16, table.shape[1], 3, 5, 1200)
    room = torch.full((need + 512,), 0x55, dtype=torch.uint8, device=dev)
    ops.paged_attention_mx4(*args, out=out, lse=lse, workspace=room[:need])
    assert bool((room[need:] == 0x55).all())
    assert bool((out[cu[-1]:] == 7).all()) and bool((lse[cu[-1]:] == 7).all())
    _check(out.cpu(), lse.cpu(), _reference(q, k, v, table, cu, ctx), rows=torch.arange(cu[-1]))
    fresh = ops.paged_attention_mx4(*args)
    assert torch.equal(fresh[:cu[-1]], out[:cu[-1]])
    small = ops.paged_attention_mx4(*args, workspace=room[:256])
    assert torch.equal(small[:cu[-1]], out[:cu[-1]])
    assert bool((ops.paged_attention_mx4(*args[:4], _i32([0, 0, 0, 0], dev), *args[5:], out=torch.full_like(out, 5.0)) == 5).all())


def _step(gen, lens, heads, kv, dim, rot, axes, dtype, spare=2):
    cu = [0] + np.cumsum([n for n, _ in lens]).tolist()
    T = cu[-1] + spare
    q, k, v = (_normal(gen, T, h, dim, dtype=dtype) for h in (heads, kv, kv))
    positions = torch.randint(0, 600, (axes, T), generator=gen, dtype=torch.int32)
    angle = torch.rand(600, rot // 2, generator=gen, dtype=torch.float64) * 6.28
    rope = torch.stack([angle.cos(), angle.sin()], -1).reshape(600, rot).float()
    return q, k, v, positions, rope, [i % axes for i in range(rot // 2)]


@pytest.mark.parametrize("lens", [[(1, 1)], [(1, 17), (1, 64), (3, 2), (0, 9), (1, 33)], [(130, 200), (67, 67)]], ids=str)
@pytest.mark.parametrize("heads,kv,dim,rot,pairing,norm", [(8, 2, 256, 64, "halves", True), (4, 4, 128, 128, "adjacent", False),
                                                           (12, 3, 64, 32, "halves", False), (7, 1, 64, 64, "adjacent", True),
                                                           (16, 5, 128, 96, "halves", True), (2, 9, 256, 256, "halves", False)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_append(dev, dtype, heads, kv, dim, rot, pairing, norm, lens):
    from spock_amd import ops
    print(f"[mx4 append {dtype} {heads}/{kv}x{dim} rot {rot} {pairing} norm {norm} {lens}]", flush=True)
    t = DT[dtype]
    gen = torch.Generator().manual_seed(dim + rot + len(lens))
    page = [16, 20, 1, 64][(heads + len(lens)) % 4]
    cu, ctx, table, pages = _tables(lens, page, heads)
    q, k, v, positions, rope, axis = _step(gen, lens, heads, kv, dim, rot, 3, t)
    k, v = (x * torch.exp(torch.randn(x.shape[0], x.shape[1], 1, generator=gen)).to(t) for x in (k, v))
    qw, kw = ((torch.randn(dim, generator=gen) * 0.2).to(t) for _ in range(2)) if norm else (None, None)
    if len(lens) > 2:
        table[2, 0] = pages  # a token without a page
    pools = [_pool(gen, pages, page, kv, dim) for _ in range(2)]
    zero = torch.zeros(pages, page, kv, dim, dtype=torch.float64)
    _, wk, wv = R.mrope_append(q, k, v, positions, rope, axis, zero + math.nan, zero + math.nan, table, cu, ctx, qw, kw, pairing=pairing)
    order = list(ORDERS)[(heads + len(lens)) % 3]
    mine = [_on(dev, m, order) for m in pools]
    on = lambda x: None if x is None else x.to(dev)  # noqa: E731
    out = torch.full((q.shape[0], heads, dim), 9.0, dtype=t, device=dev)
    got = ops.mrope_append_mx4(on(q), on(k), on(v), on(positions), on(rope), axis, *mine, on(table), _i32(cu, dev), _i32(ctx, dev),
                               q_norm_weight=on(qw), k_norm_weight=on(kw), pairing=pairing, out=out)
    assert bool((got[cu[-1]:] == 9).all())
    plain = [torch.zeros(pages, page, kv, dim, dtype=t, device=dev) for _ in range(2)]
    want = ops.mrope_append(on(q), on(k), on(v), on(positions), on(rope), axis, *plain, on(table), _i32(cu, dev), _i32(ctx, dev),
                            q_norm_weight=on(qw), k_norm_weight=on(kw), pairing=pairing)
    assert torch.equal(got[:cu[-1]], want[:cu[-1]])
    for have, held, rows in zip(mine, pools, (wk, wv)):
        codes, scales = M.quantize(torch.nan_to_num(rows), M.MOST[t])
        written = ~torch.isnan(rows).any(-1)  # [pages][page][kv]
        codes = torch.where(written[..., None], codes, held[0])
        scales = torch.where(written[..., None], scales, held[1])
        assert torch.equal(have.scales.cpu(), scales)
        # -0 and 0 are one value
        assert torch.equal(M.values(have.codes.cpu(), scales), M.values(codes, scales))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_append_not_numbers(dev, dtype):
    """Infinities and NaN in keys and values make their blocks no numbers (a rotated key: both of the pair's), and no others;
    what a norm's weight takes past the type is cut."""
    from spock_amd import ops
    t = DT[dtype]
    gen = torch.Generator().manual_seed(4)
    lens = [(6, 6)]
    cu, ctx, table, pages = _tables(lens, 16, 4)
    q, k, v, positions, rope, axis = _step(gen, lens, 4, 2, 128, 64, 1, t, spare=0)
    kw = torch.zeros(128).to(t)
    kw[100] = 60000.0 if dtype == "f16" else 1e38
    k[0, 0, 3] = math.inf      # rotates with 35: blocks 0 and 1
    k[1, 1, 70] = math.nan     # does not rotate: block 2
    v[2, 0, 127] = -math.inf
    v[3, 1, 0] = math.nan
    mine = ops.mx4_cache(pages, 16, 2, 128, dev)
    ops.mrope_append_mx4(q.to(dev), k.to(dev), v.to(dev), positions.to(dev), rope.to(dev), axis, *mine, table.to(dev), _i32(cu, dev),
                         _i32(ctx, dev))
    pg = int(table[0, 0])
    ks, vs = mine[0].scales.cpu()[pg], mine[1].scales.cpu()[pg]
    none = torch.zeros(16, 2, 4, dtype=torch.bool)
    none[0, 0, :2] = none[1, 1, 2] = True
    assert torch.equal(ks == 255, none)
    none = torch.zeros(16, 2, 4, dtype=torch.bool)
    none[2, 0, 3] = none[3, 1, 0] = True
    assert torch.equal(vs == 255, none)
    assert not mine[0].codes.cpu()[pg, 0, 0, :32].any() and not mine[1].codes.cpu()[pg, 2, 0, 48:].any()
    ops.mrope_append_mx4(q.to(dev), k.to(dev).nan_to_num(1, 1, 1) * 8, v.to(dev), positions.to(dev), rope.to(dev), axis, *mine, table.to(dev),
                         _i32(cu, dev), _i32(ctx, dev), k_norm_weight=kw.to(dev))
    assert int(mine[0].scales.cpu()[pg][:6].max()) <= M.MOST[t] + 127
    assert bool(torch.isfinite(ops.mx4_dequantize(ops.Mx4(*(x.transpose(1, 2).contiguous() for x in mine[0])), t)).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_append_past_the_type(dev, dtype):
    """Keys that a norm's weight takes past what the type's scales hold, in bf16 also past fp32: the largest code of the largest
    scale, with their signs, and the block's others against that scale."""
    from spock_amd import ops
    t, gen = DT[dtype], torch.Generator().manual_seed(6)
    cu, ctx, table, pages = _tables([(9, 9)], 16, 6)
    q, k, v, positions, rope, axis = _step(gen, [(9, 9)], 4, 2, 128, 64, 1, t, spare=0)
    kw = torch.zeros(128).to(t)
    kw[[3, 100]] = 60000.0 if dtype == "f16" else 3.2e38  # one that rotates with 35, and one that does not
    k[:, :, 100] = torch.where(torch.arange(18).view(9, 2) % 3 == 0, -6.0, 5.0).to(t)
    k[5, 1, 100] = 0.6  # at the type's end, not past it
    zero = torch.full((pages, 16, 2, 128), math.nan, dtype=torch.float64)
    rows = R.mrope_append(q, k, v, positions, rope, axis, zero, zero, table, cu, ctx, None, kw)[1][int(table[0, 0]), :9]
    most = 6 * 2.0 ** M.MOST[t]
    assert float(rows.abs().max()) > (2 * most if dtype == "f16" else 2.0 ** 129) and bool((rows[:, :, 96:].abs() > most).any(-1).any())
    codes, scales = M.quantize(rows, M.MOST[t])
    assert int(scales.max()) == M.MOST[t] + 127
    mine = ops.mx4_cache(pages, 16, 2, 128, dev)
    ops.mrope_append_mx4(q.to(dev), k.to(dev), v.to(dev), positions.to(dev), rope.to(dev), axis, *mine, table.to(dev), _i32(cu, dev),
                         _i32(ctx, dev), k_norm_weight=kw.to(dev))
    have = [x.cpu()[int(table[0, 0]), :9] for x in mine[0]]
    assert torch.equal(have[1], scales)
    assert torch.equal(M.values(*have), M.values(codes, scales))
    cut = M.values(codes, scales).abs() == most
    assert bool(cut[:, :, 100].sum() >= 17) and torch.equal(M.values(*have)[cut].sign(), rows[cut].sign())


def test_python_refusals(dev):
    from spock_amd import ops
    from spock_amd._lib import SpockError
    k, v = ops.mx4_cache(4, 16, 2, 64, dev)
    assert k.codes.shape == (4, 16, 2, 32) and v.scales.shape == (4, 16, 2, 2)
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device=dev)
    table, cu, ctx = _i32([[0, 1]], dev), _i32([0, 1], dev), _i32([5], dev)
    assert ops.paged_attention_mx4(q, k, v, table, cu, ctx, 1, 5).shape == q.shape
    wrong = ops.mx4_cache(4, 16, 2, 128, dev)[0]
    flat = ops.Mx4(v.codes.contiguous(), v.scales)
    for a in ((q, k.codes, v.codes), (q, k, wrong), (q, wrong, wrong), (q.float(), k, v), (q, k, flat), (q[0], k, v),
              (q, ops.Mx4(k.codes, k.codes), v), (q, k, ops.Mx4(v.codes.cpu(), v.scales)), (q, ops.Mx4(k.codes.view(torch.int8), k.scales), v)):
        with pytest.raises(SpockError):
            ops.paged_attention_mx4(*a, table, cu, ctx, 1, 5)
    with pytest.raises(SpockError):
        ops.paged_attention_mx4(q, k, v, table.long(), cu, ctx, 1, 5)


def test_a_serving_step_in_four_bits(dev):
    """Projections with weights in 4 bits, rotation and store, attention and the output projection into the residual
    stream: as they are used, in one graph, replayed as the sequences grow; every replay is the eager result, and the
    first is the definition's."""
    from spock_amd import ops
    t, dim, heads, kv, hidden, page = torch.bfloat16, 64, 4, 2, 256, 16
    gen = torch.Generator().manual_seed(12)
    lens = [(1, 40), (3, 70), (1, 1)]
    cu, ctx, table, pages = _tables([(n, c + 16) for n, c in lens], page, 12)
    ctx = [c for _, c in lens]
    T = cu[-1]
    wqkv = M.quantize(torch.randn((heads + 2 * kv) * dim, hidden, generator=gen) * 0.06)
    wo = M.quantize(torch.randn(hidden, heads * dim, generator=gen) * 0.06)
    pools = [_pool(gen, pages, page, kv, dim, spread=0.0) for _ in range(2)]
    _, _, _, positions, rope, axis = _step(gen, lens, heads, kv, dim, 32, 1, t, spare=0)
    x = torch.randn(T, hidden, generator=gen).to(t)
    qkv4, o4 = (ops.Mx4(*(m.to(dev) for m in w)) for w in (wqkv, wo))
    xd, posd, roped, tabled, cud, ctxd = x.to(dev), positions.to(dev), rope.to(dev), table.to(dev), _i32(cu, dev), _i32(ctx, dev)
    space = torch.empty(ops.paged_attention_mx4_workspace_bytes(T, heads, kv, dim, page, table.shape[1], 3, 3, 400), dtype=torch.uint8, device=dev)

    def step(k4, v4, workspace=None):
        rows = ops.mx4_matmul(xd, qkv4).view(T, heads + 2 * kv, dim)
        q, k, v = rows.split([heads, kv, kv], 1)
        q = ops.mrope_append_mx4(q, k, v, posd, roped, axis, k4, v4, tabled, cud, ctxd)
        out = ops.paged_attention_mx4(q, k4, v4, tabled, cud, ctxd, 3, 400, workspace=workspace)
        return q, ops.mx4_matmul(out.view(T, heads * dim), o4, residual=xd)

    eager, graphed = [_on(dev, m) for m in pools], [_on(dev, m) for m in pools]
    rows = ops.mx4_matmul(xd, qkv4).cpu().view(T, heads + 2 * kv, dim)
    q, y = step(*eager)
    # the definition, from this step's own projections and queries
    k64, v64 = (M.cached(*m, t) for m in pools)
    _, wk, wv = R.mrope_append(rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:], positions, rope, axis,
                               torch.full_like(k64, math.nan), torch.full_like(v64, math.nan), table, cu, ctx)
    for m, w, held in zip(eager, (wk, wv), (k64, v64)):
        new = ~torch.isnan(w)
        held[new] = M.values(*M.quantize(torch.nan_to_num(w)))[new]
        assert torch.equal(M.cached(m.codes.cpu(), m.scales.cpu(), t), held)
    want, _, bound = R.attention(q.cpu(), k64, v64, table, cu, ctx)
    o = M.values(*wo)
    flat, fb = want.reshape(T, -1), bound.reshape(T, -1)
    exact = flat @ o.T + x.double()
    size = flat.abs() @ o.abs().T + x.double().abs()
    err = (y.cpu().double() - exact).abs()
    assert bool((err <= fb @ o.abs().T + 2.0 ** -8 * exact.abs() * 1.01 + 300 * 2.0 ** -24 * size).all())
    for a, b in zip(graphed, eager):  # the same start for the replays
        for u, w in zip(a, b):
            u.copy_(w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*graphed, workspace=space)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*graphed, workspace=space)
    for k in range(4):
        ctxd.add_(torch.tensor([1, 3, 1], dtype=torch.int32, device=dev))
        posd.add_(1)
        xd.copy_(torch.randn(T, hidden, generator=gen).to(t))
        want = [w.clone() for w in step(*eager)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)
        for a, b in zip(graphed, eager):
            for u, w in zip(a, b):
                assert torch.equal(u, w)
