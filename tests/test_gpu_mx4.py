"""GPU parity of quantisation to 4 bits and of the products with such weights against the definitions in 64 bits
(mx4_ref.py).

Bars: codes, scales and values are exact.  A product is one rounding of its result (2^-11 fp16, 2^-8 bf16,
relative), after in_dim + 4 fp32 roundings at most (products of the operands are exact, each sum is rounded once and
the waves' sums and the residual add four more), each 2^-24 of sum |x| |w| (+ |residual|)."""
import functools
import math

import pytest
import torch

import mx4_ref as M

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _same(have, want):
    return bool(((have == want) | (torch.isnan(have) & torch.isnan(want))).all())


def _rows(gen, rows, cols, dtype, spread=3.0):
    x = torch.randn(rows, cols, generator=gen) * torch.exp(spread * torch.randn(rows, cols // 32, generator=gen)).repeat_interleave(32, -1)
    return x.to(dtype)


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (16, 1024), (257, 96), (5, 3584), (1031, 160)])
@pytest.mark.parametrize("dtype", list(DT))
def test_quantize(dev, dtype, rows, cols):
    from spock_amd import ops
    print(f"[mx4 quantize {dtype} {rows}x{cols}]", flush=True)
    x = _rows(torch.Generator().manual_seed(rows), rows, cols, DT[dtype])
    m = ops.mx4_quantize(x.to(dev))
    codes, scales = M.quantize(x)
    assert torch.equal(m.scales.cpu(), scales) and torch.equal(m.codes.cpu(), codes)
    for to in DT.values():
        assert _same(ops.mx4_dequantize(m, to).cpu().double(), M.values(codes, scales, to))


@pytest.mark.parametrize("dtype", list(DT))
def test_quantize_edges(dev, dtype):
    """Ties, the last quarter of a binade, subnormal and the largest magnitudes, signed zeros, infinities and NaN."""
    from spock_amd import ops
    t = DT[dtype]
    big, tiny = torch.finfo(t).max, torch.finfo(t).smallest_normal
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, 0.0, -0.0, 0.26, 0.24, 4.99, 5.01])
    rows = [torch.cat([s * ties * 2.0 ** e, -s * ties * 2.0 ** e]) for e in (-3, 0, 5) for s in (1, -1)]
    rows += [torch.full((32,), big), torch.full((32,), -big), torch.full((32,), tiny), torch.full((32,), tiny / 4), torch.zeros(32),
             torch.cat([torch.full((1,), tiny / 4), torch.zeros(31)]), torch.linspace(-big / 2, big / 2, 32)]
    for v in (math.inf, -math.inf, math.nan):
        for at in (0, 13, 31):
            r = torch.linspace(-3, 3, 32)
            r[at] = v
            rows.append(r)
    x = torch.stack(rows).to(t)
    x = torch.cat([x, x.flip(0)], -1)  # a block that is no number beside one that is
    m = ops.mx4_quantize(x.to(dev))
    codes, scales = M.quantize(x)
    assert torch.equal(m.scales.cpu(), scales)
    assert torch.equal(m.codes.cpu(), codes)


def test_dequantize_every_code_and_scale(dev):
    from spock_amd import ops
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)           # 16 blocks of all pairs
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    m = ops.Mx4(codes.to(dev), scales.to(dev))
    for t in DT.values():
        assert _same(ops.mx4_dequantize(m, t).cpu().double(), M.values(codes, scales, t))


def test_strides_shapes_and_streams(dev):
    """Rows apart in memory, several leading dimensions, none, no rows, given outputs, another stream."""
    from spock_amd import ops
    from spock_amd._lib import SpockError
    gen = torch.Generator().manual_seed(5)
    wide = _rows(gen, 20, 256, torch.float16).to(dev)
    x = wide[:, 32:160]
    codes = torch.full((20, 96), 0x55, dtype=torch.uint8, device=dev)
    scales = torch.full((20, 9), 0x55, dtype=torch.uint8, device=dev)
    m = ops.mx4_quantize(x, out=ops.Mx4(codes[:, 16:80], scales[:, 3:7]))
    rc, rs = M.quantize(x.cpu())
    assert torch.equal(m.codes.cpu(), rc) and torch.equal(m.scales.cpu(), rs)
    assert bool((codes[:, :16] == 0x55).all()) and bool((codes[:, 80:] == 0x55).all())
    assert bool((scales[:, :3] == 0x55).all()) and bool((scales[:, 7:] == 0x55).all())
    out = torch.full((20, 192), -1.0, dtype=torch.bfloat16, device=dev)
    ops.mx4_dequantize(m, out=out[:, 8:136])
    assert torch.equal(out[:, 8:136].cpu().double(), M.values(rc, rs, torch.bfloat16))
    assert bool((out[:, :8] == -1).all()) and bool((out[:, 136:] == -1).all())
    y = _rows(gen, 24, 64, torch.float32)
    n = ops.mx4_quantize(y.view(2, 3, 4, 64).to(dev))
    assert n.codes.shape == (2, 3, 4, 32) and torch.equal(n.codes.cpu().view(24, 32), M.quantize(y)[0])
    assert ops.mx4_dequantize(n).shape == (2, 3, 4, 64)
    one = ops.mx4_quantize(y[0].to(dev))
    assert one.codes.shape == (32,) and torch.equal(one.codes.cpu(), M.quantize(y[:1])[0][0])
    none = ops.mx4_quantize(y[:0].to(dev))
    assert none.codes.shape == (0, 32) and ops.mx4_dequantize(none).shape == (0, 64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.mx4_quantize(y.to(dev))
    s.synchronize()
    assert torch.equal(other.codes.cpu(), M.quantize(y)[0])
    for bad in (lambda: ops.mx4_quantize(wide[:, :100]), lambda: ops.mx4_quantize(wide.double()), lambda: ops.mx4_quantize(wide.T),
                lambda: ops.mx4_quantize(wide[:, 1:129]), lambda: ops.mx4_quantize(x, out=ops.Mx4(codes, scales)),
                lambda: ops.mx4_dequantize(ops.Mx4(codes[:, :64], scales[:, :3])), lambda: ops.mx4_dequantize(m, torch.float64),
                lambda: ops.mx4_dequantize(ops.Mx4(codes.cpu(), scales)), lambda: ops.mx4_dequantize(m, out=out)):
        with pytest.raises(SpockError):
            bad()


@pytest.mark.parametrize("shape", [(5, 16, 2, 64), (3, 7, 1, 128), (1, 20, 3, 32), (4, 1, 1, 256)], ids=str)
def test_pools_as_rows(dev, shape):
    """What mx4_cache makes, whose memory has another order than its dimensions, is quantised into and read back as it is."""
    from spock_amd import ops
    from spock_amd._lib import SpockError
    gen = torch.Generator().manual_seed(shape[1])
    pool, other = ops.mx4_cache(*shape, dev)
    x = _rows(gen, math.prod(shape[:3]), shape[3], torch.bfloat16).view(shape)
    codes, scales = M.quantize(x)
    there = torch.empty(shape[0], shape[2], shape[1], shape[3], dtype=x.dtype, device=dev).transpose(1, 2).copy_(x)
    assert ops.mx4_quantize(there, out=pool) is pool
    fresh = ops.mx4_quantize(there)
    for m in (pool, fresh):
        assert m.codes.shape == codes.shape and torch.equal(m.codes.cpu(), codes) and torch.equal(m.scales.cpu(), scales)
    for t in DT.values():
        have = ops.mx4_dequantize(pool, t)
        assert have.shape == x.shape and torch.equal(have.cpu().double(), M.values(codes, scales, t))
    hold = torch.zeros_like(there)
    assert ops.mx4_dequantize(pool, out=hold) is hold and torch.equal(hold.cpu().double(), M.values(codes, scales, x.dtype))
    some = ops.mx4_dequantize(ops.Mx4(*(t[1:] for t in pool)))
    assert torch.equal(some.cpu().double(), M.values(codes, scales, torch.bfloat16)[1:])
    assert torch.equal(other.codes, torch.zeros_like(other.codes))
    if shape[1] > 1 and shape[2] > 1:  # another order, gaps
        for bad in (lambda: ops.mx4_quantize(x.to(dev), out=pool), lambda: ops.mx4_dequantize(pool, out=x.to(dev)),
                    lambda: ops.mx4_dequantize(ops.Mx4(*(t[:, 1:] for t in pool))),
                    lambda: ops.mx4_dequantize(ops.Mx4(pool.codes, pool.scales.contiguous()))):
            with pytest.raises(SpockError):
                bad()


def _product(x, w, residual, dtype, four):
    """(result, bound) in 64 bits; x, w as values."""
    y = x @ w.T
    size = x.abs() @ w.abs().T
    if residual is not None:
        y, size = y + residual.double(), size + residual.double().abs()
    return y, HALF[dtype] * y.abs() * (1 + HALF[dtype]) + (x.shape[-1] + 4) * 2.0 ** -24 * size * (1 + HALF[dtype])


def _check(have, want, bound, floor=0.0):
    have = have.cpu().double()
    ok = ((have - want).abs() <= bound + floor) | (torch.isnan(have) & torch.isnan(want)) | (have == want)
    assert bool(ok.all()), (float(((have - want).abs() / (bound + 1e-30))[~ok].max()), torch.nonzero(~ok)[:4].tolist())


# one row and a few, the ends of the row groups, more than one group of rows and of columns, depths that end inside a
# step, columns that end inside a tile
SHAPES = [(1, 1, 32), (1, 17, 64), (2, 1024, 1024), (7, 33, 96), (16, 48, 4096), (17, 1024, 3584), (33, 200, 160), (64, 64, 128),
          (65, 130, 288), (100, 257, 1024), (129, 512, 512), (300, 1000, 992), (515, 129, 2048), (777, 771, 224)]


@pytest.mark.parametrize("rows,out,depth", SHAPES)
@pytest.mark.parametrize("four", [False, True], ids=["x16", "x4"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_matmul(dev, dtype, four, rows, out, depth):
    from spock_amd import ops
    print(f"[mx4 matmul {dtype} {'x4' if four else 'x16'} {rows}x{out}x{depth}]", flush=True)
    t, gen = DT[dtype], torch.Generator().manual_seed(rows * 7 + out)
    x = _rows(gen, rows, depth, t, spread=0.7)
    w = M.quantize(_rows(gen, out, depth, torch.float32, spread=0.7) * 0.05)
    residual = torch.randn(rows, out, generator=gen).to(t) if rows % 2 else None
    xv, mine = x.double(), x.to(dev)
    if four:
        m = M.quantize(x)
        xv, mine = M.values(*m), ops.Mx4(*(v.to(dev) for v in m))
    got = ops.mx4_matmul(mine, ops.Mx4(*(v.to(dev) for v in w)), residual=None if residual is None else residual.to(dev), dtype=t)
    assert got.dtype == t and got.shape == (rows, out)
    _check(got, *_product(xv, M.values(*w), residual, t, four))


# many rows: tiles of 128 x 128 and of 256 x 256, ends inside a tile, depths that end inside a block of stages
MANY = [(1300, 1030, 96), (1303, 1025, 512), (1290, 1057, 1568), (3601, 3590, 160), (3590, 3603, 1024), (3845, 3329, 544)]


@pytest.mark.parametrize("rows,out,depth", MANY)
@pytest.mark.parametrize("four", [False, True], ids=["x16", "x4"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_matmul_many_rows(dev, dtype, four, rows, out, depth):
    """Rows apart in memory, of scales also by odd numbers of bytes; one block of w is no number, and the
    residual is out where out lies inside a larger tensor."""
    from spock_amd import ops
    print(f"[mx4 matmul {dtype} {'x4' if four else 'x16'} {rows}x{out}x{depth}]", flush=True)
    t, gen = DT[dtype], torch.Generator().manual_seed(rows + depth)
    apart = depth % 512 == 0 and rows % 2 == 1  # scales that are not aligned though their rows are long enough

    def on(m):
        codes, scales = m
        if apart:
            codes, scales = torch.cat([codes, codes[:, :16]], 1).to(dev), torch.cat([scales[:, :1], scales, scales[:, :2]], 1).to(dev)
            return ops.Mx4(codes[:, :depth // 2], scales[:, 1:1 + depth // 32])
        return ops.Mx4(codes.to(dev), scales.to(dev))

    x = _rows(gen, rows, depth, t, spread=0.5)
    w = M.quantize(_rows(gen, out, depth, torch.float32, spread=0.5) * 0.05)
    w[1][out - 2, -1] = 255
    xv, mine = x.double(), torch.cat([x, x[:, :8]], 1).to(dev)[:, :depth]
    if four:
        m = M.quantize(x)
        xv, mine = M.values(*m), on(m)
    hold = torch.full((rows, out + 9), 3.0, dtype=t, device=dev)
    res = torch.randn(rows, out, generator=gen).to(t)
    hold[:, 4:4 + out] = res.to(dev)
    ops.mx4_matmul(mine, on(w), residual=hold[:, 4:4 + out], out=hold[:, 4:4 + out])
    want, bound = _product(xv.to(dev), M.values(*w).to(dev), res.to(dev), t, four)
    _check(hold[:, 4:4 + out], want.cpu(), bound.cpu())
    assert bool(torch.isnan(hold[:, 4 + out - 2]).all()) and not bool(torch.isnan(hold[:, 4:4 + out - 2]).any())
    assert bool((hold[:, :4] == 3).all()) and bool((hold[:, 4 + out:] == 3).all())


# what a program calls for one row and a few, with weights of every size: each form of the kernel for few rows with scales by
# the dword (depths of whole steps of 128) and by the byte
FEW = [(rows, out, depth) for out in (131200, 13000, 6500, 1100) for rows in (1, 4, 16) for depth in (256, 160)] + \
    [(33, 2200, 384), (33, 2200, 96), (40, 6000, 128), (40, 6000, 96), (20, 150, 512)]
# tiles with scales of aligned 16 bytes, in several groups of stages, the last not whole
LONG = [(1302, 1026, 2560), (1302, 1026, 512), (3590, 3603, 2560), (3590, 3603, 512)]


def _form(four, rows, out, depth, aligned=True):
    """Which kernel a product takes, as its rule in csrc/mx4.hip has it."""
    tiles, big = -(-out // 16) * -(-rows // 16), -(-out // 256) * -(-rows // 256)
    if rows <= 16 or tiles < (2200 if four else 5000):
        form = (4, 1) if tiles >= 8192 else (4, 4) if tiles >= 800 else (2, 4) if tiles >= 400 else (1, 4)
        return ("few", 4 if rows <= 4 and not four else 16, *form, 4 if depth % 128 == 0 and aligned else 1)
    return ("tiles", 256 if big >= 200 else 128, 16 if depth % 512 == 0 and aligned else 1)


@functools.lru_cache(maxsize=1)
def _weights(out, depth):
    """Codes of all kinds and scales from 2^-6 to 1, and their values."""
    gen = torch.Generator().manual_seed(out + depth)
    codes = torch.randint(0, 256, (out, depth // 2), generator=gen, dtype=torch.uint8)
    scales = torch.randint(121, 128, (out, depth // 32), generator=gen).to(torch.uint8)
    return codes, scales, M.values(codes, scales)


@pytest.mark.parametrize("rows,out,depth", FEW + LONG)
@pytest.mark.parametrize("four", [False, True], ids=["x16", "x4"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_matmul_forms(dev, dtype, four, rows, out, depth):
    from spock_amd import ops
    print(f"[mx4 matmul form {dtype} {'x4' if four else 'x16'} {rows}x{out}x{depth}]", flush=True)
    t, gen = DT[dtype], torch.Generator().manual_seed(rows)
    codes, scales, wv = _weights(out, depth)
    if four:
        m = torch.randint(0, 256, (rows, depth // 2), generator=gen, dtype=torch.uint8), \
            torch.randint(124, 128, (rows, depth // 32), generator=gen).to(torch.uint8)
        xv, mine = M.values(*m), ops.Mx4(*(v.to(dev) for v in m))
    else:
        x = torch.randn(rows, depth, generator=gen).to(t)
        xv, mine = x.double(), x.to(dev)
    res = torch.randn(rows, out, generator=gen).to(t).to(dev) if rows % 3 else None
    got = ops.mx4_matmul(mine, ops.Mx4(codes.to(dev), scales.to(dev)), residual=res, dtype=t)
    _check(got, *(v.cpu() for v in _product(xv.to(dev), wv.to(dev), res, t, four)))


@pytest.mark.parametrize("rows,out", [(4, 70), (40, 70), (1300, 1030)])
def test_matmul_weights_past_fp16(dev, rows, out):
    """Rows in fp16: a weight enters as mx4_dequantize gives it there, rounded to fp16's steps where its scale is below
    2^-23, infinite where it passes 65504, whatever its scale."""
    from spock_amd import ops
    print(f"[mx4 matmul past fp16 {rows}x{out}]", flush=True)
    gen, depth = torch.Generator().manual_seed(rows), 128
    codes = torch.randint(0, 256, (out, depth // 2), generator=gen, dtype=torch.uint8)
    scales = torch.randint(127 - 27, 127 - 22, (out, depth // 32), generator=gen).to(torch.uint8)
    scales[::3] = torch.randint(127 + 13, 127 + 17, scales[::3].shape, generator=gen).to(torch.uint8)
    codes[::6] &= 0x99  # magnitudes of 0 and 0.5: finite up to scales of 2^16
    x = torch.randn(rows, depth, generator=gen).to(torch.float16)
    x[:, ::2] *= 2.0 ** -9
    x[0, 5] = 0.0  # times an infinity: NaN
    wv = M.values(codes, scales, torch.float16)
    assert bool(torch.isinf(wv).any()) and bool(torch.isfinite(wv[::6]).all()) and bool((M.values(codes, scales)[1::3] != wv[1::3]).any())
    got = ops.mx4_matmul(x.to(dev), ops.Mx4(codes.to(dev), scales.to(dev))).cpu()
    want, bound = _product(x.double(), wv, None, torch.float16, False)
    low, want16 = want.abs() + bound, want.to(torch.float16)
    near = torch.isfinite(want) & (low > 65504)  # next to fp16's end, where the sum's own error decides
    _check(torch.where(near, want16, got), torch.where(near | (want.abs() > 65504), want16.double(), want), bound, floor=2.0 ** -25)
    assert bool((torch.isnan(got) == torch.isnan(want)).all())


@pytest.mark.parametrize("four", [False, True], ids=["x16", "x4"])
@pytest.mark.parametrize("rows", [3, 40, 200])
def test_matmul_strides_and_in_place(dev, rows, four):
    """Operands that are parts of larger ones; out is the residual; what lies around out is left."""
    from spock_amd import ops
    t, gen = torch.bfloat16, torch.Generator().manual_seed(rows)
    x = _rows(gen, rows, 512, t, spread=0.5).to(dev)
    w = M.quantize(_rows(gen, 99, 512, torch.float32, spread=0.5))
    xs, ws = x[:, 64:352], ops.Mx4(w[0].to(dev)[:, 32:176], w[1].to(dev)[:, 2:11])
    wv = M.values(w[0][:, 32:176], w[1][:, 2:11])
    xv = xs.cpu().double()
    if four:
        m = ops.mx4_quantize(x)
        xs = ops.Mx4(m.codes[:, 32:176], m.scales[:, 2:11])
        xv = M.values(xs.codes.cpu(), xs.scales.cpu())
    hold = torch.full((rows, 130), 3.0, dtype=t, device=dev)
    res = torch.randn(rows, 99, generator=gen).to(t)
    hold[:, 7:106] = res.to(dev)
    got = ops.mx4_matmul(xs, ws, residual=hold[:, 7:106], out=hold[:, 7:106])
    assert got.data_ptr() == hold[:, 7:106].data_ptr()
    _check(hold[:, 7:106], *_product(xv, wv, res, t, four))
    assert bool((hold[:, :7] == 3).all()) and bool((hold[:, 106:] == 3).all())


@pytest.mark.parametrize("rows,out", [(5, 1100), (1300, 1100)])
@pytest.mark.parametrize("four", [False, True], ids=["x16", "x4"])
def test_matmul_rows_far_apart(dev, four, rows, out):
    """Rows 4 MB apart, more than 2^32 bytes in all: the same bits as side by side."""
    from spock_amd import ops
    gen, apart, depth = torch.Generator().manual_seed(rows), 2 ** 22, 544

    def far(t):
        size = t.element_size()
        hold = torch.empty(t.shape[0] * apart // size, dtype=t.dtype, device=dev).as_strided(t.shape, (apart // size, 1))
        return hold.copy_(t)

    x = _rows(gen, rows, depth, torch.bfloat16, spread=0.5).to(dev)
    w = ops.mx4_quantize(_rows(gen, out, depth, torch.float32, spread=0.5).to(dev))
    near = ops.mx4_quantize(x) if four else x
    want = ops.mx4_matmul(near, w)
    got = far(torch.zeros_like(want))
    spread = ops.Mx4(*map(far, near)) if four else far(near)
    ops.mx4_matmul(spread, ops.Mx4(*map(far, w)), out=got)
    assert torch.equal(got, want)
    if four:
        assert torch.equal(ops.mx4_dequantize(spread), ops.mx4_dequantize(near))
        again = ops.Mx4(*(far(torch.zeros_like(t)) for t in near))
        ops.mx4_quantize(far(x), out=again)
        assert torch.equal(again.codes, near.codes) and torch.equal(again.scales, near.scales)


@pytest.mark.parametrize("rows", [2, 70, 300])
@pytest.mark.parametrize("four", [False, True], ids=["x16", "x4"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_matmul_not_numbers(dev, dtype, four, rows):
    """An infinity in x, a block of w and of x4 that is no number: only their own rows and columns have it, also where
    the depth ends inside a step."""
    from spock_amd import ops
    t, gen = DT[dtype], torch.Generator().manual_seed(rows)
    depth, out = 160, 70
    x = _rows(gen, rows, depth, t, spread=0.3)
    w = M.quantize(_rows(gen, out, depth, torch.float32, spread=0.3))
    w[1][5, 4] = 255                     # of the last, short step
    w[1][64, 0] = 255
    x[1, 3] = math.inf                   # rows in 4 bits: their block is no number
    xv, mine = x.double(), x.to(dev)
    if four:
        m = M.quantize(x)
        xv, mine = M.values(*m), ops.Mx4(*(v.to(dev) for v in m))
    got = ops.mx4_matmul(mine, ops.Mx4(*(v.to(dev) for v in w)), dtype=t).cpu().double()
    want = xv @ M.values(*w).T
    for r in range(rows):
        for c in range(out):
            if not math.isfinite(float(want[r, c])):
                assert (math.isnan(got[r, c]) and math.isnan(want[r, c])) or got[r, c] == want[r, c], (r, c)
    fine = torch.isfinite(want)
    assert bool(torch.isfinite(got[fine]).all())
    xf, wf = torch.nan_to_num(xv, 0, 0, 0), torch.nan_to_num(M.values(*w), 0, 0, 0)
    y, bound = _product(xf, wf, None, t, four)
    assert bool(((got - y).abs() <= bound)[fine].all())


@pytest.mark.parametrize("four", [False, True], ids=["x16", "x4"])
def test_matmul_scales_of_all_sizes(dev, four):
    """Weights from 2^-20 to 2^12 in fp16, and from 2^-100 to 2^100 in bf16, whose products meet in fp32."""
    from spock_amd import ops
    gen = torch.Generator().manual_seed(3)
    for t, lo, hi in ((torch.float16, -20, 12), (torch.bfloat16, -100, 100)):
        for rows in (4, 150):
            codes = torch.randint(0, 256, (50, 64), generator=gen, dtype=torch.uint8)
            scales = torch.randint(lo + 127, hi + 127, (50, 1), generator=gen).repeat(1, 4).to(torch.uint8)
            x = torch.randn(rows, 128, generator=gen).to(t) * 2.0 ** -6
            xv, mine = x.double(), x.to(dev)
            if four:
                m = M.quantize(x)
                xv, mine = M.values(*m), ops.Mx4(*(v.to(dev) for v in m))
            got = ops.mx4_matmul(mine, ops.Mx4(codes.to(dev), scales.to(dev)), dtype=t)
            # below fp16's smallest normal a result is rounded to 2^-24
            _check(got, *_product(xv, M.values(codes, scales, t), None, t, four), floor=2.0 ** -25 if t is torch.float16 else 0.0)


def test_matmul_refusals(dev):
    from spock_amd import ops
    from spock_amd._lib import SpockError
    x = torch.zeros(4, 64, dtype=torch.float16, device=dev)
    w = ops.mx4_quantize(torch.zeros(8, 64, device=dev))
    wide = ops.mx4_quantize(torch.zeros(8, 96, device=dev))
    ok = ops.mx4_matmul(x, w)
    assert ok.shape == (4, 8) and ops.mx4_matmul(x[:0], w).shape == (0, 8)
    assert ops.mx4_matmul(x.view(2, 2, 64), w).shape == (2, 2, 8) and ops.mx4_matmul(x[0], w).shape == (8,)
    assert ops.mx4_matmul(w, w).dtype == torch.bfloat16 and ops.mx4_matmul(w, w, dtype=torch.float16).dtype == torch.float16
    for bad in (lambda: ops.mx4_matmul(x, wide), lambda: ops.mx4_matmul(x.float(), w), lambda: ops.mx4_matmul(x, w, dtype=torch.bfloat16),
                lambda: ops.mx4_matmul(x, x), lambda: ops.mx4_matmul(x, w, residual=ok.float()), lambda: ops.mx4_matmul(x, w, residual=ok[:2]),
                lambda: ops.mx4_matmul(x, w, out=ok[:2]), lambda: ops.mx4_matmul(w, w, dtype=torch.float32),
                lambda: ops.mx4_matmul(x.T, w), lambda: ops.mx4_matmul(x, ops.Mx4(w.codes[None], w.scales[None]))):
        with pytest.raises(SpockError):
            bad()


def test_products_in_a_graph_and_on_two_streams(dev):
    """Quantisation and products captured once and replayed on new inputs, beside eager calls on another stream."""
    from spock_amd import ops
    gen = torch.Generator().manual_seed(9)
    w = ops.mx4_quantize((torch.randn(304, 512, generator=gen) * 0.05).to(dev))
    w2 = ops.mx4_quantize((torch.randn(512, 320, generator=gen)[:, :320] * 0.05).to(dev))
    x = torch.randn(37, 512, generator=gen).to(torch.bfloat16).to(dev)

    def step(x):
        h = ops.mx4_matmul(x, w)[:, :288]
        return ops.mx4_matmul(ops.mx4_quantize(h), ops.Mx4(w2.codes[:, :144], w2.scales[:, :9]), residual=x)

    step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(x)
    side = torch.cuda.Stream()
    for k in range(4):
        x.copy_(torch.randn(37, 512, generator=gen).to(torch.bfloat16))
        want = step(x).clone()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            again = step(x)
        torch.cuda.synchronize()
        assert torch.equal(held, want) and torch.equal(again, want)
