"""GPU runs of the paged operators on views with dimensions of one, whose
strides no access multiplies: one token inside an odd row, one KV head of an
odd stride, one page."""
import pytest
import torch

import paged_ref as R
from test_gpu_paged import _check, _i32, _normal

pytestmark = pytest.mark.gpu


def _odd(t, dims, dev):
    """t on the device with odd strides in `dims`, all of size one."""
    t = t.to(dev)
    strides = [(1001 + 2 * i if i in dims else n) for i, n in enumerate(t.stride())]
    return t.as_strided(t.shape, strides, t.storage_offset())


@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 128), (4, 1, 64), (8, 2, 256)])
@pytest.mark.parametrize("n,pages,page", [(1, 5, 16), (3, 1, 64), (1, 1, 64), (2, 60, 1)])
def test_strides_of_single_dimensions_are_not_read(dev, heads, kv, dim, n, pages, page):
    from spock_amd import ops
    print(f"[single dimensions {heads}/{kv}x{dim} {n} tokens, {pages} pages of {page}]", flush=True)
    gen = torch.Generator().manual_seed(dim + n)
    kc, vc = (_normal(gen, pages, page, kv, dim, dtype=torch.float16) for _ in range(2))
    q, k, v = (_normal(gen, n, h, dim, dtype=torch.float16) for h in (heads, kv, kv))
    table = torch.randperm(pages, generator=gen).to(torch.int32)[None]
    cu, ctx = [0, n], [min(50, pages * page)]
    rows = lambda t, h: _odd(t, [i for i, s in enumerate((n, h)) if s == 1], dev)
    shape = (pages, page, kv)
    one = [i for i, s in enumerate(shape) if s == 1]
    dk, dv = _odd(kc, one, dev), vc.to(dev)             # K and V differ in the strides that are not read
    rope = torch.tensor([[0.6, 0.8] * 16], device=dev)
    pos = torch.zeros(1, n, dtype=torch.int32)
    want = R.mrope_append(q, k, v, pos, rope.cpu(), [0] * 16, kc, vc, table, cu, ctx)
    out = torch.empty(n, heads, dim, dtype=torch.float16, device=dev)
    got = ops.mrope_append(rows(q, heads), rows(k, kv), rows(v, kv), pos.to(dev), rope, [0] * 16, dk, dv, table.to(dev), _i32(cu, dev),
                           _i32(ctx, dev), out=_odd(out, [0] if n == 1 else [], dev))
    torch.cuda.synchronize()
    # two products and a sum in fp32, one rounding
    assert bool(((got.cpu().double() - want[0]).abs() <= 2.0 ** -11 * want[0].abs() + 2.0 ** -20).all())
    assert torch.equal(dv.cpu().double(), want[2])
    ref = R.attention(q, dk.cpu().contiguous(), dv.cpu(), table, cu, ctx)
    o, lse = ops.paged_attention(rows(q, heads), dk, dv, table.to(dev), _i32(cu, dev), _i32(ctx, dev), n, ctx[0], return_lse=True)
    torch.cuda.synchronize()
    _check(o.cpu(), lse.cpu(), ref)
