"""GPU runs of paged_attention over infinities and NaN among the values that a
row sees: softmax . V says what they give, wherever in the context they lie.

An infinity times a weight that rounds to zero (below 2^-30 of the row's largest
in fp16, 2^-125 in bf16) is NaN; scores of these inputs are normal with deviation
1, so no weight comes near that."""
import math

import pytest
import torch

import paged_ref as R
from test_gpu_paged import DT, _attend, _check, _normal, _tables

pytestmark = pytest.mark.gpu


def _put(cache, table, s, pos, what):
    cache[int(table[s][pos // cache.shape[1]]), pos % cache.shape[1]] = what


# one row, the rows of a few drafts, of a chunk; short contexts, and ones that are split into ranges
@pytest.mark.parametrize("n,ctx", [(1, 300), (1, 5000), (9, 300), (9, 5000), (40, 300), (150, 700)])
@pytest.mark.parametrize("dtype,heads,kv,dim", [("f16", 8, 2, 256), ("bf16", 8, 2, 128), ("f16", 12, 3, 64), ("bf16", 8, 2, 256)])
def test_values_that_every_row_sees(dev, dtype, heads, kv, dim, n, ctx):
    print(f"[visible infinities {dtype} {heads}/{kv}x{dim} {n}:{ctx}]", flush=True)
    gen = torch.Generator().manual_seed(dim + n)
    cu, lens, table, pages = _tables([(n, ctx), (1, 200)], 16, dim + n)
    kc, vc = (_normal(gen, pages, 16, kv, dim, dtype=DT[dtype]) for _ in range(2))
    q = _normal(gen, cu[-1], heads, dim, dtype=DT[dtype])
    # an early key's whole row, one element of another, both signs in one dimension, a NaN, one in the middle
    one = torch.full((kv, dim), math.nan)
    one[:] = vc[int(table[0][0]), 5].float()
    one[0] = math.inf
    _put(vc, table, 0, 5, one.to(DT[dtype]))
    for pos, h, d, x in ((17, kv - 1, 3, -math.inf), (40, kv - 1, 9, math.inf), (97, kv - 1, 9, -math.inf), (64, kv - 1, 20, math.nan),
                         (ctx // 2, kv - 1, 31, math.inf)):
        vc[int(table[0][pos // 16]), pos % 16, h, d] = x
    ref = R.attention(q, kc, vc, table, cu, lens)
    out, lse = _attend(dev, q, kc, vc, table, cu, lens)
    want, have = ref[0], out.double()
    assert torch.equal(torch.isnan(want), torch.isnan(have))
    assert torch.equal(want[torch.isinf(want)], have[torch.isinf(want)]) and torch.equal(torch.isinf(want), torch.isinf(have))
    assert bool(torch.isinf(want).any())
    _check(out, lse, ref)
