"""GPU runs of mrope_append with the positions of text on several axes."""
import pytest
import torch

from test_gpu_paged import _i32, _mrope_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[(1, 9)], [(5, 37), (1, 20), (18, 18)]], ids=str)
def test_one_row_expanded_to_all_axes(dev, lens):
    from spock_amd import _lib, ops
    print(f"[mrope expanded positions {lens}]", flush=True)
    q, k, v, pos, rope, kc, vc, table, cu, ctx, (qw, kw) = _mrope_inputs("f16", 8, 2, 128, 64, 3, lens, 16, 7, True)
    row = pos[:1].to(dev)
    axis = [i % 3 for i in range(32)]
    got = []
    for p in (row.expand(3, -1), row.repeat(3, 1), row[0].expand(3, -1)):
        dk, dv = kc.to(dev), vc.to(dev)
        out = ops.mrope_append(q.to(dev), k.to(dev), v.to(dev), p, rope.to(dev), axis, dk, dv, table.to(dev), _i32(cu, dev), _i32(ctx, dev),
                               q_norm_weight=qw.to(dev), k_norm_weight=kw.to(dev))
        torch.cuda.synchronize()
        got.append((out, dk, dv))
    for x in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(x, got[0]))
    with pytest.raises(_lib.SpockError, match="axis"):
        ops.mrope_append(q.to(dev), k.to(dev), v.to(dev), row.expand(3, -1), rope.to(dev), [3] * 32, dk, dv, table.to(dev), _i32(cu, dev), _i32(ctx, dev))
