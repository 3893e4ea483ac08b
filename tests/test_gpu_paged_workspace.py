"""GPU runs of the paged operators on one workspace that was sized for the
largest call and holds anything: every smaller call is as with one of its own,
and nothing behind the size is written."""
import numpy as np
import pytest
import torch

from test_gpu_paged import DT, _i32, _normal, _tables

pytestmark = pytest.mark.gpu

GUARD = 4096


def _kept(need, dev):
    """A workspace of NaN with a guard behind it."""
    return torch.full((need + GUARD,), 0xFF, dtype=torch.uint8, device=dev)


@pytest.mark.parametrize("dtype,heads,kv,dim", [("f16", 8, 2, 256), ("bf16", 12, 3, 64)])
def test_attention_on_the_largest_calls_workspace(dev, dtype, heads, kv, dim):
    from spock_amd import ops
    gen = torch.Generator().manual_seed(dim)
    page, cols, most_c = 16, 320, 5000
    need = ops.paged_attention_workspace_bytes(600, heads, kv, dim, page, cols, 8, 500, most_c)
    ws = _kept(need, dev)
    for lens in ([(1, 5000)], [(9, 4900)], [(33, 2000)], [(500, 5000)], [(17, 300), (1, 4000)], [(1, 700 + 500 * i) for i in range(8)],
                 [(100, 900), (200, 5000), (3, 4000), (1, 1)]):
        print(f"[kept workspace {dtype} {heads}/{kv}x{dim} {lens}]", flush=True)
        cu, ctx, table, pages = _tables(lens, page, dim)
        kc, vc = (_normal(gen, pages, page, kv, dim, dtype=DT[dtype]).to(dev) for _ in range(2))
        q = _normal(gen, cu[-1], heads, dim, dtype=DT[dtype]).to(dev)
        args = (q, kc, vc, table.to(dev), _i32(cu, dev), _i32(ctx, dev), max(n for n, _ in lens), max(ctx))
        want = ops.paged_attention(*args, return_lse=True)
        have = ops.paged_attention(*args, return_lse=True, workspace=ws[:need])
        torch.cuda.synchronize()
        assert torch.equal(want[0], have[0]) and torch.equal(want[1], have[1])
        assert bool((ws[need:] == 0xFF).all())
    assert bool((ws[:need] != 0xFF).any())


def test_a_call_takes_no_more_than_it_needs(dev):
    """Without a workspace of the caller's: a prompt whose tiles fill the chip takes none, not what smaller calls would."""
    from spock_amd import ops
    gen = torch.Generator().manual_seed(2)
    cu, ctx, table, pages = _tables([(4096, 4096)], 64, 2)
    kc, vc = (_normal(gen, pages, 64, 4, 64, dtype=torch.float16).to(dev) for _ in range(2))
    q = _normal(gen, 4096, 64, 64, dtype=torch.float16).to(dev)
    out = torch.empty_like(q)
    args = (q, kc, vc, table.to(dev), _i32(cu, dev), _i32(ctx, dev), 4096, 4096)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.paged_attention(*args, out=out)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() == before
    assert ops.paged_attention_workspace_bytes(4096, 64, 4, 64, 64, table.shape[1], 1, 4096, 4096) > 2 ** 26


def test_verification_on_the_largest_calls_workspace(dev):
    from spock_amd import ops
    from test_gpu_verify import _call, _case, _check, _inputs, _want
    vocab = 9001
    need = ops.verify_workspace_bytes(vocab, 40, 200)
    ws = _kept(need, dev)
    for v, rows in ((9001, [5] * 40), (9001, [5] * 8), (9001, [1]), (9000, [9, 1, 3]), (70, [2] * 40), (4097, [7] * 20)):
        print(f"[kept workspace verify {v} x {len(rows)}]", flush=True)
        c = _case(v + len(rows), v, rows, "f16", temps=(1.0, 0.0, 0.7))
        got = _call(_inputs(c, dev), workspace=ws[:need])
        torch.cuda.synchronize()
        _check(got, _want(c))
        assert bool((ws[need:] == 0xFF).all())


def test_workspaces_that_are_no_buffer_are_refused(dev):
    """Views with gaps or repeats, whose bytes in a row are not their own, and other devices."""
    from spock_amd import _lib, ops
    from test_gpu_verify import _call, _case, _inputs
    need = ops.paged_attention_workspace_bytes(1, 8, 2, 64, 16, 320, 1, 1, 5000)
    cu, ctx, table, pages = _tables([(1, 5000)], 16, 0)
    c = torch.zeros(pages, 16, 2, 64, dtype=torch.float16, device=dev)
    q = torch.zeros(1, 8, 64, dtype=torch.float16, device=dev)
    args = (q, c, c, table.to(dev), _i32(cu, dev), _i32(ctx, dev), 1, 5000)
    v = _inputs(_case(1, 64, [2, 2], "f16"), dev)
    for size, call in ((need, lambda ws: ops.paged_attention(*args, workspace=ws)),
                       (ops.verify_workspace_bytes(64, 2, 4), lambda ws: _call(v, workspace=ws))):
        call(torch.empty(size, dtype=torch.uint8, device=dev))
        for ws in (torch.empty(2 * size, dtype=torch.uint8, device=dev)[::2], torch.empty(1, dtype=torch.uint8, device=dev).expand(size),
                   torch.empty(size, dtype=torch.uint8)):
            with pytest.raises(_lib.SpockError, match="workspace"):
                call(ws)
    torch.cuda.synchronize()
