"""Sizes and bounds of 2^31 and more, which the library's 32-bit fields would take without a word as other ones: sizes are refused
before anything is called, bounds are the largest.  The tensors are views that repeat a few bytes; nothing of such a size is allocated, and no GPU is needed."""
import ctypes as C

import pytest
import torch

BIG = 2 ** 32 + 5  # 5 in 32 bits


@pytest.fixture
def ops(monkeypatch):
    from spock_amd import ops
    monkeypatch.setattr(ops, "_device", lambda what, t: t.get_device())  # CPU tensors pass for one device's
    monkeypatch.setattr(ops, "_call", lambda *a: pytest.fail("called"))
    monkeypatch.setattr(ops, "_launch", lambda *a: pytest.fail("called"))
    return ops


def _refused(call, text):
    from spock_amd._lib import SpockError
    with pytest.raises(SpockError, match=text):
        call()


def _wide(rows, n, dtype):
    return torch.zeros(1, dtype=dtype).expand(rows, n)


def _four(ops, rows, n):
    return ops.Mx4(torch.zeros(n // 2, dtype=torch.uint8).expand(rows, -1), torch.zeros(n // 32, dtype=torch.uint8).expand(rows, -1))


@pytest.mark.parametrize("rows,out", [(BIG, 1), (1, BIG), (2 ** 31, 1)])
@pytest.mark.parametrize("four", [False, True])
def test_matmul(ops, four, rows, out):
    x = _four(ops, rows, 32) if four else torch.zeros(32, dtype=torch.bfloat16).expand(rows, 32)
    _refused(lambda: ops.mx4_matmul(x, _four(ops, out, 32), out=_wide(rows, out, torch.bfloat16)), "rows|out")


def test_rows_of_many_values(ops):
    n = 2 ** 32 + 32
    codes, scales = torch.zeros(1, dtype=torch.uint8).expand(n // 2), torch.zeros(1, dtype=torch.uint8).expand(n // 32)
    contiguous = pytest.MonkeyPatch()
    contiguous.setattr(ops, "_row_stride", lambda what, name, t: t.shape[-1])
    try:
        _refused(lambda: ops.mx4_quantize(torch.zeros(1).expand(n), out=ops.Mx4(codes, scales)), "row")
        _refused(lambda: ops.mx4_dequantize(ops.Mx4(codes, scales), out=torch.zeros(1).expand(n)), "row")
    finally:
        contiguous.undo()


def _step(ops, tokens=1, heads=2, pages=1, max_pages=1):
    q = torch.zeros(64, dtype=torch.float16).expand(tokens, heads, 64)
    cache = [torch.zeros(64, dtype=torch.float16).expand(pages, 16, 2, 64) for _ in range(2)]
    four = [ops.Mx4(torch.zeros(32, dtype=torch.uint8).expand(pages, 16, 2, 32), torch.zeros(2, dtype=torch.uint8).expand(pages, 16, 2, 2))
            for _ in range(2)]
    table = torch.zeros(1, max_pages, dtype=torch.int32) if max_pages < 100 else torch.zeros(1, 1, dtype=torch.int32).as_strided((1, max_pages), (1, 1))
    return q, cache, four, (table, torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("name", ["max_query_len", "max_context_len", "window"])
@pytest.mark.parametrize("value,held", [(BIG, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 40, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 32 + 1, -1)])
def test_attention_bounds(ops, monkeypatch, four, name, value, held):
    """A bound bounds no less when it is the largest that there is, and a window no less wide; a negative one stays refused."""
    q, cache, mx4, rest = _step(ops)
    bounds = dict(max_query_len=1, max_context_len=16, window=0)
    bounds[name] = value
    fn, pools = (ops.paged_attention_mx4, mx4) if four else (ops.paged_attention, cache)
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda dev, what, fn, a, s: seen.append(a._obj))
    monkeypatch.setattr(ops, "_call", lambda fn, a, dev, what: seen.append(a))
    fn(q, *pools, *rest, **bounds)
    assert getattr(seen[0], name) == held
    if held < 0:
        from spock_amd import _lib
        assert _lib.lib().spk_paged_attention_workspace_size(C.byref(seen[0])) == 0 and b"window" in _lib.lib().spk_last_error()


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("sizes", [dict(tokens=BIG), dict(heads=BIG), dict(pages=BIG)], ids=str)
def test_steps(ops, four, sizes):
    q, cache, mx4, rest = _step(ops, **sizes)
    attend, append, pools = (ops.paged_attention_mx4, ops.mrope_append_mx4, mx4) if four else (ops.paged_attention, ops.mrope_append, cache)
    _refused(lambda: attend(q, *pools, *rest, 1, 16, out=q), next(iter(sizes)))
    kv = q[:, :1].expand(-1, 2, -1)
    positions = torch.zeros(1, 1, dtype=torch.int32).expand(1, q.shape[0])
    _refused(lambda: append(q, kv, kv, positions, torch.zeros(4, 32), [0] * 16, *pools, *rest, out=q), next(iter(sizes)))


@pytest.mark.parametrize("at", range(7))
def test_workspaces(ops, at):
    sizes = [4, 8, 2, 64, 16, 10, 2, 4, 160, 0]
    sizes[at] = BIG
    for fn in (ops.paged_attention_workspace_bytes, ops.paged_attention_mx4_workspace_bytes):
        _refused(lambda: fn(*sizes), "below 2\\^31")
    sizes = [4, 8, 2, 64, 16, 10, 2, 4, 160, 0]
    for at in (7, 8):
        for fn in (ops.paged_attention_workspace_bytes, ops.paged_attention_mx4_workspace_bytes):
            assert fn(*sizes[:at], BIG, *sizes[at + 1:]) == fn(*sizes[:at], 2 ** 31 - 1, *sizes[at + 1:]) > 0
