"""The 4-bit operators without a GPU: the reference itself, and what the entry points refuse before any launch."""
import ctypes as C

import pytest
import torch

import mx4_ref as M
import test_gpu_mx4 as G


def test_the_reference_is_the_format():
    codes = torch.arange(256, dtype=torch.uint8).reshape(16, 16)
    scales = torch.full((16, 1), 127, dtype=torch.uint8)
    v = M.values(codes, scales)
    assert v[0, :4].tolist() == [0.0, 0.0, 0.5, 0.0] and v[15, -1] == -6.0
    assert sorted(set(v.flatten().tolist())) == sorted({s * g for s in (1, -1) for g in M.GRID.tolist()})
    x = torch.zeros(1, 32)
    x[0, :10] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.75, 7.9])
    c, s = M.quantize(x)
    assert s.tolist() == [[127]]
    assert M.values(c, s)[0, :10].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -1.0, 6.0]
    c, s = M.quantize(torch.tensor([[8.0] + [0.0] * 31, [float("nan")] + [1.0] * 31, [0.0] * 32, [2.0 ** -140] * 32]))
    assert s[:, 0].tolist() == [128, 255, 0, 0] and not c[1].any() and not c[2].any()


def _matmul(_lib, **over):
    m = lambda at: _lib.SpkMx4(at, 32, at, 2)  # noqa: E731
    f = dict(dtype=_lib.SPK_F16, rows=3, out_dim=5, in_dim=64, x=256, x_stride=64, x4=m(256), w=m(256), residual=None,
             residual_stride=0, out=512, out_stride=5)
    f.update(over)
    return _lib.SpkMx4MatmulArgs(*[f[n] for n, _ in _lib.SpkMx4MatmulArgs._fields_])


def _four(**over):
    from spock_amd import _lib
    f = dict(codes=256, code_stride=32, scales=256, scale_stride=2)
    f.update(over)
    return _lib.SpkMx4(*[f[n] for n, _ in _lib.SpkMx4._fields_])


BAD = [(lambda: dict(dtype=0), -5), (lambda: dict(dtype=3), -5), (lambda: dict(in_dim=0), -2), (lambda: dict(in_dim=48), -2),
       (lambda: dict(rows=-1), -2), (lambda: dict(out_dim=-1), -2), (lambda: dict(w=_four(codes=None)), -1),
       (lambda: dict(w=_four(scales=None)), -1), (lambda: dict(w=_four(codes=264)), -4), (lambda: dict(w=_four(code_stride=40)), -4),
       (lambda: dict(w=_four(code_stride=16)), -2), (lambda: dict(w=_four(scale_stride=1)), -2), (lambda: dict(x=264), -4),
       (lambda: dict(x_stride=65), -4), (lambda: dict(x_stride=56), -2), (lambda: dict(x=None, x4=_four(codes=None)), -1),
       (lambda: dict(x=None, x4=_four(code_stride=16)), -2), (lambda: dict(out=None), -1), (lambda: dict(out=513), -4),
       (lambda: dict(out_stride=4), -2), (lambda: dict(residual=512, residual_stride=4), -2),
       (lambda: dict(rows=2 ** 30 + 1), -2), (lambda: dict(out_dim=2 ** 30 + 1), -2), (lambda: dict(rows=2 ** 20, out_dim=2 ** 19), -2),
       (lambda: dict(residual=512, residual_stride=6), -5), (lambda: dict(residual=513, residual_stride=5), -4)]


@pytest.mark.parametrize("over,code", BAD)
def test_matmul_refusals(over, code):
    from spock_amd import _lib
    a = _matmul(_lib, **over())
    assert _lib.lib().spk_mx4_matmul(C.byref(a), None) == code, _lib.lib().spk_last_error()


@pytest.mark.parametrize("over", [dict(rows=0), dict(out_dim=0)])
def test_matmul_of_nothing(over):
    from spock_amd import _lib
    a = _matmul(_lib, **{**over, "x": None, "out": None})
    assert _lib.lib().spk_mx4_matmul(C.byref(a), None) == 0
    assert _lib.lib().spk_mx4_matmul(None, None) == -1


@pytest.mark.parametrize("name", ["spk_mx4_quantize", "spk_mx4_dequantize"])
@pytest.mark.parametrize("over,code", [(dict(dtype=5), -5), (dict(rows=-1), -2), (dict(cols=48), -2), (dict(cols=-32), -2),
                                       (dict(x=None), -1), (dict(x=264), -4), (dict(stride=65), -4), (dict(stride=32), -2),
                                       (dict(rows=2 ** 31), -2), (dict(rows=2 ** 28, cols=64), -2), (dict(m=None), -1),
                                       (dict(m=dict(codes=None)), -1), (dict(m=dict(scales=None)), -1), (dict(m=dict(codes=8)), -4),
                                       (dict(m=dict(code_stride=24)), -4), (dict(m=dict(code_stride=16)), -2),
                                       (dict(m=dict(scale_stride=1)), -2), (dict(rows=0, x=None), 0), (dict(cols=0, x=None), 0)])
def test_quantize_refusals(name, over, code):
    from spock_amd import _lib
    f = dict(x=256, dtype=_lib.SPK_F16, stride=64, rows=3, cols=64, m={})
    f.update(over)
    m = None if f["m"] is None else C.byref(_four(**f["m"]))
    fn = getattr(_lib.lib(), name)
    if name.endswith("dequantize"):
        rc = fn(m, f["rows"], f["cols"], f["dtype"], f["x"], f["stride"], None)
    else:
        rc = fn(f["x"], f["dtype"], f["stride"], f["rows"], f["cols"], m, None)
    assert rc == code, _lib.lib().spk_last_error()


def _cache(_lib, **over):
    f = dict(dtype=_lib.SPK_F16, num_kv_heads=2, head_dim=64, page_size=16, num_pages=4, max_pages=4, num_seqs=1,
             total_tokens=1, k_cache=256, v_cache=256, page_stride=1024, token_stride=64, head_stride=32,
             block_table=256, table_stride=4, cu_seqlens=256, context_lens=256)
    f.update(over)
    return _lib.SpkPagedCache(*[f[n] for n, _ in _lib.SpkPagedCache._fields_])


PAGED = [(dict(dtype=0), {}, -5), (dict(head_dim=96), {}, -2), (dict(k_cache=None), {}, -1), (dict(k_cache=264), {}, -4),
         (dict(token_stride=72), {}, -4), (dict(head_stride=40), {}, -4), (dict(page_stride=1032), {}, -4),
         (dict(page_stride=2 ** 32), {}, -2), ({}, None, -1), ({}, dict(k_scales=None), -1), ({}, dict(v_scales=None), -1),
         ({}, dict(page_stride=-1), -2), ({}, dict(token_stride=2 ** 32), -2), ({}, dict(head_stride=-2), -2)]


@pytest.mark.parametrize("over,scales,code", PAGED)
def test_paged_refusals(over, scales, code):
    from spock_amd import _lib
    lib = _lib.lib()
    f = dict(k_scales=256, v_scales=256, page_stride=64, token_stride=4, head_stride=2)
    s = None if scales is None else C.byref(_lib.SpkPagedScales(*{**f, **scales}.values()))
    a = _lib.SpkPagedAttnArgs(_cache(_lib, **over), 4, 1, 64, 0, 0.0, 256, 256, 64, None, 0, 0, 256, 256, 64, None, None, 0)
    assert lib.spk_paged_attention_mx4(C.byref(a), s, None) == code, lib.spk_last_error()
    m = _lib.SpkMropeArgs(_cache(_lib, **over), 4, 32, 0, 1, bytes(16), 256, 1, 256, 8, 0.0, 256, 256, 64, 256, 128, 64, 256, 128, 64,
                          None, None, 256, 256, 64)
    assert lib.spk_mrope_append_mx4(C.byref(m), s, None) == code, lib.spk_last_error()


def test_paged_workspaces():
    """Enough for every smaller call, and none where nothing is joined."""
    from spock_amd import _lib, ops
    lib = _lib.lib()
    for tokens, heads, kv, dim, seqs, q, c, window in ((64, 8, 2, 256, 64, 1, 16000, 0), (9, 8, 2, 128, 1, 9, 5000, 0),
                                                       (4096, 16, 4, 128, 4, 2048, 6000, 0), (300, 7, 1, 64, 3, 100, 9000, 128)):
        pages = -(-c // 16)
        most = ops.paged_attention_mx4_workspace_bytes(tokens, heads, kv, dim, 16, pages, seqs, q, c, window)
        for t in (tokens, tokens // 2 + 1, 1):
            for n in (seqs, 1):
                for length in (c, c // 3, 100):
                    for mq in (q, 1):
                        a = ops._attention_sizes(t, heads, kv, dim, 16, pages, n, mq, length, window)
                        assert lib.spk_paged_attention_mx4_workspace_need(C.byref(a)) <= most
    a = ops._attention_sizes(1, 8, 2, 256, 16, 8, 1, 1, 128, 0)
    assert lib.spk_paged_attention_mx4_workspace_need(C.byref(a)) == 0


def test_python_refusals():
    from spock_amd import ops
    from spock_amd._lib import SpockError
    x = torch.zeros(2, 64)
    m = ops.Mx4(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8))
    for call in (lambda: ops.mx4_quantize(x), lambda: ops.mx4_dequantize(m), lambda: ops.mx4_dequantize(x),
                 lambda: ops.mx4_matmul(x, m), lambda: ops.mx4_matmul(m, m)):
        with pytest.raises(SpockError):
            call()


def test_every_form_of_the_product_is_tested():
    """Each kernel that the rule of spk_mx4_matmul chooses among has a shape in the tests on the GPU."""
    for four in (False, True):
        have = {G._form(four, *x) for x in G.FEW + G.LONG + G.SHAPES} | {G._form(four, *x, x[0] % 2 == 0) for x in G.MANY}
        want = {("few", xr, *form, sb) for xr in ((16,) if four else (4, 16)) for form in ((4, 1), (4, 4), (2, 4), (1, 4)) for sb in (4, 1)}
        want |= {("tiles", size, sb) for size in (128, 256) for sb in (16, 1)}
        assert have == want, want - have
