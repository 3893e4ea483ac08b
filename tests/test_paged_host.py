"""The paged step without a GPU: the index arithmetic of csrc/paged.hpp,
compiled for the host, over tables and lengths that point outside the
buffers, and the refusals of the entry points before any launch."""
import ctypes as C
import subprocess

import numpy as np
import pytest

from conftest import ROOT

SHIM = r'''
#include "paged.hpp"
using namespace spk_paged;
extern "C" {
int first_wrong_quotient(uint32_t d, const uint32_t* p, int n) {
  const PageDiv v = page_div(d);
  for (int i = 0; i < n; ++i) if (divide(v, p[i]) != p[i] / d) return i;
  return -1;
}
// the slots of every position of every sequence: how many lie outside a pool of `elements`, how many have a page
void walk(const int32_t* table, long stride, const int32_t* cu, const int32_t* ctx, int seqs, int total, int page_size,
          int pages, int max_pages, long page_stride, long token_stride, long elements, long row, long* out) {
  Cache c{table, cu, ctx, stride, 0, (uint32_t)page_stride, (uint32_t)token_stride, seqs, total, page_size, pages,
          max_pages, page_div(page_size)};
  out[0] = out[1] = out[2] = out[3] = 0;
  for (int s = 0; s < seqs; ++s) {
    const Seq q = seq_at(c, s);
    if (q.first < 0 || q.n < 0 || q.first + q.n > total || q.ctx < 0 || q.ctx > (long)max_pages * page_size) ++out[0];
    out[3] += q.n;
    for (int p = 0; p < q.ctx; ++p) {
      const long at = offset_of(c, s, p);
      if (at < 0) continue;
      ++out[1];
      if (at + row > elements) ++out[2];
    }
  }
}
void sees(int first, int n, int ctx, int i, int window, int* lo, int* hi) { visible(Seq{first, n, ctx}, i, window, lo, hi); }
}
'''


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "shim.cpp").write_text(SHIM)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(ROOT / "spock_amd" / "csrc"),
                        str(d / "shim.cpp"), "-o", str(d / "shim.so")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return C.CDLL(str(d / "shim.so"))


@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 8, 16, 20, 60, 64, 255, 256, 257, 528, 65535, 2 ** 20 + 1, 2 ** 30 + 3, 2 ** 31 - 65])
def test_division_by_the_page_size(shim, d):
    rng = np.random.default_rng(d)
    multiples = np.arange(0, min((2 ** 31 - 1) // d, 20000) + 1, dtype=np.int64) * d
    p = np.concatenate([np.arange(4096), multiples, multiples - 1, multiples + 1, (2 ** 31 - 1) // d * d - np.arange(2),
                        rng.integers(0, 2 ** 31, 20000), 2 ** 31 - 1 - np.arange(4096)])
    p = np.ascontiguousarray(p[(p >= 0) & (p < 2 ** 31)].astype(np.uint32))
    shim.first_wrong_quotient.argtypes = [C.c_uint32, C.c_void_p, C.c_int]
    i = shim.first_wrong_quotient(d, p.ctypes.data, p.size)
    assert i == -1, (d, int(p[i]))


@pytest.mark.parametrize("seed", range(6))
def test_tables_and_lengths_from_outside(shim, seed):
    rng = np.random.default_rng(seed)
    seqs, page_size, pages, max_pages = 9, int(rng.choice([1, 3, 16, 20])), 13, 7
    heads, dim, total = 2, 64, 40
    table = rng.integers(0, pages, (seqs, max_pages)).astype(np.int32)
    bad = rng.random(table.shape) < 0.3
    table[bad] = rng.choice([-1, pages, pages + 1, -2 ** 31, 2 ** 31 - 1], bad.sum())
    cu = rng.integers(-50, 90, seqs + 1).astype(np.int32)
    cu[rng.integers(0, seqs + 1)] = -2 ** 31
    ctx = rng.integers(-5, max_pages * page_size + 50, seqs).astype(np.int32)
    ctx[0], ctx[1] = 2 ** 31 - 1, -2 ** 31
    out = (C.c_long * 4)()
    row = heads * dim
    shim.walk.argtypes = [C.c_void_p, C.c_long, C.c_void_p, C.c_void_p] + [C.c_int] * 5 + [C.c_long] * 4 + [C.c_void_p]
    shim.walk(table.ctypes.data, max_pages, cu.ctypes.data, ctx.ctypes.data, seqs, total, page_size, pages, max_pages,
              page_size * row, row, pages * page_size * row, row, out)
    lens = np.clip(ctx, 0, max_pages * page_size)
    fine = sum(int(((table[s] >= 0) & (table[s] < pages))[np.arange(n) // page_size].sum()) for s, n in enumerate(lens))
    assert out[0] == 0 and out[2] == 0 and out[1] == fine


def test_visible_ranges(shim):
    lo, hi = C.c_int(), C.c_int()
    for n, ctx in ((1, 0), (1, 1), (3, 2), (5, 5), (4, 100), (7, 0)):
        for window in (0, 1, 2, 50, 1000):
            for i in range(n):
                shim.sees(0, n, ctx, i, window, C.byref(lo), C.byref(hi))
                p = ctx - n + i
                keys = [j for j in range(ctx) if j <= p and (not window or j > p - window)]
                assert list(range(lo.value, hi.value)) == keys


def _cache(_lib, **over):
    f = dict(dtype=_lib.SPK_F16, num_kv_heads=2, head_dim=64, page_size=16, num_pages=4, max_pages=4, num_seqs=1,
             total_tokens=1, k_cache=256, v_cache=256, page_stride=2048, token_stride=128, head_stride=64,
             block_table=256, table_stride=4, cu_seqlens=256, context_lens=256)
    f.update(over)
    return _lib.SpkPagedCache(*[f[n] for n, _ in _lib.SpkPagedCache._fields_])


BAD_CACHE = [(dict(dtype=0), -5), (dict(dtype=3), -5), (dict(head_dim=96), -2), (dict(num_kv_heads=0), -2),
             (dict(page_size=0), -2), (dict(num_pages=0), -2), (dict(max_pages=0), -2), (dict(num_seqs=-1), -2),
             (dict(total_tokens=-1), -2), (dict(max_pages=2 ** 27), -2), (dict(k_cache=None), -1),
             (dict(v_cache=None), -1), (dict(block_table=None), -1), (dict(cu_seqlens=None), -1),
             (dict(context_lens=None), -1), (dict(k_cache=264), -4), (dict(token_stride=100), -4),
             (dict(head_stride=-64), -4), (dict(page_stride=2047), -4), (dict(page_stride=2 ** 32), -2), (dict(token_stride=2 ** 32), -2), (dict(num_seqs=2, table_stride=3), -2)]


@pytest.mark.parametrize("over,code", BAD_CACHE)
def test_cache_refusals(over, code):
    from spock_amd import _lib
    lib = _lib.lib()
    a = _lib.SpkPagedAttnArgs(_cache(_lib, **over), 4, 1, 64, 0, 0.0, 256, 256, 64, None, 0, 0, 256, 256, 64, None, None, 0)
    assert lib.spk_paged_attention(C.byref(a), None) == code, lib.spk_last_error()
    m = _lib.SpkMropeArgs(_cache(_lib, **over), 4, 32, 0, 1, bytes(16), 256, 1, 256, 10, 0.0, 256, 256, 64, 256, 128, 64,
                          256, 128, 64, None, None, 256, 256, 64)
    assert lib.spk_mrope_append(C.byref(m), None) == code, lib.spk_last_error()


@pytest.mark.parametrize("over,code", [
    (dict(num_q_heads=5), -2), (dict(num_q_heads=0), -2), (dict(max_query_len=-1), -2), (dict(window=-1), -2),
    (dict(max_context_len=-1), -2), (dict(q=None), -1), (dict(out=None), -1), (dict(q=258), -4), (dict(out=258), -4),
    (dict(gate=258), -4), (dict(gate=256, gate_head_stride=4), -4), (dict(q_token_stride=257), -4),
    (dict(out_head_stride=63), -4), (dict(max_context_len=60000, max_pages=4000), -1)])
def test_attention_refusals(over, code):
    from spock_amd import _lib
    lib = _lib.lib()
    assert lib.spk_paged_attention(None, None) == -1
    assert lib.spk_paged_attention_workspace_size(None) == 0
    over = dict(over)
    a = _lib.SpkPagedAttnArgs(_cache(_lib, max_pages=over.pop("max_pages", 4), table_stride=4000), 4, 1, 64, 0, 0.0, 256, 256,
                              64, None, 256, 64, 256, 256, 64, None, None, 0)
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.spk_paged_attention(C.byref(a), None) == code, lib.spk_last_error()
    if "max_context_len" in over and code == -1:  # the workspace is what was missing
        assert b"workspace" in lib.spk_last_error() and lib.spk_paged_attention_workspace_size(C.byref(a)) > 0
        a.workspace, a.workspace_bytes = 256, 16
        assert lib.spk_paged_attention(C.byref(a), None) == -5
        a.workspace, a.workspace_bytes = 264, 1 << 30
        assert lib.spk_paged_attention(C.byref(a), None) == -5


@pytest.mark.parametrize("over,code", [
    (dict(num_q_heads=0), -2), (dict(rot_dim=0), -2), (dict(rot_dim=24), -2), (dict(rot_dim=80), -2), (dict(pairing=2), -5),
    (dict(num_axes=0), -2), (dict(num_axes=5), -2), (dict(pair_axis=None), -1), (dict(pair_axis=bytes([0] * 15 + [3])), -5),
    (dict(rope_rows=0), -2), (dict(positions=None), -1), (dict(rope=None), -1), (dict(q=None), -1), (dict(k=None), -1),
    (dict(v=None), -1), (dict(q_out=None), -1), (dict(positions_stride=0), -2), (dict(q=258), -4), (dict(k_norm_w=258), -4),
    (dict(rope=257), -4), (dict(v_token_stride=4), -4), (dict(out_head_stride=-64), -4)])
def test_mrope_refusals(over, code):
    from spock_amd import _lib
    lib = _lib.lib()
    assert lib.spk_mrope_append(None, None) == -1
    a = _lib.SpkMropeArgs(_cache(_lib), 4, 32, 0, 3, bytes(16), 256, 1, 256, 10, 0.0, 256, 256, 64, 256, 128, 64,
                          256, 128, 64, None, None, 256, 256, 64)
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.spk_mrope_append(C.byref(a), None) == code, lib.spk_last_error()


def test_more_rows_than_a_launch_holds():
    from spock_amd import _lib
    lib = _lib.lib()
    for tokens, seqs, bound, context in ((120_000_000, 120_000_000, 1, 64), (120_000_000, 1, 1, 60000)):
        a = _lib.SpkPagedAttnArgs(_cache(_lib, num_kv_heads=16, head_stride=64, token_stride=1024, total_tokens=tokens, num_seqs=seqs,
                                         max_pages=4000, table_stride=4000), 16, bound, context, 0, 0.0, 256, 256, 64, None, 0, 0,
                                  256, 256, 64, None, 256, 1 << 62)
        assert lib.spk_paged_attention(C.byref(a), None) == -2 and b"launch" in lib.spk_last_error(), lib.spk_last_error()
    m = _lib.SpkMropeArgs(_cache(_lib, total_tokens=70_000_000), 4, 32, 0, 1, bytes(16), 256, 70_000_000, 256, 10, 0.0, 256, 256, 64,
                          256, 128, 64, 256, 128, 64, None, None, 256, 256, 64)
    assert lib.spk_mrope_append(C.byref(m), None) == -2


def test_nothing_to_do():
    from spock_amd import _lib
    lib = _lib.lib()
    for empty in (dict(num_seqs=0), dict(total_tokens=0)):
        a = _lib.SpkPagedAttnArgs(_cache(_lib, **empty), 4, 1, 64)
        assert lib.spk_paged_attention(C.byref(a), None) == 0 and lib.spk_paged_attention_workspace_size(C.byref(a)) == 0
        m = _lib.SpkMropeArgs(_cache(_lib, **empty), 4, 32, 0, 1, bytes(16), None, 0, None, 10)
        assert lib.spk_mrope_append(C.byref(m), None) == 0


def test_struct_layouts():
    from spock_amd import _lib
    assert C.sizeof(_lib.SpkPagedCache) == 104 and _lib.SpkPagedCache.k_cache.offset == 32
    assert C.sizeof(_lib.SpkMropeArgs) == 272 and _lib.SpkMropeArgs.q.offset == 160
    assert C.sizeof(_lib.SpkPagedAttnArgs) == 224 and _lib.SpkPagedAttnArgs.q.offset == 128


def test_host_tensors_are_refused():
    import torch
    from spock_amd import _lib, ops
    z = torch.zeros
    q, c, i = z(1, 4, 64, dtype=torch.float16), z(2, 16, 2, 64, dtype=torch.float16), z(2, dtype=torch.int32)
    with pytest.raises(_lib.SpockError, match="device tensors"):
        ops.paged_attention(q, c, c, z(1, 2, dtype=torch.int32), i, i[:1], 1, 32)


@pytest.mark.parametrize("over,code", [
    (dict(kind=2), -5), (dict(dtype=3), -5), (dict(vocab=0), -2), (dict(vocab=2 ** 31 - 1), -2), (dict(num_seqs=-1), -2),
    (dict(total_tokens=65536), -2), (dict(num_seqs=65536), -2), (dict(kind=1, temperature=256), -5), (dict(context_out=256), -1),
    (dict(cu_seqlens=None), -1), (dict(accepted=None), -1), (dict(tokens=None), -1), (dict(target=None), -1),
    (dict(u_accept=None), -1), (dict(u_sample=None), -1), (dict(out_tokens=None), -1), (dict(target_stride=99), -2),
    (dict(draft=256, draft_stride=99), -2), (dict(target=257), -4), (dict(draft=257, draft_stride=100), -4),
    (dict(out_tokens=256, tokens=256), -5), (dict(workspace=None), -1), (dict(workspace_bytes=8), -5), (dict(workspace=264), -5)])
def test_verify_refusals(over, code):
    from spock_amd import _lib
    lib = _lib.lib()
    assert lib.spk_verify_drafts(None, None) == -1
    a = _lib.SpkVerifyArgs(0, _lib.SPK_F16, 100, 2, 6, 256, 256, 256, 100, None, 0, None, 256, 256, 512, 256, None, None, None, 256, 1 << 20)
    for k, v in over.items():
        setattr(a, k, v)
    assert lib.spk_verify_drafts(C.byref(a), None) == code, lib.spk_last_error()


def test_verify_nothing_to_do():
    from spock_amd import _lib
    a = _lib.SpkVerifyArgs(0, _lib.SPK_F16, 100, 0, 0)
    assert _lib.lib().spk_verify_drafts(C.byref(a), None) == 0
    assert _lib.lib().spk_verify_drafts_workspace_size(100, 0, 4) == 0
    assert C.sizeof(_lib.SpkVerifyArgs) == 152 and _lib.SpkVerifyArgs.workspace.offset == 136
