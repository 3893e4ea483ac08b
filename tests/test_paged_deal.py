"""How paged_attention deals its rows and keys to workgroups, without a GPU:
csrc/paged_deal.hpp compiled for the host, the 64 lanes of a wave as contexts
that take turns at every operation that they do together.  Every piece of work
is dealt once, ranges cover the keys, and nothing that lengths or offsets hold
leads out of a launch, a workspace or a sequence."""
import ctypes as C
import subprocess

import numpy as np
import pytest

from conftest import ROOT

SHIM = r'''
#include <ucontext.h>
#include <string.h>
#include "paged_deal.hpp"
using namespace spk_paged;

// 64 lanes in turn: a lane leaves what it brings to an operation and goes on when all have.
static ucontext_t main_ctx, lane_ctx[64];
static char stacks[64][65536];
static int now, left[2][64], turn[64], live;
static bool torn;   // lanes met in different operations
static int kinds[2][64];
static void (*body)(int);
static void next_lane() {
  const int from = now;
  now = (now + 1) % 64;
  swapcontext(&lane_ctx[from], &lane_ctx[now]);
}
static const int* meet(int kind, int v) {
  const int me = now, at = turn[me]++ & 1;
  left[at][me] = v;
  kinds[at][me] = kind;
  next_lane();
  for (int i = 0; i < 64; ++i) torn |= kinds[at][i] != kind;
  return left[at];
}
static void enter() {
  body(now);
  if (--live) next_lane();  // all end in the same turn, lane 0 first
}
static void run(void (*f)(int)) {
  body = f;
  live = 64;
  memset(turn, 0, sizeof turn);
  for (int i = 0; i < 64; ++i) {
    getcontext(&lane_ctx[i]);
    lane_ctx[i].uc_stack.ss_sp = stacks[i];
    lane_ctx[i].uc_stack.ss_size = sizeof stacks[i];
    lane_ctx[i].uc_link = &main_ctx;
    makecontext(&lane_ctx[i], enter, 0);
  }
  now = 0;
  swapcontext(&main_ctx, &lane_ctx[0]);
}
struct Wave {
  static int first(int v) { return meet(1, v)[0]; }
  static int at(int v, int lane) { const int* x = meet(2, v); if ((unsigned)lane > 63) { torn = true; lane = 0; } return x[lane]; }
  static int count(bool b) { const int* x = meet(3, b); int n = 0; for (int i = 0; i < 64; ++i) n += x[i]; return n; }
  static int sum(int v) { const int* x = meet(4, v); unsigned n = 0; for (int i = 0; i < 64; ++i) n += x[i]; return (int)n; }
  static int max(int v) { const int* x = meet(5, v); int n = x[0]; for (int i = 1; i < 64; ++i) n = x[i] > n ? x[i] : n; return n; }
  static int scan(int v) { const int me = now; const int* x = meet(6, v); unsigned n = 0; for (int i = 0; i <= me; ++i) n += x[i]; return (int)n; }
};

static Deal deal;
static Share share[64];
static int number, last, seq[64], tile[64];
static bool found[64];
static void one_share(int lane) { found[lane] = find_share<Wave>(deal, number, lane, &share[lane]); }
static void one_tile(int lane) { found[lane] = find_tile<Wave>(deal, number, last, lane, &seq[lane], &tile[lane]); }

extern "C" {
// out[0..8): shares, share_rows, many, tiles, splits, chunk, join, join_few
size_t plan(const int* sizes, const int* cu, const int* ctx, int* out) {
  SpkPagedAttnArgs p{};
  p.num_q_heads = sizes[0];
  p.cache.num_kv_heads = sizes[1];
  p.cache.head_dim = sizes[2];
  p.cache.page_size = sizes[3];
  p.cache.max_pages = sizes[4];
  p.cache.num_seqs = sizes[5];
  p.cache.total_tokens = sizes[6];
  p.max_query_len = sizes[7];
  p.max_context_len = sizes[8];
  p.window = sizes[9];
  const Plan r = plan_of(p);
  const int v[8] = {r.shares, r.share_rows, r.many, r.tiles, r.splits, r.chunk, r.join, r.join_few};
  memcpy(out, v, sizeof v);
  if (cu) {
    Cache c{};
    c.cu = cu;
    c.ctx = ctx;
    c.num_seqs = sizes[5];
    c.total_tokens = sizes[6];
    c.page_size = sizes[3];
    c.max_pages = sizes[4];
    c.div = page_div(sizes[3]);
    deal = deal_of(p, r, c);
  }
  return workspace_of(p, r);
}
// rows of out: found, seq, tile, kvh, range, ranges, keys, lo, first; 1 where the lanes agreed
int share_of(int at, int* out) {
  number = at;
  torn = false;
  run(one_share);
  for (int i = 1; i < 64; ++i) torn |= found[i] != found[0] || (found[0] && memcmp(&share[i], &share[0], sizeof(Share)));
  out[0] = found[0];
  if (found[0]) memcpy(out + 1, &share[0], sizeof(Share));
  return !torn;
}
int tile_of(int at, int* out) {
  number = at;
  last = out[0] - 1;
  torn = false;
  run(one_tile);
  for (int i = 1; i < 64; ++i) torn |= found[i] != found[0] || (found[0] && (seq[i] != seq[0] || tile[i] != tile[0]));
  out[0] = found[0];
  out[1] = seq[0];
  out[2] = tile[0];
  return !torn;
}
size_t bound(const int* sizes) {
  SpkPagedAttnArgs p{};
  p.num_q_heads = sizes[0];
  p.cache.num_kv_heads = sizes[1];
  p.cache.head_dim = sizes[2];
  p.cache.page_size = sizes[3];
  p.cache.max_pages = sizes[4];
  p.cache.num_seqs = sizes[5];
  p.cache.total_tokens = sizes[6];
  p.max_query_len = sizes[7];
  p.max_context_len = sizes[8];
  p.window = sizes[9];
  return workspace_bound(p);
}
int keys_of(int lo, int hi) { return range_keys(deal, lo, hi); }
}
'''


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("deal")
    (d / "shim.cpp").write_text(SHIM)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fwrapv", "-w", "-I", str(ROOT / "spock_amd" / "csrc"),
                        str(d / "shim.cpp"), "-o", str(d / "shim.so")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    lib = C.CDLL(str(d / "shim.so"))
    lib.plan.restype = lib.bound.restype = C.c_size_t
    return lib


PLAN = ("shares", "share_rows", "many", "tiles", "splits", "chunk", "join", "join_few")


class Call:
    """The plan of a call, and its lengths as the device sees them."""

    def __init__(self, shim, cu, ctx, heads=8, kv=2, dim=128, page=16, max_pages=4000, total=None, max_q=None, max_c=None, window=0):
        self.shim, self.kv, self.window = shim, kv, window
        self.total = int(cu[-1]) if total is None else total
        self.cu, self.ctx = np.ascontiguousarray(cu, np.int32), np.ascontiguousarray(ctx, np.int32)
        S = len(ctx)
        first = np.clip(self.cu[:-1].astype(np.int64), 0, self.total)
        self.n = np.clip(self.cu[1:].astype(np.int64), first, self.total) - first
        self.length = np.clip(self.ctx.astype(np.int64), 0, max_pages * page)
        self.rows = self.n * (heads // kv)
        max_q = int(self.n.max(initial=0)) if max_q is None else max_q
        max_c = int(self.length.max(initial=0)) if max_c is None else max_c
        sizes = (C.c_int * 10)(heads, kv, dim, page, max_pages, S, self.total, max_q, max_c, window)
        out = (C.c_int * 8)()
        self.bytes = shim.plan(sizes, self.cu.ctypes.data_as(C.c_void_p), self.ctx.ctypes.data_as(C.c_void_p), out)
        for name, v in zip(PLAN, out):
            setattr(self, name, v)

    def sees(self, s, i):
        hi = max(0, int(self.length[s] - self.n[s] + i) + 1)
        return (max(0, hi - self.window) if self.window else 0), hi

    def share_of(self, at):
        out = (C.c_int * 9)()
        assert self.shim.share_of(at, out) == 1, at
        return dict(zip(("seq", "tile", "kvh", "range", "ranges", "keys", "lo", "first"), out[1:])) if out[0] else None

    def tile_of(self, at):
        out = (C.c_int * 3)(self.tiles, 0, 0)
        assert self.shim.tile_of(at, out) == 1, at
        return (out[1], out[2]) if out[0] else None

    def check_shares(self, exact=True):
        few = (self.rows > 0) & (self.rows < self.many)
        want = {(s, t, h) for s in np.nonzero(few)[0] for t in range(-(-int(self.rows[s]) // self.share_rows)) for h in range(self.kv)}
        got, ends = {}, 0
        for at in range(self.shares):
            x = self.share_of(at)
            if x is None:
                ends = 1
                continue
            assert not ends, at                                   # none after the last
            piece = (x["seq"], x["tile"], x["kvh"])
            assert piece in want and 0 <= x["range"] < x["ranges"] and x["first"] == at - x["range"], (at, x)
            lo, hi = self.sees(x["seq"], 0)[0] & ~31, self.sees(x["seq"], int(self.n[x["seq"]]) - 1)[1]
            assert x["lo"] == lo and x["keys"] > 0 and x["keys"] % 128 == 0 and x["keys"] * x["ranges"] >= hi - lo, (at, x)
            got.setdefault(piece, []).append(x["range"])
        if exact:
            assert set(got) == want
            assert all(v == list(range(len(v))) for v in got.values())
            if not self.join:
                assert all(len(v) == 1 for v in got.values())
            assert self.shares == 0 or ends or sum(map(len, got.values())) <= self.shares
        return got

    def check_tiles(self, exact=True):
        many = self.rows >= self.many
        want = {(s, t) for s in np.nonzero(many)[0] for t in range(-(-int(self.rows[s]) // 256))}
        got, before, group = [], None, 0
        for at in range(self.tiles):
            x = self.tile_of(at)
            if x is None:
                continue
            assert x in want, (at, x)
            s, t = x
            group = int(self.rows[s] // self.n[s])
            first, end = 256 * t, min(256 * t + 256, int(self.rows[s]))
            lo, hi = self.sees(s, first // group)[0], self.sees(s, (end - 1) // group)[1]
            keys = self.shim.keys_of(lo, hi)
            assert keys > 0 and keys * self.splits >= hi - (lo & ~31), (at, x)
            if len(self.ctx) <= 256 and exact:
                assert before is None or hi <= before + 128, (at, x)  # the most keys first, to within a level of 128
                before = hi
            got.append(x)
        assert len(set(got)) == len(got)
        if exact:
            assert set(got) == want


def _cu(lens):
    return np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32), np.array([c for _, c in lens], np.int32)


@pytest.mark.parametrize("lens,kw", [
    ([(1, 1)], {}), ([(1, 1500)], {}), ([(1, 130001)], dict(heads=32, kv=8, max_pages=9000)), ([(9, 9)], dict(heads=7, kv=1)),
    ([(1, c) for c in range(300, 16000, 250)], {}), ([(9, 1000 + 500 * i) for i in range(16)], {}),
    ([(0, 10), (3, 0), (4, 2), (1, 50), (0, 0), (2, 2)], {}), ([(2048, 16384)], {}),
    ([(4001, 4001), (1061, 1061), (2504, 3007), (61, 5000), (1, 2222), (1, 777)], dict(heads=16, kv=4, page=64)),
    ([(300, 900), (1, 700), (0, 5), (500, 400), (90, 1500), (257, 257), (2, 2), (64, 128)], dict(window=200)),
    ([(40, 300), (1, 300), (70, 70), (3, 2)], dict(window=31)), ([(33, 40000)], {}), ([(32, 40000)], {}), ([(17, 64)], dict(max_c=64)),
    ([(1 + i % 4, 5 * i) for i in range(256)], {}), ([(1 + i % 4, 5 * i) for i in range(257)], {}),
    ([((90, 3, 0)[i % 3], 10 + 3 * i) for i in range(300)], {}),
    ([(5, 900)] * 40, dict(max_c=1)), ([(5, 900)] * 40, dict(max_q=1, max_c=100)), ([(60, 900)] * 3, dict(max_q=1)),
    ([(3, 70), (100, 150)], dict(max_q=5000, max_c=100000)), ([(1, 2000)], dict(max_q=5000))],
    ids=lambda v: None if isinstance(v, dict) else "+".join("%d:%d" % x for x in v[:4]) + ("..%d" % len(v) if len(v) > 4 else ""))
def test_everything_is_dealt_once(shim, lens, kw):
    call = Call(shim, *_cu(lens), **kw)
    call.check_shares()
    call.check_tiles()


@pytest.mark.parametrize("seed", range(12))
def test_lengths_at_random(shim, seed):
    rng = np.random.default_rng(seed)
    S = int(rng.choice([1, 2, 7, 64, 65, 200]))
    lens = [(int(rng.choice([0, 1, 4, 30, 100, 400], p=[.1, .4, .2, .1, .1, .1])), int(rng.integers(0, 5000))) for _ in range(S)]
    heads, kv = [(8, 2), (16, 4), (7, 1), (4, 4), (40, 2)][seed % 5]
    call = Call(shim, *_cu(lens), heads=heads, kv=kv, page=int(rng.choice([1, 16, 20])), window=int(rng.choice([0, 0, 50, 2000])))
    call.check_shares()
    call.check_tiles()


@pytest.mark.parametrize("seed", range(8))
def test_lengths_and_offsets_from_outside(shim, seed):
    """Offsets that overlap or lie outside, lengths past the table: no share or tile that is not a sequence's."""
    rng = np.random.default_rng(100 + seed)
    S = int(rng.choice([3, 9, 70, 300]))
    cu = rng.integers(-50, 700, S + 1).astype(np.int32)
    cu[rng.integers(0, S + 1)], cu[rng.integers(0, S + 1)] = -2 ** 31, 2 ** 31 - 1
    ctx = rng.integers(-5, 5000, S).astype(np.int32)
    ctx[0], ctx[-1] = 2 ** 31 - 1, -2 ** 31
    call = Call(shim, cu, ctx, total=500, max_pages=100, max_q=int(rng.choice([1, 40, 500])), max_c=1000)
    call.check_shares(exact=False)
    call.check_tiles(exact=False)


def test_lengths_next_to_the_largest(shim):
    """Contexts of nearly 2^31 positions: the tried length of a range stays below it."""
    call = Call(shim, *_cu([(1, 2 ** 31 - 2 ** 21)] * 256), heads=8, kv=8, page=2 ** 20, max_pages=2047)
    assert call.join
    call.check_shares()


def test_more_ranges_of_the_largest_length_than_it_lacks_to_two_to_the_31(shim):
    call = Call(shim, *_cu([(0, 0)] * 70000 + [(1, 2 ** 31 - 2 ** 13)]), heads=1, kv=1, page=2 ** 12, max_pages=2 ** 19 - 2)
    for at in (0, 1, 5000):
        x = call.share_of(at)
        assert x["seq"] == 70000 and x["range"] == at and x["ranges"] > 2 ** 13 and x["keys"] % 128 == 0
        assert x["keys"] > 0 and 0 <= x["keys"] * x["ranges"] - (2 ** 31 - 2 ** 13) < 129 * x["ranges"]


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 256), (16, 4, 128), (7, 1, 64), (40, 2, 64), (4, 4, 128)])
@pytest.mark.parametrize("most", [(8192, 64, 8192, 32768, 0), (300, 300, 9, 5000, 0), (4096, 1, 4096, 131072, 0), (2000, 16, 500, 20000, 1024),
                                  (64, 64, 1, 200, 0), (700, 3, 600, 1200, 0)], ids=str)
def test_a_workspace_of_the_largest_sizes_serves_the_smaller(shim, heads, kv, dim, most):
    out = (C.c_int * 8)()

    def sizes(T, S, q, c, w):
        return (C.c_int * 10)(heads, kv, dim, 16, 10000, S, T, q, c, w)

    kept, largest = shim.bound(sizes(*most)), 0
    rng = np.random.default_rng(most[0] + heads)
    T, S, q, c, w = most
    log = lambda top: int(round(np.exp(rng.uniform(0, np.log(top)))))
    tried = [most] + [(log(T), log(S), log(q), log(c), w) for _ in range(6000)]
    tried += [(t, min(s, S), min(t, q), x, w) for t in list(range(1, min(T, 400))) + list(range(400, T + 1, 97)) for s in (1, 8) for x in (c, c // 3 + 1)]
    if w == 0:
        tried += [(log(T), log(S), log(q), c, log(5000)) for _ in range(500)]
    for x in tried:
        need = shim.plan(sizes(*x), None, None, out)
        assert need <= kept and need <= shim.bound(sizes(*x)), (x, need, kept)
        assert shim.bound(sizes(*x)) <= kept, x
        largest = max(largest, need)
    # and not much more than the largest need of them
    assert kept <= 3.5 * largest + 4096, (kept, largest)


def test_the_size_that_the_library_tells(shim):
    """Through the entry point: one that a smaller call needs more of than a larger one does."""
    from spock_amd import ops
    args = dict(heads=8, kv_heads=2, head_dim=256, page_size=16, max_pages=2048, num_seqs=1, max_context_len=32768)
    kept = ops.paged_attention_workspace_bytes(tokens=8192, max_query_len=8192, **args)
    for n in (1, 4, 9, 16, 32, 33, 100, 500, 2048, 4000, 8000):
        assert 0 < ops.paged_attention_workspace_bytes(tokens=n, max_query_len=n, **args) <= kept


def test_the_size_needs_no_buffers():
    from spock_amd import _lib, ops
    lib = _lib.lib()
    cache = _lib.SpkPagedCache(_lib.SPK_BF16, 2, 256, 16, 100, 2048, 3, 40)
    a = _lib.SpkPagedAttnArgs(cache, 8, 20, 32768)
    want = ops.paged_attention_workspace_bytes(40, 8, 2, 256, 16, 2048, 3, 20, 32768)
    assert lib.spk_paged_attention_workspace_size(C.byref(a)) == want > 0
    assert lib.spk_paged_attention(C.byref(a), None) == -1      # the call itself does need them
    for bad in (dict(num_q_heads=7), dict(window=-1), dict(max_context_len=-1)):
        b = _lib.SpkPagedAttnArgs(cache, 8, 20, 32768)
        for k, v in bad.items():
            setattr(b, k, v)
        assert lib.spk_paged_attention_workspace_size(C.byref(b)) == 0


def test_what_one_call_needs(shim):
    """The need of the call alone, as the plan and the refusal of a misaligned workspace have it."""
    import re
    from spock_amd import _lib
    lib = _lib.lib()
    assert lib.spk_paged_attention_workspace_need(None) == 0
    out = (C.c_int * 8)()
    for tokens, seqs, q, c in ((1, 1, 1, 32768), (9, 1, 9, 32768), (8192, 1, 8192, 32768), (16384, 1, 16384, 131072), (64, 64, 1, 16000), (700, 6, 500, 3000)):
        cache = _lib.SpkPagedCache(_lib.SPK_F16, 2, 256, 16, 100, 8192, seqs, tokens, 256, 256, 16384, 1024, 256, 256, 8192, 256, 256)
        a = _lib.SpkPagedAttnArgs(cache, 8, q, c, 0, 0.0, 256, 256, 256, None, 0, 0, 256, 256, 256, None, 264, 1 << 60)
        need = lib.spk_paged_attention_workspace_need(C.byref(a))
        assert need == shim.plan((C.c_int * 10)(8, 2, 256, 16, 8192, seqs, tokens, q, c, 0), None, None, out)
        assert need <= lib.spk_paged_attention_workspace_size(C.byref(a))
        if need:    # else it would be launched
            assert lib.spk_paged_attention(C.byref(a), None) == -5
            assert int(re.search(rb"(\d+) needed", lib.spk_last_error()).group(1)) == need
    assert lib.spk_paged_attention_workspace_need(C.byref(a)) > 0
