"""How paged_attention_mx4 deals its rows and keys, without a GPU: test_paged_deal's checks of csrc/paged_deal.hpp with the plan
for a cache in 4 bits, whose pieces of few rows have 16 and which keeps up to 2 head_dim rows of a sequence in them."""
import ctypes as C
import subprocess

import numpy as np
import pytest

import test_paged_deal as D
from conftest import ROOT


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("deal_mx4")
    source = D.SHIM.replace("plan_of(p)", "plan_mx4(p)").replace("workspace_bound(p)", "workspace_bound_mx4(p)")
    assert source.count("_mx4(p)") == 2
    (d / "shim.cpp").write_text(source)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-fwrapv", "-w", "-I", str(ROOT / "spock_amd" / "csrc"),
                        str(d / "shim.cpp"), "-o", str(d / "shim.so")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    lib = C.CDLL(str(d / "shim.so"))
    lib.plan.restype = lib.bound.restype = C.c_size_t
    return lib


@pytest.mark.parametrize("lens,kw", [
    ([(1, 1)], {}), ([(1, 1500)], {}), ([(1, 130001)], dict(heads=32, kv=8, max_pages=9000)), ([(9, 9)], dict(heads=7, kv=1)),
    ([(1, c) for c in range(300, 16000, 250)], {}), ([(9, 1000 + 500 * i) for i in range(16)], dict(dim=256)),
    ([(0, 10), (3, 0), (4, 2), (1, 50), (0, 0), (2, 2)], {}), ([(2048, 16384)], {}), ([(64, 900)] * 5, {}), ([(65, 900)] * 5, {}),
    ([(300, 900), (1, 700), (0, 5), (500, 400), (90, 1500), (257, 257), (2, 2), (64, 128)], dict(window=200)),
    ([(60, 300 + i) for i in range(60)], dict(heads=16, kv=4)), ([(1 + i % 4, 5 * i) for i in range(257)], dict(heads=32, kv=8)),
    ([(5, 900)] * 40, dict(max_c=1)), ([(60, 900)] * 3, dict(max_q=1)), ([(3, 70), (100, 150)], dict(max_q=5000, max_c=100000))],
    ids=lambda v: None if isinstance(v, dict) else "+".join("%d:%d" % x for x in v[:4]) + ("..%d" % len(v) if len(v) > 4 else ""))
def test_everything_is_dealt_once(shim, lens, kw):
    call = D.Call(shim, *D._cu(lens), **kw)
    call.check_shares()
    call.check_tiles()


@pytest.mark.parametrize("seed", range(8))
def test_lengths_at_random(shim, seed):
    rng = np.random.default_rng(seed)
    S = int(rng.choice([1, 2, 7, 64, 65, 200]))
    lens = [(int(rng.choice([0, 1, 4, 30, 100, 400], p=[.1, .4, .2, .1, .1, .1])), int(rng.integers(0, 5000))) for _ in range(S)]
    heads, kv, dim = [(8, 2, 256), (16, 4, 128), (7, 1, 64), (4, 4, 128), (40, 2, 64)][seed % 5]
    call = D.Call(shim, *D._cu(lens), heads=heads, kv=kv, dim=dim, page=int(rng.choice([1, 16, 20])), window=int(rng.choice([0, 0, 50, 2000])))
    call.check_shares()
    call.check_tiles()


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 256), (16, 4, 128), (7, 1, 64), (32, 8, 128)])
@pytest.mark.parametrize("most", [(8192, 64, 8192, 32768, 0), (300, 300, 9, 5000, 0), (32768, 512, 64, 4096, 0), (2000, 16, 500, 20000, 1024),
                                  (64, 64, 1, 200, 0), (700, 3, 600, 1200, 0)], ids=str)
def test_a_workspace_of_the_largest_sizes_serves_the_smaller(shim, heads, kv, dim, most):
    out = (C.c_int * 8)()

    def sizes(T, S, q, c, w):
        return (C.c_int * 10)(heads, kv, dim, 16, 10000, S, T, q, c, w)

    kept = shim.bound(sizes(*most))
    rng = np.random.default_rng(most[0] + heads)
    T, S, q, c, w = most
    log = lambda top: int(round(np.exp(rng.uniform(0, np.log(top)))))  # noqa: E731
    for x in [most] + [(log(T), log(S), log(q), log(c), w) for _ in range(6000)]:
        need = shim.plan(sizes(*x), None, None, out)
        assert need <= kept and need <= shim.bound(sizes(*x)), (x, need, kept)
        assert shim.bound(sizes(*x)) <= kept, x


@pytest.mark.parametrize("heads,kv,dim,seqs,new,ctx", [(32, 8, 128, 512, 64, 4096), (32, 8, 128, 512, 64, 256), (32, 8, 128, 1024, 1, 1500),
                                                       (8, 2, 256, 256, 64, 9000), (32, 8, 128, 64, 2, 4096)])
def test_pieces_that_fill_the_chip_are_not_all_split(shim, heads, kv, dim, seqs, new, ctx):
    """Where the pieces alone are rounds of the chip's workgroups, one round more carries what is split of them: no second
    share, with its part of the workspace and of the join, for every piece."""
    out = (C.c_int * 8)()
    need = shim.plan((C.c_int * 10)(heads, kv, dim, 16, 10000, seqs, seqs * new, new, ctx, 0), None, None, out)
    pieces = kv * (seqs * new * (heads // kv) // 16 + seqs)
    most = pieces + 2 * 768
    assert out[D.PLAN.index("share_rows")] == 16 and pieces <= out[0] <= most
    assert need <= most * 16 * (dim + 2) * 4 + seqs * new * heads * 8 + 1024
