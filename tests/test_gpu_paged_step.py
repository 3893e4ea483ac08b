"""GPU runs of the paged serving operators as they are used: a step of drafted
tokens through all three, captured and replayed with the lengths that the step
before left on the device; batches of more sequences than a wave looks at
together; bounds that do not hold; two calls at once.  Bars as in
test_gpu_paged.py and test_gpu_verify.py."""
import numpy as np
import pytest
import torch

import paged_ref as R
import verify_ref as V
from test_gpu_paged import DT, _attend, _check, _i32, _normal, _tables
from test_gpu_verify import _case, _check as _check_verify, _run

pytestmark = pytest.mark.gpu


def test_drafted_steps_through_all_three_operators(dev):
    """Rotation and store, attention, verification, and the accepted lengths as the next step's, in one graph: every
    step as the definitions say of what the step before left, eager steps in between."""
    from spock_amd import ops
    print("[drafted steps]", flush=True)
    gen = torch.Generator().manual_seed(5)
    rows, page, heads, kv, dim, cols = [5, 3, 1, 9], 16, 8, 2, 256, 14
    S, T, vocab = len(rows), sum(rows), heads * dim     # the attention's output of a token serves as its logits
    cu = [0] + np.cumsum(rows).tolist()
    table = torch.from_numpy(np.random.default_rng(1).permutation(S * cols + 3)[:S * cols].reshape(S, cols).astype(np.int32))
    angle = torch.arange(400)[:, None].double() * 1e4 ** (-torch.arange(32).double() / 32)
    rope = torch.stack([angle.cos(), angle.sin()], -1).reshape(400, 64).float()
    axis = [i % 3 for i in range(32)]
    f16 = torch.float16
    shapes = {"q": (T, heads, dim), "k": (T, kv, dim), "v": (T, kv, dim), "draft": (T, vocab)}
    buf = {n: torch.zeros(*s, dtype=f16, device=dev) for n, s in shapes.items()}
    kc, vc = (_normal(gen, S * cols + 3, page, kv, dim, dtype=f16).to(dev) for _ in range(2))
    pos, tokens = torch.zeros(3, T, dtype=torch.int32, device=dev), torch.zeros(T, dtype=torch.int32, device=dev)
    u, us = torch.zeros(T, device=dev), torch.zeros(S, device=dev)
    temp = torch.tensor([1.0, 0.02, 0.5, 0.0], device=dev)
    dtable, dcu, drope, dn = table.to(dev), _i32(cu, dev), rope.to(dev), _i32(rows, dev)
    ctx = _i32([100, 3, 1, 60], dev)                    # with this step's rows
    left = torch.zeros(S, dtype=torch.int32, device=dev)
    qo, out = torch.zeros(T, heads, dim, dtype=f16, device=dev), torch.zeros(T, heads, dim, dtype=f16, device=dev)
    lse, logp = torch.zeros(T, heads, device=dev), torch.zeros(T, device=dev)
    got, accepted = torch.zeros(T, dtype=torch.int32, device=dev), torch.zeros(S, dtype=torch.int32, device=dev)
    ws = torch.empty(max(1, ops.paged_attention_workspace_bytes(T, heads, kv, dim, page, cols, S, 9, cols * page)), dtype=torch.uint8, device=dev)
    wv = torch.empty(ops.verify_workspace_bytes(vocab, S, T), dtype=torch.uint8, device=dev)

    def step():
        ops.mrope_append(buf["q"], buf["k"], buf["v"], pos, drope, axis, kc, vc, dtable, dcu, ctx, out=qo)
        ops.paged_attention(qo, kc, vc, dtable, dcu, ctx, 9, cols * page, out=out, lse=lse, workspace=ws)
        ops.verify_drafts(out.view(T, vocab), tokens, dcu, u, us, draft=buf["draft"], temperature=temp, context_lens=ctx,
                          out_tokens=got, accepted=accepted, logprobs=logp, context_out=left, workspace=wv)

    def fill():
        for n, t in buf.items():
            t.copy_(_normal(gen, *t.shape, dtype=f16, std=0.3 if n == "draft" else 1.0))
        pos.copy_(torch.randint(0, 400, (3, T), generator=gen, dtype=torch.int32))
        tokens.copy_(torch.randint(0, vocab, (T,), generator=gen, dtype=torch.int32))
        u.copy_(torch.rand(T, generator=gen) * 0.9)
        us.copy_(torch.rand(S, generator=gen))

    def check(before, at):
        lens = at.tolist()
        cpu = lambda t: t.cpu()
        rq, rk, rv = R.mrope_append(cpu(buf["q"]), cpu(buf["k"]), cpu(buf["v"]), cpu(pos), rope, axis, *before, table, cu, lens)
        assert torch.equal(vc.cpu().double(), rv)
        assert bool(((kc.cpu().double() - rk).abs() <= 2.0 ** -11 * rk.abs() + 2.0 ** -19).all())
        assert bool(((qo.cpu().double() - rq).abs() <= 2.0 ** -11 * rq.abs() + 2.0 ** -19).all())
        _check(out.cpu(), lse.cpu(), R.attention(qo.cpu(), kc.cpu(), vc.cpu(), table, cu, lens))
        want = V.verify(out.view(T, vocab).float().cpu().numpy(), tokens.cpu().numpy(), np.array(cu, np.int32), u.cpu().numpy(),
                        us.cpu().numpy(), draft=buf["draft"].float().cpu().numpy(), kind="logits", temperature=temp.cpu().numpy(),
                        context=np.array(lens, np.int32))
        _check_verify((got, accepted, logp, left), want)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    some = 0
    for replay in range(6):
        fill()
        before, at = (kc.cpu(), vc.cpu()), ctx.cpu()
        graph.replay()
        torch.cuda.synchronize()
        check(before, at)
        kept = out.clone(), got.clone(), left.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, kept[0]) and torch.equal(got, kept[1]) and torch.equal(left, kept[2])
        some += int(accepted.sum())
        ctx.copy_(left + dn)                            # the next step's rows behind what was accepted
    assert some > 0


@pytest.mark.parametrize("long", [0, 3])
@pytest.mark.parametrize("dtype,heads,kv,dim", [("f16", 8, 2, 64), ("bf16", 16, 1, 128)])
def test_more_sequences_than_are_looked_at_together(dev, dtype, heads, kv, dim, long):
    print(f"[300 sequences {dtype} {heads}/{kv}x{dim} long {long}]", flush=True)
    rng = np.random.default_rng(dim + long)
    lens = [(int(n), int(n + c)) for n, c in zip(rng.integers(0, 4, 300), rng.integers(0, 90, 300))]
    for i in range(long):
        lens[(7, 150, 299)[i]] = ((90, 300), (270, 270), (33, 700))[i]
    gen = torch.Generator().manual_seed(dim)
    cu, ctx, table, pages = _tables(lens, 16, dim)
    kc, vc = (_normal(gen, pages, 16, kv, dim, dtype=DT[dtype]) for _ in range(2))
    q = _normal(gen, cu[-1], heads, dim, dtype=DT[dtype], std=2.0)
    ref = R.attention(q, kc, vc, table, cu, ctx)
    _check(*_attend(dev, q, kc, vc, table, cu, ctx), ref)
    _check(*_attend(dev, q, kc, vc, table, cu, ctx, max_c=100000), ref)


@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("dtype,heads,kv,dim", [("f16", 8, 2, 64), ("bf16", 12, 3, 128), ("f16", 4, 1, 256)])
def test_prompts_of_mixed_lengths(dev, dtype, heads, kv, dim, window):
    """Every row of prompts that are cut into tiles in the order of their keys, with short sequences, one without rows
    and one with more new tokens than positions among them."""
    lens = [(300, 900), (1, 700), (0, 5), (500, 400), (90, 1500), (257, 257), (2, 2), (64, 128)]
    print(f"[mixed prompts {dtype} {heads}/{kv}x{dim} window {window}]", flush=True)
    gen = torch.Generator().manual_seed(dim + window)
    cu, ctx, table, pages = _tables(lens, 20, dim)
    kc, vc = (_normal(gen, pages, 20, kv, dim, dtype=DT[dtype]) for _ in range(2))
    q = _normal(gen, cu[-1], heads, dim, dtype=DT[dtype], std=2.0)
    _check(*_attend(dev, q, kc, vc, table, cu, ctx, window=window), R.attention(q, kc, vc, table, cu, ctx, window=window))


@pytest.mark.parametrize("max_q", [1, 3, 17, 64, 5000])
@pytest.mark.parametrize("lens", [[(40, 90)], [(1, 300)], [(3, 70), (100, 150), (1, 30)], [(9, 400), (20, 60)]], ids=str)
def test_query_bound_does_not_change_the_result(dev, lens, max_q):
    print(f"[query bound {max_q} {lens}]", flush=True)
    gen = torch.Generator().manual_seed(max_q)
    cu, ctx, table, pages = _tables(lens, 16, max_q)
    kc, vc = (_normal(gen, pages, 16, 2, 128, dtype=torch.float16) for _ in range(2))
    q = _normal(gen, cu[-1], 8, 128, dtype=torch.float16)
    ref = R.attention(q, kc, vc, table, cu, ctx)
    for max_c in (max(ctx), 9000):
        _check(*_attend(dev, q, kc, vc, table, cu, ctx, max_q=max_q, max_c=max_c), ref)


def test_two_calls_at_once(dev):
    """Calls on two streams, each with its own outputs and workspace, are as one after the other."""
    from spock_amd import ops
    print("[two calls at once]", flush=True)
    gen = torch.Generator().manual_seed(8)
    calls = []
    for lens in ([(1, 3000), (4, 500)], [(300, 2000)]):
        cu, ctx, table, pages = _tables(lens, 16, len(lens))
        kc, vc = (_normal(gen, pages, 16, 2, 128, dtype=torch.float16).to(dev) for _ in range(2))
        q = _normal(gen, cu[-1], 8, 128, dtype=torch.float16).to(dev)
        n = max(b - a for a, b in zip(cu, cu[1:]))
        need = ops.paged_attention_workspace_bytes(cu[-1], 8, 2, 128, 16, table.shape[1], len(lens), n, max(ctx))
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        calls.append((lambda out, q=q, kc=kc, vc=vc, t=table.to(dev), cu=_i32(cu, dev), c=_i32(ctx, dev), n=n, m=max(ctx), ws=ws:
                      ops.paged_attention(q, kc, vc, t, cu, c, n, m, out=out, workspace=ws), torch.empty_like(q)))
    want = []
    for call, out in calls:
        call(out)
        torch.cuda.synchronize()
        want.append(out.clone())
    streams = [torch.cuda.Stream() for _ in calls]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for (call, out), s in zip(calls, streams):
            with torch.cuda.stream(s):
                out.zero_()
                call(out)
        torch.cuda.synchronize()
        for (_, out), w in zip(calls, want):
            assert torch.equal(out, w)


@pytest.mark.parametrize("u", [0.0, 0.4, 0.999999])
def test_draw_from_more_pieces_than_threads(dev, u):
    """A vocabulary whose pieces take two passes of the workgroup that draws."""
    print(f"[draw from 1,300,001 entries at {u}]", flush=True)
    c = _case(3, 1300001, [2], "f16")
    c["u_sample"][:] = u
    _run(c, dev)
