"""GPU parity of spk_verify_drafts against the definition in 64 bits
(verify_ref.py).  Tokens, counts and lengths are equal; log-probabilities are
off by at most 10 fp32 roundings of the row's sum of exponentials (the
exponential's unit in the last place, three levels of an 8-term sum) and one
of the result."""
import numpy as np
import pytest
import torch

import verify_ref as R

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _case(seed, vocab, rows, dtype, kind="logits", draft=True, near=0.5, std=2.5, temps=(1.0,)):
    """Targets, drafters near them, and tokens drawn from the drafters' rows."""
    rng = np.random.default_rng(seed)
    T, S = sum(rows), len(rows)
    x = rng.normal(size=(T, vocab)) * std
    y = x + rng.normal(size=(T, vocab)) * near
    temp = np.array([temps[s % len(temps)] for s in range(S)], np.float32)
    hot = np.repeat(np.where(temp > 0, temp, 1e-2), rows)[:, None]
    if kind == "probs":
        x, y = (np.exp(z) / np.exp(z).sum(-1, keepdims=True) for z in (x, y))
    target, drafts = (torch.from_numpy(z).to(DT[dtype]) for z in (x, y))
    z = (np.log(np.maximum(drafts.double().numpy(), 1e-30)) if kind == "probs" else drafts.double().numpy()) / hot
    drawn = (z + rng.gumbel(size=z.shape)).argmax(-1)
    tokens = np.concatenate([[0], drawn[:-1]]).astype(np.int32) if T else np.zeros(0, np.int32)
    return dict(target=target, draft=drafts if draft else None, tokens=tokens, cu=np.concatenate([[0], np.cumsum(rows)]).astype(np.int32),
                u_accept=rng.random(T, dtype=np.float32), u_sample=rng.random(S, dtype=np.float32), kind=kind,
                temperature=temp if kind == "logits" else None, context=rng.integers(50, 5000, S).astype(np.int32))


def _np(t):
    return None if t is None else t.float().numpy()


def _want(c):
    return R.verify(_np(c["target"]), c["tokens"], c["cu"], c["u_accept"], c["u_sample"], draft=_np(c["draft"]), kind=c["kind"],
                    temperature=c["temperature"], context=c["context"])


def _inputs(c, dev):
    d = {k: torch.from_numpy(c[k]).to(dev) if isinstance(c[k], np.ndarray) else c[k] for k in c}
    d["target"] = d["target"].to(dev)
    d["draft"] = None if d["draft"] is None else d["draft"].to(dev)
    return d


def _call(d, **kw):
    from spock_amd import ops
    return ops.verify_drafts(d["target"], d["tokens"], d["cu"], d["u_accept"], d["u_sample"], draft=d["draft"], kind=d["kind"],
                             temperature=d["temperature"], context_lens=d["context"], **kw)


def _check(got, want):
    tokens, accepted, logp, ctx = (x.cpu().numpy() for x in got)
    rows = want[0] != -99
    assert np.array_equal(accepted, want[1]), (accepted, want[1])
    assert np.array_equal(tokens[rows], want[0][rows]), (tokens[rows], want[0][rows])
    assert np.array_equal(ctx, want[3])
    a, b = logp[rows].astype(np.float64), want[2][rows]
    same = (a == b) | (np.isnan(a) & np.isnan(b))
    off = np.where(same, 0.0, np.abs(np.where(same, 0, a) - np.where(same, 0, b)))
    assert np.all(off <= 10 * 2.0 ** -23 + 2.0 ** -24 * np.abs(np.where(same, 0, b))), off.max()


def _run(c, dev, **kw):
    got = _call(_inputs(c, dev), **kw)
    torch.cuda.synchronize()
    _check(got, _want(c))
    return got


@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 1000, 4095, 4096, 4097, 12289, 50021])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_logits(dev, dtype, vocab):
    print(f"[verify logits {dtype} {vocab}]", flush=True)
    for seed, (rows, draft, temps) in enumerate([([1], True, (1.0,)), ([5, 3, 1, 0, 9], True, (0.7, 1.0, 1.3)),
                                                 ([4, 4, 2], False, (1.0, 0.0)), ([2] * 70, True, (0.0, 0.9, -1.0))]):
        _run(_case(seed + vocab, vocab, rows, dtype, draft=draft, temps=temps, near=0.3 if seed % 2 else 1.0), dev)


@pytest.mark.parametrize("vocab", [3, 513, 4096, 9001])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("draft", [True, False])
def test_probs(dev, draft, dtype, vocab):
    print(f"[verify probs {dtype} {vocab} {draft}]", flush=True)
    for seed, rows in enumerate([[1], [6, 2, 1, 4], [3] * 30]):
        _run(_case(seed + vocab, vocab, rows, dtype, kind="probs", draft=draft, std=1.5), dev)


def test_large_vocabulary(dev):
    _run(_case(3, 248320, [5, 1, 3], "f16", temps=(0.8, 0.0, 1.0)), dev)
    _run(_case(4, 248321, [2, 2], "f32", temps=(1.0,)), dev)


def test_many_drawn_tokens(dev):
    """Flat distributions over many tokens: the drawn one lies between close running sums every time."""
    for dtype in ("f16", "f32"):
        _run(_case(5, 30000, [2] * 120, dtype, std=0.5, near=0.2), dev)
        _run(_case(6, 30000, [1] * 120, dtype, std=0.3), dev)


def test_equality_is_a_refusal_and_sums_are_strict(dev):
    """Probabilities and numbers that binary fractions hold exactly: u q == p refuses, C == u total goes on."""
    V = 8
    target = torch.tensor([[.25, .25, 0, .25, .25, 0, 0, 0]] * 6)
    draft = torch.tensor([[.5, 0, .5, 0, 0, 0, 0, 0]] * 6)
    tokens = np.array([9, 0, 7, 0, 5, 2], np.int32)  # pairs (input, draft): drafts 0, 0, 2
    c = dict(target=target, draft=draft, tokens=tokens, cu=np.array([0, 2, 4, 6], np.int32),
             u_accept=np.array([.5, 0, .25, 0, 0, 0], np.float32), u_sample=np.array([0.0, .75, 1 / 3], np.float32), kind="probs",
             temperature=None, context=np.array([10, 20, 30], np.int32))
    got = _run(c, dev)
    # .5 * .5 == .25 refuses, residual {1, 3, 4}: u = 0 takes the first with weight; .25 * .5 < .25 accepts, C = .75 goes on to 4;
    # p = 0 refuses at u = 0
    assert got[0].cpu().tolist() == [1, -1, 0, 4, 3, -1] and got[1].cpu().tolist() == [0, 1, 0]
    for u, token in ((0.0, 0), (.25, 1), (.499, 1), (.5, 3), (.75, 4), (0.9999999, 4), (1.0, 4), (2.0, 4)):
        one = dict(c, target=target[:1], draft=None, tokens=tokens[:1], cu=np.array([0, 1], np.int32), u_accept=c["u_accept"][:1],
                   u_sample=np.array([u], np.float32), context=c["context"][:1])
        assert _run(one, dev)[0].item() == token


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_masked_and_broken_rows(dev, dtype):
    """Logits of -inf, rows without a finite logit, NaN and +inf: refused and, drawn from, -1; the largest masked."""
    lowest = torch.finfo(DT[dtype]).min
    c = _case(7, 5000, [3] * 8, dtype, temps=(1.0, 1.0, 0.0, 0.5))
    t, q = c["target"], c["draft"]
    t[0, 100:] = -float("inf")
    t[3, :] = -float("inf")
    t[4, 17] = float("nan")
    t[7, :] = -float("inf")
    t[9, 3] = float("inf")
    t[12, 1:] = lowest
    t[13, :] = lowest
    q[15, 40] = float("nan")
    t[18, ::2] = -float("inf")
    q[18, 1::2] = -float("inf")
    _run(c, dev)


def test_ties_take_the_lowest_index(dev):
    c = _case(8, 9000, [2] * 6, "f16", temps=(0.0,))
    for i, at in enumerate(([5, 6], [8999, 4096], [0, 8999], [4095, 4096], [777, 300, 8000], [1, 2])):
        c["target"][2 * i, at] = 50.0
        c["tokens"][2 * i + 1] = min(at) if i % 2 else max(at)
    got = _run(c, dev)
    assert got[1].cpu().tolist() == [0, 1, 0, 1, 0, 1]


def test_identical_distributions_accept_everything(dev):
    c = _case(9, 3000, [9] * 5, "bf16", near=0.0, temps=(0.6, 1.0))
    got = _run(c, dev)
    assert got[1].cpu().tolist() == [8] * 5


def test_tokens_outside_the_vocabulary_and_offsets_outside_the_rows(dev):
    c = _case(10, 600, [3, 3, 3, 3], "f32")
    c["tokens"][[1, 5, 7, 10]] = [-1, 600, 2 ** 31 - 1, -2 ** 31]
    _run(c, dev)
    c["draft"] = None
    _run(c, dev)
    c = _case(11, 600, [3, 3], "f16")
    c["cu"] = np.array([-4, 2, 900], np.int32)
    _run(c, dev)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_strides_offsets_and_rows_behind(dev, dtype):
    """Rows inside a wider buffer from an odd element on; buffers of the caller's; rows past the last sequence stay."""
    c = _case(12, 1001, [4, 2], dtype)
    want = _want(c)
    d = _inputs(c, dev)
    for name in ("target", "draft"):
        wide = torch.full((9, 1031), 60.0, dtype=DT[dtype], device=dev)
        wide[:6, 5:1006] = d[name]
        d[name] = wide[:, 5:1006]
    pad = lambda t: torch.cat([t, t[:3]])
    d["tokens"], d["u_accept"] = pad(d["tokens"]), pad(d["u_accept"])
    out, logp = torch.full((9,), 55, dtype=torch.int32, device=dev), torch.full((9,), 5.5, device=dev)
    got = _call(d, out_tokens=out, logprobs=logp, context_out=d["context"])
    torch.cuda.synchronize()
    assert got[3].data_ptr() == d["context"].data_ptr()
    _check((out[:6], got[1], logp[:6], got[3]), want)
    assert bool((out[6:] == 55).all()) and bool((logp[6:] == 5.5).all())


def test_no_rows(dev):
    c = _case(13, 100, [0, 0], "f16")
    got = _call(_inputs(c, dev))
    torch.cuda.synchronize()
    assert got[1].cpu().tolist() == [0, 0] and np.array_equal(got[3].cpu().numpy(), c["context"])


def test_captured_and_replayed_on_new_inputs(dev):
    """One captured call over buffers whose contents change, with eager calls of the same buffers between replays."""
    cases = [_case(20 + i, 7001, [4, 1, 6], "f16", temps=(0.9, 1.0, 0.0)) for i in range(4)]
    d = _inputs(cases[0], dev)
    from spock_amd import ops
    ws = torch.empty(ops.verify_workspace_bytes(7001, 3, 11), dtype=torch.uint8, device=dev)
    bufs = dict(out_tokens=torch.zeros(11, dtype=torch.int32, device=dev), accepted=torch.zeros(3, dtype=torch.int32, device=dev),
                logprobs=torch.zeros(11, device=dev), context_out=torch.zeros(3, dtype=torch.int32, device=dev), workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _call(d, **bufs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _call(d, **bufs)
    for c in cases[1:] + cases[:2]:
        new = _inputs(c, dev)
        for k, t in new.items():
            if isinstance(t, torch.Tensor):
                d[k].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        _check(got, _want(c))
        _check(_call(d), _want(c))


def test_argument_checks(dev):
    from spock_amd import _lib, ops
    c = _inputs(_case(30, 64, [2, 2], "f16"), dev)
    good = dict(target=c["target"], tokens=c["tokens"], cu_seqlens=c["cu"], u_accept=c["u_accept"], u_sample=c["u_sample"],
                draft=c["draft"], temperature=c["temperature"], context_lens=c["context"])
    ops.verify_drafts(**good)
    for over in (dict(target=c["target"].double()), dict(target=c["target"][0]), dict(draft=c["draft"].float()), dict(draft=c["draft"][:2]),
                 dict(tokens=c["tokens"].long()), dict(cu_seqlens=c["cu"][:2]), dict(u_accept=c["u_accept"].cpu()),
                 dict(u_sample=c["u_sample"].double()), dict(kind="scores"), dict(kind="probs"), dict(context_lens=c["context"][:1]),
                 dict(out_tokens=c["tokens"]), dict(target=c["target"].t().contiguous().t()), dict(accepted=torch.zeros(3, dtype=torch.int32, device=dev))):
        with pytest.raises(_lib.SpockError):
            ops.verify_drafts(**{**good, **over})
    torch.cuda.synchronize()
