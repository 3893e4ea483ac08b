"""GPU runs of verify_drafts at the ends of the temperatures' range: +inf counts
as the largest finite float, at which finite 16-bit logits are alike.

At 3e38 log2(e) / T has an error of half a denormal step (1.5e-7 relative),
times exponents below 2 here: within the ten roundings that a row's sum has."""
import numpy as np
import pytest

from test_gpu_verify import _call, _case, _check, _inputs, _want

pytestmark = pytest.mark.gpu

MOST = np.finfo(np.float32).max


def _run(c, dev):
    import torch
    got = _call(_inputs(c, dev))
    torch.cuda.synchronize()
    _check(got, _want(dict(c, temperature=np.minimum(c["temperature"], MOST))))
    return got


@pytest.mark.parametrize("vocab", [7, 5000])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_the_highest_are_uniform(dev, dtype, vocab):
    print(f"[verify at infinite temperature {dtype} {vocab}]", flush=True)
    c = _case(40 + vocab, vocab, [3, 1, 2, 4] * 5, dtype, temps=(np.inf, 3e38, 1e31, MOST))
    c["target"][4, 1:] = c["draft"][8, ::2] = -float("inf")
    got = _run(c, dev)
    assert bool((got[1].cpu()[::4] >= 0).all()) and bool((got[0].cpu()[np.cumsum([0] + [3, 1, 2, 4] * 5)[:-1]] >= 0).all())
    _run(dict(c, draft=None), dev)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_logits_as_large_as_the_temperature(dev, dtype):
    print(f"[verify large logits {dtype}]", flush=True)
    c = _case(41, 3000, [4, 2, 1] * 8, dtype, std=2e37, near=1e37, temps=(3e38, 1e38, 2e37, np.inf))
    _run(c, dev)
