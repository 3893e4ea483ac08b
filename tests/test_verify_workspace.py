"""What spk_verify_drafts refuses of its buffers, without a GPU.  What it needs of
its workspace, as its refusal of a misaligned one states it, never passes what
the size query told for a larger call."""
import ctypes as C
import re

import numpy as np
import pytest


def _need(lib, _lib, vocab, seqs, rows):
    a = _lib.SpkVerifyArgs(0, _lib.SPK_F16, vocab, seqs, rows, 256, 256, 256, vocab, None, 0, None, 256, 256, 512, 256, None, None,
                           None, 264, 1 << 40)
    assert lib.spk_verify_drafts(C.byref(a), None) == -5
    return int(re.search(rb"(\d+) needed", lib.spk_last_error()).group(1))


@pytest.mark.parametrize("vocab,seqs,rows", [(248320, 64, 384), (248320, 9, 54), (1000, 65535, 65535), (100003, 48, 192), (1, 3, 9),
                                             (1300001, 2, 2), (50021, 400, 2000)])
def test_a_workspace_of_the_largest_sizes_serves_the_smaller(vocab, seqs, rows):
    from spock_amd import _lib
    lib = _lib.lib()
    size = lib.spk_verify_drafts_workspace_size
    kept, largest = size(vocab, seqs, rows), 0
    rng = np.random.default_rng(vocab)
    log = lambda top: int(round(np.exp(rng.uniform(0, np.log(top)))))
    tried = [(vocab, seqs, rows)] + [(log(vocab), log(seqs), log(rows)) for _ in range(3000)]
    tried += [(vocab, s, r) for s in range(1, min(seqs, 70) + 1) for r in range(1, min(rows, 60) + 1)]
    for v, s, r in tried:
        need = _need(lib, _lib, v, s, r)
        assert need <= size(v, s, r) <= kept, (v, s, r, need, kept)
        largest = max(largest, need)
    assert kept <= 2 * largest + 4096, (kept, largest)


@pytest.mark.parametrize("out", ["out_tokens", "accepted", "logprobs", "context_out"])
@pytest.mark.parametrize("other", ["cu_seqlens", "tokens", "target", "draft", "temperature", "u_accept", "u_sample", "context_lens", "out_tokens",
                                   "accepted", "logprobs", "context_out"])
def test_an_output_is_no_other_buffer(out, other):
    """A workgroup would read what another one wrote."""
    from spock_amd import _lib
    lib = _lib.lib()
    if out == other or (out, other) in (("context_out", "context_lens"), ("out_tokens", "tokens")):
        return
    names = ("cu_seqlens", "tokens", "target", "draft", "temperature", "u_accept", "u_sample", "out_tokens", "accepted", "logprobs",
             "context_lens", "context_out", "workspace")
    a = _lib.SpkVerifyArgs(0, _lib.SPK_F16, 100, 2, 6)
    for i, n in enumerate(names):
        setattr(a, n, 4096 * (i + 1))
    a.target_stride = a.draft_stride = 100
    a.workspace_bytes = 1 << 20
    setattr(a, out, getattr(a, other))
    assert lib.spk_verify_drafts(C.byref(a), None) == -5 and b"output" in lib.spk_last_error(), lib.spk_last_error()
