"""Python host side of the MI355X hot path: thin wrappers that hand device
tensors (torch, ROCm) to the C ABI on the current HIP stream.

torch is only plumbing here (device memory, streams); every computation is a
hand-written gfx950 kernel behind include/spock_hip.h.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib
from ._lib import (SpkChunkArgs, SpkDecodeArgs, SpkMatvecDesc, SpkMropeArgs, SpkPagedAttnArgs, SpkPagedCache,
                   SpkVerifyArgs, check, lib)

KEY_DIM = 128
VALUE_DIM = 128
CHUNK = 64


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _dev(t: torch.Tensor, dtype=None) -> torch.Tensor:
    if not t.is_cuda:
        raise _lib.SpockError("expected a device tensor")
    if dtype is not None and t.dtype != dtype:
        raise _lib.SpockError(f"expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise _lib.SpockError("expected a contiguous tensor")
    return t


# ----------------------------------------------------------------------------
# chunk prefill
# ----------------------------------------------------------------------------
_CU_CHECKED: dict = {}


def _check_cu_dev(cu_dev: torch.Tensor, cu_host: np.ndarray, dev) -> None:
    """The launch is sized from the host copy; for packs of more than 32
    sequences the kernels find the sequences through the device copy, so the
    two must agree (the kernels keep every access in bounds either way, but a
    differing copy gives wrong results).  The comparison reads the device
    tensor back once per (buffer, torch version counter, host offsets) and is
    cached, so repeated calls stay asynchronous: offsets rewritten behind
    torch's back (through a raw pointer, without a version bump) are not seen
    again, and must not be."""
    if cu_dev.device != dev or cu_dev.dtype != torch.int32 or not cu_dev.is_contiguous():
        raise _lib.SpockError("chunk_prefill: cu_seqlens_dev must be a contiguous int32 tensor on q's device")
    if cu_dev.numel() != cu_host.size:
        raise _lib.SpockError(f"chunk_prefill: cu_seqlens_dev has {cu_dev.numel()} entries, cu_seqlens {cu_host.size}")
    key = (cu_dev.data_ptr(), cu_dev._version, cu_host.tobytes())
    if key in _CU_CHECKED:
        return
    if not np.array_equal(cu_dev.cpu().numpy(), cu_host):
        raise _lib.SpockError("chunk_prefill: cu_seqlens_dev differs from cu_seqlens")
    if len(_CU_CHECKED) > 64:
        _CU_CHECKED.clear()
    _CU_CHECKED[key] = True


def chunk_workspace_bytes(num_heads: int, total_tokens: int, num_seqs: int = 1) -> int:
    return int(lib().spk_chunk_prefill_workspace_size(num_heads, total_tokens, num_seqs, CHUNK))


def chunk_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor,
                  beta: torch.Tensor, initial_state: Optional[torch.Tensor] = None,
                  cu_seqlens: Optional[Sequence[int]] = None, use_qk_l2norm: bool = False,
                  q_scale: float = 0.0, out_core: Optional[torch.Tensor] = None,
                  out_state: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None, core_head_stride: int = 0,
                  cu_seqlens_dev: Optional[torch.Tensor] = None):
    """Gated-DeltaNet chunk prefill (spk_chunk_prefill).

    q, k: [H][N][128], v: [H][N][128] (float32 or float16, device);
    g, beta: [H][N] float32; cu_seqlens: host sequence offsets (None = one
    sequence; cu_seqlens_dev optionally holds the same offsets already on the
    device, int32).  Returns (core [H][N][128] f32, state [S][H][128][128] f32).
    """
    if q.dim() != 3:
        raise _lib.SpockError(f"chunk_prefill: q must be [H][N][128], got {tuple(q.shape)}")
    H, N, dk = q.shape
    if dk != KEY_DIM:
        raise _lib.SpockError("chunk_prefill: key_dim and value_dim must be 128")
    for name, t in (("k", k), ("v", v)):
        if tuple(t.shape) != (H, N, KEY_DIM):
            raise _lib.SpockError(f"chunk_prefill: {name} shape {tuple(t.shape)} != q shape {(H, N, KEY_DIM)}")
    for name, t in (("g", g), ("beta", beta)):
        if tuple(t.shape) != (H, N):
            raise _lib.SpockError(f"chunk_prefill: {name} shape {tuple(t.shape)} != {(H, N)}")
    dtype = q.dtype
    if dtype not in (torch.float32, torch.float16):
        raise _lib.SpockError("chunk_prefill: q/k/v must be float32 or float16")
    for t in (q, k, v):
        _dev(t, dtype)
    _dev(g, torch.float32)
    _dev(beta, torch.float32)
    dev = q.device
    if cu_seqlens is None:
        S = 1
        cu_dev = None
        cu_host = None
        if cu_seqlens_dev is not None:
            raise _lib.SpockError("chunk_prefill: cu_seqlens_dev given without cu_seqlens")
    else:
        cu_host = np.ascontiguousarray(np.asarray(cu_seqlens, dtype=np.int32))
        S = len(cu_host) - 1
        if cu_seqlens_dev is not None:
            _check_cu_dev(cu_seqlens_dev, cu_host, dev)
            cu_dev = cu_seqlens_dev
        else:
            cu_dev = torch.from_numpy(cu_host.copy()).to(dev)
    state_elems = S * H * KEY_DIM * VALUE_DIM
    if initial_state is not None:
        _dev(initial_state, torch.float32)
        if initial_state.numel() != state_elems:
            raise _lib.SpockError(f"chunk_prefill: initial_state must hold [S={S}][H={H}][128][128] "
                                  f"= {state_elems} floats, got {initial_state.numel()}")
    hs = core_head_stride or N
    if out_core is None:
        if hs != N:
            raise _lib.SpockError("chunk_prefill: core_head_stride needs an out_core buffer")
        out_core = torch.empty((H, N, VALUE_DIM), dtype=torch.float32, device=dev)
    else:
        _dev(out_core, torch.float32)
        if hs < N or out_core.numel() < ((H - 1) * hs + N) * VALUE_DIM:
            raise _lib.SpockError(f"chunk_prefill: out_core holds {out_core.numel()} floats, "
                                  f"rows (h*{hs} + t) for H={H}, N={N} need {((H - 1) * hs + N) * VALUE_DIM}")
    if out_state is None:
        out_state = torch.empty((S, H, KEY_DIM, VALUE_DIM), dtype=torch.float32, device=dev)
    else:
        _dev(out_state, torch.float32)
        if out_state.numel() < state_elems:
            raise _lib.SpockError(f"chunk_prefill: out_state holds {out_state.numel()} floats, need {state_elems}")
    need = chunk_workspace_bytes(H, N, S)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    a = SpkChunkArgs()
    a.num_heads, a.total_tokens, a.key_dim, a.value_dim, a.chunk_size = H, N, KEY_DIM, VALUE_DIM, CHUNK
    a.use_qk_l2norm = int(bool(use_qk_l2norm))
    a.q_scale = float(q_scale)
    a.input_dtype = _lib.SPK_F32 if dtype == torch.float32 else _lib.SPK_F16
    a.q, a.k, a.v, a.g, a.beta = map(_ptr, (q, k, v, g, beta))
    a.initial_state = _ptr(initial_state)
    a.out_core = _ptr(out_core)
    a.core_head_stride = core_head_stride
    a.out_state = _ptr(out_state)
    a.cu_seqlens = _ptr(cu_dev)
    a.cu_seqlens_host = None if cu_host is None else cu_host.ctypes.data
    a.num_seqs = S
    a.workspace = _ptr(workspace)
    a.workspace_bytes = workspace.numel() * workspace.element_size()
    check(lib().spk_chunk_prefill(C.byref(a), _stream()), "spk_chunk_prefill")
    return out_core, out_state


def prefill_collect(dn_qkv: torch.Tensor, g_beta: torch.Tensor, bufs, seq_len: int, token_idx: int,
                    num_heads: int = 16) -> None:
    qo, ko, vo, go, bo = bufs
    check(lib().spk_prefill_collect(_ptr(dn_qkv), _ptr(g_beta), _ptr(qo), _ptr(ko), _ptr(vo),
                                    _ptr(go), _ptr(bo), num_heads, seq_len, token_idx, KEY_DIM,
                                    VALUE_DIM, _stream()), "spk_prefill_collect")


def chunk_last_to_fp16(src: torch.Tensor, seq_len: int, total_seq: int, num_heads: int = 16,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    if out is None:
        out = torch.empty(num_heads * VALUE_DIM, dtype=torch.float16, device=src.device)
    check(lib().spk_chunk_last_to_fp16(_ptr(src), _ptr(out), num_heads, VALUE_DIM, seq_len,
                                       total_seq, _stream()), "spk_chunk_last_to_fp16")
    return out


# ----------------------------------------------------------------------------
# decode step
# ----------------------------------------------------------------------------
_DECODE_FNS = {
    "fused": "spk_deltanet_decode_step",
    "conv_l2_qk": "spk_deltanet_conv_l2_qk",
    "gbeta_norm_gate": "spk_deltanet_recurrent_gbeta_norm_gate",
    "recurrent": "spk_deltanet_recurrent",
}


def decode_step(qkv: torch.Tensor, state: torch.Tensor, conv_state: Optional[torch.Tensor] = None,
                conv_weight: Optional[torch.Tensor] = None, a: Optional[torch.Tensor] = None,
                b: Optional[torch.Tensor] = None, a_log_bias: Optional[torch.Tensor] = None,
                z: Optional[torch.Tensor] = None, norm_weight: Optional[torch.Tensor] = None,
                layer_idx: int = 0, q_scale: float = 0.0, rms_eps: float = 0.0,
                variant: str = "fused", num_heads: int = 16) -> None:
    """In-place batched DeltaNet decode step over the leading batch dim of
    qkv [B][6144] fp16, state [B][...] fp32, conv_state [B][6144][4] fp16,
    a/b [B][16] fp16, z [B][2048] fp16."""
    B = qkv.shape[0]
    d = SpkDecodeArgs()
    d.batch, d.num_heads, d.layer_idx = B, num_heads, layer_idx
    d.q_scale, d.rms_eps = float(q_scale), float(rms_eps)
    d.qkv, d.qkv_stride = _ptr(qkv), qkv[0].numel() if B else 0
    if conv_state is not None:
        d.conv_state, d.conv_state_stride = _ptr(conv_state), conv_state[0].numel()
    d.conv_weight = _ptr(conv_weight)
    if a is not None:
        d.a, d.b, d.ab_stride = _ptr(a), _ptr(b), a[0].numel()
    d.a_log_bias = _ptr(a_log_bias)
    d.state, d.state_stride = _ptr(state), state[0].numel() if B else 0
    if z is not None:
        d.z, d.z_stride = _ptr(z), z[0].numel()
    d.norm_weight = _ptr(norm_weight)
    name = _DECODE_FNS[variant]
    check(getattr(lib(), name)(C.byref(d), _stream()), name)


# ----------------------------------------------------------------------------
# GEMV / lm_head / argmax
# ----------------------------------------------------------------------------
def matvec_f16(W: torch.Tensor, x: torch.Tensor, y: Optional[torch.Tensor] = None) -> torch.Tensor:
    out_dim, in_dim = W.shape
    if y is None:
        y = torch.empty(out_dim, dtype=torch.float16, device=W.device)
    check(lib().spk_matvec_f16(_ptr(W), _ptr(x), _ptr(y), out_dim, in_dim, _stream()),
          "spk_matvec_f16")
    return y


MATVEC_ORDERS = {"spans": 0, "strided": 1, "serial": 2}


def matvec_f16_order(W: torch.Tensor, x: torch.Tensor, order: str,
                     y: Optional[torch.Tensor] = None) -> torch.Tensor:
    """spk_matvec_f16_order: "spans" (lm_head_tiled.comp), "strided"
    (matvec_tiled.comp) or "serial" (matvec.comp) summation order."""
    out_dim, in_dim = W.shape
    if y is None:
        y = torch.empty(out_dim, dtype=torch.float16, device=W.device)
    check(lib().spk_matvec_f16_order(_ptr(W), _ptr(x), _ptr(y), out_dim, in_dim,
                                     MATVEC_ORDERS[order], _stream()),
          "spk_matvec_f16_order")
    return y


def matvec_f16_batched(items) -> None:
    """items: sequence of (W, x, y) device tensors; one call."""
    arr = (SpkMatvecDesc * len(items))()
    for i, (W, x, y) in enumerate(items):
        arr[i].W, arr[i].x, arr[i].y = _ptr(W), _ptr(x), _ptr(y)
        arr[i].out_dim, arr[i].in_dim = W.shape[0], W.shape[1]
    check(lib().spk_matvec_f16_batched(arr, len(items), _stream()), "spk_matvec_f16_batched")


def argmax_f16(vals: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    if out is None:
        out = torch.empty(1, dtype=torch.int32, device=vals.device)
    check(lib().spk_argmax_f16(_ptr(vals), vals.numel(), _ptr(out), _stream()), "spk_argmax_f16")
    return out


def lm_head_workspace_bytes(vocab: int) -> int:
    return int(lib().spk_lm_head_workspace_size(vocab))


def lm_head_argmax(W: torch.Tensor, x: torch.Tensor, logits: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    vocab, hidden = W.shape
    if out is None:
        out = torch.empty(1, dtype=torch.int32, device=W.device)
    need = lm_head_workspace_bytes(vocab)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=W.device)
    check(lib().spk_lm_head_argmax(_ptr(W), _ptr(x), vocab, hidden, _ptr(logits), _ptr(out),
                                   _ptr(workspace), workspace.numel() * workspace.element_size(),
                                   _stream()), "spk_lm_head_argmax")
    return out


# ----------------------------------------------------------------------------
# a serving step over a paged cache
# ----------------------------------------------------------------------------
_HALF = {torch.float16: _lib.SPK_F16, torch.bfloat16: _lib.SPK_BF16}
_PAIRINGS = {"halves": _lib.SPK_ROPE_HALVES, "adjacent": _lib.SPK_ROPE_ADJACENT}


def _on(what: str, name: str, t: torch.Tensor, dev: int, dtype, shape=None) -> None:
    if t.dtype is not dtype or t.get_device() != dev:
        raise _lib.SpockError(f"{what}: {name} must be {dtype} on cuda:{dev}, got {t.dtype} on {t.device}")
    if shape is not None and t.shape != shape:
        raise _lib.SpockError(f"{what}: {name} shape {tuple(t.shape)} != {tuple(shape)}")


def _flat(what: str, name: str, t: torch.Tensor, dev: int, dtype, shape) -> None:
    _on(what, name, t, dev, dtype, shape)
    if not t.is_contiguous():
        raise _lib.SpockError(f"{what}: {name} must be contiguous")


def _rows(what: str, name: str, t: torch.Tensor, dev: int, dtype, shape):
    """Token and head strides of a [tokens][heads][dim] view: any, and 0 where there is one."""
    _on(what, name, t, dev, dtype, shape)
    token, head, last = t.stride()
    if last != 1:
        raise _lib.SpockError(f"{what}: the last dimension of {name} must be contiguous")
    return (token if shape[0] > 1 else 0), (head if shape[1] > 1 else 0)


def _workspace(what: str, t: torch.Tensor, dev: int) -> None:
    """The kernels write all of its bytes in a row: of a view with gaps or repeats those are not its own."""
    if t.get_device() != dev or not t.is_contiguous():
        raise _lib.SpockError(f"{what}: workspace must be contiguous and on cuda:{dev}, got strides {t.stride()} on {t.device}")


def _device(what: str, t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise _lib.SpockError(f"{what}: expected device tensors")
    return t.get_device()


def _paged_cache(what: str, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                 cu_seqlens: torch.Tensor, context_lens: torch.Tensor) -> SpkPagedCache:
    dev, dtype = _device(what, q), q.dtype
    if q.dim() != 3 or k_cache.dim() != 4:
        raise _lib.SpockError(f"{what}: q must be [tokens][heads][dim] and the caches [pages][page_size][kv_heads][dim], "
                              f"got {tuple(q.shape)} and {tuple(k_cache.shape)}")
    if dtype not in _HALF:
        raise _lib.SpockError(f"{what}: q must be float16 or bfloat16, got {dtype}")
    shape = k_cache.shape
    pages, page_size, kv_heads, dim = shape
    tokens, _, q_dim = q.shape
    if q_dim != dim:
        raise _lib.SpockError(f"{what}: q has head_dim {q_dim}, the cache {dim}")
    _on(what, "k_cache", k_cache, dev, dtype)
    _on(what, "v_cache", v_cache, dev, dtype, shape)
    strides, v_strides = k_cache.stride(), v_cache.stride()
    if 1 in shape:  # a stride of one element is not read
        strides, v_strides = ([n if size > 1 else 0 for n, size in zip(t, shape)] for t in (strides, v_strides))
    if v_strides != strides or strides[3] != 1:
        raise _lib.SpockError(f"{what}: k_cache and v_cache need equal strides and a contiguous last dimension, "
                              f"got {k_cache.stride()} and {v_cache.stride()}")
    seqs = context_lens.numel()
    _on(what, "block_table", block_table, dev, torch.int32)
    _flat(what, "cu_seqlens", cu_seqlens, dev, torch.int32, (seqs + 1,))
    _flat(what, "context_lens", context_lens, dev, torch.int32, (seqs,))
    if block_table.dim() != 2 or block_table.shape[0] != seqs or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise _lib.SpockError(f"{what}: block_table must be [{seqs}][max_pages] with contiguous rows, "
                              f"got {tuple(block_table.shape)}")
    return SpkPagedCache(_HALF[dtype], kv_heads, dim, page_size, pages, block_table.shape[1], seqs, tokens,
                         k_cache.data_ptr(), v_cache.data_ptr(), strides[0], strides[1], strides[2],
                         block_table.data_ptr(), block_table.stride(0), cu_seqlens.data_ptr(), context_lens.data_ptr())


def _call(fn, a, dev: int, what: str) -> None:
    """fn(a) on the current stream of the tensors' device, which is made current for the launch.  (The raw handle of
    the stream costs a tenth of the torch.cuda.Stream object around it, 2 us of a 20 us call.)"""
    if torch.cuda.current_device() == dev:
        rc = fn(C.byref(a), torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(C.byref(a), torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        check(rc, what)


def mrope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, rope: torch.Tensor,
                 pair_axis: Sequence[int], k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                 cu_seqlens: torch.Tensor, context_lens: torch.Tensor, q_norm_weight: Optional[torch.Tensor] = None,
                 k_norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, pairing: str = "halves",
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary positions with several axes, and the store into the pages (spk_mrope_append).

    q [T][Hq][D], k, v [T][Hkv][D] (float16 or bfloat16, any token and head strides); positions [axes][T] int32 (for text
    also one row expanded to all axes);
    rope [rows][rot_dim] float32, (cos, sin) per pair; pair_axis: the axis of each of the rot_dim / 2 pairs (host);
    caches [pages][page_size][Hkv][D] (any page, token and head strides, the same for both); block_table
    [S][max_pages], cu_seqlens [S+1], context_lens [S] int32 on the device.  q and k are normalised first where a
    norm weight [D] is given (RMSNorm, 1 + w).  Writes the new tokens' keys and values into the caches and returns
    the queries (in `out`, which may be q; rows past cu_seqlens[S] are not written).
    """
    what = "mrope_append"
    cache = _paged_cache(what, q, k_cache, v_cache, block_table, cu_seqlens, context_lens)
    shape, dtype, dev = q.shape, q.dtype, q.get_device()
    T, heads, D = shape
    kv_shape = (T, cache.num_kv_heads, D)
    qs = _rows(what, "q", q, dev, dtype, shape)
    ks = _rows(what, "k", k, dev, dtype, kv_shape)
    vs = _rows(what, "v", v, dev, dtype, kv_shape)
    try:
        axes = bytes(list(pair_axis))
    except (TypeError, ValueError):
        raise _lib.SpockError(f"{what}: pair_axis must be a sequence of axis numbers, got {pair_axis!r}") from None
    rot = 2 * len(axes)
    rows = rope.shape[0]
    _flat(what, "rope", rope, dev, torch.float32, (rows, rot))
    num_axes = positions.shape[0]
    _on(what, "positions", positions, dev, torch.int32, (num_axes, T))
    if T > 1 and positions.stride(1) != 1:
        raise _lib.SpockError(f"{what}: positions must have contiguous rows")
    if 1 < num_axes <= 4 and positions.stride(0) == 0:  # one row broadcast to all axes
        if max(axes, default=0) >= num_axes:
            raise _lib.SpockError(f"{what}: pair_axis names axis {max(axes)} of {num_axes}")
        num_axes, axes = 1, bytes(len(axes))
    if q_norm_weight is not None:
        _flat(what, "q_norm_weight", q_norm_weight, dev, dtype, (D,))
    if k_norm_weight is not None:
        _flat(what, "k_norm_weight", k_norm_weight, dev, dtype, (D,))
    if pairing not in _PAIRINGS:
        raise _lib.SpockError(f"{what}: pairing must be one of {sorted(_PAIRINGS)}, got {pairing!r}")
    if out is None:
        out = q.new_empty(shape)
    outs = _rows(what, "out", out, dev, dtype, shape)
    a = SpkMropeArgs(cache, heads, rot, _PAIRINGS[pairing], num_axes, axes, positions.data_ptr(), positions.stride(0),
                     rope.data_ptr(), rows, eps, q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1],
                     v.data_ptr(), vs[0], vs[1], _ptr(q_norm_weight), _ptr(k_norm_weight), out.data_ptr(), outs[0], outs[1])
    _call(lib().spk_mrope_append, a, dev, what)
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    cu_seqlens: torch.Tensor, context_lens: torch.Tensor, max_query_len: int, max_context_len: int,
                    scale: float = 0.0, window: int = 0, gate: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False, lse: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None):
    """Attention of each sequence's new tokens over its pages (spk_paged_attention).

    q [T][Hq][D]; caches, tables and lengths as in mrope_append; max_query_len, max_context_len: host bounds of the
    sequences' lengths; scale 0 = 1/sqrt(D); window > 0: only the last `window` positions are seen; gate [T][Hq][D]:
    the output is multiplied by sigmoid(gate).  Returns out [T][Hq][D], or (out, lse [T][Hq] float32) with return_lse
    or an lse buffer.  Rows past cu_seqlens[S] are not written.
    workspace: paged_attention_workspace_bytes() of the largest sizes in use; one that is too small is left alone and a
    fresh one taken.
    """
    what = "paged_attention"
    cache = _paged_cache(what, q, k_cache, v_cache, block_table, cu_seqlens, context_lens)
    shape, dtype, dev = q.shape, q.dtype, q.get_device()
    qs = _rows(what, "q", q, dev, dtype, shape)
    gs = (0, 0) if gate is None else _rows(what, "gate", gate, dev, dtype, shape)
    if out is None:
        out = q.new_empty(shape)
    outs = _rows(what, "out", out, dev, dtype, shape)
    if lse is not None:
        _flat(what, "lse", lse, dev, torch.float32, shape[:2])
    elif return_lse:
        lse = q.new_empty(shape[:2], dtype=torch.float32)
    a = SpkPagedAttnArgs(cache, shape[1], max_query_len, max_context_len, window, scale, q.data_ptr(), qs[0], qs[1],
                         _ptr(gate), gs[0], gs[1], out.data_ptr(), outs[0], outs[1], _ptr(lse), None, 0)
    need = lib().spk_paged_attention_workspace_need(C.byref(a))
    if need:
        if workspace is None or workspace.numel() * workspace.element_size() < need:
            workspace = q.new_empty(need, dtype=torch.uint8)
        else:
            _workspace(what, workspace, dev)
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _call(lib().spk_paged_attention, a, dev, what)
    return out if lse is None else (out, lse)


def paged_attention_workspace_bytes(tokens: int, heads: int, kv_heads: int, head_dim: int, page_size: int,
                                    max_pages: int, num_seqs: int, max_query_len: int, max_context_len: int,
                                    window: int = 0) -> int:
    """Bytes of a workspace for paged_attention at these sizes and any smaller ones, for callers that keep one."""
    cache = SpkPagedCache(_lib.SPK_F16, kv_heads, head_dim, page_size, 1, max_pages, num_seqs, tokens, 16, 16, 0, 0, 0,
                          16, max_pages, 16, 16)
    a = SpkPagedAttnArgs(cache, heads, max_query_len, max_context_len, window)
    return int(lib().spk_paged_attention_workspace_size(C.byref(a)))


_ROWS = {**_HALF, torch.float32: _lib.SPK_F32}
_KINDS = {"logits": _lib.SPK_VERIFY_LOGITS, "probs": _lib.SPK_VERIFY_PROBS}


def verify_workspace_bytes(vocab: int, num_seqs: int, tokens: int) -> int:
    """Bytes of a workspace for verify_drafts at these sizes and any smaller ones."""
    return int(lib().spk_verify_drafts_workspace_size(vocab, num_seqs, tokens))


def verify_drafts(target: torch.Tensor, tokens: torch.Tensor, cu_seqlens: torch.Tensor, u_accept: torch.Tensor,
                  u_sample: torch.Tensor, draft: Optional[torch.Tensor] = None, kind: str = "logits",
                  temperature: Optional[torch.Tensor] = None, context_lens: Optional[torch.Tensor] = None,
                  out_tokens: Optional[torch.Tensor] = None, accepted: Optional[torch.Tensor] = None,
                  logprobs: Optional[torch.Tensor] = None, context_out: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None):
    """Accepts or refuses drafted tokens and draws the next one (spk_verify_drafts).

    target [T][vocab] (float16, bfloat16 or float32): row t is the distribution of the token after row t, as logits or
    as probabilities (`kind`); tokens [T] int32: the input token of every row; cu_seqlens [S+1] int32: the rows of each
    sequence, the last accepted token's first; draft [T][vocab]: the rows that the drafts were drawn from, None for a
    drafter that is certain; temperature [S] float32 (logits; None = 1, 0 = greedy); u_accept [T], u_sample [S] float32
    in [0, 1).  Returns (out_tokens [T] int32, accepted [S] int32, logprobs [T] float32, context_out [S] int32 or None
    without context_lens).  Rows past cu_seqlens[S] are not written.  workspace: verify_workspace_bytes() of the largest
    sizes in use; one that is too small is left alone and a fresh one taken.
    """
    what = "verify_drafts"
    dev = _device(what, target)
    if target.dim() != 2 or target.dtype not in _ROWS or (target.shape[1] > 1 and target.numel() and target.stride(1) != 1):
        raise _lib.SpockError(f"{what}: target must be [rows][vocab] float16, bfloat16 or float32 with contiguous rows, "
                              f"got {tuple(target.shape)} {target.dtype}")
    if kind not in _KINDS:
        raise _lib.SpockError(f"{what}: kind must be one of {sorted(_KINDS)}, got {kind!r}")
    T, vocab = target.shape
    rows, seqs = (T,), (u_sample.numel(),)
    S = seqs[0]
    stride, draft_stride = (target.stride(0) if T > 1 else vocab), 0
    if draft is not None:
        _on(what, "draft", draft, dev, target.dtype, (T, vocab))
        if vocab > 1 and T and draft.stride(1) != 1:
            raise _lib.SpockError(f"{what}: draft must have contiguous rows")
        draft_stride = draft.stride(0) if T > 1 else vocab
    i32, f32 = torch.int32, torch.float32
    _flat(what, "tokens", tokens, dev, i32, rows)
    _flat(what, "cu_seqlens", cu_seqlens, dev, i32, (S + 1,))
    _flat(what, "u_accept", u_accept, dev, f32, rows)
    _flat(what, "u_sample", u_sample, dev, f32, seqs)
    if temperature is not None:
        _flat(what, "temperature", temperature, dev, f32, seqs)
    if context_lens is not None:
        _flat(what, "context_lens", context_lens, dev, i32, seqs)
        if context_out is None:
            context_out = torch.empty(seqs, dtype=i32, device=target.device)
    if context_out is not None:
        _flat(what, "context_out", context_out, dev, i32, seqs)
    if out_tokens is None:
        out_tokens = torch.empty(rows, dtype=i32, device=target.device)
    if accepted is None:
        accepted = torch.empty(seqs, dtype=i32, device=target.device)
    if logprobs is None:
        logprobs = torch.empty(rows, dtype=f32, device=target.device)
    _flat(what, "out_tokens", out_tokens, dev, i32, rows)
    _flat(what, "accepted", accepted, dev, i32, seqs)
    _flat(what, "logprobs", logprobs, dev, f32, rows)
    need = lib().spk_verify_drafts_workspace_size(vocab, S, T)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=target.device)
    else:
        _workspace(what, workspace, dev)
    a = SpkVerifyArgs(_KINDS[kind], _ROWS[target.dtype], vocab, S, T, cu_seqlens.data_ptr(), tokens.data_ptr(),
                      target.data_ptr(), stride, _ptr(draft), draft_stride, _ptr(temperature), u_accept.data_ptr(),
                      u_sample.data_ptr(), out_tokens.data_ptr(), accepted.data_ptr(), logprobs.data_ptr(),
                      _ptr(context_lens), _ptr(context_out), workspace.data_ptr(), workspace.numel() * workspace.element_size())
    _call(lib().spk_verify_drafts, a, dev, what)
    return out_tokens, accepted, logprobs, context_out
