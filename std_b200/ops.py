"""torch-facing wrappers over the C ABI (one call per kernel entry point).

PyTorch only supplies device memory and the current CUDA stream here; every
call goes through libstd_b200.so.  Tensors must be CUDA, contiguous and of the
documented dtype -- there is no CPU path and no fallback.
"""

from __future__ import annotations

import math
from typing import Dict, Optional, Tuple

import torch

from . import _lib

_WS: Dict[Tuple[str, int], torch.Tensor] = {}


def _stream() -> int:
    return _stream_of(torch.cuda.current_device())


def _stream_of(device: int) -> int:
    # the raw handle of torch.cuda.current_stream(device), without building a Stream object (3 us a call)
    return torch._C._cuda_getCurrentRawStream(device)


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _check(t: torch.Tensor, dtype: torch.dtype, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (no CPU path)")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def workspace(kind: str, nbytes: int, device: torch.device) -> torch.Tensor:
    """Scratch buffer, grown on demand, one per (kind, device).

    Allocation happens outside graph capture: call each op once eagerly before
    capturing it.
    """
    key = (kind, device.index if device.index is not None else torch.cuda.current_device())
    buf = _WS.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(int(nbytes), 256), dtype=torch.uint8, device=device)
        _WS[key] = buf
    return buf


# ----------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------

def draft_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                    len_offset: int = 0, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    after_append: bool = False):
    """q [B, Hq, D] bf16; caches [B, Hkv, cap, D] bf16; lens [B] int32 (device).

    after_append=True (STD_DRAFT_AFTER_APPEND): the previous launch on the
    stream writes only q and each request's newest K/V row, so the kernel may
    start reading the older rows before it finishes."""
    B, Hq, D = q.shape
    _, Hkv, cap, _ = k_cache.shape
    for t, n in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _check(t, torch.bfloat16, n)
    _check(lens, torch.int32, "lens")
    if out is None:
        out = torch.empty_like(q)
    nb = _lib.query("std_draft_attn_workspace_bytes", B, Hq, Hkv, D, cap)
    ws = workspace("draft", nb, q.device)
    _lib.call("std_draft_attn", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lens.data_ptr(), int(len_offset),
              B, Hq, Hkv, D, cap, out.data_ptr(), _p(lse), ws.data_ptr(), ws.numel(), 1 if after_append else 0,
              _stream())
    return out


def draft_attention_indexed(q: torch.Tensor, dense_k: torch.Tensor, dense_v: torch.Tensor, idx: torch.Tensor,
                            tail_k: torch.Tensor, tail_v: torch.Tensor, lens: torch.Tensor, len_offset: int = 0,
                            out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None):
    """Draft attention over dense-cache rows idx [B, Hkv, n_idx] (int32,
    ascending) followed by the tail [B, Hkv, tail_cap, D]; keys per request =
    lens[b] + len_offset."""
    B, Hq, D = q.shape
    _, Hkv, cap_d, _ = dense_k.shape
    for t, n in ((q, "q"), (dense_k, "dense_k"), (dense_v, "dense_v"), (tail_k, "tail_k"), (tail_v, "tail_v")):
        _check(t, torch.bfloat16, n)
    _check(idx, torch.int32, "idx")
    _check(lens, torch.int32, "lens")
    if idx.shape[:2] != (B, Hkv):
        raise ValueError("idx must be [B, Hkv, n_idx]")
    if out is None:
        out = torch.empty_like(q)
    _lib.call("std_draft_attn_indexed", q.data_ptr(), dense_k.data_ptr(), dense_v.data_ptr(), cap_d, idx.data_ptr(),
              idx.shape[2], tail_k.data_ptr(), tail_v.data_ptr(), tail_k.shape[2], lens.data_ptr(), int(len_offset),
              B, Hq, Hkv, D, out.data_ptr(), _p(lse), _stream())
    return out


def verify_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                     len_offset: int, causal: bool = True, out: Optional[torch.Tensor] = None,
                     lse: Optional[torch.Tensor] = None):
    """q [B, nq, Hq, D] bf16; caches [B, Hkv, cap, D]; keys = lens[b] + len_offset."""
    B, nq, Hq, D = q.shape
    _, Hkv, cap, _ = k_cache.shape
    for t, n in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _check(t, torch.bfloat16, n)
    _check(lens, torch.int32, "lens")
    if out is None:
        out = torch.empty_like(q)
    nb = _lib.query("std_verify_attn_workspace_bytes", B, Hkv, cap)
    ws = workspace("verify", nb, q.device)
    _lib.call("std_verify_attn", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lens.data_ptr(),
              int(len_offset), nq, 1 if causal else 0, B, Hq, Hkv, D, cap, out.data_ptr(), _p(lse), ws.data_ptr(),
              ws.numel(), _stream())
    return out


def verify_attention_partial(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lens: torch.Tensor,
                             len_offset: int, causal: bool, out_f32: torch.Tensor, lse: torch.Tensor):
    """verify_attention with an fp32 output and its LSE (one key range's
    partial of a sequence-sharded verify)."""
    B, nq, Hq, D = q.shape
    _, Hkv, cap, _ = k_cache.shape
    for t, n in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _check(t, torch.bfloat16, n)
    _check(out_f32, torch.float32, "out_f32")
    _check(lse, torch.float32, "lse")
    nb = _lib.query("std_verify_attn_workspace_bytes", B, Hkv, cap)
    ws = workspace("verify", nb, q.device)
    _lib.call("std_verify_attn_partial", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lens.data_ptr(),
              int(len_offset), nq, 1 if causal else 0, B, Hq, Hkv, D, cap, out_f32.data_ptr(), lse.data_ptr(),
              ws.data_ptr(), ws.numel(), _stream())
    return out_f32


def merge_partials_f32(parts: torch.Tensor, rows: int, D: int, out: torch.Tensor,
                       lse_out: Optional[torch.Tensor] = None):
    """parts [n, stride] fp32, each [rows*D O | rows LSE] -> out [rows, D] bf16."""
    n, stride = parts.shape
    _check(parts, torch.float32, "parts")
    _lib.call("std_merge_partials_f32", parts.data_ptr(), stride, n, rows, D, out.data_ptr(), _p(lse_out), _stream())
    return out


def merge_partials(o_parts: torch.Tensor, lse_parts: torch.Tensor, out: Optional[torch.Tensor] = None,
                   lse_out: Optional[torch.Tensor] = None):
    """o_parts [n, rows, D] bf16, lse_parts [n, rows] fp32 -> out [rows, D]."""
    n, rows, D = o_parts.shape
    _check(o_parts, torch.bfloat16, "o_parts")
    _check(lse_parts, torch.float32, "lse_parts")
    if out is None:
        out = torch.empty((rows, D), dtype=torch.bfloat16, device=o_parts.device)
    _lib.call("std_merge_partials", o_parts.data_ptr(), lse_parts.data_ptr(), n, rows, D, out.data_ptr(),
              _p(lse_out), _stream())
    return out


def collect_relevance(q: torch.Tensor, k_cache: torch.Tensor, visual_pos: torch.Tensor, rel_out: torch.Tensor):
    """Collector v1 for one layer: rel_out [B, Hkv, P] fp32 at the visual
    positions gets sum over the verify rows of softmax over the visual keys of
    (group-mean query . k) / sqrt(D).  q [B, nq, Hq, D] bf16; k_cache [B, Hkv,
    cap, D] bf16; visual_pos [V] int32."""
    B, nq, Hq, D = q.shape
    _, Hkv, cap, _ = k_cache.shape
    _check(q, torch.bfloat16, "q")
    _check(k_cache, torch.bfloat16, "k_cache")
    _check(visual_pos, torch.int32, "visual_pos")
    _check(rel_out, torch.float32, "rel_out")
    V = visual_pos.numel()
    ws = workspace("collect", _lib.query("std_collect_workspace_bytes", B, Hkv, nq, V), q.device)
    _lib.call("std_collect_relevance", q.data_ptr(), k_cache.data_ptr(), visual_pos.data_ptr(), V, B, nq, Hq, Hkv, D,
              cap, rel_out.data_ptr(), rel_out.shape[-1], ws.data_ptr(), ws.numel(), _stream())
    return rel_out


# ----------------------------------------------------------------------------
# selection
# ----------------------------------------------------------------------------

def select_scores(q_text: torch.Tensor, k_rows: torch.Tensor, P: int, q_start: int,
                  scores: Optional[torch.Tensor] = None, write_probs: bool = False, scale: Optional[float] = None):
    """q_text [T, Hq, D] bf16; k_rows [Hkv, kstride, D] bf16 -> scores [Hkv, P] fp32.

    With write_probs, also returns the fp16 probabilities view [Hq, T, P].
    """
    T, Hq, D = q_text.shape
    Hkv, kstride, _ = k_rows.shape
    _check(q_text, torch.bfloat16, "q_text")
    _check(k_rows, torch.bfloat16, "k_rows")
    if scores is None:
        scores = torch.empty((Hkv, P), dtype=torch.float32, device=q_text.device)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    nb = _lib.query("std_select_workspace_bytes", T, Hq, P)
    ws = workspace("select", nb, q_text.device)
    _lib.call("std_select_scores", q_text.data_ptr(), k_rows.data_ptr(), kstride, T, Hq, Hkv, D, P, q_start,
              float(scale), scores.data_ptr(), 1 if write_probs else 0, ws.data_ptr(), ws.numel(), _stream())
    if not write_probs:
        return scores
    import ctypes

    ps = ctypes.c_longlong(0)
    _lib.call("std_select_probs_view", T, Hq, P, ctypes.byref(ps))
    probs = ws[: Hq * T * ps.value * 2].view(torch.float16).view(Hq, T, ps.value)[:, :, :P]
    return scores, probs


def topk_select(scores: torch.Tensor, visual_pos: torch.Tensor, k: int, out: Optional[torch.Tensor] = None):
    """scores [n_seg, P] fp32; visual_pos [V] int32 ascending -> [n_seg, k] int32 ascending."""
    n_seg, P = scores.shape
    _check(scores, torch.float32, "scores")
    _check(visual_pos, torch.int32, "visual_pos")
    if out is None:
        out = torch.empty((n_seg, k), dtype=torch.int32, device=scores.device)
    _lib.call("std_topk_select", scores.data_ptr(), P, n_seg, visual_pos.data_ptr(), visual_pos.numel(), k,
              out.data_ptr(), _stream())
    return out


def compact_gather(dense_cache: torch.Tensor, sparse_cache: torch.Tensor, b: int, non_visual: torch.Tensor,
                   topk: torch.Tensor):
    """caches [layers, 2, B, Hkv, cap, D]; non_visual [NV] int32; topk [layers, Hkv, K] int32."""
    layers, _, B, Hkv, cap_d, D = dense_cache.shape
    cap_s = sparse_cache.shape[4]
    _check(dense_cache, torch.bfloat16, "dense_cache")
    _check(sparse_cache, torch.bfloat16, "sparse_cache")
    _check(non_visual, torch.int32, "non_visual")
    _check(topk, torch.int32, "topk")
    _lib.call("std_compact_gather", dense_cache.data_ptr(), sparse_cache.data_ptr(), layers, B, b, Hkv, D, cap_d,
              cap_s, non_visual.data_ptr(), non_visual.numel(), topk.data_ptr(), topk.shape[-1], _stream())


# ----------------------------------------------------------------------------
# decoder pieces
# ----------------------------------------------------------------------------

def embed(table: torch.Tensor, tok: torch.Tensor, tok_start: int, n: int, out: torch.Tensor):
    B, stride = tok.shape
    _lib.call("std_embed", table.data_ptr(), table.shape[0], table.shape[1], tok.data_ptr(), stride, tok_start, n, B,
              out.data_ptr(), _stream())
    return out


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, out: torch.Tensor):
    H = x.shape[-1]
    M = x.numel() // H
    _lib.call("std_rmsnorm", x.data_ptr(), w.data_ptr(), float(eps), M, H, out.data_ptr(), _stream())
    return out


def gemm(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor, bias: Optional[torch.Tensor] = None):
    """out[M, N] = x[M, K] @ w[N, K]^T (+ bias) on the tcgen05 weight-streaming GEMM (M <= 256)."""
    M, K = x.shape
    N = w.shape[0]
    _check(x, torch.bfloat16, "x")
    _check(w, torch.bfloat16, "w")
    _check(out, torch.bfloat16, "out")
    nb = _lib.query("std_gemm_workspace_bytes", M, N, K)
    ws = workspace("gemm", nb, x.device) if nb > 0 else None
    _lib.call("std_gemm_bf16", x.data_ptr(), w.data_ptr(), _p(bias), out.data_ptr(), M, N, K, _p(ws),
              0 if ws is None else ws.numel(), _stream())
    return out


def gemm_add_rmsnorm(x: torch.Tensor, w: torch.Tensor, resid: torch.Tensor, norm_w: Optional[torch.Tensor],
                     eps: float, out: Optional[torch.Tensor], bias: Optional[torch.Tensor] = None):
    """resid <- bf16(resid + x @ w^T (+ bias)); out = rmsnorm(resid) * norm_w (norm_w None: add only).

    One GEMM plus one fused epilogue kernel; equal to gemm() then add_rmsnorm()."""
    M, K = x.shape
    N = w.shape[0]
    for t, n in ((x, "x"), (w, "w"), (resid, "resid")):
        _check(t, torch.bfloat16, n)
    nb = _lib.query("std_gemm_epilogue_workspace_bytes", M, N, K)
    ws = workspace("gemm", nb, x.device)
    _lib.call("std_gemm_add_rmsnorm", x.data_ptr(), w.data_ptr(), _p(bias), resid.data_ptr(), _p(norm_w), float(eps),
              _p(out), M, N, K, ws.data_ptr(), ws.numel(), _stream())
    return out


def gemm_argmax(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor, rows_out: Optional[int] = None, n: int = 1,
                out_stride: int = 1, out_start: int = 0, margin_out: Optional[torch.Tensor] = None):
    """Greedy argmax of x @ w^T's bf16 rows (lm_head + argmax) without storing the logits.

    Result t (< rows_out, default all rows) goes to out[(t//n)*out_stride + out_start + t%n];
    with margin_out (fp32, same indexing) also the row's top-1 minus top-2 logit."""
    M, K = x.shape
    N = w.shape[0]
    _check(x, torch.bfloat16, "x")
    _check(w, torch.bfloat16, "w")
    _check(out, torch.int32, "out")
    rows_out = M if rows_out is None else rows_out
    keys = workspace("argmax_keys", M * 8, x.device)  # zero-initialised, left zero by every call
    nb = _lib.query("std_gemm_epilogue_workspace_bytes", M, N, K)
    ws = workspace("gemm", nb, x.device)
    if margin_out is not None:
        _check(margin_out, torch.float32, "margin_out")
    _lib.call("std_gemm_argmax", x.data_ptr(), w.data_ptr(), M, N, K, rows_out, n, out_stride, out_start,
              out.data_ptr(), _p(margin_out), keys.data_ptr(), ws.data_ptr(), ws.numel(), _stream())
    return out


def gemm_rope_append(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], B: int, n: int, Hq: int,
                     Hkv: int, D: int, pos_base: torch.Tensor, pos_off: int, slot_base: torch.Tensor, slot_off: int,
                     cos_t: torch.Tensor, sin_t: torch.Tensor, q_out: torch.Tensor, k_cache: torch.Tensor,
                     v_cache: torch.Tensor):
    """qkv = x @ w^T + bias, then rope_append on it, as one GEMM + one fused epilogue kernel."""
    M, K = x.shape
    N = w.shape[0]
    if M != B * n or N != (Hq + 2 * Hkv) * D:
        raise ValueError("gemm_rope_append: x rows must be B*n and w rows (Hq + 2 Hkv) * D")
    _check(x, torch.bfloat16, "x")
    _check(w, torch.bfloat16, "w")
    cap = k_cache.shape[-2]
    nb = _lib.query("std_gemm_epilogue_workspace_bytes", M, N, K)
    ws = workspace("gemm", nb, x.device)
    _lib.call("std_gemm_rope_append", x.data_ptr(), w.data_ptr(), _p(bias), K, B, n, Hq, Hkv, D, pos_base.data_ptr(),
              int(pos_off), slot_base.data_ptr(), int(slot_off), cos_t.data_ptr(), sin_t.data_ptr(), cos_t.shape[0],
              q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), cap, ws.data_ptr(), ws.numel(), _stream())
    return q_out


def add_rmsnorm(x: torch.Tensor, delta: torch.Tensor, w: torch.Tensor, eps: float, out: torch.Tensor):
    """x <- x + delta (bf16, in place); out = rmsnorm(x) * w."""
    H = x.shape[-1]
    M = x.numel() // H
    _lib.call("std_add_rmsnorm", x.data_ptr(), delta.data_ptr(), w.data_ptr(), float(eps), M, H, out.data_ptr(),
              _stream())
    return out


def rope_append(qkv: torch.Tensor, B: int, n: int, Hq: int, Hkv: int, D: int, pos_base: torch.Tensor, pos_off: int,
                slot_base: torch.Tensor, slot_off: int, cos_t: torch.Tensor, sin_t: torch.Tensor,
                q_out: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor):
    cap = k_cache.shape[-2]
    _lib.call("std_rope_append", qkv.data_ptr(), B, n, Hq, Hkv, D, pos_base.data_ptr(), int(pos_off),
              slot_base.data_ptr(), int(slot_off), cos_t.data_ptr(), sin_t.data_ptr(), cos_t.shape[0],
              q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), cap, _stream())
    return q_out


def silu_mul(gu: torch.Tensor, out: torch.Tensor, interleaved: bool = False):
    """out = silu(gate) * up; gu columns [gate | up] or 64-feature [gate | up] blocks (interleaved)."""
    I2 = gu.shape[-1]
    M = gu.numel() // I2
    _lib.call("std_silu_mul", gu.data_ptr(), M, I2 // 2, 1 if interleaved else 0, out.data_ptr(), _stream())
    return out


def gemm_silu_mul(x: torch.Tensor, w_gu: torch.Tensor, out: torch.Tensor):
    """out[M, I] = silu(x @ gate^T) * (x @ up^T) with w_gu [2I, K] in 64-row [gate | up] blocks."""
    M, K = x.shape
    N = w_gu.shape[0]
    _check(x, torch.bfloat16, "x")
    _check(w_gu, torch.bfloat16, "w_gu")
    _check(out, torch.bfloat16, "out")
    nb = _lib.query("std_gemm_epilogue_workspace_bytes", M, N, K)
    ws = workspace("gemm", nb, x.device)
    _lib.call("std_gemm_silu_mul", x.data_ptr(), w_gu.data_ptr(), M, N // 2, K, out.data_ptr(), ws.data_ptr(),
              ws.numel(), _stream())
    return out


def add(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor):
    _lib.call("std_add", a.data_ptr(), b.data_ptr(), a.numel(), out.data_ptr(), _stream())
    return out


def argmax_rows(logits: torch.Tensor, out: torch.Tensor, n: int = 1, out_stride: int = 1, out_start: int = 0):
    V = logits.shape[-1]
    rows = logits.numel() // V
    _lib.call("std_argmax_rows", logits.data_ptr(), rows, V, n, out_stride, out_start, out.data_ptr(), _stream())
    return out


# ----------------------------------------------------------------------------
# paged K/V cache
# ----------------------------------------------------------------------------

_PAGED_DTYPES = (torch.bfloat16, torch.float16)
_PAGED_SIZES = (16, 32, 64, 128, 256)
_PAGED_WS_BYTES: Dict[int, int] = {}


def _paged_check(dtype: torch.dtype, device: int, *tensors) -> None:
    """Each (tensor, name, shape): contiguous, of this shape and type, on the
    call's device.  (These checks are most of a small call's time: one pass.)"""
    for t, name, shape in tensors:
        if t.dtype is dtype and t.get_device() == device and t.shape == shape and t.is_contiguous():
            continue
        _check(t, dtype, name)
        if t.get_device() != device:
            raise RuntimeError(f"{name} is on {t.device}, the call's other tensors on cuda:{device}")
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")


def _paged_device(t: torch.Tensor, name: str) -> int:
    """The call's device: kernels run on the current device's stream, so it
    has to be that one."""
    device = t.get_device()
    if device < 0:
        raise RuntimeError(f"{name} must be a CUDA tensor (no CPU path)")
    if device != torch._C._cuda_getDevice():  # (torch.cuda.current_device without its check that CUDA is up)
        raise RuntimeError(f"{name} is on {t.device}, but cuda:{torch.cuda.current_device()} is the current device")
    return device


def _paged_own(names: str, *tensors: torch.Tensor) -> None:
    """Memory that a call took for itself while its stream is being captured: it has
    to stay the graph's, as it does under torch.cuda.graph (from the graph's own pool).  A capture
    that torch did not begin (a loop or branch body, std_capture_while_begin and
    std_capture_if_begin) gets it from the general pool instead, which would hand it
    to others while the graph still writes it: refused."""
    if torch.cuda.get_allocator_backend() != "native":
        return
    segments = torch.cuda.memory_snapshot(include_traces=False)
    for at in (t.data_ptr() for t in tensors if t.numel() > 0):
        pools = [tuple(s["segment_pool_id"]) for s in segments if s["address"] <= at < s["address"] + s["total_size"]]
        if not pools or pools[0] == (0, 0):
            raise RuntimeError(f"a capture that torch.cuda.graph did not begin (a graph's loop or branch body) needs "
                               f"{names}: memory allocated here would not stay with the graph")


def _paged_pool(k_pages: torch.Tensor, v_pages: torch.Tensor, dtype: torch.dtype, device: int):
    if k_pages.dim() != 4:
        raise ValueError("k_pages must be [num_pages, Hkv, page_size, D]")
    shape = k_pages.shape
    _paged_check(dtype, device, (k_pages, "k_pages", shape), (v_pages, "v_pages", shape))
    if shape[2] not in _PAGED_SIZES:
        raise ValueError(f"page_size must be 16, 32, 64, 128 or 256, got {shape[2]}")
    if shape[3] not in (64, 128):
        raise ValueError(f"head dim must be 64 or 128, got {shape[3]}")
    return shape


def paged_update(past_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, n_blocks: torch.Tensor,
                 free_pages: torch.Tensor, n_free: torch.Tensor, page_size: int, max_tokens: int,
                 out: Optional[Tuple[torch.Tensor, ...]] = None):
    """One step's tables of a paged cache, from the requests' lengths.

    past_lens, new_lens [B]; block_table [B, max_blocks], n_blocks [B],
    free_pages [num_pages] and n_free [1] are updated in place (all int32 on the
    device): every request ends up with the pages that past + new tokens need,
    taken from or returned to the end of the free list, so new_lens 0 with a
    shorter past_lens rolls a request back.  Returns (cu_q [B + 1], kv_lens [B],
    slots [max_tokens], positions [max_tokens], admitted [B]); a request that the
    list cannot serve has admitted 0, kv_lens 0 and slots -1.  A step without
    requests (B 0) gives cu_q [0] and slots of -1.  What the call writes shares no
    memory with its other tensors (status 1).  `out` gives the
    five result tensors (a captured graph's static buffers; the captured body of a
    loop or branch needs it)."""
    device = _paged_device(past_lens, "past_lens")
    B, i32 = past_lens.numel(), torch.int32
    if block_table.dim() != 2:
        raise ValueError("block_table must be [B, max_blocks]")
    width, num_pages, max_tokens = block_table.shape[1], free_pages.numel(), int(max_tokens)
    page_size = int(page_size)
    if not 0 <= max_tokens < 2 ** 31:
        raise ValueError("max_tokens must be a non-negative int32")
    if not (0 <= page_size < 2 ** 31 and width < 2 ** 31 and num_pages < 2 ** 31):  # (ctypes would cut them)
        raise ValueError(f"page_size, max_blocks and num_pages must be int32, got {page_size}, {width} and {num_pages}")
    _paged_check(i32, device, (past_lens, "past_lens", (B,)), (new_lens, "new_lens", (B,)),
                 (block_table, "block_table", (B, width)), (n_blocks, "n_blocks", (B,)),
                 (free_pages, "free_pages", (num_pages,)), (n_free, "n_free", (1,)))
    if out is None:
        sizes = (B + 1, B, B, max_tokens, max_tokens)
        room = torch.empty(sum(sizes), dtype=i32, device=past_lens.device)
        if torch._C._cuda_isCurrentStreamCapturing():
            _paged_own("out=", room)
        cu_q, kv_lens, admitted, slots, positions = room.unsafe_split_with_sizes(sizes)  # (no views to keep track of)
    else:
        cu_q, kv_lens, slots, positions, admitted = out
        _paged_check(i32, device, (cu_q, "cu_q", (B + 1,)), (kv_lens, "kv_lens", (B,)),
                     (slots, "slots", (max_tokens,)), (positions, "positions", (max_tokens,)),
                     (admitted, "admitted", (B,)))
    if B == 0:  # nothing to do but to say so
        if page_size not in _PAGED_SIZES:
            raise ValueError(f"page_size must be 16, 32, 64, 128 or 256, got {page_size}")
        cu_q.zero_()
        slots.fill_(-1)
        positions.fill_(-1)
        return cu_q, kv_lens, slots, positions, admitted
    _lib.call("std_paged_update", past_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(),
              n_blocks.data_ptr(), free_pages.data_ptr(), n_free.data_ptr(), B, width, page_size, num_pages,
              max_tokens, cu_q.data_ptr(), kv_lens.data_ptr(), slots.data_ptr(), positions.data_ptr(),
              admitted.data_ptr(), _stream_of(device))
    return cu_q, kv_lens, slots, positions, admitted


def paged_rope_append(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, cos_t: torch.Tensor,
                      sin_t: torch.Tensor, q_out: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor):
    """RoPE of qkv [T, (Hq + 2 Hkv) * D]'s q and k at positions [T]; q goes to
    q_out [T, Hq, D], k and v to slots [T] of the pools [num_pages, Hkv, page,
    D].  Position -1: the row is skipped; slot -1: nothing is stored.  bf16 or
    fp16 throughout (tables cos_t, sin_t [max_pos, D / 2] too).  q_out and the pools
    share no memory with the call's other tensors (status 1)."""
    device = _paged_device(qkv, "qkv")
    dtype = qkv.dtype
    if dtype not in _PAGED_DTYPES:
        raise RuntimeError(f"qkv must be bfloat16 or float16, got {dtype}")
    if q_out.dim() != 3 or cos_t.dim() != 2:
        raise ValueError("q_out must be [T, Hq, D] and cos_t [max_pos, D / 2]")
    num_pages, Hkv, page, D = _paged_pool(k_pages, v_pages, dtype, device)
    T, Hq = q_out.shape[:2]
    max_pos = cos_t.shape[0]
    _paged_check(dtype, device, (q_out, "q_out", (T, Hq, D)), (qkv, "qkv", (T, (Hq + 2 * Hkv) * D)),
                 (cos_t, "cos_t", (max_pos, D // 2)), (sin_t, "sin_t", (max_pos, D // 2)))
    _paged_check(torch.int32, device, (positions, "positions", (T,)), (slots, "slots", (T,)))
    _lib.call("std_paged_rope_append", qkv.data_ptr(), T, Hq, Hkv, D, 1 if dtype == torch.float16 else 0,
              positions.data_ptr(), slots.data_ptr(), cos_t.data_ptr(), sin_t.data_ptr(), max_pos, q_out.data_ptr(),
              k_pages.data_ptr(), v_pages.data_ptr(), num_pages, page, _stream_of(device))
    return q_out


def _paged_workspace_bytes(D: int) -> int:
    nb = _PAGED_WS_BYTES.get(D)
    if nb is None:
        nb = _PAGED_WS_BYTES[D] = _lib.query("std_paged_attn_workspace_bytes", D)
    return nb


def paged_attention_workspace(head_dim: int, device: Optional[torch.device] = None) -> torch.Tensor:
    """A workspace for paged_attention calls of this head dim (64 or 128) on one
    stream, or captured into one graph: calls that may run at the same time need
    one each.  device defaults to the current one."""
    nb = _paged_workspace_bytes(int(head_dim))
    if nb == 0:
        raise ValueError(f"head dim must be 64 or 128, got {head_dim}")
    return torch.empty(nb, dtype=torch.uint8, device="cuda" if device is None else device)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    cu_q: torch.Tensor, kv_lens: torch.Tensor, causal: bool = True, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None):
    """Attention of each request's new tokens over its paged cache.

    q [T, Hq, D]: request b's tokens are rows cu_q[b] .. cu_q[b+1] - 1 (cu_q [B +
    1] int32); pools [num_pages, Hkv, page, D]; block_table [B, max_blocks] and
    kv_lens [B] int32, the new tokens' keys included.  Token t of n sees keys 0 ..
    kv_len - n + t (causal) or all kv_len.  bf16 or fp16; any Hq / Hkv up to 128.
    scale defaults to 1 / sqrt(D).  out [T, Hq, D], lse [T, Hq] fp32 (optional),
    which share no memory with the call's other tensors (status 1).
    Rows that see no key give 0 and -inf; rows outside every request are left
    as they were (uninitialised in an `out` made here): all of them in a step
    without requests.  workspace (optional): a
    buffer of paged_attention_workspace, which no other call may use before this
    one has run; one kept by the caller serves a whole sequence of calls.  The
    captured body of a loop or branch needs `out` and `workspace`."""
    device = _paged_device(q, "q")
    dtype = q.dtype
    if dtype not in _PAGED_DTYPES:
        raise RuntimeError(f"q must be bfloat16 or float16, got {dtype}")
    if q.dim() != 3 or block_table.dim() != 2:
        raise ValueError("q must be [T, Hq, D] and block_table [B, max_blocks]")
    T, Hq, D = q.shape
    num_pages, Hkv, page, _ = _paged_pool(k_pages, v_pages, dtype, device)
    B, width = block_table.shape
    _paged_check(dtype, device, (q, "q", (T, Hq, k_pages.shape[3])))
    if Hkv < 1 or Hq % Hkv != 0 or not 1 <= Hq // Hkv <= 128:
        raise ValueError(f"query heads ({Hq}) must be a multiple of key heads ({Hkv}), at most 128 times as many")
    _paged_check(torch.int32, device, (block_table, "block_table", (B, width)), (cu_q, "cu_q", (B + 1,)),
                 (kv_lens, "kv_lens", (B,)))
    if width >= 2 ** 31:
        raise ValueError(f"block_table has {width} entries a request, more than int32 counts")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < 2.3e38:  # (times log2 e it has to be a float)
        raise ValueError(f"scale must be positive and below 2.3e38, got {scale}")
    made = ()  # here
    if out is None:
        out = torch.empty_like(q)
        made = (out,)
    else:
        _paged_check(dtype, device, (out, "out", (T, Hq, D)))
    if lse is not None:
        _paged_check(torch.float32, device, (lse, "lse", (T, Hq)))
    nb = _paged_workspace_bytes(D)
    if workspace is None:
        # Of this call alone: the caching allocator hands it out in stream order, and
        # under torch.cuda.graph from the graph's own pool, so no two calls or graphs
        # share it.
        ws = torch.empty(nb, dtype=torch.uint8, device=q.device)
        made += (ws,)
    else:
        ws = workspace
        _paged_check(torch.uint8, device, (ws, "workspace", ws.shape))
        if ws.numel() < nb or ws.data_ptr() % 32 != 0:
            raise ValueError(f"workspace must have at least {nb} bytes and begin at a multiple of 32")
    if made and torch._C._cuda_isCurrentStreamCapturing():
        _paged_own("out= and workspace=", *made)
    if B == 0:  # every row is outside every request
        return out
    _lib.call("std_paged_attn", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(),
              cu_q.data_ptr(), kv_lens.data_ptr(), T, B, Hq, Hkv, D, 1 if dtype == torch.float16 else 0, num_pages,
              page, width, 1 if causal else 0, scale, out.data_ptr(), _p(lse), ws.data_ptr(), nb, _stream_of(device))
    return out


def device_error() -> int:
    return _lib.device_error()
