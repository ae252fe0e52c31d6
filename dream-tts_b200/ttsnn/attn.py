"""Decode attention reading the KV cache in place (crates/tts-nn/src/attn.rs)."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from ._ctx import ctx_of, packed, ptr, stream, stream_of
from .qkrope import chunk_batch, contiguous_cache, same_device


def decode_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, span: int,
                     window_start: int) -> torch.Tensor:
    """`q [b, n_kv, gqa, 128]` f32 (scale folded in) over caches `[b, n_kv, cap, 128]` f16:
    softmax over positions `[window_start, span)` (attn.rs:22-73). Returns f32 like q."""
    b, n_kv, gqa, hd = q.shape
    cap = k.shape[2]
    if span > cap:
        raise ValueError(f"span {span} exceeds capacity {cap}")
    if k.dtype != torch.float16:
        raise L.TtsError(2, "decode_attention: the cache must be f16")
    kv, table = contiguous_cache(k, v)
    spans = torch.full((b,), span, dtype=torch.int32, device=q.device)
    window = span - window_start if window_start > 0 else 0
    qc = q.to(torch.float32).contiguous()
    out = torch.empty(b, n_kv, gqa, hd, device=q.device, dtype=torch.float32)
    L.call("tts_decode_attention", ctx_of(qc), ptr(qc), b, gqa, C.byref(kv), ptr(spans),
           span, window, ptr(out), 0, stream())
    return out


def decode_attention_paged(q: torch.Tensor, kv: L.KvCache, spans: torch.Tensor, max_span: int,
                           window: int = 0, out_f16: bool = True) -> torch.Tensor:
    """Paged form: per-lane spans; q `[lanes, n_kv * gqa, 128]`."""
    lanes, heads, hd = q.shape
    gqa = heads // kv.n_kv
    out = torch.empty(lanes, heads * hd, device=q.device,
                      dtype=torch.float16 if out_f16 else torch.float32)
    L.call("tts_decode_attention", ctx_of(q), ptr(q), lanes, gqa, C.byref(kv), ptr(spans),
           int(max_span), int(window), ptr(out), 1 if out_f16 else 0, stream())
    return out


_workspace: dict[int, int] = {}  # bytes of a chunk_attention call's workspace, by device


def paged_cache(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor) -> L.KvCache:
    """One layer's pools `[pages, n_kv, block_size, 128]` f16 and block table int32
    `[lanes, max_blocks]` as the cache the paged calls take (it keeps the tensors alive)."""
    if k.shape != v.shape or k.dim() != 4 or k.dtype != torch.float16 or v.dtype != torch.float16:
        raise ValueError("paged_cache: k and v must be f16 [pages, n_kv, block_size, 128]")
    if table.dim() != 2 or table.dtype != torch.int32:
        raise ValueError("paged_cache: the block table must be int32 [lanes, max_blocks]")
    if not (k.is_contiguous() and v.is_contiguous() and table.is_contiguous()):
        raise ValueError("paged_cache: pools and table must be contiguous")
    same_device("paged_cache", k, v, table)
    pages, n_kv, bs, hd = k.shape
    kv = L.KvCache(k.data_ptr(), v.data_ptr(), table.data_ptr(), table.shape[1], bs, pages, n_kv, hd)
    kv.lanes, kv.keep = table.shape[0], (k, v, table)
    return kv


def chunk_attention(q: torch.Tensor, row_start: torch.Tensor, spans: torch.Tensor,
                    kv: L.KvCache, scale: float, window: int = 0,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a ragged chunk of new rows over their lanes' pages (their own K and V
    included, see `qkrope.rotary_append`): q `[rows, heads, 128]` f16 or f32, lane i's rows
    row_start[i] .. row_start[i + 1] at its last positions before spans[i], each seeing the
    positions up to its own (at most `window` of them, 0: all). Returns f16
    `[rows, heads * 128]` (or `out`); rows of no lane are not written."""
    if q.dim() != 3 or q.shape[2] != 128 or q.dtype not in (torch.float16, torch.float32):
        raise ValueError("chunk_attention: q must be [rows, heads, 128], f16 or f32")
    rows, heads, _ = q.shape
    if heads % kv.n_kv:
        raise ValueError(f"chunk_attention: {heads} heads over {kv.n_kv} kv heads")
    if not -2 ** 31 <= window < 2 ** 31:
        raise ValueError("chunk_attention: window must be 0 or a number of positions below 2^31")
    same_device("chunk_attention", q, row_start, spans, out)
    b = chunk_batch("chunk_attention", rows, row_start, spans, kv)
    if out is None:
        out = torch.empty(rows, heads * 128, device=q.device, dtype=torch.float16)
    elif out.numel() != q.numel() or out.dtype != torch.float16 or not out.is_contiguous():
        raise ValueError("chunk_attention: out must be contiguous f16 [rows, heads * 128]")
    if rows == 0:
        return out
    qc = packed(q)
    c = ctx_of(q)
    # from torch's allocator, so that calls on several streams or in several graphs have their own
    size = _workspace.get(q.device.index)
    if size is None:
        size = _workspace[q.device.index] = int(L.load().tts_chunk_attention_workspace(c))
    work = torch.empty(size, dtype=torch.uint8, device=q.device)
    L.call("tts_chunk_attention", c, qc.data_ptr(), int(q.dtype == torch.float16),
           heads // kv.n_kv, C.byref(b), C.byref(kv), float(scale), int(window), out.data_ptr(),
           work.data_ptr(), size, stream_of(q))
    return out
