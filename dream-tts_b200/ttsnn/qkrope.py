"""QK-norm, RoPE and the KV-cache write in one launch (crates/tts-nn/src/qkrope.rs)."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from ._ctx import ctx_of, packed, ptr, stream, stream_of


def eligible(qkv: torch.Tensor, k_cache: torch.Tensor, head_dim: int) -> bool:
    """Shapes the kernel takes (qkrope.rs:11-18): f32 activations, f16 cache, head_dim 128."""
    return (qkv.is_cuda and qkv.dtype == torch.float32 and k_cache.dtype == torch.float16
            and head_dim == 128)


def contiguous_cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[L.KvCache, torch.Tensor]:
    """The reference's per-lane cache `[b, n_kv, cap, 128]` as a paged cache: one page of
    `cap` positions per lane, page i = lane i of the (possibly narrowed) view."""
    b, n_kv, cap, hd = k_cache.shape
    for c in (k_cache, v_cache):
        if not c.is_contiguous():
            raise ValueError("qk_rope: cache must be contiguous")
    table = torch.arange(b, dtype=torch.int32, device=k_cache.device).reshape(b, 1)
    kv = L.KvCache(k_cache.data_ptr(), v_cache.data_ptr(), table.data_ptr(), 1, cap, b, n_kv, hd)
    return kv, table


def apply(qkv: torch.Tensor, norms: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
          k_cache: torch.Tensor, v_cache: torch.Tensor, heads: int, start, eps: float,
          f32_kv: bool = False) -> tuple[torch.Tensor, None]:
    """`qkv [b, 1, (heads + 2 n_kv) * 128]` f32 -> q `[b, heads, 1, 128]`; k and v are written
    as f16 into the caches `[b, n_kv, cap, 128]` at position `start` (qkrope.rs:26-69).
    `start` may also be an int32 tensor `[b]` of per-lane positions (lanes of different lengths
    in one step, which the paged decode step does; the reference uses one start per call).

    Decode only (t == 1): prefill's multi-position form is not on this path.
    """
    b, t, width = qkv.shape
    _, n_kv, cap, hd = k_cache.shape
    if t != 1:
        raise L.TtsError(2, "qk_rope: only t == 1 (a decode step) is supported")
    if f32_kv:
        raise L.TtsError(2, "qk_rope: the f32 k/v side outputs are prefill-only")
    if isinstance(start, torch.Tensor):
        pos = start.to(device=qkv.device, dtype=torch.int32).contiguous()
        if pos.numel() != b:
            raise ValueError("qk_rope: one position per lane")
        end = int(pos.max().item()) + t
    else:
        pos = torch.full((b,), int(start), dtype=torch.int32, device=qkv.device)
        end = int(start) + t
    if end > cap:
        raise ValueError(f"qk_rope: {end} positions exceed {cap}")
    if width != (heads + 2 * n_kv) * hd:
        raise ValueError("qk_rope: qkv width does not match heads and cache")
    x = qkv.reshape(b, width).contiguous()
    kv, table = contiguous_cache(k_cache, v_cache)
    q = torch.empty(b, heads, hd, device=qkv.device, dtype=torch.float32)
    nm = norms.to(torch.float32).contiguous()
    L.call("tts_qk_rope_append", ctx_of(x), ptr(x), b, heads, ptr(nm), ptr(cos.contiguous()),
           ptr(sin.contiguous()), cos.shape[0], ptr(pos), C.byref(kv), float(eps), ptr(q),
           stream())
    return q.reshape(b, heads, 1, hd), None


def chunk_batch(op: str, rows: int, row_start: torch.Tensor, spans: torch.Tensor,
                kv: L.KvCache) -> L.ChunkBatch:
    """The ragged batch of a chunk call: int32 device tensors `row_start [lanes + 1]` and
    `spans [lanes]` (tts_chunk_batch)."""
    lanes = spans.numel()
    if row_start.dtype != torch.int32 or spans.dtype != torch.int32:
        raise ValueError(f"{op}: row_start and spans must be int32")
    if row_start.numel() != lanes + 1 or not (row_start.is_contiguous() and spans.is_contiguous()):
        raise ValueError(f"{op}: row_start must hold one entry more than spans, both contiguous")
    if lanes > getattr(kv, "lanes", lanes):
        raise ValueError(f"{op}: {lanes} lanes over a block table of {kv.lanes}")
    same_device(op, row_start, *getattr(kv, "keep", ()))
    return L.ChunkBatch(lanes, rows, row_start.data_ptr(), spans.data_ptr())


def same_device(op: str, x: torch.Tensor, *others: torch.Tensor | None) -> None:
    dev = x.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"{op}: tensors on {dev} and {t.device}")


def _tables(op: str, cos: torch.Tensor, sin: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    if cos.shape != sin.shape or cos.dim() != 2:
        raise ValueError(f"{op}: cos and sin must be [positions, rotary_dim / 2] both")
    return packed(cos, torch.float32), packed(sin, torch.float32)


def rotary(x: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
           interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions on `x [rows, heads, head_dim]` (f32 or f16), row r at `positions[r]`
    (int32): the first 2 * cos.shape[1] dims of each head in half-split or interleaved pairs, the
    rest copied. x may be a column block of wider rows. Into `out` (x, or memory
    apart from it), else a new tensor."""
    if x.dim() != 3 or x.dtype not in (torch.float32, torch.float16):
        raise ValueError("rotary: x must be [rows, heads, head_dim], f32 or f16")
    rows, heads, hd = x.shape
    if positions.dtype != torch.int32 or positions.numel() != rows or not positions.is_contiguous():
        raise ValueError("rotary: one contiguous int32 position per row")
    same_device("rotary", x, positions, cos, sin, out)
    c, s = _tables("rotary", cos, sin)

    def whole(t):
        row, head, one = t.stride()  # of a dimension of one entry it says nothing
        return (one == 1 and (head == hd or heads == 1) and t.data_ptr() % 16 == 0
                and (rows == 1 or row % 8 == 0 and heads * hd <= row < 2 ** 31))

    def pitch(t):
        return t.stride(0) if rows > 1 else heads * hd

    if out is None:
        y = x.new_empty((rows, heads, hd))
    else:
        if out.shape != x.shape or out.dtype != x.dtype or not whole(out):
            raise ValueError("rotary: out must have x's shape and type, heads side by side and "
                             "16-byte aligned rows")
        y = out
    if rows == 0:
        return y
    xc = x if whole(x) else packed(x)
    length, pairs = c.shape
    L.call("tts_rotary", ctx_of(x), xc.data_ptr(), x.dtype == torch.float16, rows, heads, hd,
           pitch(xc), positions.data_ptr(), c.data_ptr(), s.data_ptr(), length, 2 * pairs,
           bool(interleaved), y.data_ptr(), pitch(y), stream_of(x))
    return y


def rotary_append(qkv: torch.Tensor, heads: int, row_start: torch.Tensor, spans: torch.Tensor,
                  cos: torch.Tensor, sin: torch.Tensor, kv: L.KvCache, interleaved: bool = False,
                  norms: torch.Tensor | None = None, eps: float = 1e-6, q_f16: bool = True,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """A ragged chunk's rows `qkv [rows, (heads + 2 n_kv) * 128]` (f32 or f16): the QK-norm if
    `norms [2, 128]` is given, the rotation at each row's position, K and V into the pages; the
    rotated q `[rows, heads, 128]` is returned, f16 or f32 (or written to `out`). Lane i's rows
    are row_start[i] .. row_start[i + 1] and spans[i] the positions it holds once they are in; rows
    before position 0 (more of them than spans[i]) are left out, of q too."""
    if qkv.dim() != 2 or qkv.dtype not in (torch.float32, torch.float16):
        raise ValueError("rotary_append: qkv must be [rows, width], f32 or f16")
    rows = qkv.shape[0]
    if qkv.shape[1] != (heads + 2 * kv.n_kv) * 128:
        raise ValueError("rotary_append: qkv width does not match heads and cache")
    if norms is not None and norms.numel() != 256:
        raise ValueError("rotary_append: norms must be [2, 128]")
    same_device("rotary_append", qkv, row_start, spans, cos, sin, norms, out)
    c, s = _tables("rotary_append", cos, sin)
    b = chunk_batch("rotary_append", rows, row_start, spans, kv)
    if out is None:
        q = torch.empty(rows, heads, 128, device=qkv.device,
                        dtype=torch.float16 if q_f16 else torch.float32)
    else:
        if (out.numel() != rows * heads * 128 or not out.is_contiguous()
                or out.dtype not in (torch.float32, torch.float16)):
            raise ValueError("rotary_append: out must be contiguous [rows, heads, 128], f32 or f16")
        q = out
    if rows == 0:
        return q
    x = packed(qkv)
    nm = None if norms is None else packed(norms, torch.float32)
    L.call("tts_rotary_append", ctx_of(x), x.data_ptr(), int(x.dtype == torch.float16), int(heads),
           C.byref(b), None if nm is None else nm.data_ptr(), float(eps), c.data_ptr(),
           s.data_ptr(), c.shape[0], 2 * c.shape[1], int(interleaved), C.byref(kv), q.data_ptr(),
           int(q.dtype == torch.float16), stream_of(x))
    return q
