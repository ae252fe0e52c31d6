"""Device-side code picking: greedy (crates/qwen3tts/src/talker.rs:154-189) and top-k sampling
with caller-supplied draws (crates/tts-nn/src/topk.rs)."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from ._ctx import as_type, ctx_of, ptr, stream, stream_of


def argmax(logits: torch.Tensor, banned: torch.Tensor | None = None) -> torch.Tensor:
    """Greedy pick per row over `[rows, n]` f32 with banned ids at -inf; ties go to the
    highest index, as Rust's `max_by` keeps the last maximum."""
    x = logits.to(torch.float32).contiguous()
    rows, n = x.reshape(-1, x.shape[-1]).shape
    out = torch.empty(rows, dtype=torch.int32, device=x.device)
    b = None
    if banned is not None:
        b = banned.to(torch.uint8).contiguous()
        if b.numel() != n:
            raise ValueError("argmax: banned mask must cover every id")
    L.call("tts_argmax", ctx_of(x), ptr(x), rows, n, ptr(b), ptr(out), stream())
    return out


def talker_pick(logits: torch.Tensor, rule, record: bool = False) -> torch.Tensor:
    """sample_with_u's greedy branch (crates/qwen3tts/src/talker.rs:154-189) on `[rows, vocab]`
    f32 under a pick rule (`rule.c`, a PickRule; counts and frames indexed by row): banned ids
    and a young eos at -inf, each id's logit penalised once per time the row emitted it, the
    last of equal maxima. With `record`, the picks join the rows' histories (talker.rs:984-996)."""
    x = logits.to(torch.float32).contiguous()
    rows, n = x.shape
    out = torch.empty(rows, dtype=torch.int32, device=x.device)
    L.call("tts_talker_pick", ctx_of(x), ptr(x), rows, n, rule.c, 1 if record else 0, ptr(out),
           stream())
    return out


MAX_N = 4096
MAX_K = 64


def sample(logits: torch.Tensor, draws: torch.Tensor, k: int, temperature: float) -> torch.Tensor:
    """One index per row of `logits` `[rows, n]` drawn from its top `k` at `temperature` with
    `draws[row]` in `[0, 1)` (crates/tts-nn/src/topk.rs:98-107): no nucleus cut, no penalty."""
    x = logits.to(torch.float32).contiguous()
    rows, n = x.shape
    d = draws.to(torch.float32).contiguous()
    if d.numel() != rows:
        raise L.TtsError(1, f"topk_sample: {d.numel()} draws for {rows} rows")
    out = torch.empty(rows, dtype=torch.int32, device=x.device)
    L.call("tts_topk_sample", ctx_of(x), ptr(x), rows, n, ptr(d), int(k), float(temperature),
           ptr(out), stream())
    return out


def _per_row(v, rows: int, dtype: torch.dtype, device: torch.device, name: str):
    """A setting for every row: None, one value for all, or a tensor of one per row."""
    if v is None:
        return None
    whole = dtype == torch.int32  # any number keeps its meaning: -1 is off, so is 2^30 for any row
    if not isinstance(v, torch.Tensor):
        v = min(max(v, -1), 2 ** 30) if whole else v
        return torch.full((rows,), v, dtype=dtype, device=device)
    if v.numel() != rows or v.device != device:
        raise ValueError(f"sample_filtered: {name} must hold one value per row, on {device}")
    if whole and v.dtype != dtype:
        v = v.to(torch.int64).clamp(-1, 2 ** 30)
    return as_type(v, dtype)


def sample_filtered(logits: torch.Tensor, draws: torch.Tensor, temperature=None, top_k=None,
                    top_p=None, min_p=None) -> torch.Tensor:
    """One id per row of `logits [rows, n]` (f32 or f16; any row stride) drawn with
    `draws[row]` in [0, 1): at `temperature` (None: 1; 0: the largest logit), from the `top_k`
    largest (0: all), of those the shortest prefix with a share `top_p` of the weight, of those
    the ids at least `min_p` times as likely as the first. Each setting is one number or a tensor
    of one per row. int32 [rows], -1 where no id can be picked (tts_filter_sample)."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.float16):
        raise ValueError("sample_filtered: logits must be [rows, n], f32 or f16")
    rows, n = logits.shape
    # (the library's row stride is an int)
    x = logits if logits.stride(1) == 1 and n <= logits.stride(0) < 2 ** 31 else logits.contiguous()
    d = _per_row(draws, rows, torch.float32, x.device, "draws")
    if d is None:
        raise ValueError("sample_filtered: draws are needed")
    each = (_per_row(temperature, rows, torch.float32, x.device, "temperature"),
            _per_row(top_k, rows, torch.int32, x.device, "top_k"),
            _per_row(top_p, rows, torch.float32, x.device, "top_p"),
            _per_row(min_p, rows, torch.float32, x.device, "min_p"))
    how = L.Sampling(*(None if t is None else t.data_ptr() for t in each))
    out = torch.empty(rows, dtype=torch.int32, device=x.device)
    if rows == 0:
        return out
    L.call("tts_filter_sample", ctx_of(x), x.data_ptr(), int(x.dtype == torch.float16), rows, n,
           x.stride(0) if rows > 1 else 0, d.data_ptr(), C.byref(how), out.data_ptr(), stream_of(x))
    return out
