"""Ragged chunk batches over paged caches for the chunk operators' tests, and their definitions
in 64 bits."""
import numpy as np

F16, F32 = 2.0 ** -11, 2.0 ** -24  # half a step of each type, relative


def batch(seed, new, held, n_kv, page, spare=3, first=0, one_page=False):
    """Lanes with new[i] rows over held[i] positions: row starts (from `first`), spans, a shuffled
    block table and pools f16 N(0, 1)."""
    rng = np.random.default_rng(seed)
    lanes = len(new)
    starts = np.concatenate([[first], first + np.cumsum(new)]).astype(np.int32)
    spans = (np.asarray(new) + np.asarray(held)).astype(np.int32)
    per = 1 if one_page else max(1, -(-int(max(spans.max(), 1)) // page))
    pages = lanes * per + spare
    table = rng.permutation(pages)[:lanes * per].reshape(lanes, per).astype(np.int32)
    k = rng.standard_normal((pages, n_kv, page, 128)).astype(np.float16)
    v = rng.standard_normal((pages, n_kv, page, 128)).astype(np.float16)
    return starts, spans, table, k, v


def lane_rows(pool, table, lane, span):
    """The lane's first `span` cached rows [span, n_kv, 128] in 64 bits (pages outside the pool 0)."""
    page = pool.shape[2]
    at = np.arange(span)
    pg = table[lane, at // page] if span else np.zeros(0, int)
    ok = (pg >= 0) & (pg < pool.shape[0])
    rows = pool[np.where(ok, pg, 0), :, at % page].astype(np.float64)
    return np.where(ok[:, None, None], rows, 0.0)


def attention(q, starts, spans, table, k, v, scale, window, out):
    """chunk_attention's definition over `out` (rows of no lane kept), and the sum of |w v| that
    bounds what rounding the weights can move."""
    out = out.astype(np.float64)
    mass = np.zeros_like(out)
    heads, n_kv = q.shape[1], k.shape[1]
    for i in range(len(spans)):
        n, span = starts[i + 1] - starts[i], int(spans[i])
        kc, vc = lane_rows(k, table, i, span), lane_rows(v, table, i, span)
        for j in range(n):
            p = span - n + j
            lo = max(0, p + 1 - window) if window else 0
            for h in range(heads):
                row, cols = starts[i] + j, slice(h * 128, h * 128 + 128)
                if p < 0:
                    out[row, cols] = 0
                    continue
                s = kc[lo:p + 1, h * n_kv // heads] @ q[row, h].astype(np.float64) * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                vv = vc[lo:p + 1, h * n_kv // heads]
                out[row, cols] = w @ vv
                mass[row, cols] = w @ np.abs(vv)
    return out, mass


def attention_bound(want, mass):
    """Weights rounded to f16 (half a step each of sum |w v|), 2^-13 of it for the f32 scores and
    exponentials, the f16 result."""
    return (F16 + 2.0 ** -13) * mass + F16 * np.abs(want) + 2.0 ** -25


def turn(x, cos, sin, rotary, interleaved):
    """The rotation of x [rows, heads, hd] in 64 bits with the rows' tables [rows, rotary / 2], and
    |a cos| + |b sin|."""
    x, c, s = x.astype(np.float64), cos[:, None].astype(np.float64), sin[:, None].astype(np.float64)
    ia = np.arange(0, rotary, 2) if interleaved else np.arange(rotary // 2)
    ib = ia + 1 if interleaved else ia + rotary // 2
    y, mass = x.copy(), np.abs(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mass[..., ia], mass[..., ib] = np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)
    return y, mass


def tables(length, rotary, base=1e4):
    ph = np.arange(length)[:, None] * base ** (-2.0 * np.arange(rotary // 2) / rotary)
    return np.cos(ph).astype(np.float32), np.sin(ph).astype(np.float32)


def sample(logits, draws, temperature=None, top_k=None, top_p=None, min_p=None):
    """sample_filtered's definition, row by row in 64 bits."""
    picks = []
    for r in range(logits.shape[0]):
        x = logits[r].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x)
        ids = np.argsort(-x, kind="stable")
        ids = ids[x[ids] > -np.inf]
        if not len(ids):
            picks.append(-1)
            continue
        t = 1.0 if temperature is None else float(temperature[r])
        if not t > 0:
            picks.append(ids[0])
            continue
        v = x[ids]
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(v == v[0], 1.0, np.exp((v - v[0]) / t))
        k = 0 if top_k is None else int(top_k[r])
        if k > 0:
            ids, w = ids[:k], w[:k]
        p = 1.0 if top_p is None else float(top_p[r])
        if p < 1:
            n = int((np.cumsum(w) < p * w.sum()).sum()) + 1
            ids, w = ids[:n], w[:n]
        m = 0.0 if min_p is None else float(min_p[r])
        if m > 0:
            n = int((w >= min(m, 1.0)).sum())
            ids, w = ids[:n], w[:n]
        c = np.cumsum(w)
        picks.append(ids[min(int((c < float(draws[r]) * c[-1]).sum()), len(ids) - 1)])
    return np.array(picks, np.int32)
