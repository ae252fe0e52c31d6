"""The serving operators for ragged chunks of new tokens over a paged KV cache: rotation and
append, attention, and the filtered draw of the next token. Each in its plain form (elementary
torch operations in 32 or 64 bits) and, where `own` is true, as a user calls the framework."""
import itertools
import math
import os
import random
import sys

import torch

own = False

HD = 128  # the paged cache's head width


def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dream-tts_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ttsnn
    return ttsnn


# ---------------------------------------------------------------- cases

def _attn(name, **kw):
    return {"name": name, "op": "attention", "window": 0, "q32": False, "pad": 0, **kw}


def _append(name, **kw):
    return {"name": name, "op": "append", "x32": True, "q32": False, "norm": False,
            "interleaved": False, "rotary": HD, "factor": 1.0, "pad": 0, **kw}


def listed():
    return [
        # a few lanes early in their answers, one new token each: launch latency counts
        _attn("attn_token_few", lanes=3, new=1, new_min=1, held=140, held_min=20, n_kv=8, gqa=2, page=16),
        # a full decode batch deep into long documents, one token a lane: bound by reading the cache
        _attn("attn_token_long", lanes=48, new=1, new_min=1, held=8000, held_min=600, n_kv=8, gqa=2, page=32),
        # prompts of different lengths joining lanes that already hold some, sliding window, odd
        # lengths, pages that end inside a tile, rows of padding behind the last lane
        _attn("attn_chunk_ragged", lanes=13, new=701, new_min=0, held=1900, held_min=0, n_kv=4, gqa=4,
              page=24, window=1000, q32=True, pad=5),
        # one chunk of a long prompt over what is cached already: bound by the tensor cores
        _attn("attn_prompt_long", lanes=1, new=4096, new_min=4096, held=12288, held_min=12288,
              n_kv=8, gqa=2, page=64),
        # a decode batch's rows rotated, normed and appended
        _append("append_token", lanes=48, new=1, new_min=1, held=3000, held_min=10, heads=16, n_kv=8,
                page=16, norm=True, table=4096),
        # the chunk of a ragged prompt batch with the model's QK-norm
        _append("append_chunk", lanes=21, new=900, new_min=1, held=2100, held_min=0, heads=16, n_kv=8,
                page=32, norm=True, table=4096),
        # interleaved pairs over half of each head, scaled positions, f16 rows, padding behind
        _append("append_partial", lanes=7, new=1501, new_min=3, held=9000, held_min=0, heads=28, n_kv=4,
                page=8, rotary=64, interleaved=True, x32=False, factor=4.0, table=16384, pad=9),
        # the rotation alone at a narrow head, a short text
        {"name": "rotate_small", "op": "rotate", "rows": 77, "heads": 12, "hd": 64, "rotary": 64,
         "interleaved": False, "x32": True, "factor": 1.0, "table": 2048},
        # a long document's rows at far positions, part of an odd head width
        {"name": "rotate_far", "op": "rotate", "rows": 12345, "heads": 20, "hd": 96, "rotary": 48,
         "interleaved": True, "x32": False, "factor": 8.0, "table": 131072},
        # a codebook head's logits for a few lanes, top-k
        {"name": "sample_codes", "op": "sample", "rows": 8, "n": 2048, "x32": True, "k": 50, "p": 1.0,
         "min_p": 0.0, "banned": 0.0},
        # a text vocabulary, every request with its own settings, some ids banned
        {"name": "sample_mixed", "op": "sample", "rows": 48, "n": 32003, "x32": False, "k": 200, "p": 0.8,
         "min_p": 0.02, "banned": 0.05},
        # a large batch over a large vocabulary, nucleus only
        {"name": "sample_large", "op": "sample", "rows": 192, "n": 151851, "x32": True, "k": 0, "p": 0.9,
         "min_p": 0.0, "banned": 0.0},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "rotate", "sample", "sample"])
    if op == "attention":
        c = {"op": op, "lanes": _log(rng, 1, 64), "new": _log(rng, 1, 4096), "held": _log(rng, 1, 12288),
             "n_kv": rng.choice([1, 2, 4, 8]), "gqa": rng.choice([1, 2, 3, 4, 7, 8]),
             "page": rng.choice([8, 16, 24, 32, 64, 128]),
             "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]), "q32": rng.random() < 0.3, "pad": rng.randrange(3)}
        c["n_kv"] = min(c["n_kv"], 32 // c["gqa"]) or 1
        c["new_min"], c["held_min"] = rng.choice([0, 1, c["new"]]), rng.choice([0, c["held"]])
        limit = 16 * 4096 * 16384
        while c["lanes"] * c["n_kv"] * c["gqa"] * c["new"] * (c["new"] + c["held"]) > limit // 2:
            side = "lanes" if c["lanes"] > 1 else "new" if c["new"] > 1 else "held"
            c[side] = (c[side] + 1) // 2
            c["new_min"], c["held_min"] = min(c["new_min"], c["new"]), min(c["held_min"], c["held"])
        while c["lanes"] * c["n_kv"] * (c["new"] + c["held"]) > 48 * 8 * 6000:
            c["lanes"] = (c["lanes"] + 1) // 2
        return c
    if op == "append":
        c = {"op": op, "lanes": _log(rng, 1, 64), "new": _log(rng, 1, 1500), "held": _log(rng, 1, 9000),
             "heads": rng.choice([4, 8, 16, 28]), "n_kv": rng.choice([2, 4, 8]), "page": rng.choice([5, 8, 16, 24, 64]),
             "rotary": rng.choice([128, 128, 64, 32, 96, 24]), "interleaved": rng.random() < 0.5,
             "x32": rng.random() < 0.6, "q32": rng.random() < 0.4, "norm": rng.random() < 0.5,
             "factor": rng.choice([1.0, 2.0, 8.0]), "pad": rng.randrange(4), "table": 16384}
        c["heads"] = c["heads"] if c["heads"] % c["n_kv"] == 0 else 16
        while c["lanes"] * c["new"] * (c["heads"] + c["n_kv"]) > 9000 * 24:
            c["lanes"] = (c["lanes"] + 1) // 2 if c["lanes"] > 1 else 1
            c["new"] = c["new"] if c["lanes"] > 1 else min(c["new"], 1000)
        c["new_min"], c["held_min"] = rng.choice([0, 1, c["new"]]), rng.choice([0, c["held"]])
        return c
    if op == "rotate":
        hd = rng.choice([32, 64, 80, 96, 128, 192, 256])
        return {"op": op, "rows": _log(rng, 1, 12000), "heads": rng.randint(1, 1900 // hd), "hd": hd,
                "rotary": 8 * rng.randint(1, hd // 8), "interleaved": rng.random() < 0.5,
                "x32": rng.random() < 0.5, "factor": rng.choice([1.0, 4.0]), "table": 131072}
    n = _log(rng, 2, 151851)
    return {"op": op, "rows": _log(rng, 1, 190), "n": n, "x32": rng.random() < 0.6,
            "k": rng.choice([0, 1, _log(rng, 1, 1000), n + 1]), "p": rng.choice([1.0, round(rng.uniform(0.05, 1.0), 3)]),
            "min_p": rng.choice([0.0, round(rng.uniform(0.0, 0.3), 3)]), "banned": rng.choice([0.0, 0.1])}


def _lengths(case):
    """The lanes' new and held positions, from the case alone."""
    r = random.Random("%d %d %d %d" % (case["lanes"], case["new"], case["held"], case["n_kv"]))
    new = [r.randint(case["new_min"], case["new"]) for _ in range(case["lanes"])]
    held = [r.randint(case["held_min"], case["held"]) for _ in range(case["lanes"])]
    return new, held


# ---------------------------------------------------------------- inputs

def _chunk_state(case, g):
    """The ragged batch and its paged cache: row starts, spans, shuffled pages."""
    new, held = _lengths(case)
    starts = [0, *itertools.accumulate(new)]
    spans = [n + h for n, h in zip(new, held)]
    page, lanes = case["page"], case["lanes"]
    per = max(1, -(-max(spans) // page))
    pages = lanes * per + 3
    order = torch.randperm(pages, device="cuda", generator=g)
    table = order[:lanes * per].reshape(lanes, per)
    shape = (pages, case["n_kv"], page, HD)
    return {"row_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
            "spans": torch.tensor(spans, dtype=torch.int32, device="cuda"),
            "table": table.to(torch.int32).contiguous(), "rows": starts[-1] + case["pad"],
            "new_max": max(new), "spare": order[-1], "k": torch.randn(shape, device="cuda", generator=g, dtype=torch.float16),
            "v": torch.randn(shape, device="cuda", generator=g, dtype=torch.float16)}


def _tables(length, rotary, factor):
    """Rotary tables [length, rotary / 2] with positions divided by `factor` (angles in 64 bits)."""
    i = torch.arange(rotary // 2, device="cuda", dtype=torch.float64)
    angle = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] / factor * 1e6 ** (-2 * i / rotary)
    return torch.cos(angle).float(), torch.sin(angle).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    if case["op"] == "attention":
        s = _chunk_state(case, g)
        heads = case["n_kv"] * case["gqa"]
        # normed queries and keys: scores of a few units
        s["q"] = normal(s["rows"], heads, HD) * 2
        s["q"] = s["q"] if case["q32"] else s["q"].half()
        s["out"] = torch.zeros(s["rows"], heads * HD, device="cuda", dtype=torch.float16)
    elif case["op"] == "append":
        s = _chunk_state(case, g)
        x = normal(s["rows"], (case["heads"] + 2 * case["n_kv"]) * HD)
        s["qkv"] = x if case["x32"] else x.half()
        s["norms"] = 1 + 0.1 * normal(2, HD) if case["norm"] else None
        s["cos"], s["sin"] = _tables(case["table"], case["rotary"], case["factor"])
        s["q"] = torch.zeros(s["rows"], case["heads"], HD, device="cuda",
                             dtype=torch.float32 if case["q32"] else torch.float16)
    elif case["op"] == "rotate":
        x = normal(case["rows"], case["heads"], case["hd"])
        s = {"x": x if case["x32"] else x.half()}
        s["cos"], s["sin"] = _tables(case["table"], case["rotary"], case["factor"])
        s["positions"] = torch.randint(0, case["table"], (case["rows"],), device="cuda", generator=g, dtype=torch.int32)
    else:
        rows, n = case["rows"], case["n"]
        # a bulk of unlikely ids and a few that stand out
        x = normal(rows, n) * 2
        x += 6 * (torch.rand(rows, n, device="cuda", generator=g) < 20 / n) * torch.rand(rows, 1, device="cuda", generator=g)
        if case["banned"]:
            banned = torch.rand(n, device="cuda", generator=g) < case["banned"]
            banned[0] = False
            x.masked_fill_(banned, -math.inf)
        s = {"logits": x if case["x32"] else x.half(), "draws": torch.rand(rows, device="cuda", generator=g)}
        u = torch.rand(4, rows, device="cuda", generator=g)
        s["temperature"] = 0.5 + u[0]
        s["top_k"] = (case["k"] * (0.2 + 0.8 * u[1])).ceil().int()
        s["top_p"] = torch.where(u[2] < 0.1, 1.0, case["p"] + (1 - case["p"]) * 0.5 * u[2])
        s["min_p"] = case["min_p"] * u[3]
    s["case"] = case
    return s


# ---------------------------------------------------------------- plain forms

def _row_places(s):
    """Each row's lane (the last lane's index + 1 for rows behind them), offset and position."""
    row = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    lane = torch.searchsorted(s["row_start"][1:].contiguous(), row, right=True)
    live = lane < len(s["spans"])
    at = lane.clamp(max=len(s["spans"]) - 1)
    offset = row - s["row_start"][at]
    position = s["spans"][at] - (s["row_start"][at + 1] - s["row_start"][at]) + offset
    return live, at, offset, position


def _plain_attention(s):
    case = s["case"]
    lanes, n_kv, gqa = case["lanes"], case["n_kv"], case["gqa"]
    live, lane, offset, _ = _row_places(s)
    n = max(1, s["new_max"])
    cached = lambda pages: pages[s["table"].long()].transpose(1, 2).reshape(lanes, n_kv, -1, HD).float()  # noqa: E731
    k, v = cached(s["k"]), cached(s["v"])
    j = torch.arange(n, device="cuda")
    row = (s["row_start"][:-1, None] + j).clamp(max=s["rows"] - 1)
    q = s["q"][row.long()].float().reshape(lanes, n, n_kv, gqa, HD).permute(0, 2, 3, 1, 4).reshape(lanes, n_kv, gqa * n, HD)
    position = (s["spans"] - s["row_start"][1:] + s["row_start"][:-1])[:, None] + j
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= position[..., None]
    if case["window"]:
        seen &= key > position[..., None] - case["window"]
    x = (q @ k.transpose(2, 3)).reshape(lanes, n_kv, gqa, n, -1).mul_(HD ** -0.5)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x.exp_()
    x /= x.sum(-1, keepdim=True).clamp(min=1e-37)
    o = (x.reshape(lanes, n_kv, gqa * n, -1) @ v).reshape(lanes, n_kv, gqa, n, HD)
    o = o[lane, :, :, offset.clamp(max=n - 1)].reshape(s["rows"], -1).half()
    return torch.where(live[:, None], o, s["out"])


def _turn(x, cos, sin, rotary, interleaved):
    """Rotates the first `rotary` dims of each head of x [rows, heads, hd]; cos, sin [rows, 1, rotary / 2]."""
    if interleaved:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., rotary:]), -1)


def _plain_append(s):
    case = s["case"]
    heads, n_kv, page = case["heads"], case["n_kv"], case["page"]
    live, lane, _, position = _row_places(s)
    x = s["qkv"].float().reshape(s["rows"], heads + 2 * n_kv, HD)
    qk = x[:, :heads + n_kv]
    if case["norm"]:
        qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + 1e-6)
        qk = torch.cat((qk[:, :heads] * s["norms"][0], qk[:, heads:] * s["norms"][1]), 1)
    at = position.clamp(min=0).long()
    qk = _turn(qk, s["cos"][at][:, None], s["sin"][at][:, None], case["rotary"], case["interleaved"])
    q = torch.where(live[:, None, None], qk[:, :heads].to(s["q"].dtype), s["q"])
    # rows behind the last lane write a page of no lane with what it holds already
    block = s["table"].long()[lane, (at // page).clamp(max=s["table"].shape[1] - 1)]
    block = torch.where(live, block, s["spare"])
    slot = torch.where(live, at % page, torch.zeros_like(at))
    free = torch.logical_not(live)[:, None, None]
    for_k = torch.where(free, s["k"][block, :, slot], qk[:, heads:].half())
    for_v = torch.where(free, s["v"][block, :, slot], x[:, heads + n_kv:].half())
    s["k"][block, :, slot] = for_k
    s["v"][block, :, slot] = for_v
    return {"q": q, "k": s["k"], "v": s["v"]}


def _plain_rotate(s):
    case, at = s["case"], s["positions"].long()
    y = _turn(s["x"].float(), s["cos"][at][:, None], s["sin"][at][:, None], case["rotary"], case["interleaved"])
    return y.to(s["x"].dtype)


def _plain_sample(s):
    x = s["logits"].float()
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device="cuda")
    z = (value.double() - value[:, :1].double()) / s["temperature"].double()[:, None]
    w = z.exp()
    k = s["top_k"][:, None]
    w = torch.where((rank < k) | (k <= 0), w, 0.0)
    total = w.cumsum(1)
    p = s["top_p"].double()[:, None]
    w = torch.where((total - w < p * total[:, -1:]) | (p >= 1), w, 0.0)
    w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    total = w.cumsum(1)
    at = (total < s["draws"].double()[:, None] * total[:, -1:]).sum(1)
    return index.gather(1, at[:, None])[:, 0].int()


def _cache(ttsnn, s):
    return ttsnn.attn.paged_cache(s["k"], s["v"], s["table"])


def _own(s):
    case, ttsnn = s["case"], _framework()
    if case["op"] == "attention":
        return ttsnn.attn.chunk_attention(s["q"], s["row_start"], s["spans"], _cache(ttsnn, s),
                                          scale=HD ** -0.5, window=case["window"], out=s["out"])
    if case["op"] == "append":
        q = ttsnn.qkrope.rotary_append(s["qkv"], case["heads"], s["row_start"], s["spans"], s["cos"], s["sin"],
                                       _cache(ttsnn, s), interleaved=case["interleaved"], norms=s["norms"],
                                       eps=1e-6, out=s["q"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if case["op"] == "rotate":
        return ttsnn.qkrope.rotary(s["x"], s["positions"], s["cos"], s["sin"], interleaved=case["interleaved"])
    return ttsnn.topk.sample_filtered(s["logits"], s["draws"], s["temperature"], top_k=s["top_k"],
                                      top_p=s["top_p"], min_p=s["min_p"])


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "append": _plain_append, "rotate": _plain_rotate,
            "sample": _plain_sample}[state["case"]["op"]](state)


# ---------------------------------------------------------------- work and exact values

def work(case):
    size = lambda wide: 4 if wide else 2  # noqa: E731
    if case["op"] == "sample":
        rows, n = case["rows"], case["n"]
        return {"bytes": rows * (n * size(case["x32"]) + 24), "flops": 2 * rows * n}
    if case["op"] == "rotate":
        rows, heads, hd, rot = (case[x] for x in ("rows", "heads", "hd", "rotary"))
        return {"bytes": rows * (2 * heads * hd * size(case["x32"]) + rot * 4 + 4), "flops": 3 * rows * heads * rot}
    new, held = _lengths(case)
    rows, n_kv = sum(new), case["n_kv"]
    if case["op"] == "append":
        heads, rot = case["heads"], case["rotary"]
        wide = HD * (heads * (size(case["x32"]) + size(case["q32"])) + 2 * n_kv * (size(case["x32"]) + 2))
        return {"bytes": rows * (wide + rot * 4), "flops": rows * (heads + n_kv) * (3 * rot + (4 * HD if case["norm"] else 0))}
    heads, w = n_kv * case["gqa"], case["window"] or 1 << 40
    seen = sum(min(p + 1, w) for n, h in zip(new, held) for p in range(h, h + n))
    keys = sum(h + n - max(0, h + 1 - w) for n, h in zip(new, held) if n)
    return {"bytes": rows * heads * HD * (size(case["q32"]) + 2) + keys * n_kv * HD * 4, "flops": 4 * HD * heads * seen}


def exact(case, seed):
    def attention():
        new, held = _lengths(case)
        out = s["out"].double()
        row = 0
        for i in range(case["lanes"]):
            n, span = new[i], new[i] + held[i]
            at = torch.arange(span, device="cuda")
            page, slot = s["table"][i].long()[at // case["page"]], at % case["page"]
            p = torch.arange(held[i], span, device="cuda")[:, None]
            hidden = at[None] > p
            if case["window"]:
                hidden |= at[None] <= p - case["window"]
            for h in range(case["n_kv"] * case["gqa"] if n else 0):
                k, v = (t[page, h // case["gqa"], slot].double() for t in (s["k"], s["v"]))
                a = s["q"][row:row + n, h].double() @ k.T / math.sqrt(HD)
                a[hidden] = -math.inf
                out[row:row + n, h * HD:(h + 1) * HD] = torch.softmax(a, 1) @ v
            row += n
        return out

    def turn(x, c, s, rotary, interleaved):
        y = x.clone()
        for i in range(rotary // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
            y[..., a] = x[..., a] * c[:, None, i] - x[..., b] * s[:, None, i]
            y[..., b] = x[..., b] * c[:, None, i] + x[..., a] * s[:, None, i]
        return y

    def append():
        new, held = _lengths(case)
        heads, n_kv = case["heads"], case["n_kv"]
        q, kc, vc = s["q"].double(), s["k"].double(), s["v"].double()
        row = 0
        for i in range(case["lanes"]):
            n = new[i]
            at = torch.arange(held[i], held[i] + n, device="cuda")
            x = s["qkv"][row:row + n].double().reshape(n, heads + 2 * n_kv, HD)
            parts = [x[:, :heads], x[:, heads:heads + n_kv]]
            if case["norm"]:
                parts = [y * s["norms"][j].double() / torch.sqrt(torch.linalg.vector_norm(y, dim=-1, keepdim=True) ** 2 / HD + 1e-6)
                         for j, y in enumerate(parts)]
            parts = [turn(y, s["cos"][at].double(), s["sin"][at].double(), case["rotary"], case["interleaved"]) for y in parts]
            page, slot = s["table"][i].long()[at // case["page"]], at % case["page"]
            q[row:row + n] = parts[0]
            kc[page, :, slot], vc[page, :, slot] = parts[1], x[:, heads + n_kv:]
            row += n
        return {"q": q, "k": kc, "v": vc}

    def sample():
        picks = []
        host = {name: s[name].cpu().double().tolist() for name in ("draws", "temperature", "top_k", "top_p", "min_p")}
        for r in range(len(host["draws"])):
            x = s["logits"][r].double()
            order = torch.argsort(-x, stable=True)
            kept = order[:int(host["top_k"][r])] if host["top_k"][r] > 0 else order
            w = torch.exp(x[kept] / host["temperature"][r] - x[kept[0]] / host["temperature"][r])
            if host["top_p"][r] < 1:
                share = torch.cumsum(w, 0) / w.sum()
                last = int((share < host["top_p"][r]).sum())
                kept, w = kept[:last + 1], w[:last + 1]
            enough = int((w >= host["min_p"][r]).sum())
            kept, share = kept[:enough], torch.cumsum(w[:enough], 0) / w[:enough].sum()
            picks.append(int(kept[min(int((share < host["draws"][r]).sum()), enough - 1)]))
        return torch.tensor(picks, dtype=torch.int32)

    s = prepare(case, seed)
    if case["op"] == "attention":
        return attention()
    if case["op"] == "append":
        return append()
    if case["op"] == "rotate":
        x, at = s["x"].double(), s["positions"].long()
        return turn(x, s["cos"][at].double(), s["sin"][at].double(), case["rotary"], case["interleaved"])
    return sample()
