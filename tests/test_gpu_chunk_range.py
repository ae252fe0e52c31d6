"""Chunk attention over the whole range of its arguments: magnitudes of f32 queries, scales."""
import numpy as np
import pytest
import torch

import _chunks as ck

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def attend(tt, q, b, scale=SCALE, window=0, out=None):
    starts, spans, table, k, v = b
    kv = tt.attn.paged_cache(dev(k), dev(v), dev(table))
    o = tt.attn.chunk_attention(dev(q), dev(starts), dev(spans), kv, scale, window, out)
    return o.cpu().numpy().astype(np.float64)


def score_error(q, b, scale):
    """What f32 scores may be off by: of the largest sum of |scale q_d k_d| of a row and a position
    128 products and sums of half a step each and 2^-22 of what two f16 pieces leave of a query's
    element, 2^-39 of its row's largest where that is more."""
    starts, spans, table, k, v = b
    n_kv, most = k.shape[1], 0.0
    gqa = q.shape[1] // n_kv
    for i in range(len(spans)):
        kc = np.abs(ck.lane_rows(k, table, i, int(spans[i])))
        rows = np.abs(q[starts[i]:starts[i + 1]].astype(np.float64)).reshape(-1, n_kv, gqa, 128)
        for h in range(n_kv if len(kc) and len(rows) else 0):
            most = max(most, (rows[:, h] @ kc[:, h].T).max() * (128 * 2.0 ** -24 + 2.0 ** -22)
                       + 2.0 ** -39 * (rows[:, h].max(-1)[..., None] * kc[:, h].sum(-1)).max())
    return most * abs(scale)


def within(q, b, got, scale):
    """attention_bound, and twice (weights and their sum) what the scores may be off by."""
    want, mass = ck.attention(q, *b, scale, 0, np.zeros(got.shape))
    slack = 2 * score_error(q, b, scale) * mass
    off = np.abs(got - want) - ck.attention_bound(want, mass) - slack
    assert not np.isnan(got).any() and off.max() <= 0, (off.max(), np.argwhere(off > 0)[:4])


@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e-7, 1e-5, 1e-3, 30.0, 1e5, 1e9, 1e37])
def test_f32_queries_of_any_size(tt, size):
    """The same scores from queries of any magnitude, `scale` making up for it."""
    b = ck.batch(61, [1, 40, 150, 3, 2, 70, 1], [200, 30, 0, 129, 7, 300, 400], 2, 16)
    q = (np.random.default_rng(62).standard_normal((int(b[0][-1]), 4, 128)) * size).astype(np.float32)
    scale = float(np.float32(SCALE / size))
    within(q, b, attend(tt, q, b, scale), scale)
    tt.check()


@pytest.mark.parametrize("gqa,seed", [(2, 63), (8, 64)])
def test_f32_queries_of_a_size_for_each_row(tt, gqa, seed):
    """Rows of very different magnitudes beside one another, in runs of every kind."""
    rng = np.random.default_rng(seed)
    new = rng.choice([1, 1, 2, 4, 5, 15, 17, 33, 64, 70, 129, 0], 300)
    b = ck.batch(seed, new, rng.choice([0, 0, 3, 60, 130, 300], 300), 2, 16)
    q = rng.standard_normal((int(b[0][-1]), 2 * gqa, 128))
    q *= rng.choice([1e-20, 1e-6, 0.01, 0.3, 1, 3], (q.shape[0], q.shape[1], 1))
    q = q.astype(np.float32)
    within(q, b, attend(tt, q, b), SCALE)
    tt.check()


def test_f32_queries_of_a_size_for_each_dim(tt):
    """Dims a million times smaller than their row's largest, beside keys as much larger."""
    starts, spans, table, k, v = ck.batch(65, [40, 1], [200, 300], 2, 16)
    small = np.arange(128) % 2 == 1
    k[..., ~small] *= 2.0 ** -10
    k[..., small] *= 2.0 ** 10
    q = np.random.default_rng(66).standard_normal((41, 4, 128))
    q[..., ~small] *= 2.0 ** 10
    q[..., small] *= 2.0 ** -10
    b = (starts, spans, table, k, v)
    q = q.astype(np.float32)
    within(q, b, attend(tt, q, b), SCALE)


def test_f32_queries_of_zero_infinity_and_nan(tt):
    """Rows of zeros weigh all positions alike; a row with an infinity or NaN is NaN, alone."""
    b = ck.batch(69, [60, 1, 2], [30, 100, 3], 2, 16)
    q = np.random.default_rng(70).standard_normal((63, 4, 128)).astype(np.float32)
    q[[3, 60], :] = 0
    q[5, 1, 7] = np.nan
    q[40, 2, 100] = np.inf
    got = attend(tt, q, b).reshape(63, 4, 128)
    assert np.isnan(got[5, 1]).all() and np.isnan(got[40, 2]).all()
    q[5, 1], q[40, 2], got[5, 1], got[40, 2] = 0, 0, 0, 0
    want, mass = ck.attention(q, *b, SCALE, 0, np.zeros((63, 512)))
    want, mass = want.reshape(63, 4, 128), mass.reshape(63, 4, 128)
    want[5, 1], want[40, 2] = 0, 0
    slack = 2 * score_error(q, b, SCALE) * mass
    assert (np.abs(got - want) <= ck.attention_bound(want, mass) + slack).all()
    tt.check()


@pytest.mark.parametrize("q32,size,scale", [(False, 1, 2e38), (True, 1, 2e38), (True, 1e38, 2e38),
                                            (True, 1e38, 1.0), (False, 1, 1e30), (True, 1, -2e38),
                                            (False, 1, 1e9), (True, 1, 3e10), (True, 1e5, 7e6),
                                            (False, 1, -1e12), (True, 1e9, 1.3)])
def test_scores_past_f32(tt, q32, size, scale):
    """Scores far apart, past f32's range: the largest takes it all. Rows whose two largest scores
    are nearer than f32 sums tell apart are left out; a few queries of 1e38 are infinite as f32, their
    rows NaN."""
    b = ck.batch(67, [30, 1, 2], [60, 200, 3], 2, 16)
    q = (np.random.default_rng(68).standard_normal((33, 4, 128)) * size)
    with np.errstate(over="ignore"):
        q = q.astype(np.float32 if q32 else np.float16)
    got = attend(tt, q, b, scale)
    starts, spans, table, k, v = b
    told = 0
    for i in range(3):
        kc, vc = ck.lane_rows(k, table, i, int(spans[i])), ck.lane_rows(v, table, i, int(spans[i]))
        for j in range(starts[i + 1] - starts[i]):
            p = spans[i] - (starts[i + 1] - starts[i]) + j
            for h in range(4):
                if not np.isfinite(q[starts[i] + j, h]).all():
                    assert np.isnan(got[starts[i] + j, h * 128:h * 128 + 128]).all()
                    continue
                s = kc[:p + 1, h // 2] @ q[starts[i] + j, h].astype(np.float64) * np.sign(scale)
                at = np.argsort(s)
                size_of = np.abs(kc[:p + 1, h // 2]) @ np.abs(q[starts[i] + j, h].astype(np.float64))
                if len(at) > 1 and s[at[-1]] - s[at[-2]] < 2.0 ** -15 * size_of.max():
                    continue
                told += 1
                # the lone weight is 2^(8 + the rounding of c s), itself rounded to f16 (half a step)
                # while the f32 sum has it whole: attention_bound of a mass of |v|
                lone = vc[at[-1], h // 2]
                off = np.abs(got[starts[i] + j, h * 128:h * 128 + 128] - lone)
                assert (off <= ck.attention_bound(lone, np.abs(lone))).all()
    assert told > 100
    tt.check()


@pytest.mark.parametrize("q32", [False, True])
@pytest.mark.parametrize("new,gqa", [(3, 1), (70, 4)])
def test_scores_far_below_f32s_steps_then_ordinary_ones(tt, new, gqa, q32):
    """Scores of -1e9 and less at a row's first positions, scores of a few units behind them, which
    alone weigh."""
    starts, spans, table, k, v = ck.batch(71, [new], [900 - new], 1, 32)
    at = np.arange(900)
    k[table[0, at // 32], 0, at % 32, 0] = 0
    level = (starts, spans, table, k.copy(), v)
    k[table[0, at[:700] // 32], 0, at[:700] % 32, 0] = -60000
    q = np.random.default_rng(72).standard_normal((new, gqa, 128))
    q[..., 0] = 60000
    q = q.astype(np.float32 if q32 else np.float16)
    b = (starts, spans, table, k, v)
    got = attend(tt, q, b, 2.0)
    want, mass = ck.attention(q, *b, 2.0, 0, np.zeros(got.shape))
    assert (np.abs(got - want) <= ck.attention_bound(want, mass) + 2 * score_error(q, level, 2.0) * mass).all()
    tt.check()


@pytest.mark.parametrize("q32", [False, True])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3, 2 ** 30, 5])
def test_windows_of_any_size_over_rows_before_position_0(tt, window, q32):
    """Lanes with (many) more new rows than positions beside ordinary ones."""
    starts, spans, table, k, v = ck.batch(73, [3, 20, 300, 1], [0, 400, 10, 129], 2, 16)
    spans[0], spans[2] = 0, 7
    q = np.random.default_rng(74).standard_normal((324, 4, 128)).astype(np.float32 if q32 else np.float16)
    b = (starts, spans, table, k, v)
    got = attend(tt, q, b, window=window, out=torch.full((324, 512), 9.0, device="cuda", dtype=torch.float16))
    wide = starts.astype(np.int64)  # numpy's int32 would wrap as well
    want, mass = ck.attention(q, wide, spans, table, k, v, SCALE, window, np.zeros(got.shape))
    slack = 2 * score_error(q, b, SCALE) * mass
    assert (np.abs(got - want) <= ck.attention_bound(want, mass) + slack).all()
    assert (got[:3] == 0).all() and (got[23:316] == 0).all()
    tt.check()


@pytest.mark.parametrize("q32", [False, True])
@pytest.mark.parametrize("page,window", [(8, 1), (8, 100), (16, 37), (24, 300), (64, 130), (128, 129), (32, 32)])
def test_pages_before_the_window_may_be_gone(tt, page, window, q32):
    """Block-table entries of pages that lie wholly before every row's window name no page of the
    pool: nothing is reported and no row changes, with NaN among the values beside them too."""
    new, held = [1, 1, 40, 1, 170, 3], [900, 333, 500, 129, 260, 700]
    b = ck.batch(75, new, held, 2, page)
    starts, spans, table, k, v = b
    for i in range(6):
        first = max(0, held[i] + 1 - window)  # the first position that a row of the lane sees
        gone = np.arange(first // page)
        table[i, gone] = np.where(gone % 3 == 0, -1, np.where(gone % 3 == 1, k.shape[0], 2 ** 30))
        if first % page:
            at = np.arange(first // page * page, first)
            v[table[i, at // page], :, at % page] = np.nan
    q = np.random.default_rng(76).standard_normal((int(starts[-1]), 4, 128)).astype(np.float32 if q32 else np.float16)
    got = attend(tt, q, b, window=window)
    tt.check()
    want, mass = ck.attention(q, *b, SCALE, window, np.zeros(got.shape))
    slack = 2 * score_error(q, (starts, spans, np.clip(table, 0, k.shape[0] - 1), k, v), SCALE) * mass
    off = np.abs(got - want) - ck.attention_bound(want, mass) - slack
    assert not np.isnan(got).any() and off.max() <= 0, (off.max(), np.argwhere(off > 0)[:4])


@pytest.mark.parametrize("q32", [False, True])
@pytest.mark.parametrize("window", [0, 130000])
def test_values_not_finite_beside_long_spans(tt, window, q32):
    """A NaN that one row of a tile sees, over 131072 positions: the tile's other rows are summed
    again, in every lane, without a wait of the CTA's other warps running out."""
    lanes, new, span, page = 74, 128, 131072, 64
    g = torch.Generator(device="cuda").manual_seed(77)
    k, v = (torch.randn(span // page, 2, page, 128, device="cuda", generator=g).half() for _ in range(2))
    v += 2  # so that a sum of them is not near 0
    table = torch.arange(span // page, dtype=torch.int32, device="cuda").repeat(lanes, 1)
    bad = max(0, span - new + 1 - window) if window else span - 1  # of the first row, or the last
    v[bad // page, :, bad % page] = float("nan")
    one = torch.randn(new, 4, 128, device="cuda", generator=g)
    one = one if q32 else one.half()
    starts = torch.arange(lanes + 1, dtype=torch.int32, device="cuda") * new
    spans = torch.full((lanes,), span, dtype=torch.int32, device="cuda")
    got = tt.attn.chunk_attention(one.repeat(lanes, 1, 1), starts, spans, tt.attn.paged_cache(k, v, table), SCALE,
                                  window).reshape(lanes, new, 4, 128)
    tt.check()
    at, p = torch.arange(span, device="cuda"), torch.arange(span - new, span, device="cuda")[:, None]
    seen = (at <= p) & (at > p - window if window else at >= 0)
    alone = 0 if window else new - 1
    keep = [r for r in range(new) if r != alone]
    for h in range(4):
        kc, vc = (t[:, h // 2].reshape(span, 128).double() for t in (k, v))
        vc[bad] = 0
        w = torch.softmax((one[:, h].double() @ kc.T * SCALE).masked_fill(~seen, -torch.inf), 1)
        want, mass = w @ vc, w @ vc.abs()
        # attention_bound, and f32 sums of 65536 products (half a warp's) and 2048 weights in a row
        bound = (ck.F16 + 2.0 ** -13 + 67584 * ck.F32) * mass + ck.F16 * want.abs() + 2.0 ** -25
        assert (got[:, :, h].double() - want).abs().sub(bound)[:, keep].max() <= 0
        assert torch.isnan(got[:, alone, h]).all()


def test_unaligned_and_one_row_views(tt):
    """Views that start between 16-byte boundaries, and single rows and heads of any stride, give
    what their copies give."""
    off = lambda t, n=1: torch.cat([t.new_zeros(n), t.flatten()])[n:].view(t.shape)
    g = torch.Generator(device="cuda").manual_seed(79)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)
    cos, sin = (dev(t) for t in ck.tables(90, 64))
    pos = torch.arange(5, dtype=torch.int32, device="cuda") * 7
    for x in (rand(5, 3, 64), rand(5, 3, 64).half()):
        want = tt.qkrope.rotary(x, pos, cos, sin)
        assert torch.equal(tt.qkrope.rotary(off(x), pos, off(cos), off(sin, 3)), want)
        assert torch.equal(tt.qkrope.rotary(x.flatten()[64:256].as_strided((1, 3, 64), (5, 64, 1)), pos[:1], cos, sin),
                           tt.qkrope.rotary(x.flatten()[64:256].clone().view(1, 3, 64), pos[:1], cos, sin))
        assert torch.equal(tt.qkrope.rotary(x[:, 1:2], pos, cos, sin), want[:, 1:2])
    starts, spans, table, k, v = ck.batch(80, [5], [20], 1, 8)
    sd, pd, norms = dev(starts), dev(spans), rand(2, 128)
    for x in (rand(5, 4 * 128), rand(5, 4 * 128).half()):
        out = []
        for qkv, c, s, w in ((x, cos, sin, norms), (off(x), off(cos), off(sin), off(norms, 2))):
            kv = tt.attn.paged_cache(dev(k), dev(v), dev(table))
            q = tt.qkrope.rotary_append(qkv, 2, sd, pd, c, s, kv, norms=w)
            out += [q, kv.keep[0], kv.keep[1], tt.attn.chunk_attention(off(q) if qkv is not x else q, sd, pd, kv, SCALE)]
        assert all(torch.equal(a, b) for a, b in zip(out[:4], out[4:], strict=True))
    logits = rand(300, 1).t()
    u = torch.full((1,), 0.6, device="cuda")
    assert torch.equal(tt.topk.sample_filtered(logits, u), tt.topk.sample_filtered(logits.clone().reshape(1, 300), u))
    tt.check()


def test_filtered_draw_over_rows_far_apart(tt):
    """A row stride past 31 bits."""
    flat = torch.zeros(2 ** 31 + 4096, dtype=torch.float16, device="cuda")
    x = flat.as_strided((2, 1000), (2 ** 31 + 8, 1))
    x.copy_(torch.randn(2, 1000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(81)))
    u = torch.tensor([0.3, 0.8], device="cuda")
    want = ck.sample(x.cpu().numpy(), u.cpu().numpy(), top_k=np.array([40, 0]))
    got = tt.topk.sample_filtered(x, u, top_k=torch.tensor([40, 2 ** 40], device="cuda"))
    assert np.array_equal(got.cpu().numpy(), want)


def test_rows_before_position_0_in_both_calls(tt):
    """A lane with more new rows than positions is no error: the append leaves the first ones out,
    the attention gives 0 for them; a span below 0 is reported by both."""
    starts, spans, table, k, v = ck.batch(82, [6, 3], [0, 5], 1, 8)
    spans[0] = 4
    g = torch.Generator(device="cuda").manual_seed(83)
    x = torch.randn(9, 4 * 128, device="cuda", generator=g)
    cos, sin = (dev(t) for t in ck.tables(30, 128))
    kd, vd, sd, pd = dev(k), dev(v), dev(starts), dev(spans)
    kv = tt.attn.paged_cache(kd, vd, dev(table))
    q = torch.full((9, 2, 128), 5.0, device="cuda", dtype=torch.float16)
    tt.qkrope.rotary_append(x, 2, sd, pd, cos, sin, kv, out=q)
    o = tt.attn.chunk_attention(q, sd, pd, kv, SCALE)
    tt.check()
    assert (q[:2] == 5).all() and not (q[2:] == 5).all(-1).any() and (o[:2] == 0).all()
    # rows 2 .. 5 are at positions 0 .. 3: as four rows of their own
    k2, v2 = dev(k), dev(v)
    kv2 = tt.attn.paged_cache(k2, v2, dev(table))
    q2 = tt.qkrope.rotary_append(x[2:], 2, sd.sub(2).clamp(min=0), pd, cos, sin, kv2)
    assert torch.equal(q2, q[2:]) and torch.equal(k2, kd) and torch.equal(v2, vd)
    assert torch.equal(tt.attn.chunk_attention(q2, sd.sub(2).clamp(min=0), pd, kv2, SCALE), o[2:])
    tt.check()
    bad = pd.clone()
    bad[0] = -1
    for call in (lambda: tt.qkrope.rotary_append(x, 2, sd, bad, cos, sin, kv),
                 lambda: tt.attn.chunk_attention(q, sd, bad, kv, SCALE)):
        call()
        with pytest.raises(tt.TtsError, match="out of range"):
            tt.check()


def test_rows_and_pages_past_32_bits(tt):
    """Rows and pages whose elements lie past 2^31 of their buffers, in both chunk calls."""
    rows, heads, n_kv, page = 1_060_000, 16, 8, 64  # 2^31 elements: 1,048,576 rows of q, 32768 pages
    starts, spans, table, k, v = ck.batch(84, [30, 1, 300], [100, 400, 0], n_kv, page)
    g = torch.Generator(device="cuda").manual_seed(85)
    first = rows - 331
    sd, pd = dev(starts + np.int32(first)), dev(spans)
    far = dev(table + np.int32(33000))
    pools = [torch.empty(33000 + len(k), n_kv, page, 128, device="cuda", dtype=torch.float16) for _ in range(2)]
    for pool, near in zip(pools, (k, v)):
        pool[33000:].copy_(dev(near))
    x = torch.empty(rows, (heads + 2 * n_kv) * 128, device="cuda", dtype=torch.float16)
    x[first:].copy_(torch.randn(331, x.shape[1], device="cuda", generator=g))
    cos, sin = (dev(t) for t in ck.tables(500, 128))
    q = torch.empty(rows, heads, 128, device="cuda", dtype=torch.float16)
    out = torch.empty(rows, heads * 128, device="cuda", dtype=torch.float16)
    kv = tt.attn.paged_cache(*pools, far)
    tt.qkrope.rotary_append(x, heads, sd, pd, cos, sin, kv, out=q)
    tt.attn.chunk_attention(q, sd, pd, kv, SCALE, out=out)
    tt.check()
    kd, vd = dev(k), dev(v)
    kv = tt.attn.paged_cache(kd, vd, dev(table))
    want_q = tt.qkrope.rotary_append(x[first:].clone(), heads, dev(starts), pd, cos, sin, kv)
    want = tt.attn.chunk_attention(want_q, dev(starts), pd, kv, SCALE)
    assert torch.equal(q[first:], want_q) and torch.equal(pools[0][33000:], kd) and torch.equal(pools[1][33000:], vd)
    assert torch.equal(out[first:], want)


@pytest.mark.parametrize("q32", [False, True])
@pytest.mark.parametrize("new,held,window", [([200, 1, 300, 2], [100, 4000, 900, 30], 0), ([150, 40], [600, 90], 70)])
def test_values_at_f16s_largest(tt, new, held, window, q32):
    """A mean of values of +-65504 is no larger: roundings of the weights make none infinite."""
    b = ck.batch(86, new, held, 8, 32)
    starts, spans, table, k, v = b
    v[:] = np.float16(65504)
    v[..., 1::2] *= -1
    for seed in range(87, 91):
        q = np.random.default_rng(seed).standard_normal((int(starts[-1]), 16, 128)) * 2
        got = attend(tt, q.astype(np.float32 if q32 else np.float16), b, window=window)
        tt.check()
        off = np.abs(got - np.tile(v[0, 0, 0].astype(np.float64), 16))
        # each weight is half a step of f16 off at most (2^-11), 2^-13 as in attention_bound
        assert (off <= 65504 * (2.0 ** -11 + 2.0 ** -13)).all(), off.max()
    v[table[0, 0], :, 0] = np.inf  # seen by lane 0's rows alone, where the window reaches it
    got = attend(tt, q.astype(np.float32 if q32 else np.float16), b, window=window)
    assert np.isfinite(got[starts[1]:]).all() and np.isfinite(got[:starts[1]]).all() == (window > 0)
