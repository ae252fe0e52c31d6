"""The chunk operators (rotary, rotary_append, chunk_attention) on a B200 against their
definitions in 64 bits. Bounds count roundings: half a step of a type is torch.finfo(t).eps / 2."""
import numpy as np
import pytest
import torch

import _chunks as ck

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.detach().cpu().numpy().astype(np.float64)


def attend(tt, q, b, window=0, out=None, scale=SCALE, table=None):
    starts, spans, tab, k, v = b
    kv = tt.attn.paged_cache(dev(k), dev(v), dev(tab if table is None else table))
    return tt.attn.chunk_attention(dev(q), dev(starts), dev(spans), kv, scale, window, out)


def check_attention(tt, q, b, window=0, clean=True):
    starts, spans, table, k, v = b
    out = np.full((q.shape[0], q.shape[1] * 128), 7.0, np.float16)
    got = host(attend(tt, q, b, window, dev(out)))
    if clean:
        tt.check()
    want, mass = ck.attention(q, starts, spans, table, k, v, SCALE, window, out)
    off = np.abs(got - want) - ck.attention_bound(want, mass)
    assert not np.isnan(got).any() and off.max() <= 0, (off.max(), np.argwhere(off > 0)[:4])


CASES = [  # new, held, n_kv, gqa, page, window
    ([1], [0], 1, 1, 8, 0), ([1], [127], 2, 2, 16, 0), ([1, 1, 1], [128, 129, 700], 8, 2, 32, 0),
    ([5, 0, 1, 33], [0, 9, 250, 95], 2, 4, 24, 0), ([64, 65, 127], [64, 0, 1], 2, 2, 64, 0),
    ([130, 3], [300, 0], 1, 8, 128, 0), ([40], [17], 1, 16, 8, 0), ([50, 7], [3, 260], 2, 3, 40, 0),
    ([200], [60], 2, 2, 16, 1), ([200, 1, 1], [60, 400, 3], 2, 2, 16, 64),
    ([300], [0], 1, 2, 16, 129), ([1, 1], [1000, 555], 2, 7, 8, 300), ([257], [511], 1, 2, 32, 0),
]


@pytest.mark.parametrize("q32", [False, True])
@pytest.mark.parametrize("new,held,n_kv,gqa,page,window", CASES)
def test_chunk_attention(tt, new, held, n_kv, gqa, page, window, q32):
    b = ck.batch(len(new) + sum(held), new, held, n_kv, page)
    rows = int(b[0][-1]) + 3
    q = np.random.default_rng(5).standard_normal((rows, n_kv * gqa, 128)) * 2
    check_attention(tt, q.astype(np.float32 if q32 else np.float16), b, window)


def test_chunk_attention_one_odd_page_per_lane(tt):
    """One contiguous page per lane may have any size; rows may start behind row 0."""
    b = ck.batch(3, [30, 1, 77], [200, 333, 0], 2, 345, one_page=True, first=4)
    q = np.random.default_rng(6).standard_normal((int(b[0][-1]) + 1, 4, 128)).astype(np.float16)
    check_attention(tt, q, b)


def test_chunk_attention_long_cache_few_rows(tt):
    b = ck.batch(4, [1, 3], [9000, 5000], 2, 64)
    q = np.random.default_rng(7).standard_normal((4, 4, 128)).astype(np.float16) * 3
    check_attention(tt, q, b)


def test_chunk_attention_more_rows_than_positions(tt):
    """Rows before position 0 see nothing and are zero."""
    starts, spans, table, k, v = ck.batch(5, [20, 6], [0, 4], 2, 8)
    spans[0] = 7
    q = np.random.default_rng(8).standard_normal((26, 4, 128)).astype(np.float16)
    check_attention(tt, q, (starts, spans, table, k, v))
    spans[:] = 0
    assert (host(attend(tt, q, (starts, spans, table, k, v))) == 0).all()
    tt.check()


@pytest.mark.parametrize("window", [0, 20])
def test_chunk_attention_never_reads_unseen_positions(tt, window):
    """NaN and infinities behind the span, at later rows' positions and before the window reach no
    row that does not see them."""
    new, held = [30, 1, 140], [50, 77, 10]
    b = ck.batch(9, new, held, 2, 16)
    starts, spans, table, k, v = b
    q = np.random.default_rng(10).standard_normal((int(starts[-1]), 4, 128)).astype(np.float16)
    want, mass = ck.attention(q, *b, SCALE, window, np.zeros((q.shape[0], 512)))
    bound = ck.attention_bound(want, mass)
    for in_k, val in ((True, np.nan), (True, np.inf), (False, np.nan), (False, -np.inf)):
        bad = (k if in_k else v).copy()
        for i in range(3):
            unseen = np.arange(spans[i], table.shape[1] * 16)  # behind the span
            if new[i] > 2:                                     # the last two rows alone see it
                unseen = np.append(unseen, spans[i] - 2)
            if window:                                         # before every row's window
                unseen = np.append(unseen, np.arange(max(0, spans[i] - new[i] + 1 - window)))
            bad[table[i, unseen // 16], :, unseen % 16] = val
        got = host(attend(tt, q, (starts, spans, table, bad if in_k else k, v if in_k else bad), window))
        tt.check()
        for i in range(3):
            rows = slice(starts[i], starts[i + 1] - (2 if new[i] > 2 else 0))
            assert (np.abs(got[rows] - want[rows]) <= bound[rows]).all(), (in_k, val, i)
            if new[i] > 2 and val != np.inf:
                assert not np.isfinite(got[starts[i + 1] - 2:starts[i + 1]]).any()


@pytest.mark.parametrize("rise", [1.0, -1.0, 0.0])
@pytest.mark.parametrize("new,gqa", [(3, 1), (70, 4)])
def test_chunk_attention_rising_scores(tt, rise, new, gqa):
    """Scores that climb by hundreds of nats along the positions (the softmax's reference has to
    follow inside a unit and from unit to unit), fall as steeply, or jump at a few places."""
    b = ck.batch(31, [new], [900 - new], 1, 32)
    starts, spans, table, k, v = b
    at = np.arange(900)
    size = (at / 3 if rise > 0 else (900 - at) / 3) if rise else np.where(at % 97 == 60, at / 5.0, 0)
    row = np.zeros((900, 128))
    row[:, 0] = size * SCALE ** -1 / 8
    row[:, 1:] = np.random.default_rng(32).standard_normal((900, 127)) * 0.1
    k[table[0, at // 32], 0, at % 32] = row.astype(np.float16)
    q = np.random.default_rng(33).standard_normal((new, gqa, 128)).astype(np.float32)
    q[..., 0] = 8
    check_attention(tt, q.astype(np.float16), b)
    check_attention(tt, q, b)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_chunk_attention_scales(tt, scale):
    b = ck.batch(34, [33, 1], [200, 150], 2, 16)
    starts, spans, table, k, v = b
    q = np.random.default_rng(35).standard_normal((34, 4, 128)).astype(np.float16)
    got = host(attend(tt, q, b, scale=scale))
    want, mass = ck.attention(q, *b, scale, 0, np.zeros((34, 512)))
    # f32 scores of up to ~100: their rounding (2^-24 each of 128 products and sums) adds to the bound
    slack = 2.0 ** -24 * 128 * 40 * abs(scale) * mass
    assert (np.abs(got - want) <= ck.attention_bound(want, mass) + slack).all()


@pytest.mark.parametrize("scale", [-0.2, 0.7])
def test_chunk_attention_scales_of_f32_queries(tt, scale):
    b = ck.batch(36, [33, 1, 150, 2, 1, 1], [200, 150, 0, 7, 300, 1], 2, 16)
    q = np.random.default_rng(37).standard_normal((188, 4, 128)).astype(np.float32)
    got = host(attend(tt, q, b, scale=scale))
    want, mass = ck.attention(q, *b, scale, 0, np.zeros((188, 512)))
    # f32 scores of up to ~30: their rounding (2^-24 each of 128 products and sums) adds to the bound,
    # and so does what two f16 pieces leave of a query (2^-22 of it)
    slack = (2.0 ** -24 * 128 + 2.0 ** -22) * 40 * abs(scale) * mass
    assert (np.abs(got - want) <= ck.attention_bound(want, mass) + slack).all()


def test_chunk_attention_two_streams_at_once(tt):
    """Calls that overlap on the GPU have a workspace each."""
    args = []
    for seed, (new, held) in ((36, ([1, 2], [5000, 4000])), (37, ([90, 260], [700, 0]))):
        starts, spans, table, k, v = ck.batch(seed, new, held, 2, 32)
        q = np.random.default_rng(seed).standard_normal((int(starts[-1]), 4, 128)).astype(np.float16)
        kv = tt.attn.paged_cache(dev(k), dev(v), dev(table))
        args.append((dev(q), dev(starts), dev(spans), kv, SCALE))
    want = [tt.attn.chunk_attention(*a) for a in args]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                got.append(tt.attn.chunk_attention(*a))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))
    tt.check()


def test_chunk_attention_many_lanes(tt):
    """As many lanes as a call takes, most of them with one row or none."""
    rng = np.random.default_rng(38)
    new, held = rng.integers(0, 3, 1024), rng.integers(0, 40, 1024)
    new[500], held[77] = 90, 700
    b = ck.batch(39, new, held, 1, 8)
    q = rng.standard_normal((int(b[0][-1]), 2, 128)).astype(np.float16)
    check_attention(tt, q, b)


@pytest.mark.parametrize("gqa,q32,seed", [(2, False, 41), (2, True, 42), (8, False, 43)])
def test_chunk_attention_runs_of_every_kind(tt, gqa, q32, seed):
    """Single rows, a few rows, one query tile, two and several, of one unit or more, in any order."""
    rng = np.random.default_rng(seed)
    new = rng.choice([1, 1, 2, 4, 5, 15, 17, 33, 64, 70, 129, 0], 400)
    held = rng.choice([0, 0, 3, 60, 130, 300], 400)
    b = ck.batch(seed, new, held, 2, 16)
    q = rng.standard_normal((int(b[0][-1]), 2 * gqa, 128))
    check_attention(tt, q.astype(np.float32 if q32 else np.float16), b)


def test_chunk_attention_one_long_chunk(tt):
    """More work tiles than a warp looks through at once, more lanes behind them."""
    b = ck.batch(44, [1, 4300, 2, 500], [60, 70, 3, 0], 1, 16)
    q = np.random.default_rng(45).standard_normal((int(b[0][-1]), 2, 128)).astype(np.float16)
    check_attention(tt, q, b, window=150)


def test_chunk_attention_shared_pages_and_unaligned_sectors(tt):
    """Lanes over the same prefix pages; q and out on 16-byte, not 32-byte, boundaries."""
    starts, spans, table, k, v = ck.batch(46, [40, 30, 1], [64, 64, 64], 2, 16)
    table[1, :4] = table[2, :4] = table[0, :4]
    q = np.random.default_rng(47).standard_normal((71, 4, 128)).astype(np.float16)
    b = (starts, spans, table, k, v)
    want = attend(tt, q, b)
    mine = torch.empty(q.size + 8, device="cuda", dtype=torch.float16)
    out = torch.empty(q.size + 16, device="cuda", dtype=torch.float16).fill_(3)
    view, at = mine[8:].view(q.shape), out[8:-8].view(71, 512)
    view.copy_(dev(q))
    kv = tt.attn.paged_cache(dev(k), dev(v), dev(table))
    tt.attn.chunk_attention(view, dev(starts), dev(spans), kv, SCALE, out=at)
    tt.check()
    assert torch.equal(at, want) and (out[:8] == 3).all() and (out[-8:] == 3).all()
    exact, mass = ck.attention(q, *b, SCALE, 0, np.zeros((71, 512)))
    assert (np.abs(host(want) - exact) <= ck.attention_bound(exact, mass)).all()


def test_chunk_attention_pages_outside_pool(tt):
    b = ck.batch(11, [9, 40], [70, 30], 2, 16)
    starts, spans, table, k, v = b
    table[0, 1], table[1, 4] = -1, k.shape[0]
    q = np.random.default_rng(12).standard_normal((49, 2, 128)).astype(np.float16)
    check_attention(tt, q, b, clean=False)
    with pytest.raises(tt.TtsError, match="outside the pool"):
        tt.check()


def test_chunk_attention_bad_device_data(tt):
    """Descending row starts void the call; a span beyond the table skips its lane."""
    starts, spans, table, k, v = ck.batch(13, [4, 5, 6], [9, 9, 9], 2, 16)
    q = np.random.default_rng(14).standard_normal((15, 2, 128)).astype(np.float16)
    for bad in ([0, 9, 4, 15], [-1, 4, 9, 15], [0, 4, 9, 16]):
        out = torch.full((15, 256), 3.0, dtype=torch.float16, device="cuda")
        attend(tt, q, (np.array(bad, np.int32), spans, table, k, v), out=out)
        with pytest.raises(tt.TtsError, match="row starts"):
            tt.check()
        assert (out == 3).all()
    want = host(attend(tt, q, (starts, spans, table, k, v)))
    spans[1] = table.shape[1] * 16 + 1
    out = torch.full((15, 256), 3.0, dtype=torch.float16, device="cuda")
    got = host(attend(tt, q, (starts, spans, table, k, v), out=out))
    with pytest.raises(tt.TtsError, match="span"):
        tt.check()
    assert (got[4:9] == 3).all() and np.array_equal(got[:4], want[:4])
    assert np.array_equal(got[9:], want[9:])


def test_chunk_attention_captured_and_on_another_stream(tt):
    b = ck.batch(15, [40, 1, 9], [90, 800, 0], 2, 16)
    starts, spans, table, k, v = b
    q = dev(np.random.default_rng(16).standard_normal((50, 4, 128)).astype(np.float16))
    kd, vd, td = dev(k), dev(v), dev(table)
    kv = tt.attn.paged_cache(kd, vd, td)
    sd, pd = dev(starts), dev(spans)
    want = tt.attn.chunk_attention(q, sd, pd, kv, SCALE)
    out, two = torch.zeros_like(want), torch.zeros_like(want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            tt.attn.chunk_attention(q, sd, pd, kv, SCALE, out=out)
        with torch.cuda.graph(g2, stream=side):
            tt.attn.chunk_attention(q, sd, pd, kv, SCALE, out=two)
        for _ in range(3):
            g.replay()
            g2.replay()
    eager = tt.attn.chunk_attention(q, sd, pd, kv, SCALE)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(two, want) and torch.equal(eager, want)
    # new lengths under the same graph
    starts2, spans2 = np.array([0, 1, 2, 50], np.int32), np.array([60, 700, 48], np.int32)
    sd.copy_(dev(starts2))
    pd.copy_(dev(spans2))
    g.replay()
    torch.cuda.synchronize()
    want2, mass = ck.attention(q.cpu().numpy(), starts2, spans2, table, k, v, SCALE, 0,
                               out.cpu().numpy())
    assert (np.abs(host(out) - want2) <= ck.attention_bound(want2, mass)).all()
    tt.check()


@pytest.mark.parametrize("hd,rotary,interleaved,f16", [
    (64, 64, False, False), (64, 32, True, True), (80, 40, False, True), (96, 96, True, False),
    (128, 64, False, False), (128, 8, True, True), (256, 256, False, True), (8, 8, True, False)])
def test_rotary(tt, hd, rotary, interleaved, f16):
    rng = np.random.default_rng(hd + rotary)
    rows, heads, length = 37, 5, 20000
    cos, sin = ck.tables(length, rotary)
    pos = rng.integers(0, length, rows).astype(np.int32)
    pos[:2] = 0, length - 1
    x = rng.standard_normal((rows, heads, hd)).astype(np.float16 if f16 else np.float32)
    want, mass = ck.turn(x, cos[pos], sin[pos], rotary, interleaved)
    bound = 3 * ck.F32 * mass + (ck.F16 * np.abs(want) + 2.0 ** -25 if f16 else 0)
    args = (dev(pos), dev(cos), dev(sin), interleaved)
    got = tt.qkrope.rotary(dev(x), *args)
    assert got.dtype == (torch.float16 if f16 else torch.float32)
    assert (np.abs(host(got) - want) <= bound).all()
    # a column block of wider rows, in place: the columns beside it stay
    wide = torch.full((rows, heads * hd + 16), 5.0, device="cuda", dtype=got.dtype)
    view = wide[:, 8:8 + heads * hd].unflatten(1, (heads, hd))
    view.copy_(dev(x))
    tt.qkrope.rotary(view, *args, out=view)
    assert torch.equal(view, got) and (wide[:, :8] == 5).all() and (wide[:, -8:] == 5).all()
    tt.check()


def test_rotary_into_other_columns_of_the_same_rows(tt):
    rng = np.random.default_rng(51)
    wide = dev(rng.standard_normal((37, 2, 3, 64)).astype(np.float32))
    pos, (cos, sin) = dev(rng.integers(0, 90, 37).astype(np.int32)), (dev(t) for t in ck.tables(90, 64))
    before = wide[:, 0].clone()
    want = tt.qkrope.rotary(before, pos, cos, sin)
    tt.qkrope.rotary(wide[:, 0], pos, cos, sin, out=wide[:, 1])
    tt.check()
    assert torch.equal(wide[:, 0], before) and torch.equal(wide[:, 1], want)


def test_rotary_positions_outside_the_tables(tt):
    cos, sin = ck.tables(10, 16)
    x = dev(np.ones((4, 2, 16), np.float32))
    out = torch.full_like(x, 9.0)
    pos = torch.tensor([3, -1, 10, 9], dtype=torch.int32, device="cuda")
    tt.qkrope.rotary(x, pos, dev(cos), dev(sin), out=out)
    with pytest.raises(tt.TtsError, match="RoPE table"):
        tt.check()
    assert (out[1:3] == 9).all() and not (out[0] == 9).any() and not (out[3] == 9).any()


@pytest.mark.parametrize("x16,q16,norm,rotary,interleaved,page,heads,n_kv", [
    (False, True, True, 128, False, 16, 4, 2), (True, True, False, 64, True, 5, 7, 1),
    (False, False, True, 24, True, 8, 3, 3), (True, False, False, 128, False, 33, 16, 8),
    (False, False, False, 96, False, 7, 28, 4)])
def test_rotary_append(tt, x16, q16, norm, rotary, interleaved, page, heads, n_kv):
    new, held = [3, 0, 1, 40], [0, 5, 60, 17]
    starts, spans, table, k, v = ck.batch(heads + page, new, held, n_kv, page, first=2)
    rows = int(starts[-1]) + 2
    rng = np.random.default_rng(rotary)
    x = rng.standard_normal((rows, heads + 2 * n_kv, 128)).astype(np.float16 if x16 else np.float32)
    norms = rng.uniform(0.5, 1.5, (2, 128)).astype(np.float32)
    cos, sin = ck.tables(100, rotary)
    kd, vd = dev(k), dev(v)
    q = torch.full((rows, heads, 128), 4.0, device="cuda", dtype=torch.float16 if q16 else torch.float32)
    tt.qkrope.rotary_append(dev(x.reshape(rows, -1)), heads, dev(starts), dev(spans), dev(cos), dev(sin),
                            tt.attn.paged_cache(kd, vd, dev(table)), interleaved,
                            dev(norms) if norm else None, 1e-6, out=q)
    tt.check()
    wq, wk, wv = np.full(q.shape, 4.0), k.astype(np.float64), v.astype(np.float64)
    bq, bk = np.zeros(q.shape), np.zeros(k.shape)
    for i in range(4):
        for j in range(new[i]):
            row, p = starts[i] + j, spans[i] - new[i] + j
            y = x[row:row + 1].astype(np.float64)
            if norm:
                w = np.repeat(norms.astype(np.float64), [heads, n_kv], 0)
                y[:, :heads + n_kv] *= w / np.sqrt((y[:, :heads + n_kv] ** 2).mean(-1, keepdims=True) + 1e-6)
            z, mass = ck.turn(y[:, :heads + n_kv], cos[p:p + 1], sin[p:p + 1], rotary, interleaved)
            # three f32 roundings of the turn; the norm's 128-term f32 sum stays within 2^-18
            bound = (2.0 ** -18 if norm else 3 * ck.F32) * mass
            pg = table[i, p // page]
            wq[row], wk[pg, :, p % page], wv[pg, :, p % page] = z[0, :heads], z[0, heads:], y[0, heads + n_kv:]
            bq[row] = bound[0, :heads] + (ck.F16 * np.abs(z[0, :heads]) + 2.0 ** -25 if q16 else 0)
            bk[pg, :, p % page] = bound[0, heads:] + ck.F16 * np.abs(z[0, heads:]) + 2.0 ** -25
    assert (np.abs(host(q) - wq) <= bq).all()
    assert (np.abs(host(kd) - wk) <= bk).all()
    assert np.array_equal(vd.cpu().numpy(), wv.astype(np.float16))


def test_rotary_append_bad_device_data(tt):
    """Pages outside the pool and positions outside the tables skip their rows, descending starts
    the whole call."""
    starts, spans, table, k, v = ck.batch(21, [4, 4], [4, 4], 1, 8)
    cos, sin = ck.tables(7, 128)
    x = dev(np.ones((8, 3 * 128), np.float32))
    table[1, 0] = k.shape[0]
    kd, vd = dev(k), dev(v)
    q = torch.full((8, 1, 128), 4.0, device="cuda")
    kv = tt.attn.paged_cache(kd, vd, dev(table))
    tt.qkrope.rotary_append(x, 1, dev(starts), dev(spans), dev(cos), dev(sin), kv, out=q)
    with pytest.raises(tt.TtsError, match="RoPE table.*outside the pool"):
        tt.check()
    q = host(q)
    assert (q[3:] == 4).all() and not (q[:3] == 4).all(-1).any()  # row 3 is at position 7
    before = kd.clone()
    tt.qkrope.rotary_append(x, 1, dev(starts[::-1].copy()), dev(spans), dev(cos), dev(sin), kv)
    with pytest.raises(tt.TtsError, match="row starts"):
        tt.check()
    assert torch.equal(before, kd)


def test_refusals(tt):
    starts, spans, table, k, v = ck.batch(22, [2], [3], 2, 8)
    kv = tt.attn.paged_cache(dev(k), dev(v), dev(table))
    sd, pd = dev(starts), dev(spans)
    q = torch.zeros(2, 4, 128, device="cuda", dtype=torch.float16)
    go = tt.attn.chunk_attention
    with pytest.raises(ValueError, match="heads over"):
        go(q[:, :3], sd, pd, kv, SCALE)
    with pytest.raises(ValueError, match="f16 or f32"):
        go(q.bfloat16(), sd, pd, kv, SCALE)
    with pytest.raises(ValueError, match="int32"):
        go(q, sd.long(), pd, kv, SCALE)
    with pytest.raises(ValueError, match="one entry more"):
        go(q, sd[:1], pd, kv, SCALE)
    with pytest.raises(ValueError, match="block table of"):
        go(q, dev(np.zeros(4, np.int32)), dev(np.zeros(3, np.int32)), kv, SCALE)
    with pytest.raises(tt.TtsError, match="window"):
        go(q, sd, pd, kv, SCALE, window=-1)
    with pytest.raises(tt.TtsError, match="finite scale"):
        go(q, sd, pd, kv, float("nan"))
    with pytest.raises(tt.TtsError, match="gqa"):
        go(torch.zeros(2, 34, 128, device="cuda"), sd, pd, kv, SCALE)
    odd = tt.attn.paged_cache(torch.zeros(4, 2, 12, 128, device="cuda", dtype=torch.float16),
                              torch.zeros(4, 2, 12, 128, device="cuda", dtype=torch.float16),
                              torch.zeros(1, 2, device="cuda", dtype=torch.int32))
    with pytest.raises(tt.TtsError, match="multiple of 8"):
        go(q, sd, pd, odd, SCALE)
    none = torch.zeros(0, 4, 128, device="cuda", dtype=torch.float16)
    assert go(none, dev(np.zeros(2, np.int32)), pd, kv, SCALE).shape == (0, 512)
    cos, sin = (dev(t) for t in ck.tables(8, 20))
    x = torch.zeros(2, 1, 64, device="cuda")
    with pytest.raises(tt.TtsError, match="rotary_dim"):
        tt.qkrope.rotary(x, pd.repeat(2), cos, sin)
    with pytest.raises(ValueError, match="position per row"):
        tt.qkrope.rotary(x, pd, cos, sin)
    with pytest.raises(tt.TtsError, match="rotary_dim"):
        tt.qkrope.rotary(x[..., :16], pd.repeat(2), cos, sin)
    with pytest.raises(ValueError, match="width"):
        tt.qkrope.rotary_append(torch.zeros(2, 640, device="cuda"), 4, sd, pd, cos, sin, kv)
    with pytest.raises(ValueError, match="cuda"):
        go(q, sd.cpu(), pd, kv, SCALE)
    tt.check()


def test_a_prompt_in_chunks_then_tokens(tt):
    """Projection, rotation and append, attention and the draw as a serving loop runs them: two
    lanes' prompts in chunks of different sizes, then single tokens, over a page pool's cache; each
    attention against the definition on the device's own q and pages, each pick against the
    definition on the device's own logits, and the chunks' pages against one whole chunk's."""
    from qwen3tts.stack import Geometry, PagedKv
    heads, n_kv, dim, vocab, page = 4, 2, 256, 1000, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)
    wqkv = tt.Proj(rand((heads + 2 * n_kv) * 128, dim) * 0.06)
    wo, head = tt.Proj(rand(dim, heads * 128) * 0.05), rand(vocab, dim) * 0.3
    norms = rand(2, 128) * 0.1 + 1
    cos, sin = tt.rope_table_scaled(512, 128, 1e4, "yarn", 4.0, 128)
    geo = Geometry(dim=dim, layers=2, heads=heads, n_kv=n_kv, ffn=256, rope_len=512)
    prompts = [rand(150, dim), rand(77, dim)]
    plans = [[(150, 77)], [(64, 0), (1, 70), (80, 6), (5, 1)]]
    pages = []
    for plan in plans:
        pool = PagedKv(geo, 2, 80, page, 32)
        for lane in range(2):
            pool.admit(lane, 200)
        kv = tt.attn.paged_cache(pool.k[1], pool.v[1], pool.table)
        held = [0, 0]

        def step(rows):
            n = [len(r) for r in rows]
            held[:] = [h + m for h, m in zip(held, n)]
            starts, spans = np.array([0, n[0], sum(n)], np.int32), np.array(held, np.int32)
            sd, pd = dev(starts), dev(spans)
            q = tt.qkrope.rotary_append(wqkv(torch.cat(rows)), heads, sd, pd, cos, sin, kv, norms=norms)
            o = tt.attn.chunk_attention(q, sd, pd, kv, SCALE)
            want, mass = ck.attention(q.cpu().numpy(), starts, spans, pool.table.cpu().numpy(),
                                      pool.k[1].cpu().numpy(), pool.v[1].cpu().numpy(), SCALE, 0,
                                      np.zeros(o.shape))
            assert (np.abs(host(o) - want) <= ck.attention_bound(want, mass)).all()
            return wo(o.float()), starts

        done = [0, 0]
        for chunk in plan:
            y, starts = step([prompts[i][done[i]:done[i] + chunk[i]] for i in range(2)])
            done = [d + c for d, c in zip(done, chunk)]
        assert held == [150, 77]
        pages.append([pool.k[1][pool.table[i].long()].transpose(1, 2).reshape(-1, n_kv, 128)[:held[i]]
                      for i in range(2)])
        for _ in range(3):
            logits = y[dev(starts[1:].astype(np.int64)) - 1] @ head.T
            u = torch.rand(2, device="cuda", generator=g)
            how = (np.float32([0.7, 1.1]), np.int32([50, 0]), np.float32([0.9, 0.95]), np.float32([0, 0.02]))
            pick = tt.topk.sample_filtered(logits, u, *(dev(h) for h in how))
            assert np.array_equal(pick.cpu().numpy(), ck.sample(logits.cpu().numpy(), u.cpu().numpy(), *how))
            x = head[pick.long()]
            y, starts = step([x[:1], x[1:]])
        assert pool.free_pages() == 80 - 2 * 25
    tt.check()
    # the projection sums a row in another order when it shares its call with other rows; one f16 step
    for a, b in zip(*pages):
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -9, atol=2 ** -9)
