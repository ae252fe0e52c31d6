"""topk.sample_filtered on a B200 against its definition in 64 bits: the picks are equal."""
import numpy as np
import pytest
import torch

import _chunks as ck

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def same(tt, x, u, **how):
    got = tt.topk.sample_filtered(dev(x), dev(u), **{n: dev(v) for n, v in how.items()})
    want = ck.sample(x, u, **how)
    assert np.array_equal(got.cpu().numpy(), want), np.argwhere(got.cpu().numpy() != want).ravel()[:8]


def inputs(rows, n, seed=0, f16=False):
    rng = np.random.default_rng(seed + n)
    x = (rng.standard_normal((rows, n)) * 2.5).astype(np.float16 if f16 else np.float32)
    u = rng.random(rows).astype(np.float32)
    u[0] = 0
    u[-1] = np.float32(1 - 2.0 ** -24)
    return rng, x, u


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (9, 31), (40, 257), (33, 2048), (17, 5003), (6, 32003),
                                    (3, 151851), (2, 262144)])
def test_every_filter_together(tt, rows, n, f16):
    rng, x, u = inputs(rows, n, 1, f16)
    same(tt, x, u)
    same(tt, x, u, temperature=rng.uniform(0.3, 2, rows).astype(np.float32),
         top_k=rng.integers(0, min(n, 300) + 2, rows).astype(np.int32),
         top_p=rng.uniform(0.1, 1.1, rows).astype(np.float32),
         min_p=rng.uniform(-0.05, 0.2, rows).astype(np.float32))


@pytest.mark.parametrize("how", ["temperature", "top_k", "top_p", "min_p"])
def test_each_filter_alone(tt, how):
    rng, x, u = inputs(64, 4099, 2)
    x[:32] = np.round(x[:32] * 2) / 2  # many ids share a logit
    v = {"temperature": rng.uniform(0.01, 50, 64), "top_k": rng.integers(1, 4200, 64),
         "top_p": rng.uniform(0, 1, 64), "min_p": rng.uniform(0, 1, 64)}[how]
    same(tt, x, u, **{how: v.astype(np.int32 if how == "top_k" else np.float32)})


def test_equal_logits(tt):
    """All ids alike: the draw alone decides, cuts fall inside the tie, lowest ids first."""
    x = np.full((50, 1000), -3.25, np.float32)
    x[25:, 500:] = 4
    x[10] = 0.0
    x[10, ::2] = -0.0
    u = (np.arange(50) / 50 + 0.003).astype(np.float32)
    same(tt, x, u)
    same(tt, x, u, top_k=np.arange(1, 51).astype(np.int32))
    same(tt, x, u, top_p=np.linspace(0.0011, 0.999, 50).astype(np.float32))
    same(tt, x, u, top_k=np.full(50, 700, np.int32), top_p=np.full(50, 0.3, np.float32),
         min_p=np.full(50, 0.5, np.float32))


@pytest.mark.parametrize("n", [5003, 32003, 151851])
def test_more_equal_logits_than_a_list_holds(tt, n):
    """Thousands of ids share a logit (counted along the ids), a few values only, or lie so close
    together beside one far off that their bin is narrowed by their bits, around zero too."""
    rng = np.random.default_rng(n)
    rows = 14
    x = np.full((rows, n), -3.25, np.float32)
    x[2:4] = np.round(rng.standard_normal((2, n)) * 2) / 2
    x[4:6] = rng.integers(0, 2, (2, n)) * 0.5
    x[6:10] = rng.standard_normal((4, n)) * 1e-3
    x[8:10] += 7
    x[6:10, n // 3] = 40
    x[10:12] = rng.standard_normal((2, n)) * 1e-30
    x[12:] = rng.standard_normal((2, n)) * 1e-3 - 100
    x[12:, n - 1] = 1e8
    u = rng.random(rows).astype(np.float32)
    u[3], u[4] = 0, np.float32(1 - 2.0 ** -24)
    t = np.full(rows, 20, np.float32)
    t[12:] = 1e7
    same(tt, x, u, temperature=t)
    same(tt, x, u, temperature=t, top_k=rng.integers(1500, n, rows).astype(np.int32))
    same(tt, x, u, temperature=t, top_p=rng.uniform(0.2, 0.999, rows).astype(np.float32))
    same(tt, x, u, temperature=t, top_k=rng.integers(1500, n, rows).astype(np.int32),
         top_p=rng.uniform(0.2, 0.999, rows).astype(np.float32), min_p=np.full(rows, 0.1, np.float32))
    with np.errstate(over="ignore"):
        half = x.astype(np.float16)
    same(tt, half, u, top_p=np.full(rows, 0.7, np.float32))


def test_settings_at_their_ends(tt):
    rng, x, u = inputs(10, 333, 3)
    nan = np.float32(np.nan)
    same(tt, x, u, temperature=np.array([0, -1, nan, 1e-30, 1e30, 1e-3, 0, 1, 2, 5], np.float32))
    same(tt, x, u, top_k=np.array([0, -5, 1, 333, 334, 2 ** 31 - 1, 332, 2, 1, 1], np.int32))
    same(tt, x, u, top_p=np.array([0, -1, nan, 1, 2, 1 - 2.0 ** -24, 1e-30, 0.5, 0.9, 0], np.float32))
    same(tt, x, u, min_p=np.array([0, -1, nan, 1, 2, 1e-30, 1e-9, 0.5, 0.9, 1], np.float32))


def test_masked_and_infinite_logits(tt):
    rng, x, u = inputs(12, 777, 4)
    x[0], x[1] = -np.inf, np.nan
    x[2, :776] = -np.inf
    x[3, 5:700] = np.nan
    x[4, [9, 99, 600]] = np.inf
    x[5] = np.inf
    x[6] = -np.finfo(np.float32).max
    x[7, ::3] = -np.finfo(np.float32).max
    x[8, 3] = np.finfo(np.float32).max
    x[9] = 1e-40
    x[9, 7] = 0
    for how in ({}, {"top_k": np.full(12, 2, np.int32)}, {"top_p": np.full(12, 0.6, np.float32)},
                {"min_p": np.full(12, 0.3, np.float32)}, {"temperature": np.zeros(12, np.float32)}):
        same(tt, x, u, **how)


def test_strides_numbers_and_streams(tt):
    """A view of wider rows at an odd offset, plain numbers for settings, another stream, a graph."""
    rng, wide, u = inputs(20, 1501, 5)
    x = dev(wide)[:, 1:1400]
    want = ck.sample(wide[:, 1:1400], u, np.full(20, 0.8, np.float32), np.full(20, 40, np.int32),
                     np.full(20, 0.9, np.float32), np.full(20, 0.05, np.float32))
    ud = dev(u)
    go = lambda: tt.topk.sample_filtered(x, ud, 0.8, 40, 0.9, 0.05)
    assert np.array_equal(go().cpu().numpy(), want)
    half = dev(wide.astype(np.float16))[:, 1:1400]
    assert np.array_equal(tt.topk.sample_filtered(half, ud, 0.8).cpu().numpy(),
                          ck.sample(wide.astype(np.float16)[:, 1:1400], u, np.full(20, 0.8, np.float32)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = go()
        g.replay()
        side.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)
    # one row whose stride says nothing, and logits shared by every row
    assert tt.topk.sample_filtered(x[:1], ud[:1]).shape == (1,)
    shared = x[:1].expand(20, -1)
    assert np.array_equal(tt.topk.sample_filtered(shared, ud).cpu().numpy(),
                          ck.sample(np.repeat(wide[:1, 1:1400], 20, 0), u))


def test_the_topk_samplers_walk(tt, orc):
    """With top-k alone the pick is tts_topk_sample's, up to its f32 sums at a border."""
    rng, x, u = inputs(256, 2048, 6)
    a = tt.topk.sample(dev(x), dev(u), 50, 0.9)
    b = tt.topk.sample_filtered(dev(x), dev(u), 0.9, 50)
    assert (a != b).sum() <= 1


def test_refusals(tt):
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    for bad in (lambda: tt.topk.sample_filtered(x.bfloat16(), u), lambda: tt.topk.sample_filtered(x, u[:1]),
                lambda: tt.topk.sample_filtered(x, None), lambda: tt.topk.sample_filtered(x, u, top_k=u[:1]),
                lambda: tt.topk.sample_filtered(x, u.cpu())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(tt.TtsError, match="262144"):
        tt.topk.sample_filtered(torch.zeros(1, 262145, device="cuda"), u[:1])
    assert tt.topk.sample_filtered(x[:0], u[:0]).shape == (0,)
    tt.check()
