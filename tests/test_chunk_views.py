"""What the chunk operators and the filtered draw hand to the library for tensors of unusual
strides, starts and types: the calls are caught and their arguments read back on the CPU."""

import ctypes as C

import numpy as np
import pytest
import torch

from ttsnn import attn, qkrope, topk
from ttsnn import _lib as L


@pytest.fixture
def calls(monkeypatch):
    """The arguments of every library call, pointers and numbers as the library would see them."""
    seen = []
    for m in (attn, qkrope, topk):
        monkeypatch.setattr(m, "ctx_of", lambda t: 0)
        monkeypatch.setattr(m, "stream_of", lambda t: 0)
    monkeypatch.setattr(L, "call", lambda name, *args: seen.append((name, args)))
    return seen


def wide(shape, strides, dtype=torch.float16):
    """A tensor of these strides with no memory behind it."""
    return torch.empty_strided(shape, strides, dtype=dtype, device="meta")


@pytest.mark.parametrize("stride", [2 ** 31 - 8, 2 ** 31, 2 ** 31 + 8, 2 ** 32 + 64, 2 ** 33])
def test_row_strides_past_31_bits(calls, stride):
    """A stride that the library's int cannot hold never reaches it: the rows are copied, and an
    output of such rows is refused."""
    at = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device="meta")
    topk.sample_filtered(wide((3, 40), (stride, 1)), at(3))
    ldl = calls[-1][1][5]
    assert ldl == (stride if stride < 2 ** 31 else 40)
    x = wide((3, 2, 16), (stride, 16, 1))
    pos = at(3, dtype=torch.int32)
    qkrope.rotary(x, pos, at(9, 8), at(9, 8))
    assert calls[-1][1][6] == (stride if stride < 2 ** 31 else 32) and calls[-1][1][14] == 32
    if stride < 2 ** 31:
        qkrope.rotary(at(3, 2, 16, dtype=torch.float16), pos, at(9, 8), at(9, 8), out=x)
        assert calls[-1][1][14] == stride
    else:
        with pytest.raises(ValueError, match="out must"):
            qkrope.rotary(at(3, 2, 16, dtype=torch.float16), pos, at(9, 8), at(9, 8), out=x)


def values(pointer, dtype, n):
    """What a caught call's pointer holds."""
    return np.ctypeslib.as_array(C.cast(pointer, C.POINTER(dtype)), (n,)).copy()


@pytest.mark.parametrize("top_k,want", [
    (torch.tensor([5, 0, -3, 2 ** 31 - 1]), [5, 0, -1, 2 ** 18]),
    (torch.tensor([2 ** 32 + 5, 2 ** 31, 2 ** 62, -2 ** 40]), [2 ** 18, 2 ** 18, 2 ** 18, -1]),
    (torch.tensor([5.0, 1e10, float("inf"), -float("inf")]), [5, 2 ** 18, None, -1]),
    (torch.tensor([7, 0, 9, 255], dtype=torch.uint8), [7, 0, 9, 255]),
    (2 ** 31, [2 ** 18] * 4), (2 ** 63 - 1, [2 ** 18] * 4), (-2 ** 40, [-1] * 4), (50, [50] * 4)])
def test_top_k_of_any_size(monkeypatch, calls, top_k, want):
    """A top_k beyond int32 keeps its meaning (at least as many ids as there are, or off): it is
    not cut to its low bits. `want` 2^18 stands for any number no smaller than a row may be long,
    None for that or off."""
    got = []

    def call(name, *args):
        how = C.cast(args[7], C.POINTER(L.Sampling)).contents
        got.extend(values(how.top_k, C.c_int, 4).tolist())

    monkeypatch.setattr(L, "call", call)
    topk.sample_filtered(torch.zeros(4, 9), torch.zeros(4), top_k=top_k)
    for g, w in zip(got, want, strict=True):
        assert g <= 0 if w == -1 else g >= w if w == 2 ** 18 else w is None and (g <= 0 or g >= 2 ** 18) or g == w


def off_by(n, *shape, dtype=torch.float32):
    """A contiguous tensor `n` elements behind a 16-byte boundary."""
    t = torch.randn(n + 64 + int(np.prod(shape)), generator=torch.Generator().manual_seed(len(shape)))
    t = t.to(dtype)
    skip = (-t.data_ptr() % 16) // t.element_size() + n
    return t[skip:skip + int(np.prod(shape))].view(*shape)


def held(monkeypatch, name, take):
    """take(args) of the next call of `name`, read while its tensors live."""
    got = []

    def call(called, *args):
        assert called == name
        got.append(take(args))

    monkeypatch.setattr(L, "call", call)
    return got


def f32(pointer, n):
    assert pointer % 16 == 0
    return values(pointer, C.c_float, n)


def lane(n):
    kv = attn.paged_cache(torch.zeros(2, 1, 16, 128).half(), torch.zeros(2, 1, 16, 128).half(),
                          torch.zeros(1, 2, dtype=torch.int32))
    return torch.tensor([0, n], dtype=torch.int32), torch.tensor([n], dtype=torch.int32), kv


@pytest.mark.parametrize("off", [0, 1, 3])
def test_inputs_that_start_between_16_byte_boundaries(monkeypatch, calls, off):
    """Contiguous views at an odd offset are brought to a boundary, not refused."""
    x, cos, sin = off_by(off, 3, 2, 16), off_by(off, 9, 8), off_by(off, 9, 8)
    got = held(monkeypatch, "tts_rotary", lambda a: [f32(a[1], 96), f32(a[8], 72), f32(a[9], 72)])
    qkrope.rotary(x, torch.zeros(3, dtype=torch.int32), cos, sin)
    for g, t in zip(got[0], (x, cos, sin), strict=True):
        assert np.array_equal(g, t.numpy().ravel())
    starts, spans, kv = lane(3)
    qkv, norms = off_by(off, 3, 3 * 128), off_by(off, 2, 128)
    got = held(monkeypatch, "tts_rotary_append", lambda a: [f32(a[1], 3 * 384), f32(a[5], 256), f32(a[7], 72),
                                                           f32(a[8], 72)])
    qkrope.rotary_append(qkv, 1, starts, spans, cos, sin, kv, norms=norms)
    for g, t in zip(got[0], (qkv, norms, cos, sin), strict=True):
        assert np.array_equal(g, t.numpy().ravel())
    q = off_by(off, 3, 2, 128)
    monkeypatch.setitem(attn._workspace, q.device.index, 64)
    got = held(monkeypatch, "tts_chunk_attention", lambda a: f32(a[1], 768))
    attn.chunk_attention(q, starts, spans, kv, 1.0)
    assert np.array_equal(got[0], q.numpy().ravel())


def test_strides_of_one_row_or_head_say_nothing(monkeypatch, calls):
    """A dimension of one entry may have any stride, torch calls such a tensor contiguous."""
    column = torch.randn(100, 1).t()
    assert column.stride() == (1, 1) and column.is_contiguous()
    got = held(monkeypatch, "tts_filter_sample", lambda a: (a[5], values(a[1], C.c_float, 100)))
    topk.sample_filtered(column, torch.zeros(1))
    assert got[0][0] in (0, 100) and np.array_equal(got[0][1], column[0].numpy())
    cos, sin, pos = torch.zeros(9, 8), torch.zeros(9, 8), torch.zeros(1, dtype=torch.int32)
    for x in (torch.randn(40)[:32].as_strided((1, 2, 16), (3, 16, 1)),  # one row
              torch.randn(9, 5, 16)[:1, :1], torch.randn(40).as_strided((1, 1, 16), (7, 5, 1))):
        n = x.numel()
        got = held(monkeypatch, "tts_rotary", lambda a: (a[6], a[14], f32(a[1], n)))
        out = torch.empty(48).as_strided(x.shape, (5, 16 if x.shape[1] > 1 else 3, 1))
        for y in (None, x, out):
            qkrope.rotary(x, pos, cos, sin, out=y)
        assert all(g[0] == g[1] == n and np.array_equal(g[2], x.numpy().ravel()) for g in got) and len(got) == 3
    x = torch.randn(5, 9, 16)[:, :1]  # several rows of one head: still strided
    got = held(monkeypatch, "tts_rotary", lambda a: (a[6], a[14]))
    qkrope.rotary(x, torch.zeros(5, dtype=torch.int32), cos, sin)
    assert got == [(144, 16)]


@pytest.fixture(scope="module")
def lib():
    import build
    build.build()
    return L.load()


@pytest.mark.parametrize("which", ["k_pages", "v_pages"])
def test_outputs_inside_the_pools_are_refused(lib, which):
    """No GPU call is made: addresses far apart, then one buffer's end or start inside a pool."""
    ctx = C.cast(C.create_string_buffer(256), C.c_void_p)
    pool, page_bytes = 1 << 30, 8 * 2 * 16 * 256  # 8 pages of 2 kv heads, 16 positions
    kv = L.KvCache(1 << 40, 1 << 41, 4096, 4, 16, 8, 2, 128)
    setattr(kv, which, pool)
    b = L.ChunkBatch(2, 8, 4096, 4096)
    q, out, work, size = 1 << 33, 1 << 34, 1 << 35, 1 << 40
    chunk = lambda q, out, work: lib.tts_chunk_attention(ctx, q, 1, 2, C.byref(b), C.byref(kv), 1.0, 0, out, work,
                                                         size, None)
    append = lambda x, q: lib.tts_rotary_append(ctx, x, 0, 4, C.byref(b), None, 1e-6, 4096, 4096, 64, 64, 0,
                                                C.byref(kv), q, 0, None)
    rows = 8 * 4 * 128  # elements of q
    for call in (lambda: chunk(q, pool, work), lambda: chunk(q, pool - rows * 2 + 16, work),
                 lambda: chunk(q, pool + page_bytes - 16, work), lambda: chunk(q, out, pool - 16),
                 lambda: chunk(q, out, out - 64), lambda: chunk(q, out, q + rows * 2 - 16)):
        assert call() == 1 and "apart from one another" in L.last_error()
    for call in (lambda: append(pool + 16, q), lambda: append(pool - 16, q), lambda: append(q, pool + page_bytes - 16),
                 lambda: append(q, pool - rows * 4 + 16)):
        assert call() == 1 and "apart from the pools" in L.last_error()
