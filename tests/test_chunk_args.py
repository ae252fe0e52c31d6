"""Argument checks of the chunk operators and the filtered draw, and the scaled rotary tables: no
GPU call is made (every check comes before the context is used)."""
import ctypes as C
import math

import numpy as np
import pytest

import ttsnn
from ttsnn import _lib as L


@pytest.fixture(scope="module")
def lib():
    import build
    build.build()
    return L.load()


CTX = C.cast(C.create_string_buffer(256), C.c_void_p)
A = 4096  # an aligned address that is never read


def refused(lib, status, text, name, *args):
    rc = getattr(lib, name)(*args)
    assert rc == status and text in L.last_error(), (rc, L.last_error())


def kv(**kw):
    f = dict(k_pages=A, v_pages=A, block_table=A, max_blocks=4, block_size=16, num_blocks=8, n_kv=2,
             head_dim=128)
    f.update(kw)
    return C.byref(L.KvCache(*(f[n] for n, _ in L.KvCache._fields_)))


def lanes(n=2, rows=8, starts=A, spans=A):
    return C.byref(L.ChunkBatch(n, rows, starts, spans))


@pytest.mark.parametrize("status,text,change", [
    (1, "NULL", dict(q=0)), (1, "NULL", dict(out=0)), (1, "batch pointers", dict(b=lanes(starts=0))),
    (1, "lanes must", dict(b=lanes(0))), (1, "rows >= 0", dict(b=lanes(rows=-1))),
    (2, "1024", dict(b=lanes(1025))), (1, "head_dim", dict(kv=kv(head_dim=64))),
    (1, "NULL", dict(kv=kv(k_pages=0))), (1, "aligned", dict(kv=kv(v_pages=A + 8))),
    (2, "multiple of 8", dict(kv=kv(block_size=12))), (2, "2^31", dict(kv=kv(max_blocks=2 ** 30))),
    (1, "aligned", dict(q=A + 2)), (2, "gqa", dict(gqa=0)), (2, "gqa", dict(gqa=17)),
    (1, "window", dict(window=-1)), (1, "scale", dict(scale=math.inf)),
    (2, "pool rows", dict(kv=kv(num_blocks=2 ** 27))), (2, "rows", dict(b=lanes(rows=2 ** 29))),
    (1, "aligned", dict(work=A + 8)), (1, "workspace", dict(work=0)), (1, "workspace", dict())])
def test_chunk_attention_refuses(lib, status, text, change):
    f = dict(q=A, f16=1, gqa=2, b=lanes(), kv=kv(), scale=1.0, window=0, out=A, work=A)
    f.update(change)
    refused(lib, status, text, "tts_chunk_attention", CTX, f["q"], f["f16"], f["gqa"], f["b"], f["kv"],
            f["scale"], f["window"], f["out"], f["work"], 1 << 10, None)


@pytest.mark.parametrize("status,text,change", [
    (1, "NULL", dict(x=0)), (1, "heads", dict(heads=0)), (2, "rotary_dim", dict(rotary=132)),
    (2, "rotary_dim", dict(rotary=12)), (2, "rotary_dim", dict(rotary=0)), (1, "rope_len", dict(length=0)),
    (1, "interleaved", dict(inter=2)), (1, "aligned", dict(q=A + 4)), (1, "tables", dict(cos=A + 4)),
    (1, "batch pointers", dict(b=lanes(spans=0))), (1, "NULL", dict(kv=kv(block_table=0)))])
def test_rotary_append_refuses(lib, status, text, change):
    f = dict(x=A, heads=4, b=lanes(), cos=A, length=64, rotary=64, inter=0, kv=kv(), q=A)
    f.update(change)
    refused(lib, status, text, "tts_rotary_append", CTX, f["x"], 0, f["heads"], f["b"], None, 1e-6, f["cos"],
            A, f["length"], f["rotary"], f["inter"], f["kv"], f["q"], 0, None)


@pytest.mark.parametrize("status,text,change", [
    (1, "NULL", dict(pos=0)), (2, "head_dim", dict(hd=264)), (2, "head_dim", dict(hd=20)),
    (2, "rotary_dim", dict(rotary=72)), (1, "strides", dict(ldx=120)), (1, "strides", dict(ldx=132)),
    (1, "strides", dict(ldx=136, y=A)), (1, "aligned", dict(x=A + 4)), (1, "heads", dict(heads=0)),
    (1, "rows", dict(rows=-1))])
def test_rotary_refuses(lib, status, text, change):
    f = dict(x=A, rows=3, heads=2, hd=64, ldx=0, pos=A, rotary=64, y=2 * A)
    f.update(change)
    refused(lib, status, text, "tts_rotary", CTX, f["x"], 0, f["rows"], f["heads"], f["hd"], f["ldx"], f["pos"],
            A, A, 10, f["rotary"], 0, f["y"], 0, None)


@pytest.mark.parametrize("status,text,change", [
    (1, "NULL", dict(x=0)), (1, "NULL", dict(u=0)), (1, "rows", dict(rows=0)), (1, "n >= 1", dict(n=0)),
    (1, "ldl", dict(ldl=99)), (2, "262144", dict(n=262145))])
def test_filter_sample_refuses(lib, status, text, change):
    f = dict(x=A, rows=3, n=100, ldl=0, u=A)
    f.update(change)
    refused(lib, status, text, "tts_filter_sample", CTX, f["x"], 0, f["rows"], f["n"], f["ldl"], f["u"], None,
            A, None)


def test_scaled_tables():
    """Each kind against its formula written out; the phases are rounded once, to f32."""
    n, r, base, f = 300, 64, 1e4, 4.0
    t, i = np.arange(n)[:, None], np.arange(r // 2)
    plain = base ** (-2 * i / r)

    def check(want, scale=1.0, **kw):
        c, s = ttsnn.rope_table_scaled(n, r, base, factor=f, device="cpu", **kw)
        assert c.shape == s.shape == (n, r // 2)
        # half a step of f32, and the phase's own 64-bit rounding (below 300 radians)
        assert np.abs(c.numpy() - scale * np.cos(t * want)).max() <= scale * (2.0 ** -24 + 1e-12)
        assert np.abs(s.numpy() - scale * np.sin(t * want)).max() <= scale * (2.0 ** -24 + 1e-12)

    check(plain / f, kind="linear")
    slow = (base * f ** (r / (r - 2))) ** (-2 * i / r)
    check(slow, kind="ntk")
    assert math.isclose(slow[-1], plain[-1] / f)
    low = max(0, math.floor(r * math.log(512 / (32 * 2 * math.pi)) / (2 * math.log(base))))
    high = min(r - 1, math.ceil(r * math.log(512 / (2 * math.pi)) / (2 * math.log(base))))
    mix = np.clip((i - low) / (high - low), 0, 1)
    yarn = plain * (1 - mix) + plain / f * mix
    check(yarn, 0.1 * math.log(f) + 1, kind="yarn", original=512)
    check(yarn, 2.0, kind="yarn", original=512, mscale=2.0)
    assert (mix[:low + 1] == 0).all() and mix[-1] == 1
    same = ttsnn.rope_table_scaled(n, r, base, device="cpu")
    ref = ttsnn.rope_table_f32(n, r, base, device="cpu")
    assert all(np.abs(a.numpy() - b.numpy()).max() <= 2.0 ** -23 for a, b in zip(same, ref))


def test_overlapping_buffers_are_refused(lib):
    """Outputs over inputs that other blocks may still read."""
    for f16, out in ((1, A), (1, A + 8 * 4 * 256 - 16), (0, A + 8 * 4 * 512 - 16)):
        refused(lib, 1, "apart from q", "tts_chunk_attention", CTX, A, f16, 2, lanes(), kv(), 1.0, 0, out, A,
                1 << 40, None)
    for q in (A, A + 8 * 8 * 512 - 16, A - 16):
        refused(lib, 1, "apart from qkv", "tts_rotary_append", CTX, A, 0, 4, lanes(), None, 1e-6, A, A, 64, 64, 0,
                kv(), q, 0, None)
    for y, ld in ((A + 16, 0), (A + 512, 0), (A + 16, 256), (A + 512 - 16, 256), (A + 1024 - 16, 256)):
        refused(lib, 1, "apart from it", "tts_rotary", CTX, A, 0, 3, 2, 64, ld, A, A, A, 10, 64, 0, y, ld, None)


def test_cache_on_another_device_is_refused():
    import torch
    at = lambda *shape, dtype=torch.float16: torch.zeros(*shape, dtype=dtype, device="meta")
    cache = ttsnn.attn.paged_cache(at(4, 2, 8, 128), at(4, 2, 8, 128), at(1, 4, dtype=torch.int32))
    starts, spans = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    with pytest.raises(ValueError, match="meta"):
        ttsnn.attn.chunk_attention(torch.zeros(2, 4, 128), starts, spans, cache, 1.0)
    with pytest.raises(ValueError, match="meta"):
        ttsnn.qkrope.rotary_append(torch.zeros(2, 1024), 4, starts, spans, torch.zeros(8, 64),
                                   torch.zeros(8, 64), cache)
    with pytest.raises(ValueError, match="2\\^31"):
        ttsnn.attn.chunk_attention(torch.zeros(2, 4, 128), starts, spans, cache, 1.0, window=2 ** 32 + 5)


@pytest.mark.parametrize("kw", [dict(kind="other"), dict(kind="yarn"), dict(factor=0.0), dict(rotary_dim=7),
                                dict(length=0), dict(kind="ntk", rotary_dim=2),
                                dict(kind="yarn", original=100, beta_fast=1.0)])
def test_scaled_tables_refuse(kw):
    args = dict(length=10, rotary_dim=8, base=1e4, device="cpu")
    args.update(kw)
    with pytest.raises(ValueError):
        ttsnn.rope_table_scaled(**args)
