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
