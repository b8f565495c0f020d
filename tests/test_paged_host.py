"""What the paged cache's calls refuse before they reach a GPU: through the C ABI, and through the Python entry points."""
import ctypes

import pytest
import torch

import gpuk_b200 as gpuk
from gpuk_b200 import cabi

P = 1 << 20      # an aligned address that is never followed


def _pages(**more):
    values = dict(k=P, v=P, page_stride=8192, head_stride=1024, row_stride=64, num_pages=4, kv_heads=2, page_size=16, head_dim=64, dtype=cabi.DTYPE_BF16)
    values.update(more)
    return ctypes.byref(cabi.Pages(**values))


def _plan(**more):
    v = dict(lens=P, new=P, tables=P, stride=4, width=4, held=P, free=P, capacity=4, count=P, parents=None, batch=2, total=8, page=16, words=0, starts=P, positions=P, slots=P,
             masks=None, held_out=P, count_out=P)
    v.update(more)
    return cabi.lib.gpuk_paged_plan(*v.values(), None)


@pytest.mark.parametrize("more,status,text", [
    ({"batch": -1}, cabi.ERR_INVALID_ARGUMENT, "sizes"), ({"total": -1}, cabi.ERR_INVALID_ARGUMENT, "sizes"), ({"width": -1}, cabi.ERR_INVALID_ARGUMENT, "sizes"),
    ({"page": 24}, cabi.ERR_UNSUPPORTED, "powers of two"), ({"page": 0}, cabi.ERR_UNSUPPORTED, "powers of two"), ({"page": 1 << 17}, cabi.ERR_UNSUPPORTED, "powers of two"),
    ({"batch": 4097}, cabi.ERR_UNSUPPORTED, "4096"), ({"parents": P}, cabi.ERR_INVALID_ARGUMENT, "masks"), ({"masks": P, "words": 1}, cabi.ERR_INVALID_ARGUMENT, "masks"),
    ({"parents": P, "masks": P, "words": 9}, cabi.ERR_INVALID_ARGUMENT, "8 words"), ({"width": 1 << 28}, cabi.ERR_UNSUPPORTED, "too large"),
    ({"batch": 4096, "width": 1 << 20}, cabi.ERR_UNSUPPORTED, "too large"), ({"lens": None}, cabi.ERR_INVALID_ARGUMENT, "null"), ({"starts": None}, cabi.ERR_INVALID_ARGUMENT, "null"),
    ({"free": None}, cabi.ERR_INVALID_ARGUMENT, "null"), ({"slots": None}, cabi.ERR_INVALID_ARGUMENT, "null"), ({"total": 1 << 30}, cabi.ERR_UNSUPPORTED, "too many")])
def test_plan_refusals(more, status, text):
    assert _plan(**more) == status and text in cabi.last_error()


def _attention(pages=None, **more):
    v = dict(q=P, qt=256, qh=64, pages=pages or _pages(), tables=P, stride=4, width=4, lens=P, starts=P, masks=None, words=0, out=P, ot=256, oh=64, batch=2, tokens=8, heads=4,
             max_len=64, max_new=0, scale=0.125, ws=None, bytes=0)
    v.update(more)
    return cabi.lib.gpuk_paged_attention(*v.values(), None)


@pytest.mark.parametrize("more,status,text", [
    ({"pages": _pages(dtype=cabi.DTYPE_F32)}, cabi.ERR_UNSUPPORTED, "bf16 and fp16"), ({"pages": _pages(head_dim=96)}, cabi.ERR_UNSUPPORTED, "64 and 128"),
    ({"pages": _pages(kv_heads=0)}, cabi.ERR_INVALID_ARGUMENT, "sizes"), ({"heads": 5}, cabi.ERR_UNSUPPORTED, "whole number"), ({"heads": 258}, cabi.ERR_UNSUPPORTED, "at most 128"),
    ({"pages": _pages(page_size=4)}, cabi.ERR_UNSUPPORTED, "powers of two"), ({"pages": _pages(page_size=48)}, cabi.ERR_UNSUPPORTED, "powers of two"),
    ({"masks": P, "words": 9}, cabi.ERR_UNSUPPORTED, "8"), ({"masks": P}, cabi.ERR_INVALID_ARGUMENT, "sizes"), ({"scale": 0.0}, cabi.ERR_INVALID_ARGUMENT, "scale"),
    ({"scale": -1.0}, cabi.ERR_INVALID_ARGUMENT, "scale"), ({"scale": float("nan")}, cabi.ERR_INVALID_ARGUMENT, "scale"), ({"scale": float("inf")}, cabi.ERR_INVALID_ARGUMENT, "scale"),
    ({"tokens": (1 << 24) + 1}, cabi.ERR_UNSUPPORTED, "2\\^24"), ({"tokens": -1}, cabi.ERR_INVALID_ARGUMENT, "sizes"), ({"max_new": -1}, cabi.ERR_INVALID_ARGUMENT, "sizes"), ({"q": None}, cabi.ERR_INVALID_ARGUMENT, "null"),
    ({"tables": None}, cabi.ERR_INVALID_ARGUMENT, "null"), ({"pages": _pages(num_pages=0)}, cabi.ERR_INVALID_ARGUMENT, "no pages"), ({"width": 0}, cabi.ERR_INVALID_ARGUMENT, "no pages"),
    ({"q": P + 8}, cabi.ERR_INVALID_ARGUMENT, "aligned"), ({"pages": _pages(v=P + 2)}, cabi.ERR_INVALID_ARGUMENT, "aligned"), ({"qt": 12}, cabi.ERR_INVALID_ARGUMENT, "strides"),
    ({"qh": 0}, cabi.ERR_INVALID_ARGUMENT, "strides"), ({"pages": _pages(row_stride=68)}, cabi.ERR_INVALID_ARGUMENT, "strides"), ({"width": 1 << 28}, cabi.ERR_UNSUPPORTED, "too wide")])
def test_attention_refusals(more, status, text):
    import re
    assert _attention(**more) == status and re.search(text, cabi.last_error())


def test_attention_of_nothing():
    assert _attention(tokens=0) == cabi.OK and _attention(batch=0) == cabi.OK
    bytes_ = ctypes.c_int64(7)
    assert cabi.lib.gpuk_paged_attention_workspace(_pages(), 2, 0, 4, 100000, ctypes.byref(bytes_)) == cabi.OK and bytes_.value == 0
    assert cabi.lib.gpuk_paged_attention_workspace(_pages(head_dim=32), 2, 1, 4, 100000, ctypes.byref(bytes_)) == cabi.ERR_UNSUPPORTED


def _rope(**more):
    v = dict(x=P, t=128, h=64, out=P, ot=128, oh=64, positions=P, turns=P, amplitude=1.0, tokens=3, heads=2, head_dim=64, rotary=64, layout=0, dtype=0)
    v.update(more)
    return cabi.lib.gpuk_rope(*v.values(), None)


@pytest.mark.parametrize("more,status", [
    ({"head_dim": 40, "rotary": 32}, cabi.ERR_UNSUPPORTED), ({"rotary": 24}, cabi.ERR_UNSUPPORTED), ({"rotary": 80}, cabi.ERR_UNSUPPORTED), ({"rotary": 0}, cabi.ERR_UNSUPPORTED),
    ({"head_dim": 512, "rotary": 512}, cabi.ERR_UNSUPPORTED), ({"dtype": 2}, cabi.ERR_UNSUPPORTED), ({"layout": 3}, cabi.ERR_INVALID_ARGUMENT), ({"tokens": -1}, cabi.ERR_INVALID_ARGUMENT),
    ({"x": P + 4}, cabi.ERR_INVALID_ARGUMENT), ({"out": None}, cabi.ERR_INVALID_ARGUMENT), ({"positions": None}, cabi.ERR_INVALID_ARGUMENT), ({"t": 100}, cabi.ERR_INVALID_ARGUMENT)])
def test_rope_refusals(more, status):
    assert _rope(**more) == status


def _rope_paged(pages=None, **more):
    v = dict(q=P, qt=128, qh=64, k=P, kt=128, kh=64, v=P, vt=128, vh=64, out=P, ot=128, oh=64, positions=P, slots=P, turns=P, amplitude=1.0, pages=pages or _pages(), tokens=3,
             heads=2, rotary=64, layout=0)
    v.update(more)
    return cabi.lib.gpuk_rope_paged(*v.values(), None)


@pytest.mark.parametrize("more,status", [
    ({"slots": None}, cabi.ERR_INVALID_ARGUMENT), ({"k": None}, cabi.ERR_INVALID_ARGUMENT), ({"v": P + 8}, cabi.ERR_INVALID_ARGUMENT), ({"pages": _pages(page_size=12)}, cabi.ERR_UNSUPPORTED),
    ({"pages": _pages(kv_heads=-1)}, cabi.ERR_INVALID_ARGUMENT), ({"pages": _pages(head_stride=4)}, cabi.ERR_INVALID_ARGUMENT), ({"layout": -1}, cabi.ERR_INVALID_ARGUMENT)])
def test_rope_paged_refusals(more, status):
    assert _rope_paged(**more) == status


def _keep(pages=None, **more):
    v = dict(pages=pages or _pages(), layers=2, stride=65536, tables=P, ts=4, width=4, lens=P, paths=P, ps=3, depth=3, out=P, batch=2)
    v.update(more)
    return cabi.lib.gpuk_paged_keep(*v.values(), None)


@pytest.mark.parametrize("more,status", [
    ({"layers": 0}, cabi.ERR_INVALID_ARGUMENT), ({"depth": -1}, cabi.ERR_INVALID_ARGUMENT), ({"lens": None}, cabi.ERR_INVALID_ARGUMENT), ({"out": None}, cabi.ERR_INVALID_ARGUMENT),
    ({"stride": 12}, cabi.ERR_INVALID_ARGUMENT), ({"pages": _pages(k=P + 8)}, cabi.ERR_INVALID_ARGUMENT), ({"pages": _pages(head_dim=20)}, cabi.ERR_UNSUPPORTED),
    ({"pages": _pages(page_size=3)}, cabi.ERR_UNSUPPORTED), ({"layers": 40000}, cabi.ERR_UNSUPPORTED)])
def test_keep_refusals(more, status):
    assert _keep(**more) == status


def test_the_entry_points_take_cuda_tensors_only():
    ints, x, pages = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    longs, f = torch.zeros(3, dtype=torch.int64), gpuk.rope_frequencies(64)
    for call in (lambda: gpuk.paged_plan(ints, ints, torch.zeros(3, 4, dtype=torch.int32), ints, ints, ints, 16, 3), lambda: gpuk.rope(x, longs, f),
                 lambda: gpuk.rope_paged(x, x, x, longs, longs, f, pages, pages), lambda: gpuk.paged_attention(x, pages, pages, torch.zeros(2, 4, dtype=torch.int32), ints[:2], ints),
                 lambda: gpuk.paged_keep(pages, pages, torch.zeros(3, 4, dtype=torch.int32), ints, torch.zeros(3, 2, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_frequencies_refuse_what_they_cannot_be():
    for bad in (dict(rotary=7), dict(rotary=0), dict(rotary=64, scaling={"kind": "cubic", "factor": 2.0}), dict(rotary=64, scaling={"kind": "linear", "factor": 0.0}),
                dict(rotary=2, scaling={"kind": "base", "factor": 2.0}), dict(rotary=64, scaling={"kind": "bands", "factor": 2.0, "low": 4.0, "high": 1.0, "original": 100})):
        with pytest.raises(ValueError, match="gpuk"):
            gpuk.rope_frequencies(**bad)
    with pytest.raises(ValueError, match="order of rotary pairs"):
        gpuk.rope(None, None, gpuk.rope_frequencies(16), layout="thirds")
    with pytest.raises(ValueError, match="positive"):
        gpuk.paged_attention(None, None, None, None, None, None, scale=-1.0)


def test_fixed_point_turns():
    """Half a unit of 2^-64 of a turn, and what the double in front of it holds."""
    for rotary, theta in ((128, 10000.0), (32, 500000.0)):
        f, _ = gpuk.paged.scaled_frequencies(rotary, theta)
        turns = gpuk.rope_frequencies(rotary, theta).turns
        for x, t in zip(f.tolist(), turns.tolist()):
            assert abs((t % 2 ** 64) / 2 ** 64 - x / (2 * 3.141592653589793)) <= x * 2.0 ** -52 + 2.0 ** -65
