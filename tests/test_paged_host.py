"""What the paged-cache operators refuse, and the pieces that need no GPU."""

from __future__ import annotations

import math

import pytest
import torch

import flash_attention_triton_b200 as fa
from flash_attention_triton_b200 import _lib

BF16 = torch.bfloat16


def cache_arguments(batch=3, pages=7, page=16, kv_heads=2, d=64, width=4, dtype=BF16):
    return {"k_cache": torch.zeros(pages, page, kv_heads, d, dtype=dtype),
            "v_cache": torch.zeros(pages, page, kv_heads, d, dtype=dtype),
            "block_table": torch.zeros(batch, width, dtype=torch.int32),
            "lengths": torch.ones(batch, dtype=torch.int32)}


def decode_arguments(**kwargs):
    a = cache_arguments()
    return {"q": torch.zeros(3, 4, 64, dtype=BF16), **a, **kwargs}


def append_arguments(**kwargs):
    a = cache_arguments()
    return {"k": torch.zeros(3, 2, 64, dtype=BF16), "v": torch.zeros(3, 2, 64, dtype=BF16), **a, **kwargs}


@pytest.mark.parametrize("change,error,text", [
    ({}, AssertionError, "CUDA device"),
    ({"q": torch.zeros(2, 4, 64, dtype=BF16)}, ValueError, "one row for each sequence"),
    ({"q": torch.zeros(3, 3, 64, dtype=BF16)}, ValueError, "multiple of the cache's heads"),
    ({"q": torch.zeros(3, 0, 64, dtype=BF16)}, ValueError, "multiple of the cache's heads"),
    ({"q": torch.zeros(3, 4, 32, dtype=BF16)}, ValueError, "headdim"),
    ({"q": torch.zeros(3, 4, 64, dtype=torch.float16)}, ValueError, "type of the cache"),
    ({"q": None}, TypeError, "q must be a tensor"),
    ({"block_table": torch.zeros(3, 4, dtype=torch.int64)}, ValueError, "int32"),
    ({"block_table": torch.zeros(3, 8, dtype=torch.int32)[:, ::2]}, ValueError, "contiguous"),
    ({"block_table": torch.zeros(3, 0, dtype=torch.int32)}, ValueError, "no entries"),
    ({"lengths": torch.ones(4, dtype=torch.int32)}, ValueError, "one entry for each sequence"),
    ({"lengths": torch.ones(3)}, ValueError, "int32"),
    ({"k_cache": torch.zeros(7, 16, 2, 64)}, ValueError, "fp16 or bf16"),
    ({"k_cache": torch.zeros(7, 8, 2, 64, dtype=BF16)}, ValueError, "same shape"),
    ({"v_cache": torch.zeros(7, 16, 2, 128, dtype=BF16)[..., ::2]}, ValueError, "contiguous in its last"),
    ({"v_cache": torch.zeros(7 * 16 * 2 * 64 + 1, dtype=BF16)[1:].view(7, 16, 2, 64)}, ValueError, "aligned"),
    ({"v_cache": torch.zeros(1, 16, 2, 64, dtype=BF16).expand(7, 16, 2, 64)}, ValueError, "multiples of 8"),
])
def test_decode_refuses(change, error, text):
    with torch.no_grad(), pytest.raises(error, match=text):
        fa.flash_attention_decode(**decode_arguments(**change))


@pytest.mark.parametrize("change,error,text", [
    ({}, AssertionError, "CUDA device"),
    ({"k": torch.zeros(3, 4, 64, dtype=BF16)}, ValueError, "heads of the cache"),
    ({"v": torch.zeros(3, 2, 32, dtype=BF16)}, ValueError, "heads of the cache"),
    ({"v": torch.zeros(3, 2, 64)}, ValueError, "type of the cache"),
    ({"k": torch.zeros(5, 2, 64, dtype=BF16), "v": torch.zeros(5, 2, 64, dtype=BF16)}, ValueError, "one token"),
    ({"cu_seqlens": torch.zeros(3, dtype=torch.int32)}, ValueError, "one entry more"),
    ({"cu_seqlens": torch.zeros(4, dtype=torch.int64)}, ValueError, "int32"),
    ({"q": torch.zeros(3, 3, 64, dtype=BF16)}, ValueError, "multiple of the cache's heads"),
    ({"q": torch.zeros(4, 4, 64, dtype=BF16)}, ValueError, "q must be"),
    ({"cos": torch.zeros(100, 16)}, ValueError, "go together"),
    ({"cos": torch.zeros(100, 12), "sin": torch.zeros(100, 12)}, ValueError, "multiple of 16"),
    ({"cos": torch.zeros(100, 40), "sin": torch.zeros(100, 40)}, ValueError, "up to the head dimension"),
    ({"cos": torch.zeros(100, 16).double(), "sin": torch.zeros(100, 16)}, ValueError, "fp32"),
    ({"cos": torch.zeros(0, 16), "sin": torch.zeros(0, 16)}, ValueError, "fp32"),
])
def test_append_refuses(change, error, text):
    with pytest.raises(error, match=text):
        fa.append_kv_cache(**append_arguments(**change))


def test_no_graph_is_lost_in_silence():
    with pytest.raises(ValueError, match="no_grad"):
        fa.flash_attention_decode(**decode_arguments(q=torch.zeros(3, 4, 64, dtype=BF16, requires_grad=True)))
    with pytest.raises(ValueError, match="no_grad"):
        fa.append_kv_cache(**append_arguments(k=torch.zeros(3, 2, 64, dtype=BF16, requires_grad=True)))


@pytest.mark.parametrize("d", [4, 44, 264])
def test_head_dims(d):
    with pytest.raises(ValueError, match="head dimension"):
        fa.flash_attention_decode(torch.zeros(3, 4, d, dtype=BF16), **cache_arguments(d=d))


def test_workspace_size():
    lib = _lib.lib()
    # 16 bytes for every (sequence, key head) or CTA, whichever are fewer, 4 for every CTA (in fours), and two places for each
    # CTA: m, l and o of each row; no more CTAs than units of 64 keys
    assert lib.fa2_decode_workspace_bytes(1, 8, 2, 128, 16, 4) == 2 * 16 + 4 * 4 + 2 * 2 * 4 * 130 * 4
    assert lib.fa2_decode_workspace_bytes(1, 8, 2, 64, 16, 4) == 1 * 16 + 4 * 4 + 1 * 2 * (2 * 4) * 66 * 4  # two key heads at once
    assert lib.fa2_decode_workspace_bytes(1, 40, 2, 128, 16, 8) == 4 * 16 + 8 * 4 + 8 * 2 * 16 * 130 * 4  # 20 heads: two passes of 16 rows
    assert lib.fa2_decode_workspace_bytes(1, 3, 2, 64, 16, 4) == 0
    assert lib.fa2_decode_workspace_bytes(1, 8, 2, 64, 1 << 16, 1 << 16) == 0


@pytest.mark.parametrize("change,code", [
    ({"q": 0}, -1), ({"table": 0}, -1), ({"D": 12}, -2), ({"dtype": 2}, -3), ({"q": 0x1008}, -4), ({"batch": 0}, -5),
    ({"width": 1 << 30}, -5), ({"width": 1 << 26, "batch": 200}, -5), ({"scale": math.inf}, -9), ({"bytes": 16}, -10), ({"Hq": 7}, -13),
    ({"strides": [128, 64, 2048, 128, 60, 2048, 128, 64, 4]}, -12), ({"strides": [128, 32, 2048, 128, 64, 2048, 128, 64, 4]}, -12),
])
def test_decode_codes(change, code):
    import ctypes
    a = {"q": 0x1000, "k": 0x1000, "v": 0x1000, "out": 0x1000, "table": 0x1000, "lengths": 0x1000, "ws": 0x1000, "bytes": 1 << 24,
         "batch": 2, "Hq": 4, "Hkv": 2, "D": 64, "pages": 3, "page": 16, "width": 4, "dtype": 1, "scale": 0.125, "strides": None, **change}
    st = (ctypes.c_longlong * 9)(*a["strides"]) if a["strides"] else None
    assert _lib.lib().fa2_decode(a["q"], a["k"], a["v"], a["out"], a["table"], a["lengths"], a["ws"], a["bytes"], a["batch"], a["Hq"],
                                 a["Hkv"], a["D"], a["pages"], a["page"], a["width"], a["dtype"], a["scale"], st, None) == code


@pytest.mark.parametrize("change,code", [
    ({"k": 0}, -1), ({"q_out": 0}, -1), ({"Hq": 3}, -13), ({"tokens": 3}, -5), ({"rotary": 24}, -14), ({"cos": 0}, -14),
    ({"rotary": 80}, -14), ({"k_cache": 0x1004}, -4), ({"pages": 0}, -5),
])
def test_append_codes(change, code):
    a = {"q": 0x1000, "k": 0x1000, "v": 0x1000, "q_out": 0x1000, "k_out": 0, "k_cache": 0x1000, "v_cache": 0x1000, "table": 0x1000,
         "lengths": 0x1000, "cu": 0, "cos": 0x1000, "sin": 0x1000, "tokens": 2, "batch": 2, "Hq": 4, "Hkv": 2, "D": 64, "pages": 3,
         "page": 16, "width": 4, "positions": 9, "rotary": 32, "interleaved": 0, "dtype": 1, **change}
    assert _lib.lib().fa2_kv_append(*a.values(), None, None) == code


def test_rotary_tables():
    cos, sin = fa.rotary_tables(200000, 32, base=500000.0)
    assert cos.shape == sin.shape == (200000, 16) and cos.dtype == torch.float32
    p, j = 199999, 3
    angle = p * 500000.0 ** (-2 * j / 32)
    assert abs(cos[p, j].item() - math.cos(angle)) < 1e-7 and abs(sin[p, j].item() - math.sin(angle)) < 1e-7
    with pytest.raises(ValueError, match="multiple of 16"):
        fa.rotary_tables(10, 24)


def test_a_cache_that_cannot_be_written_is_refused():
    """The copy that stands for a negating view would be written in its place."""
    a = append_arguments()
    for name in ("k_cache", "v_cache"):
        with pytest.raises(ValueError, match=f"{name} must not be a negating view"):
            fa.append_kv_cache(**{**a, name: torch._neg_view(a[name])})
    with torch.no_grad(), pytest.raises(ValueError, match="q must be a plain tensor"):
        torch.vmap(lambda q: fa.flash_attention_decode(**{**decode_arguments(), "q": q}))(decode_arguments()["q"][None])
