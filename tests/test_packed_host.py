"""What flash_attention_packed refuses, and the formulas of its tests against differences."""

from __future__ import annotations

import pytest
import torch

import flash_attention_triton_b200 as fa
from flash_attention_triton_b200 import _lib
from packed_helpers import exact_packed

BF16 = torch.bfloat16


def arguments(**kwargs):
    return {"q": torch.zeros(10, 4, 64, dtype=BF16), "k": torch.zeros(10, 2, 64, dtype=BF16), "v": torch.zeros(10, 2, 64, dtype=BF16),
            "cu_seqlens": torch.tensor([0, 10], dtype=torch.int32), **kwargs}


@pytest.mark.parametrize("change,error,text", [
    ({}, AssertionError, "CUDA device"),
    ({"q": torch.zeros(10, 3, 64, dtype=BF16)}, ValueError, "multiple of kv_heads"),
    ({"q": torch.zeros(10, 0, 64, dtype=BF16)}, ValueError, "multiple of kv_heads"),
    ({"q": torch.zeros(9, 4, 64, dtype=BF16)}, ValueError, "q must be"),
    ({"q": torch.zeros(1, 10, 4, 64, dtype=BF16)}, ValueError, "q must be"),
    ({"v": torch.zeros(10, 1, 64, dtype=BF16)}, ValueError, "kv_heads"),
    ({"q": torch.zeros(10, 4, 64)}, ValueError, "fp16 or bf16"),
    ({"q": torch.zeros(10, 4, 64, dtype=torch.float16)}, ValueError, "all the same"),
    ({"cu_seqlens": torch.tensor([0, 10])}, ValueError, "int32"),
    ({"cu_seqlens": torch.tensor([0], dtype=torch.int32)}, ValueError, "one entry more"),
    ({"cu_seqlens": torch.tensor([[0, 10]], dtype=torch.int32)}, ValueError, "one dimension"),
    ({"cu_seqlens": [0, 10]}, TypeError, "tensor"),
    ({"softmax_scale": -1.0}, ValueError, "finite"),
    ({"softmax_scale": float("nan")}, ValueError, "finite"),
    ({"softmax_scale": "x"}, TypeError, "number"),
])
def test_refuses(change, error, text):
    with pytest.raises(error, match=text):
        fa.flash_attention_packed(**arguments(**change))


@pytest.mark.parametrize("d", [4, 20, 136, 256])
def test_head_dims(d):
    t = torch.zeros(10, 2, d, dtype=BF16)
    with pytest.raises(ValueError, match="head dimension"):
        fa.flash_attention_packed(t, t, t, torch.tensor([0, 10], dtype=torch.int32))


@pytest.mark.parametrize("change,code", [
    ({"q": 0}, -1), ({"plan": 0}, -1), ({"cu": 0}, -1), ({"D": 136}, -2), ({"D": 12}, -2), ({"dtype": 5}, -3), ({"k": 0x1008}, -4),
    ({"rows": (1 << 24) + 1}, -5), ({"batch": 0}, -5), ({"rows": 1 << 24, "Hq": 8000, "Hkv": 1}, -5), ({"scale": 0.0}, -9), ({"Hq": 3}, -13),
    ({"strides": [100, 64, 128, 64, 128, 64]}, -12), ({"strides": [256, 64, 0, 64, 128, 64]}, -12),
])
def test_forward_codes(change, code):
    import ctypes
    a = {"q": 0x1000, "k": 0x1000, "v": 0x1000, "o": 0x1000, "lse": 0x1000, "cu": 0x1000, "plan": 0x1000, "rows": 10, "batch": 1, "Hq": 4,
         "Hkv": 2, "D": 64, "dtype": 1, "scale": 0.125, "strides": None, **change}
    a["strides"] = (ctypes.c_longlong * 6)(*a["strides"]) if a["strides"] else None
    assert _lib.lib().fa2_packed_fwd(*a.values(), None) == code


@pytest.mark.parametrize("change,code", [({"dv": 0}, -1), ({"D": 200}, -2), ({"bytes": 100}, -10), ({"ws": 0}, -10), ({"Hq": 5}, -13)])
def test_backward_codes(change, code):
    a = {n: 0x1000 for n in ("q", "k", "v", "o", "dout", "lse", "dq", "dk", "dv", "cu", "plan", "ws")}
    a |= {"bytes": 1 << 24, "rows": 10, "batch": 1, "Hq": 4, "Hkv": 2, "D": 64, "dtype": 1, "scale": 0.125, "strides": None, **change}
    assert _lib.lib().fa2_packed_bwd(*a.values(), None) == code


def test_sizes():
    lib = _lib.lib()
    tiles = 1000 // 128 + 3  # at most, of 1000 rows in 3 sequences
    assert lib.fa2_packed_plan_bytes(1000, 3) == 16 + 2 * 16 * tiles
    assert lib.fa2_packed_bwd_workspace_bytes(1000, 3, 4) == tiles * 4 * (256 + 4) * 4 + 16
    assert lib.fa2_packed_plan_bytes(-1, 3) == lib.fa2_packed_plan_bytes(10, 0) == 0


def test_formulas_of_the_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    lengths = [5, 1, 0, 9]
    q, k, v, do = (torch.randn(15, h, 8, generator=g, dtype=torch.float64) for h in (4, 2, 2, 4))
    exact = {n: t for n, (t, _) in exact_packed(q, k, v, lengths, do).items()}
    inputs = {"dq": q, "dk": k, "dv": v}
    for name, t in inputs.items():
        for index in [(0, 0, 0), (4, 1, 3), (5, 0, 2), (14, 1, 7), (10, 1, 1)]:
            step, ends = 1e-5, []
            for sign in (1, -1):
                moved = t.clone()
                moved[index] += sign * step
                o = exact_packed(*(moved if x is t else x for x in (q, k, v)), lengths)["o"][0]
                ends.append((o * do).sum().item())
            # central differences: step^2 times a third derivative, 1e-16 / step of the sums' roundings
            assert abs((ends[0] - ends[1]) / (2 * step) - exact[name][index].item()) < 1e-8


def test_transforms_and_tangents_are_refused():
    """A tangent would be lost in silence otherwise."""
    import torch.autograd.forward_ad as fwad

    a = arguments()
    with fwad.dual_level(), pytest.raises(ValueError, match="q must be a plain tensor"):
        fa.flash_attention_packed(**{**a, "q": fwad.make_dual(a["q"], torch.ones_like(a["q"]))})
    with pytest.raises(ValueError, match="v must be a plain tensor"):
        torch.func.grad(lambda v: fa.flash_attention_packed(**{**a, "v": v}).float().sum())(a["v"])
    with pytest.raises(ValueError, match="q must be a plain tensor"):
        torch.vmap(lambda q: fa.flash_attention_packed(**{**a, "q": q}))(a["q"][None])
