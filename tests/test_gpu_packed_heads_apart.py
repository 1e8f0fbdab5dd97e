"""fp16 gradients of query heads that share a key head but not the size of their dO."""

from __future__ import annotations

import math

import pytest
import torch

from flash_attention_triton_b200 import _lib, flash_attention_packed
from packed_helpers import exact_packed

pytestmark = pytest.mark.gpu
FP16 = torch.float16


@pytest.fixture(autouse=True)
def _no_status():
    yield
    assert _lib.device_status() == 0


def inputs(lengths, heads, kv_heads, d, seed=0):
    g = torch.Generator().manual_seed(seed)
    cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    return [torch.randn(sum(lengths), h, d, generator=g).to(FP16).cuda() for h in (heads, kv_heads, kv_heads, heads)] + [cu]


def gradients(q, k, v, do, cu):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    return torch.autograd.grad(flash_attention_packed(*leaves, cu), leaves, do)


@pytest.mark.parametrize("lengths,heads,kv_heads,d", [([2048, 300], 4, 1, 64), ([2048, 300], 8, 2, 128), ([2000], 3, 1, 32), ([40] * 50, 4, 2, 96)])
def test_each_head_has_the_error_of_its_own_size(lengths, heads, kv_heads, d):
    """The bound of a head's dQ is the one that it has alone: dO of the heads beside it, up to 2^12 times larger, is no part of it."""
    q, k, v, do, cu = inputs(lengths, heads, kv_heads, d)
    powers = [0, -8, -12, -4]
    for h in range(heads):
        do[:, h] = (do[:, h].double() * 2.0 ** powers[h % 4]).to(FP16)
    dq = gradients(q, k, v, do, cu)[0]
    for h in range(heads):
        j = h * kv_heads // heads
        one = slice(h, h + 1), slice(j, j + 1)
        want, tolerance = exact_packed(q[:, one[0]], k[:, one[1]], v[:, one[1]], lengths, do[:, one[0]])["dq"]
        off = (dq[:, one[0]].double() - want).abs()
        assert (off <= tolerance).all(), (h, (off / tolerance).max().item())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("other", [math.inf, math.nan, 2.0**-12, 1024.0, 0.0])
def test_a_head_does_not_see_the_gradient_of_another(other, d):
    q, k, v, do, cu = inputs([700, 130], 4, 2, d)
    clean = gradients(q, k, v, do, cu)[0]
    do = do.clone()
    do[:, 1], do[5, 2] = other, other
    got = gradients(q, k, v, do, cu)[0]
    assert torch.equal(got[:, [0, 3]], clean[:, [0, 3]])
