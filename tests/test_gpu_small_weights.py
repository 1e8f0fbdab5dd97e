"""Rows whose weight lies almost all on one key of small value, so that many small weights make the result.

One key stands 17.5 nats above the others, with zeros as its values; the others are like each other, with values about 1.  Of
8 192 keys these are 2.1e-4 of the output, in weights of 2^-25.2 each.
"""

from __future__ import annotations

import math

import pytest
import torch

from flash_attention_triton_b200 import _lib, flash_attention_packed, flash_attention_v2
from paged_helpers import Cache, fa

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SCALE = 0.125


@pytest.fixture(autouse=True)
def _no_status():
    yield
    assert _lib.device_status() == 0


def rows(n, heads, kv_heads, d, dtype, nats=17.5, seed=0, queries=None):
    """q, k, v, dO; the first key is the one above the others."""
    g = torch.Generator().manual_seed(seed)
    q = 0.25 * torch.randn(queries or n, heads, d, generator=g)
    k, v = torch.randn(n, kv_heads, d, generator=g), 1 + 0.1 * torch.randn(n, kv_heads, d, generator=g)
    do = 1 + 0.1 * torch.randn(queries or n, heads, d, generator=g)
    q[:, :, 0], k[:, :, 0], k[0] = 8.0, 0.0, 0.0
    k[0, :, 0] = nats  # 8 x nats x SCALE
    v[0] = 0.0
    return [t.to(dtype).cuda() for t in (q, k, v, do)]


def exact(q, k, v, causal=True):
    """Output, sum of weights x |v| and the weights of one head, in 64 bits."""
    s = q.double() @ k.double().T * SCALE
    if causal:
        s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu_(1 + k.shape[0] - q.shape[0]), -math.inf)
    p = torch.softmax(s, 1)
    return p @ v.double(), p @ v.double().abs(), p


def bound(dtype, out, absolute, n, d, values):
    """The output's rounding, and that of the weights; a score's d additions in 32 bits of at most 20 and the polynomial that stands in for some
    exponentials, in a weight and in their sum; sums of n terms.  At fp16 a weight carries 2^11 beside a row whose largest
    is at least 1, so below the normal numbers it is off by 2^-36; the last term is half a step of fp16's smallest numbers."""
    half = torch.finfo(dtype).eps / 2
    e = (d + 8) * 2.0**-24 * 20 + 1e-4
    tiny = 2.0**-36 * n * values if dtype == FP16 else 0.0
    return half * out.abs() + (half + 2 * e + n * 2.0**-24) * absolute + tiny + 2.0**-25


def check(got, q, k, v, causal=True):
    out, absolute, _ = exact(q, k, v, causal)
    off = (got.double() - out).abs()
    tolerance = bound(got.dtype, out, absolute, k.shape[0], k.shape[1], v.double().abs().max().item())
    assert (off <= tolerance).all(), ((off / tolerance).max().item(), off.max().item())


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("n,heads,kv_heads,d", [(8192, 2, 1, 64), (8192, 3, 1, 128), (8192, 1, 1, 32), (3000, 2, 2, 96), (500, 4, 2, 64)])
def test_packed_forward(n, heads, kv_heads, d, dtype):
    q, k, v, _ = rows(n, heads, kv_heads, d, dtype)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        o = flash_attention_packed(q, k, v, cu, SCALE)
    for h in range(heads):
        j = h * kv_heads // heads
        check(o[:, h], q[:, h], k[:, j], v[:, j])


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("n,d", [(8192, 64), (8192, 128), (8192, 32), (8192, 256), (1000, 64), (1000, 32)])
def test_dense_forward(n, d, dtype):
    """The same arithmetic, in tiles of 64 keys up to 1024 rows of head dims up to 64."""
    q, k, v, _ = rows(n, 1, 1, d, dtype)
    with torch.no_grad():
        o = flash_attention_v2(*(t.transpose(0, 1)[None] for t in (q, k, v)), SCALE)
    check(o[0, 0], q[:, 0], k[:, 0], v[:, 0])


def test_the_largest_weights_come_late():
    """The running maximum climbs by just less than what asks for a rescale, tile after tile: the weights stay within fp16."""
    n, d = 2048, 64
    q, k, v, do = rows(n, 2, 1, d, FP16, nats=0.0)
    k[:, :, 0] = (torch.arange(n, device="cuda") // 64 * 1.3)[:, None].to(FP16)  # 1.9 in logarithms to 2 for every 64 keys
    v[0] = 1.0
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        o = flash_attention_packed(q, k, v, cu, SCALE)
        dense = flash_attention_v2(*(t.transpose(0, 1)[None].expand(1, 2, n, d) for t in (q, k, v)), SCALE)
    for h in range(2):
        check(o[:, h], q[:, h], k[:, 0], v[:, 0])
        check(dense[0, h], q[:, h], k[:, 0], v[:, 0])


@pytest.mark.parametrize("n,heads,kv_heads,d", [(8192, 2, 1, 64), (4096, 4, 1, 128), (8192, 1, 1, 32)])
def test_packed_value_gradient(n, heads, kv_heads, d):
    """dV of a key is its column of weights times dO: P comes from lse, at most 1, and carries 2^14, so
    below the normal numbers it is off by 2^-39."""
    q, k, v, do = rows(n, heads, kv_heads, d, FP16)
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dv = torch.autograd.grad(flash_attention_packed(*leaves, cu, SCALE), leaves, do)[2]
    q, k, v = (t.detach() for t in leaves)
    for j in range(kv_heads):
        want, group = torch.zeros(n, d, dtype=torch.float64, device="cuda"), heads // kv_heads
        for h in range(j * group, (j + 1) * group):
            want += exact(q[:, h], k[:, j], v[:, j])[2].T @ do[:, h].double()
        e = (d + 8) * 2.0**-24 * 20 + 1e-4
        # (dO is positive, so the sum of magnitudes is the result)
        tolerance = 2.0**-11 * want + (2.0**-11 + 2 * e + group * n * 2.0**-24) * want + 2.0**-39 * group * n * do.max().item() + 2.0**-25
        off = (dv[:, j].double() - want).abs()
        assert (off <= tolerance).all(), ((off / tolerance).max().item(), off.max().item())


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("held,heads,kv_heads,d,page", [([2048] * 400, 3, 1, 64, 16), ([131072], 2, 1, 64, 64), ([8192, 2048] * 40, 4, 2, 128, 16),
                                                        ([4096] * 80, 16, 1, 256, 32), ([1500] * 200, 4, 4, 40, 24), ([900] * 90, 2, 1, 64, 1)])
def test_decode(held, heads, kv_heads, d, page, dtype):
    """Here a warp loses the share of its own keys only, where it holds the one above the others."""
    n = max(held)
    q, k, v, _ = rows(n, heads, kv_heads, d, dtype, queries=len(held))
    cache = Cache([0] * len(held), held, page, kv_heads, d, dtype)
    for s, count in enumerate(held):
        at = cache.places(s, range(count))
        cache.k[at], cache.v[at] = k[:count], v[:count]
    o = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths(held), SCALE)
    for count in set(held):
        s = [i for i, x in enumerate(held) if x == count]
        for h in range(heads):
            j = h * kv_heads // heads
            check(o[s, h], q[s, h], k[:count, j], v[:count, j], causal=False)
