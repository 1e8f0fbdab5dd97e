"""flash_attention_decode at the edges of its arguments."""

from __future__ import annotations

import math

import pytest
import torch

from flash_attention_triton_b200 import _lib
from paged_helpers import Cache, decode_tolerance, exact_decode, fa

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _no_status():
    yield
    assert _lib.device_status() == 0


def normal(*shape, dtype, seed=1):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("batch,late", [(1, 0), (3, 1), (700, 699)])
def test_a_length_beyond_the_block_table_sets_the_status(batch, late, page):
    """The keys that have a place count; the status word says that there are others."""
    held = [5 * page] * batch
    cache = Cache(held, held, page, 2, 64, BF16)
    q = normal(batch, 4, 64, dtype=BF16)
    clean = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    assert _lib.device_status() == 0
    for more in (1, 1000, 2**31 - 2 - 5 * page):
        lengths = cache.lengths()
        lengths[late] += more
        out = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, lengths)
        assert _lib.device_status() == 0x40002
        assert torch.equal(out, clean)


def test_a_length_beyond_the_block_table_raises_where_asked(monkeypatch):
    cache = Cache([64], [64], 16, 2, 64, BF16)
    q = normal(1, 4, 64, dtype=BF16)
    monkeypatch.setenv("FA2_B200_CHECK_STATUS", "1")
    fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths([64]))
    with pytest.raises(_lib.Fa2Error, match="outside the cache"):
        fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths([65]))


def test_the_largest_length_stands_for_the_whole_table():
    cache = Cache([80, 48], [80, 80], 16, 2, 64, BF16)
    q = normal(2, 4, 64, dtype=BF16)
    want = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths())
    assert torch.equal(fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths([2**31 - 1, 48])), want)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("where", [200, 500, 5000, 9999, 19000])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("peak", ["front", "back"])
def test_a_value_of_vanishing_weight_is_not_lost(peak, value, where, heads, kv_heads, d):
    """Some keys are 200 nats above the others: 0 x NaN and 0 x infinity are NaN in whichever of the parts that are joined they stand."""
    n, scale = 20000, 8.0 / d
    cache = Cache([n], [n], 16, kv_heads, d, BF16)
    q = torch.ones(1, heads, d, dtype=BF16, device="cuda")
    k = normal(n, kv_heads, d, dtype=torch.float32) * 0.01
    k[slice(0, 100) if peak == "front" else slice(n - 100, n)] = 25.0
    cache.k[cache.places(0, range(n))] = k.to(BF16)
    assert fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths(), scale).isfinite().all()
    cache.v[cache.places(0, [where])] = value
    out = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths(), scale)
    assert not out.isfinite().any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale", [1e-30, 1e-38, 1e-40])
def test_tiny_scales(scale, dtype):
    """All weights are alike, normal number or not."""
    cache = Cache([300, 1, 7000], [300, 1, 7000], 16, 2, 64, dtype)
    q = normal(3, 4, 64, dtype=dtype)
    out = fa.flash_attention_decode(q, cache.k, cache.v, cache.table, cache.lengths(), scale)
    want, absolute, largest = exact_decode(q, cache.keys, cache.values, scale)
    assert ((out.double() - want).abs() <= decode_tolerance(dtype, want, absolute, largest, 64, 7000)).all()
