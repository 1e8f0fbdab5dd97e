"""append_kv_cache where cu_seqlens are wrong."""

from __future__ import annotations

import pytest
import torch

from flash_attention_triton_b200 import _lib
from paged_helpers import Cache, fa

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_status():
    yield
    assert _lib.device_status() == 0


def call(bounds, tokens, lengths, room=64):
    """(k, rows of the rotated keys, the cache before and after) of a call with these cu_seqlens."""
    g = torch.Generator().manual_seed(1)
    cache = Cache([0] * len(lengths), [room] * len(lengths), 16, 2, 64, BF16)
    k = torch.randn(tokens, 2, 64, generator=g).to(BF16).cuda()
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    before = cache.k.clone()
    _, out = fa.append_kv_cache(k, k, cache.k, cache.v, cache.table, cache.lengths(lengths), cu_seqlens=cu, return_k=True)
    return k, out, before, cache


@pytest.mark.parametrize("behind", [0, 40])  # sequences: up to 32 are looked up at once
@pytest.mark.parametrize("bounds", [[0, 10, 20, 31], [0, 10, 20, 2**31 - 1], [-1, 10, 20, 30], [0, 10, 20, -5]])
def test_sequences_that_leave_the_rows_are_left_out(bounds, behind):
    """Of 30 tokens those of the other sequences are written, and the status word says that some were not."""
    padded = bounds + [min(max(bounds[-1], 0), 30)] * behind
    k, out, before, cache = call(padded, 30, [10, 10, 20] + [0] * behind)
    assert _lib.device_status() == 0x80001
    seen = torch.zeros(30, dtype=torch.bool, device="cuda")
    seen[10:20] = True
    seen[slice(20, 30) if bounds[0] < 0 else slice(0, 10)] = True
    if any(b < a for a, b in zip(padded, padded[1:])):  # they fall as well, and a search among many misses some: nothing else is written
        seen &= (out != 0).flatten(1).any(1)
    assert torch.equal(out[seen], k[seen]) and (out[~seen] == 0).all()
    at = cache.places(1, range(10))
    assert torch.equal(cache.k[at].view(torch.int16), torch.where(seen[10:20, None, None], k[10:20], before[at]).view(torch.int16))
    left = 0 if bounds[0] < 0 else 2
    at = cache.places(left, range([10, 10, 20][left]))
    if padded[left] <= padded[left + 1]:
        assert torch.equal(cache.k[at].view(torch.int16), before[at].view(torch.int16))


@pytest.mark.parametrize("batch", [3, 32, 33, 500])
def test_sequences_that_fall_set_the_status(batch):
    bounds = list(range(0, 2 * batch + 1, 2))
    bounds[-2] = bounds[-3] - 1
    call(bounds, 2 * batch, [2] * batch)
    assert _lib.device_status() == 0x80001


@pytest.mark.parametrize("batch", [1, 32, 33, 500])
def test_sequences_as_they_should_be_set_none(batch):
    k, out, _, _ = call([0, *range(2, 2 * batch + 1, 2)], 2 * batch + 7, [2] * batch)
    assert torch.equal(out[: 2 * batch], k[: 2 * batch]) and (out[2 * batch :] == 0).all()
