"""A prompt and a decoding step of a serving program, each captured once and replayed with other lengths."""

from __future__ import annotations

import pytest
import torch

from flash_attention_triton_b200 import _lib, append_kv_cache, flash_attention_decode, flash_attention_packed, rotary_tables
from packed_helpers import exact_packed
from paged_helpers import Cache, cu_seqlens_of, decode_tolerance, exact_decode

pytestmark = pytest.mark.gpu
HEADS, KV_HEADS, D, PAGE, ROOM, PLACES = 8, 2, 64, 16, 200, 4


@pytest.fixture(autouse=True)
def _no_status():
    yield
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_captured_prompts_and_steps(dtype):
    """Four places of a batch; the prompts of a replay, in a buffer of fixed size, leave some of them empty."""
    g = torch.Generator(device="cuda").manual_seed(3)
    cos, sin = rotary_tables(ROOM, D, device="cuda")
    cache = Cache([0] * PLACES, [ROOM] * PLACES, PAGE, KV_HEADS, D, dtype)
    rows = 300
    fused = torch.zeros(rows, HEADS + 2 * KV_HEADS, D, dtype=dtype, device="cuda")
    step = torch.zeros(PLACES, HEADS + 2 * KV_HEADS, D, dtype=dtype, device="cuda")
    cu, lengths = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (PLACES + 1, PLACES))

    def prompt():
        q, k, v = fused.split([HEADS, KV_HEADS, KV_HEADS], 1)
        q, k = append_kv_cache(k, v, cache.k, cache.v, cache.table, lengths, cu_seqlens=cu, q=q, cos=cos, sin=sin, return_k=True)
        return q, k, flash_attention_packed(q, k, v, cu)

    def token():
        lengths.add_(lengths > 0)
        q, k, v = step.split([HEADS, KV_HEADS, KV_HEADS], 1)
        q, _ = append_kv_cache(k, v, cache.k, cache.v, cache.table, lengths, q=q, cos=cos, sin=sin)
        return q, flash_attention_decode(q, cache.k, cache.v, cache.table, lengths)

    graphs, out = [], []
    with torch.no_grad():
        for call in (prompt, token):
            call()  # nothing is in the batch yet
            torch.cuda.synchronize()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                out.append(call())
    (pq, pk, po), (tq, to) = out
    for prompts in ([130, 1, 0, 64], [0, 0, 7, 0], [100, 100, 50, 50], [0, 0, 0, 0]):
        fused.normal_(generator=g)
        cu.copy_(cu_seqlens_of(prompts))
        lengths.copy_(torch.tensor(prompts, dtype=torch.int32))
        graphs[0].replay()
        want, tolerance = exact_packed(pq[: sum(prompts)], pk[: sum(prompts)], fused[: sum(prompts), HEADS + KV_HEADS :], prompts)["o"]
        assert ((po[: sum(prompts)].double() - want).abs() <= tolerance).all() and (po[sum(prompts) :] == 0).all()
        for more in (1, 2, 3):
            step.normal_(generator=g)
            graphs[1].replay()
            held = [n + more if n else 0 for n in prompts]
            assert lengths.tolist() == held
            keys, values = ([t[cache.places(s, range(n))] if n else t[0, :0] for s, n in enumerate(held)] for t in (cache.k, cache.v))
            for s, n in enumerate(held):
                if n:
                    assert torch.equal(values[s][-1], step[s, HEADS + KV_HEADS :])
            want, absolute, largest = exact_decode(tq, keys, values)
            off = (to.double() - want).abs()
            assert (off <= decode_tolerance(dtype, want, absolute, largest, D, max(held))).all()
