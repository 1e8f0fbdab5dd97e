"""Packed prompts, the cache and single tokens together, as a serving program runs them."""

from __future__ import annotations

import pytest
import torch

from flash_attention_triton_b200 import (_lib, append_kv_cache, flash_attention_decode, flash_attention_packed,
                                         flash_attention_v2, rotary_tables)
from packed_helpers import exact_packed
from paged_helpers import Cache, cu_seqlens_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,heads,kv_heads,d,rotary,interleaved,page", [
    (torch.bfloat16, 8, 2, 64, 64, False, 16), (torch.float16, 6, 2, 128, 64, True, 24), (torch.bfloat16, 3, 3, 80, 32, False, 8)])
def test_prompts_then_tokens(dtype, heads, kv_heads, d, rotary, interleaved, page):
    """Every row of the finished texts, whichever operator formed it, against attention over the whole text."""
    prompts, texts = [130, 1, 0, 257, 64], [140, 12, 9, 258, 64]  # a place that is empty at first, a text that is only a prompt
    steps = max(t - p for p, t in zip(prompts, texts))
    g = torch.Generator().manual_seed(7)
    tokens = [[torch.randn(n, h, d, generator=g).to(dtype).cuda() for h in (heads, kv_heads, kv_heads)] for n in texts]
    cache = Cache([0] * 5, texts, page, kv_heads, d, dtype)
    cos, sin = rotary_tables(max(texts), rotary, device="cuda")
    turned = [[torch.zeros_like(t) for t in text] for text in tokens]
    out = [torch.zeros_like(text[0]) for text in tokens]

    fused = torch.cat([torch.cat(text, 1)[:p] for text, p in zip(tokens, prompts)])
    q, k, v = fused.split([heads, kv_heads, kv_heads], 1)
    cu, lengths = cu_seqlens_of(prompts), cache.lengths(prompts)
    q, k = append_kv_cache(k, v, cache.k, cache.v, cache.table, lengths, cu_seqlens=cu, q=q, cos=cos, sin=sin, interleaved=interleaved,
                           return_k=True)
    o = flash_attention_packed(q, k, v, cu)
    row = 0
    for s, p in enumerate(prompts):
        for dst, src in zip((turned[s][0], turned[s][1], turned[s][2], out[s]), (q, k, v, o)):
            dst[:p] = src[row : row + p]
        row += p
    at = list(prompts)
    for _ in range(steps):
        live = [at[s] < texts[s] for s in range(5)]
        # finished texts are empty places of the batch: length 0
        q, k, v = (torch.stack([text[i][min(at[s], texts[s] - 1)] for s, text in enumerate(tokens)]) for i in range(3))
        lengths = cache.lengths([at[s] + 1 if live[s] else 0 for s in range(5)])
        q, k = append_kv_cache(k, v, cache.k, cache.v, cache.table, lengths, q=q, cos=cos, sin=sin, interleaved=interleaved, return_k=True)
        o = flash_attention_decode(q, cache.k, cache.v, cache.table, lengths)
        for s in range(5):
            if live[s]:
                for dst, src in zip((turned[s][0], turned[s][1], turned[s][2], out[s]), (q, k, v, o)):
                    dst[at[s]] = src[s]
                at[s] += 1
            else:
                assert (o[s] == 0).all()
    assert at == texts and _lib.device_status() == 0
    q, k, v = (torch.cat([t[i] for t in turned]) for i in range(3))
    want, tolerance = exact_packed(q, k, v, texts)["o"]
    assert ((torch.cat(out).double() - want).abs() <= tolerance).all()
    for s in range(5):  # what stands in the cache is what the prompts and tokens were turned into
        places = cache.places(s, range(texts[s]))
        assert torch.equal(cache.k[places], turned[s][1]) and torch.equal(cache.v[places], turned[s][2])


def test_packed_texts_and_the_dense_operator_agree():
    """Texts of one length: the same values, forward and backward, whether packed or as a batch."""
    batch, n, heads, d = 3, 200, 4, 64
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(batch * n, heads, d, generator=g).to(torch.float16).cuda() for _ in range(4))
    want = exact_packed(q, k, v, [n] * batch, do)
    results = []
    for packed in (True, False):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        if packed:
            o = flash_attention_packed(*leaves, cu_seqlens_of([n] * batch))
        else:
            o = flash_attention_v2(*(t.view(batch, n, heads, d).transpose(1, 2) for t in leaves)).transpose(1, 2).reshape(batch * n, heads, d)
        results.append([o.detach(), *torch.autograd.grad(o, leaves, do)])
    for name, a, b in zip(want, *results):
        value, tolerance = want[name]
        assert ((a.double() - value).abs() <= tolerance).all() and ((b.double() - value).abs() <= tolerance).all(), name
