"""A paged cache with its contents by position, and the operators' formulas in 64 bits, for the tests."""

from __future__ import annotations

import math

import torch

import flash_attention_triton_b200 as fa


def cu_seqlens_of(lengths, device="cuda"):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=device)


class Cache:
    """Pages handed out in no order; every slot that no sequence's ``held`` positions use is NaN."""

    def __init__(self, held, room, page, kv_heads, d, dtype, seed=0, layout="slots", spare=3, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.page, self.held, self.room = page, list(held), list(room)
        used = [-(-max(n, 0) // page) for n in room]
        width = max(1, *used)
        pages = sum(used) + spare
        order = torch.randperm(pages, generator=g).tolist()
        table = torch.full((len(used), width), pages + 7, dtype=torch.int32)  # what is not handed out is no page
        for s, n in enumerate(used):
            for i in range(n):
                table[s, i] = order.pop()
        self.table = table.cuda()
        shape = (pages, page, kv_heads, d) if layout == "slots" else (pages, kv_heads, page, d)
        self.k, self.v = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2))
        if layout == "heads":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.keys = [(spread * torch.randn(max(n, 0), kv_heads, d, generator=g)).to(dtype).cuda() for n in held]
        self.values = [torch.randn(max(n, 0), kv_heads, d, generator=g).to(dtype).cuda() for n in held]
        for s in range(len(used)):
            if held[s] > 0:
                at = self.places(s, range(held[s]))
                self.k[at], self.v[at] = self.keys[s], self.values[s]

    def places(self, s, positions):
        p = torch.tensor(list(positions), device="cuda")
        return self.table[s, p // self.page].long(), p % self.page

    def lengths(self, values=None):
        return torch.tensor(self.held if values is None else values, dtype=torch.int32, device="cuda")


def exact_decode(q, keys, values, scale=None):
    """(output, the weighted sum of |values|, the largest sum of |q k| scale) in 64 bits, sequence by sequence."""
    out, absolute, largest = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64), 0.0
    batch, heads, d = q.shape
    scale = scale or 1 / math.sqrt(d)
    for s in range(batch):
        k, v = keys[s].double(), values[s].double()
        if k.shape[0] == 0:
            continue
        group = heads // k.shape[1]
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        x = q[s].double()
        p = torch.softmax(torch.einsum("hd,nhd->hn", x, k) * scale, 1)
        out[s] = torch.einsum("hn,nhd->hd", p, v)
        absolute[s] = torch.einsum("hn,nhd->hd", p, v.abs())
        largest = max(largest, (torch.einsum("hd,nhd->hn", x.abs(), k.abs()).max() * scale).item())
    return out, absolute, largest


def decode_tolerance(dtype, out, absolute, largest, d, longest):
    """Element by element: the output's rounding; a weight rounded to 16 bits (fp16: half a step, 2^-11; bf16: a sum of two
    terms, the first within 2^-8 of p (1 - 2^-8), so the second is at most p (1 - (1 - 2^-8)^2) < 2^-7 p and its half
    step, 2^-8 of it, at most 2^-15 p); a score's d additions in 32 bits, which the exponential turns into
    a relative error of numerator and denominator; the longest chain of additions of a running sum (one for each
    64 keys of a warp, those of a product and of the joins) with its rescales."""
    half = torch.finfo(dtype).eps / 2
    weight = half if dtype == torch.float16 else 2.0**-15
    score = (d + 8) * 2.0**-24 * (largest + 1)
    chain = (longest / 64 + 200) * 2 * 2.0**-24
    return half * out.abs() + (weight + 2 * score + chain) * absolute + 2.0**-24


def rotated(x, cos, sin, positions, interleaved):
    """x [tokens, heads, d] turned by the tables' rows, in 64 bits."""
    x = x.double().clone()
    if cos is None:
        return x
    half = cos.shape[1]
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    at = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., at[0]].clone(), x[..., at[1]].clone()
    x[..., at[0]], x[..., at[1]] = a * c - b * s, b * c + a * s
    return x


def rotation_tolerance(dtype, want, source):
    """The rounding of the result, and of two products and their sum in 32 bits, each at most |x1| + |x2|; the last
    term is half a step of fp16's smallest numbers."""
    return torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0**-10) + 3 * 2.0**-24 * 2 * source.double().abs().max() + 2.0**-25


__all__ = ["Cache", "cu_seqlens_of", "decode_tolerance", "exact_decode", "fa", "rotated", "rotation_tolerance"]
