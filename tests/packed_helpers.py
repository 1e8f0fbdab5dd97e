"""Attention over packed sequences and its gradients by the formulas in 64 bits, with the bounds of their errors."""

from __future__ import annotations

import math

import torch


def exact_packed(q, k, v, lengths, do=None, scale=None):
    """Per sequence and head, on the tensors' device: ``{name: (value, tolerance)}`` for o and, with ``do``, dq, dk and dv.

    The tolerances bound the kernels' roundings element by element, with half = half a step of the 16-bit type:

    * a score: d additions in 32 bits of at most sum |q k| scale, the exponent's own rounding, the polynomial that stands in
      for some exponentials (7.5e-5); as the relative error ``e`` of a weight, twice where it is divided by their sum;
    * a weight P rounded to 16 bits (half), or below fp16's normal numbers off by 2^-25 where the row's largest is at least 1;
    * o: sum P |v| (half + 2 e), then its own rounding;
    * dV: sum P |dO| (half + e); P comes from lse, so no sum of weights divides it a second time;
    * delta: O is rounded and carries the error of P: sum |dO| (tolerance of o);
    * dS = P (dP - delta) scale, rounded: |dS| (half + e) + P scale (error of delta and dP); fp16: 2^-24 max|dO| below normal;
    * dK, dQ: that, times |q| or |k|, summed; then their own rounding, once;
    * sums of n terms in 32 bits: n 2^-24 of the sum of magnitudes.
    """
    half = torch.finfo(q.dtype).eps / 2
    tiny = 2.0**-25 if q.dtype == torch.float16 else 0.0
    heads, kv_heads, d = q.shape[1], k.shape[1], q.shape[2]
    scale = scale or 1 / math.sqrt(d)
    group = heads // kv_heads
    Q, K, V = (t.double() for t in (q, k, v))
    names = ("o",) if do is None else ("o", "dq", "dk", "dv")
    shapes = {"o": Q, "dq": Q, "dk": K, "dv": K}
    value, error = ({n: torch.zeros_like(shapes[n]) for n in names} for _ in range(2))
    row = 0
    top = do.double().abs().max().item() if do is not None and do.numel() else 0.0
    for n in lengths:
        if n == 0:
            continue
        rows = slice(row, row + n)
        row += n
        seen = torch.ones(n, n, device=q.device, dtype=torch.bool).tril()
        count = n * 2.0**-24
        for h in range(heads):
            j = h // group
            x, y, z = Q[rows, h], K[rows, j], V[rows, j]
            s = (x @ y.T) * scale
            e = (d + 8) * 2.0**-24 * ((x.abs() @ y.abs().T) * scale * seen).max().item() + 1e-4
            p = torch.softmax(s.masked_fill(~seen, -math.inf), 1)
            o = p @ z
            a = p @ z.abs()
            oe = (half + 2 * e + count) * a + tiny * (seen.double() @ z.abs())
            value["o"][rows, h], error["o"][rows, h] = o, half * o.abs() + oe
            if do is None:
                continue
            g = do[rows, h].double()
            value["dv"][rows, j] += p.T @ g
            error["dv"][rows, j] += (half + e + group * count) * (p.T @ g.abs()) + tiny * (seen.double().T @ g.abs())
            dp = g @ z.T
            delta = (g * o).sum(1, keepdim=True)
            de = (g.abs() * (half * o.abs() + oe)).sum(1, keepdim=True) + d * 2.0**-23 * (g.abs() @ z.abs().T)
            ds = p * (dp - delta) * scale
            dse = ds.abs() * (half + e) + p * scale * de + seen * tiny * 2 * top
            value["dq"][rows, h] = ds @ y
            error["dq"][rows, h] = dse @ y.abs() + count * (ds.abs() @ y.abs())
            value["dk"][rows, j] += ds.T @ x
            error["dk"][rows, j] += dse.T @ x.abs() + group * count * (ds.abs().T @ x.abs())
    for n in names[1:]:
        error[n] += half * value[n].abs()
    floor = 2.0**-24  # half a step of fp16's smallest numbers
    return {n: (value[n], error[n] + floor) for n in names}
