"""Causal attention over packed sequences of different lengths, with fewer key and value heads than query heads."""

from __future__ import annotations

import torch

from . import _lib


def flash_attention_packed(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    softmax_scale: float | None = None,
) -> torch.Tensor:
    """Causal attention within each of the sequences that lie one behind the other in ``q``, ``k`` and ``v``.

    Args:
        q: ``[tokens, heads, headdim]``, fp16 or bf16; head dims are multiples of 8 up to 128.
        k, v: ``[tokens, kv_heads, headdim]``; query head ``h`` goes with key head ``h * kv_heads // heads``.  Slices of one
            fused projection are read in place.
        cu_seqlens: int32 ``[batch + 1]`` on the device: rows ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1`` are sequence ``s``.
            It is read by the kernels, so a captured call follows what is written into it between replays.
        softmax_scale: scaling factor (default and 0.0: ``1/sqrt(headdim)``).

    Returns:
        The output, dense, of the shape and type of ``q``.  Rows behind the last sequence (a buffer of fixed size) are zeros,
        and so are their gradients, whatever these rows hold.

    Differentiable once in ``q``, ``k`` and ``v``; the gradients of a key head are summed over its query heads in 32 bits, in
    a fixed order, so the same call gives the same bits.  ``cu_seqlens`` that fall or leave the rows give zeros and set the
    device's status word (``FA2_B200_CHECK_STATUS=1`` raises).  The reference has no counterpart.
    """
    return _lib.host().packed(q, k, v, cu_seqlens, softmax_scale)
