"""The key-value cache of a serving program: new tokens into its pages, and attention of one new token over them.

A cache is a pair of fp16 or bf16 tensors ``[pages, page_size, kv_heads, headdim]`` (any strides with a contiguous last
dimension, so a ``[pages, kv_heads, page_size, headdim]`` buffer seen through ``transpose(1, 2)`` serves as well).
Position ``p`` of sequence ``s`` stands in page ``block_table[s, p // page_size]``, slot ``p % page_size``.  ``lengths``
says how many positions of each sequence the cache holds, those of the step's new tokens included, so a decoding step
counts it up once and then hands the same tensor to :func:`append_kv_cache` and :func:`flash_attention_decode` in every
layer.  A length of 0 marks an empty place of the batch.

The kernels read ``block_table``, ``lengths`` and ``cu_seqlens`` on the device, so a captured step follows what is written
into them between replays.  A page number outside the cache, or a position beyond the block table or the rotation
tables, is left out and sets the device's status word, which ``FA2_B200_CHECK_STATUS=1`` turns into an ``Fa2Error`` after
the call.  The reference has no counterpart of these operators.
"""

from __future__ import annotations

import torch

from . import _lib


def rotary_tables(
    positions: int, rotary: int, base: float = 10000.0, device: torch.device | str | None = None
) -> tuple[torch.Tensor, torch.Tensor]:
    """Cosines and sines of ``position * base ** (-2 j / rotary)``, fp32 ``[positions, rotary // 2]`` each.

    Formed in fp64: an fp32 angle of position 100 000 is off by up to 0.004 radians.
    """
    if rotary <= 0 or rotary % 16:
        raise ValueError(f"the rotated columns must be a multiple of 16, not {rotary}")
    j = torch.arange(rotary // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2.0 * j / rotary)
    return angle.cos().float(), angle.sin().float()


def append_kv_cache(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    cu_seqlens: torch.Tensor | None = None,
    q: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    interleaved: bool = False,
    return_k: bool = False,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """Write the keys and values of new tokens into the cache, rotated by their positions on the way.

    Args:
        k, v: ``[tokens, kv_heads, headdim]``, the type of the cache; head dims are multiples of 8 up to 256.
        k_cache, v_cache: the cache, written in place.
        block_table: int32 ``[batch, width]``.
        lengths: int32 ``[batch]``, positions in the cache once this call's tokens are in it.
        cu_seqlens: int32 ``[batch + 1]``: rows ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1`` are the last positions of
            sequence ``s``.  ``None``: one token for each sequence.  Tokens of a sequence that leaves the rows are left out, and the
            status word is set; so it is where the entries fall, and which tokens are written then is not said.
        q: ``[tokens, heads, headdim]``, rotated by the same positions into a new tensor.
        cos, sin: fp32 ``[positions, rotated columns / 2]`` (:func:`rotary_tables`): the first columns of every key and
            query are rotated, the others kept.  ``None``: nothing is rotated.
        interleaved: rotate the pairs of columns ``(2 j, 2 j + 1)`` instead of ``(j, j + rotated / 2)``.
        return_k: also return the keys as they were written, for the attention of a whole prompt
            (:func:`flash_attention_packed`).

    Returns:
        ``(q, k)`` rotated, dense; ``None`` for what was not asked for.  Rows of tokens with a negative position and rows
        behind the last sequence are zeros there and are not written to the cache.

    Two tokens of a call must not have the same slot.  There is no gradient.
    """
    return _lib.host().kv_append(
        k, v, k_cache, v_cache, block_table, lengths, cu_seqlens, q, cos, sin, interleaved, return_k)


def flash_attention_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    softmax_scale: float | None = None,
) -> torch.Tensor:
    """Attention of one new token a sequence over the first ``lengths[s]`` positions of its cache.

    Args:
        q: ``[batch, heads, headdim]``; query head ``h`` reads key head ``h * kv_heads // heads``.
        k_cache, v_cache: the cache, of the type of ``q``; head dims are multiples of 8 up to 256.
        block_table: int32 ``[batch, width]``.
        lengths: int32 ``[batch]``; the output of a sequence without positions is zero.  ``2**31 - 1`` stands for as many as the
            block table has room for; any other length beyond that counts as that many and sets the status word.
        softmax_scale: scaling factor (default and 0.0: ``1/sqrt(headdim)``).

    Returns:
        The output, dense ``[batch, heads, headdim]``; the same call gives the same bits.  There is no gradient.
    """
    return _lib.host().decode(q, k_cache, v_cache, block_table, lengths, softmax_scale)
