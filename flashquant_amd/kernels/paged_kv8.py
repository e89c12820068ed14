"""A paged cache at 8 bits: the rotary store into it, tokens read back, and attention over it.

A row, the ``D`` values of a token and KV head, is kept as e4m3 codes and one power of two: ``key_cache`` and ``value_cache``
(num_blocks, block_size, H_KV, D) ``torch.float8_e4m3fn``, ``key_scales`` and ``value_scales`` (num_blocks, H_KV, block_size)
``torch.float8_e8m0fnu``; a value is its code times the scale of its row.  Half the memory and traffic of 16-bit pages, on the same
block tables and slots (no counterpart in the reference, which packs to 4 bits or leaves layers to other backends).  The caches may be
strided (halves of one tensor, heads before tokens) at multiples of 16 bytes, the scales of 8."""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from flashquant_amd.kernels._native import native, require_gpu


def rotary_paged_store8(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    slot_mapping: torch.Tensor,
    inv_freq: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    *,
    interleaved: bool = False,
    scale: float = 1.0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``rotary_paged_store`` into an 8-bit cache: rotary positions on ``q`` (tokens, H_Q, D) and ``k`` (tokens, H_KV, D), float16 or
    bfloat16, the rotated keys and ``v`` quantised into flat slots ``slot_mapping``, in one launch; returns the rotated queries
    (``out``: new memory, or ``q`` itself).  D 64, 128 or 256.

    A row's power of two is the least that brings its largest finite magnitude to 448, the largest code, or below (from 2**-118 to
    2**120); codes are rounded to nearest even from the float32 values, so they are off by 2**-4 of a value at most, or by 2**-17 of the
    row's largest where that is more.  Infinite values become NaN.  Tokens beyond ``len(slot_mapping)`` and slots outside the cache are
    not stored; two tokens of one slot race.  Keys, values, scales and the other operands share no memory.  No gradient is recorded."""
    require_gpu(q, "q")
    return native().rotary_paged_store8(q, k, v, positions, slot_mapping, inv_freq, key_cache, value_cache, key_scales, value_scales,
                                        interleaved, scale, out)


def paged_kv8_read(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    num_tokens: int,
    *,
    starts: Optional[torch.Tensor] = None,
    dtype: torch.dtype = torch.bfloat16,
    out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens of an 8-bit cache as rows of ``dtype`` (float16 or bfloat16): ``(keys, values)`` of shape (num_tokens, H_KV, D).  Sequence s
    (``block_table`` (num_seqs, max_blocks) int32) gives its tokens from ``starts[s]`` on (int32; 0 without) to rows ``cu_seqlens[s]`` ..
    ``cu_seqlens[s + 1]`` (int32, not decreasing, num_seqs + 1 of them); ``num_tokens`` is the room for all of them.

    Values are exact in bfloat16 and rounded in float16; what is beyond the type's largest number comes back as that.  Rows of tokens on
    pages outside the cache (an entry of -1), or beyond the table, are 0.  Rows behind the last sequence are 0; in ``out`` = (keys,
    values), contiguous, they are left as they were.  No gradient is recorded."""
    require_gpu(key_cache, "key_cache")
    return native().paged_kv8_read(key_cache, value_cache, key_scales, value_scales, block_table, cu_seqlens, num_tokens, starts, dtype, out)


def paged_kv8_decode(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    sm_scale: Optional[float] = None,
    *,
    window: int = 0,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    workspace: Optional[torch.Tensor] = None,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``paged_kv_decode`` over an 8-bit cache: single-token attention of ``q`` (num_seqs, H_Q, D), float16 or bfloat16, through
    ``block_table`` (num_seqs, max_blocks) and ``seq_lens`` (num_seqs,), int32, the new token counted.  Keys and values are what the
    cache stands for, without another rounding.

    ``window``, ``out``, ``return_lse`` and ``workspace`` (at least ``_C.paged_kv8_decode_workspace_bytes(...)`` bytes) as there; so are
    tokens on pages outside the cache, rows that see nothing and seen values that are NaN."""
    require_gpu(q, "q")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[-1])
    result, lse = native().paged_kv8_decode(q, key_cache, value_cache, key_scales, value_scales, block_table, seq_lens, sm_scale, window, out,
                                            return_lse, workspace)
    return (result, lse) if return_lse else result
