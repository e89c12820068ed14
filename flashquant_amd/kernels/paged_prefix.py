"""Attention for a batch whose sequences begin with the same pages (a system prompt, a document that many ask about, several answers to
one prompt), at 16 or 8 bits; no counterpart in the reference."""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from flashquant_amd.kernels._native import native, require_gpu


def paged_prefix_decode(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    prefix_ids: torch.Tensor,
    prefix_lens: torch.Tensor,
    sm_scale: Optional[float] = None,
    *,
    key_scales: Optional[torch.Tensor] = None,
    value_scales: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    workspace: Optional[torch.Tensor] = None,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``paged_kv_decode`` (or ``paged_kv8_decode``, with ``key_scales`` and ``value_scales``) of a batch in which sequences share their first
    pages: those are read once for all of them, on the matrix cores, and joined to what every sequence has of its own.  The result is
    that of these functions up to rounding.

    ``prefix_ids`` (num_seqs,) int32: the prefix of a sequence, or -1; in any order.  ``prefix_lens`` (num_prefixes,) int32, 1024 at most:
    tokens of a prefix, of which whole pages are shared.  The rows of ``block_table`` of a prefix's sequences begin with the same pages
    (one of them is read for all); ``seq_lens`` counts shared tokens, and a sequence shorter than its prefix is attended to by itself.

    Weights have 16 significant bits, as there, and 8-bit rows count as what they stand for.  ``out`` and ``return_lse`` as in
    ``paged_kv_decode``; ``workspace``: at least ``_C.paged_prefix_decode_workspace_bytes(num_seqs, H_Q, H_KV, head_dim, num_prefixes)``
    bytes, enough for smaller batches too; it holds nothing from one call to the next, and calls that may run at the same time need one
    each.  There is no window.  No gradient is recorded.  A sequence's last bits may depend on the others."""
    require_gpu(q, "q")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[-1])
    result, lse = native().paged_prefix_decode(q, key_cache, value_cache, block_table, seq_lens, prefix_ids, prefix_lens, sm_scale, key_scales,
                                               value_scales, out, return_lse, workspace)
    return (result, lse) if return_lse else result
