"""The tables of a paged cache made on the GPU, and attention over 16-bit pages (the layers that stay uncompressed beside packed
ones; no counterpart in the reference, whose tables and 16-bit attention are vLLM's)."""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from flashquant_amd.kernels._native import native, require_gpu


class PagedSchedule(NamedTuple):
    """What ``paged_schedule`` makes of a step: int64 ``slot_mapping`` and ``positions`` (num_tokens,), int32 ``seq_lens``
    (num_reqs,), ``cu_seqlens`` (num_reqs + 1,) and ``free_end`` (1,)."""
    slot_mapping: torch.Tensor
    positions: torch.Tensor
    seq_lens: torch.Tensor
    cu_seqlens: torch.Tensor
    free_end: torch.Tensor


def paged_schedule(
    context_lens: torch.Tensor,
    query_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_blocks: torch.Tensor,
    block_size: int,
    num_tokens: int,
    *,
    free_start: Optional[torch.Tensor] = None,
    out: Optional[PagedSchedule] = None,
    capped: bool = False,
) -> PagedSchedule:
    """Pages, slots and positions of a step's new tokens, in one launch and without a look at the lengths from the host.

    Request r has ``context_lens[r]`` tokens on the pages of ``block_table[r]`` and brings ``query_lens[r]`` new ones (int32).  Pages
    that its new tokens begin are taken from ``free_blocks`` (int32), from index ``free_start`` (an int32 tensor; 0 without) on, in
    the order of requests and tokens, and written into ``block_table`` (num_reqs, max_blocks) int32, in place.  ``free_end`` is the
    index of the first page left: the next step's ``free_start``.  Where pages run out an entry is -1, the slots of its tokens are
    -1, and ``free_end`` exceeds ``len(free_blocks)``.

    ``num_tokens``: room for the new tokens of all requests (a graph's padded batch); what is behind the last one gets slot -1 and
    position 0.  Tokens that there is no room for get neither slot nor page, but count in ``seq_lens``, ``cu_seqlens`` and ``free_end``;
    with ``capped`` they count nowhere, as if the requests had not brought them.  ``out``: what an earlier call of these sizes returned, written again; its ``free_end`` must not be this call's
    ``free_start``."""
    require_gpu(context_lens, "context_lens")
    return PagedSchedule(*native().paged_schedule(context_lens, query_lens, block_table, free_blocks, block_size, num_tokens,
                                                  free_start, out, capped))


def paged_kv_decode(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    sm_scale: Optional[float] = None,
    *,
    window: int = 0,
    out: Optional[torch.Tensor] = None,
    return_lse: bool = False,
    workspace: Optional[torch.Tensor] = None,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Single-token attention of ``q`` (num_seqs, H_Q, D) over ``key_cache`` / ``value_cache`` (num_blocks, block_size, H_KV, D), all
    float16 or bfloat16, through ``block_table`` (num_seqs, max_blocks) and ``seq_lens`` (num_seqs,), int32, the new token counted.

    ``window``: only so many of a sequence's last tokens are seen (0: all).  Tokens on pages outside the cache (an entry of -1) are
    not seen; a row that sees none is zero; a seen value that is infinite or NaN makes its coordinate infinite or NaN.  ``return_lse``
    adds the float32 logarithm of the softmax's denominator (num_seqs, H_Q), -inf for rows that see nothing.  The caches may be
    strided (halves of one tensor, heads before tokens).  ``workspace``: uint8, at least ``_C.paged_kv_decode_workspace_bytes(...)``
    bytes (of the largest call: smaller batches and narrower tables need no more), for callers that allocate nothing; it holds
    nothing from one call to the next, and calls that may run at the same time (on two streams, in two graphs) need one each.
    ``out``: contiguous, apart from the other operands.  No gradient is recorded.  A sequence's last bits may depend on the lengths of
    the others and on the table's width, which decide where it is divided."""
    require_gpu(q, "q")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(q.shape[-1])
    result, lse = native().paged_kv_decode(q, key_cache, value_cache, block_table, seq_lens, sm_scale, window, out, return_lse, workspace)
    return (result, lse) if return_lse else result
