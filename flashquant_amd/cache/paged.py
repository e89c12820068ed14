"""Paged storage driven from the GPU: one table of pages for all layers, and layers that keep their keys and values at 16 bits or
packed (TQ4) on those pages, with rotary positions applied on the way in.

The reference has the packed pages (src/flashquant/vllm/impl.py:132-138, 220-263) and leaves tables, positions and 16-bit layers to
vLLM; here a decode step is ``PageTable.schedule`` once and ``step`` per layer, without a look at lengths or pages from the host, so
that it can be captured in a graph."""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from flashquant_amd.kernels import (paged_kv_decode, paged_schedule, rotary_embedding, rotary_paged_store)
from flashquant_amd.kernels._native import native
from flashquant_amd.vllm.impl import TQ4AttentionKernels
from flashquant_amd.vllm.spec import get_kv_cache_shape


class PagedStep(NamedTuple):
    """A step's tokens: ``slot_mapping`` and ``positions`` (num_tokens,) int64, sequence by sequence; ``seq_lens`` (max_seqs,) and
    ``cu_seqlens`` (max_seqs + 1,) int32; ``block_table`` (max_seqs, max_blocks) int32; ``pages_taken`` (1,) int32: above the number
    of pages where there were too few.  Tokens without a page have slot -1, are not stored, and what their sequences' packed rows
    give is without meaning; a caller that can run out reads ``pages_taken``.

    The tokens are packed: sequences that bring none have none, wherever they are in the table, and what is behind the last token is
    padding.  ``token_table`` (num_tokens, max_blocks) and ``token_lens`` (num_tokens,) int32 hold, token by token, the pages of its
    sequence and how many tokens it sees (itself the last; padding: none); None where ``num_tokens`` is above ``max_seqs``."""
    slot_mapping: torch.Tensor
    positions: torch.Tensor
    seq_lens: torch.Tensor
    cu_seqlens: torch.Tensor
    block_table: torch.Tensor
    pages_taken: torch.Tensor
    token_table: Optional[torch.Tensor] = None
    token_lens: Optional[torch.Tensor] = None


def _rows(q: torch.Tensor, step: PagedStep) -> Tuple[torch.Tensor, torch.Tensor]:
    """Pages and lengths for single-token attention of ``q``, row by row (a step made by hand may have them by sequence)."""
    table, lens = (step.block_table, step.seq_lens) if step.token_table is None else (step.token_table, step.token_lens)
    if q.shape[0] != table.shape[0]:
        raise ValueError(f"a step attends one token of every sequence at most: {q.shape[0]} tokens, {table.shape[0]} rows of pages")
    return table, lens


class PageTable:
    """Block tables, lengths and the list of free pages of ``max_seqs`` sequences, all on the GPU."""

    def __init__(self, num_blocks: int, block_size: int, max_seqs: int, max_blocks_per_seq: int,
                 device: Optional[torch.device] = None) -> None:
        if device is None:
            device = torch.device("cuda")
        self.num_blocks = num_blocks
        self.block_size = block_size
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_seqs, max_blocks_per_seq), -1, **i32)
        self.context_lens = torch.zeros(max_seqs, **i32)
        # free pages from free_start on; what lies before has been taken.  The last element takes what is not a page.
        self._pages = torch.arange(num_blocks + 1, **i32)
        self.free_blocks = self._pages[:num_blocks]
        self.free_start = torch.zeros(1, **i32)

    def schedule(self, query_lens: torch.Tensor, num_tokens: int) -> PagedStep:
        """Gives ``query_lens[s]`` (int32) new tokens of sequence s their pages, slots and positions and counts them into the
        lengths; ``num_tokens`` is the room for all of them.  Tokens that there is no room for are left out: they take no page and
        count in no length."""
        s = paged_schedule(self.context_lens, query_lens, self.block_table, self.free_blocks, self.block_size, num_tokens,
                           free_start=self.free_start, capped=True)
        token_table, token_lens = native().paged_advance(s, self.context_lens, self.free_start, self.block_table, self.num_blocks,
                                                         self.block_size, num_tokens <= self.block_table.shape[0])
        return PagedStep(s.slot_mapping, s.positions, s.seq_lens, s.cu_seqlens, self.block_table, s.free_end, token_table, token_lens)

    def release(self, seq: int) -> None:
        """Ends sequence ``seq``: its pages are free again (the next to be taken) and its length is 0."""
        row = self.block_table[seq]
        held = (self.context_lens[seq] + self.block_size - 1) // self.block_size
        mine = (row >= 0) & (torch.arange(row.shape[0], device=row.device) < held)
        count = mine.sum(dtype=torch.int32)
        place = torch.where(mine, self.free_start - count + torch.cumsum(mine, 0) - 1, self.num_blocks)
        self._pages[place] = row
        self.free_start -= count
        self.block_table[seq] = -1
        self.context_lens[seq] = 0


class PagedKVLayer:
    """Keys and values of one attention layer at 16 bits, (num_blocks, block_size, heads, head_dim) each."""

    def __init__(self, table: PageTable, heads: int, head_dim: int, inv_freq: torch.Tensor, rotary_scale: float = 1.0, *,
                 interleaved: bool = False, window: int = 0, sm_scale: Optional[float] = None, dtype: torch.dtype = torch.bfloat16) -> None:
        device = table.block_table.device
        self.table = table
        self.keys, self.values = torch.zeros(2, table.num_blocks, table.block_size, heads, head_dim, dtype=dtype, device=device)
        self.inv_freq, self.rotary_scale, self.interleaved = inv_freq.to(device), rotary_scale, interleaved
        self.window = window
        self.sm_scale = 1.0 / math.sqrt(head_dim) if sm_scale is None else sm_scale

    def store(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep) -> torch.Tensor:
        """The step's keys and values into their slots, rotated; returns the rotated queries (num_tokens, H_Q, head_dim)."""
        return rotary_paged_store(q, k, v, step.positions, step.slot_mapping, self.inv_freq, self.keys, self.values,
                                  interleaved=self.interleaved, scale=self.rotary_scale)

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep) -> torch.Tensor:
        """``store`` of a step with at most one token of every sequence, then each one's attention over its sequence: (num_tokens, H_Q,
        head_dim); rows behind the last token are 0."""
        rows = _rows(q, step)
        return paged_kv_decode(self.store(q, k, v, step), self.keys, self.values, *rows, self.sm_scale, window=self.window)


class PagedTQ4Layer:
    """The same with packed rows, (num_blocks, block_size, heads * (head_dim + 8)) bytes, on the kernels of the serving backend."""

    def __init__(self, table: PageTable, heads: int, head_dim: int, inv_freq: torch.Tensor, rotary_scale: float = 1.0, *,
                 interleaved: bool = False, sm_scale: Optional[float] = None) -> None:
        device = table.block_table.device
        self.table = table
        self.cache = torch.zeros(get_kv_cache_shape(table.num_blocks, table.block_size, heads, head_dim), dtype=torch.uint8, device=device)
        self.inv_freq, self.rotary_scale, self.interleaved = inv_freq.to(device), rotary_scale, interleaved
        self.kernels = TQ4AttentionKernels(heads, head_dim, 1.0 / math.sqrt(head_dim) if sm_scale is None else sm_scale, device)

    def _rotated(self, q: torch.Tensor, k: torch.Tensor, step: PagedStep):
        return rotary_embedding(q, k, step.positions, self.inv_freq, interleaved=self.interleaved, scale=self.rotary_scale)

    def store(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep) -> torch.Tensor:
        """The step's keys (rotated) and values into their rows; returns the rotated queries."""
        q, k = self._rotated(q, k, step)
        self.kernels.compress_and_store(k, v, self.cache, step.slot_mapping)
        return q

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep) -> torch.Tensor:
        """At most one token of every sequence stored and attended over its sequence: (num_tokens, H_Q, head_dim); rows behind the
        last token are 0."""
        rows = _rows(q, step)
        q, k = self._rotated(q, k, step)
        return self.kernels.decode_step(q, k, v, self.cache, step.slot_mapping, *rows)

    def prefill(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep, max_query_len: int) -> torch.Tensor:
        """Several tokens of the sequences stored and attended, causal: (num_tokens, H_Q, head_dim).  ``max_query_len``: the most
        tokens of a sequence, those without room among them or not; rows behind the last token are not written."""
        return self.kernels.prefill(self.store(q, k, v, step), step.cu_seqlens, min(max_query_len, q.shape[0]), self.cache, step.block_table,
                                    step.seq_lens)
