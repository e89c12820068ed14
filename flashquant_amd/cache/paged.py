"""Paged storage driven from the GPU: one table of pages for all layers, and layers that keep their keys and values at 16 bits, at 8
bits or packed (TQ4) on those pages, with rotary positions applied on the way in.  Sequences may begin with the same pages; single
tokens then attend to these once for all.

The reference has the packed pages (src/flashquant/vllm/impl.py:132-138, 220-263) and leaves tables, positions and 16-bit layers to
vLLM; here a decode step is ``PageTable.schedule`` once and ``step`` per layer, without a look at lengths or pages from the host, so
that it can be captured in a graph."""
from __future__ import annotations

import math
from typing import List, NamedTuple, Optional, Set, Tuple

import torch

from flashquant_amd.kernels import (paged_kv8_decode, paged_kv8_read, paged_kv_decode, paged_prefix_decode, paged_schedule, rotary_embedding,
                                    rotary_paged_store, rotary_paged_store8)
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
    sequence and how many tokens it sees (itself the last; padding: none); None where ``num_tokens`` is above ``max_seqs``.  Where enough
    sequences share a prefix of the table, ``token_prefix`` (num_tokens,) int32 is the one of a token's sequence (or -1: it attends by
    itself) and ``prefix_lens`` their tokens; else both are None."""
    slot_mapping: torch.Tensor
    positions: torch.Tensor
    seq_lens: torch.Tensor
    cu_seqlens: torch.Tensor
    block_table: torch.Tensor
    pages_taken: torch.Tensor
    token_table: Optional[torch.Tensor] = None
    token_lens: Optional[torch.Tensor] = None
    token_prefix: Optional[torch.Tensor] = None
    prefix_lens: Optional[torch.Tensor] = None


def _rows(q: torch.Tensor, step: PagedStep) -> Tuple[torch.Tensor, torch.Tensor]:
    """Pages and lengths for single-token attention of ``q``, row by row (a step made by hand may have them by sequence)."""
    table, lens = (step.block_table, step.seq_lens) if step.token_table is None else (step.token_table, step.token_lens)
    if q.shape[0] != table.shape[0]:
        raise ValueError(f"a step attends one token of every sequence at most: {q.shape[0]} tokens, {table.shape[0]} rows of pages")
    return table, lens


class PageTable:
    """Block tables, lengths and the list of free pages of ``max_seqs`` sequences, all on the GPU, and up to ``max_prefixes`` prefixes
    that sequences share: whole pages that belong to the prefix and not to a sequence.

    A prefix is attended to once for all where at least three sequences share it.  Whether any is, ``schedule`` decides on the host: a
    graph captured before never attends so (its results are right), one captured after follows every prefix that comes and goes."""

    # Sequences that share a prefix of 2000 tokens, 32 heads over 8 of 128 (us, shared / every one by itself): 16 prefixes of two at 16 bits
    # 39 / 36, at 8 bits 37 / 26; 20 of three 49 / 82 and 47 / 49; 16 of four 40 / 56 and 38 / 40.  (Of 512 tokens 10 of three 18 / 12: the host
    # does not know lengths; of 6000 at 16 bits 32 of two 154 / 235.)
    _enough = 3

    def __init__(self, num_blocks: int, block_size: int, max_seqs: int, max_blocks_per_seq: int,
                 device: Optional[torch.device] = None, *, max_prefixes: int = 0) -> None:
        if device is None:
            device = torch.device("cuda")
        if not 0 <= max_prefixes <= 1024:
            raise ValueError(f"max_prefixes must be 0 to 1024, got {max_prefixes}")
        self.num_blocks = num_blocks
        self.block_size = block_size
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_seqs, max_blocks_per_seq), -1, **i32)
        self.context_lens = torch.zeros(max_seqs, **i32)
        # free pages from free_start on; what lies before has been taken.  The last element takes what is not a page.
        self._pages = torch.arange(num_blocks + 1, **i32)
        self.free_blocks = self._pages[:num_blocks]
        self.free_start = torch.zeros(1, **i32)
        # pages and tokens of the prefixes, the prefix of every sequence, and where enough share it; on the host which sequences share one,
        # which there are, and which enough share
        self.prefix_ids = torch.full((max_seqs,), -1, **i32)
        self._shared_ids = torch.full((max_seqs,), -1, **i32)
        self.prefix_lens = torch.zeros(max_prefixes, **i32)
        self._prefix_table = torch.full((max_prefixes, max_blocks_per_seq), -1, **i32)
        self._prefix_of: List[int] = [-1] * max_seqs
        self._made: List[bool] = [False] * max_prefixes
        self._shared: Set[int] = set()

    def schedule(self, query_lens: torch.Tensor, num_tokens: int) -> PagedStep:
        """Gives ``query_lens[s]`` (int32) new tokens of sequence s their pages, slots and positions and counts them into the
        lengths; ``num_tokens`` is the room for all of them.  Tokens that there is no room for are left out: they take no page and
        count in no length."""
        s = paged_schedule(self.context_lens, query_lens, self.block_table, self.free_blocks, self.block_size, num_tokens,
                           free_start=self.free_start, capped=True)
        rows = num_tokens <= self.block_table.shape[0]
        state = s, self.context_lens, self.free_start, self.block_table, self.num_blocks, self.block_size, rows
        if not self._shared:
            return PagedStep(s.slot_mapping, s.positions, s.seq_lens, s.cu_seqlens, self.block_table, s.free_end, *native().paged_advance(*state))
        token_table, token_lens, token_prefix = native().paged_advance_prefix(*state, self._shared_ids)
        return PagedStep(s.slot_mapping, s.positions, s.seq_lens, s.cu_seqlens, self.block_table, s.free_end, token_table, token_lens, token_prefix,
                         self.prefix_lens if rows else None)

    def make_prefix(self, seq: int, prefix: int) -> None:
        """The whole pages that sequence ``seq`` has by now become prefix ``prefix`` (below ``max_prefixes``, not in use), which the
        sequence shares from now on."""
        self._check(seq, prefix, made=False)
        tokens = self.context_lens[seq] // self.block_size * self.block_size
        row = self.block_table[seq]
        self.prefix_lens[prefix] = tokens
        self._prefix_table[prefix] = torch.where(torch.arange(row.shape[0], device=row.device) < tokens // self.block_size, row, -1)
        self._made[prefix] = True
        self._share(seq, prefix)

    def join_prefix(self, seq: int, prefix: int) -> None:
        """Sequence ``seq``, which has no tokens (their pages would be lost), begins with those of ``prefix``."""
        self._check(seq, prefix, made=True)
        self.block_table[seq] = self._prefix_table[prefix]
        self.context_lens[seq] = self.prefix_lens[prefix]
        self._share(seq, prefix)

    def drop_prefix(self, prefix: int) -> None:
        """Ends ``prefix``, which no sequence shares any more: its pages are free again."""
        if not 0 <= prefix < len(self._made) or not self._made[prefix]:
            raise ValueError(f"prefix {prefix} is not in use")
        if prefix in self._prefix_of:
            raise ValueError(f"sequence {self._prefix_of.index(prefix)} still shares prefix {prefix}")
        self._free(self._prefix_table[prefix] >= 0, self._prefix_table[prefix])
        self._prefix_table[prefix] = -1
        self.prefix_lens[prefix] = 0
        self._made[prefix] = False

    def release(self, seq: int) -> None:
        """Ends sequence ``seq``: its pages, but those of a prefix that it shares, are free again (the next to be taken) and its length is
        0."""
        row, prefix = self.block_table[seq], self._prefix_of[seq]
        held = (self.context_lens[seq] + self.block_size - 1) // self.block_size
        column = torch.arange(row.shape[0], device=row.device)
        mine = (row >= 0) & (column < held)
        if prefix >= 0:
            mine &= column >= self.prefix_lens[prefix] // self.block_size
            self._leave(seq, prefix)
        self._free(mine, row)
        self.block_table[seq] = -1
        self.context_lens[seq] = 0

    def _check(self, seq: int, prefix: int, made: bool) -> None:
        if not 0 <= seq < len(self._prefix_of) or not 0 <= prefix < len(self._made):
            raise ValueError(f"no sequence {seq} or no prefix {prefix}")
        if self._prefix_of[seq] >= 0:
            raise ValueError(f"sequence {seq} shares prefix {self._prefix_of[seq]} already")
        if self._made[prefix] != made:
            raise ValueError(f"prefix {prefix} is {'not ' if made else ''}in use")

    def _share(self, seq: int, prefix: int) -> None:
        self.prefix_ids[seq] = prefix
        self._prefix_of[seq] = prefix
        self._settle(prefix, seq)

    def _leave(self, seq: int, prefix: int) -> None:
        self.prefix_ids[seq] = -1
        self._shared_ids[seq] = -1
        self._prefix_of[seq] = -1
        self._settle(prefix)

    def _settle(self, prefix: int, joined: Optional[int] = None) -> None:
        """After a change of its sequences: whether ``prefix`` is attended to once for them."""
        members = [s for s, p in enumerate(self._prefix_of) if p == prefix]
        before, now = prefix in self._shared, len(members) >= self._enough
        changed = members if now != before else [joined] if now and joined is not None else []
        for s in changed:
            self._shared_ids[s] = prefix if now else -1
        (self._shared.add if now else self._shared.discard)(prefix)

    def _free(self, mine: torch.Tensor, row: torch.Tensor) -> None:
        count = mine.sum(dtype=torch.int32)
        place = torch.where(mine, self.free_start - count + torch.cumsum(mine, 0) - 1, self.num_blocks)
        self._pages[place] = row
        self.free_start -= count


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
        q = self.store(q, k, v, step)
        if step.token_prefix is not None and self.window == 0:
            return paged_prefix_decode(q, self.keys, self.values, *rows, step.token_prefix, step.prefix_lens, self.sm_scale)
        return paged_kv_decode(q, self.keys, self.values, *rows, self.sm_scale, window=self.window)


class PagedKV8Layer:
    """The same at 8 bits: e4m3 rows (num_blocks, block_size, heads, head_dim) with a power of two each (num_blocks, heads, block_size).
    ``dtype``: of queries, of keys and values on the way in, and of rows read back."""

    def __init__(self, table: PageTable, heads: int, head_dim: int, inv_freq: torch.Tensor, rotary_scale: float = 1.0, *,
                 interleaved: bool = False, window: int = 0, sm_scale: Optional[float] = None, dtype: torch.dtype = torch.bfloat16) -> None:
        device = table.block_table.device
        self.table = table
        rows = torch.zeros(2, table.num_blocks, table.block_size, heads, head_dim, dtype=torch.uint8, device=device)
        scales = torch.zeros(2, table.num_blocks, heads, table.block_size, dtype=torch.uint8, device=device)
        self.keys, self.values = rows.view(torch.float8_e4m3fn)
        self.key_scales, self.value_scales = scales.view(torch.float8_e8m0fnu)
        self.inv_freq, self.rotary_scale, self.interleaved = inv_freq.to(device), rotary_scale, interleaved
        self.window, self.dtype = window, dtype
        self.sm_scale = 1.0 / math.sqrt(head_dim) if sm_scale is None else sm_scale

    def store(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep) -> torch.Tensor:
        """The step's keys and values, rotated and quantised, into their slots; returns the rotated queries (num_tokens, H_Q, head_dim)."""
        return rotary_paged_store8(q, k, v, step.positions, step.slot_mapping, self.inv_freq, self.keys, self.values, self.key_scales,
                                   self.value_scales, interleaved=self.interleaved, scale=self.rotary_scale)

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep) -> torch.Tensor:
        """``store`` of a step with at most one token of every sequence, then each one's attention over its sequence: (num_tokens, H_Q,
        head_dim); rows behind the last token are 0."""
        rows = _rows(q, step)
        q = self.store(q, k, v, step)
        if step.token_prefix is not None and self.window == 0:
            return paged_prefix_decode(q, self.keys, self.values, *rows, step.token_prefix, step.prefix_lens, self.sm_scale,
                                       key_scales=self.key_scales, value_scales=self.value_scales)
        return paged_kv8_decode(q, self.keys, self.values, self.key_scales, self.value_scales, *rows, self.sm_scale, window=self.window)

    def read(self, cu_seqlens: torch.Tensor, num_tokens: int, starts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Keys (rotated) and values of the table's sequences, (num_tokens, heads, head_dim) each: of sequence s its tokens from
        ``starts[s]`` (0 without) on, to rows ``cu_seqlens[s]`` .. ``cu_seqlens[s + 1]``, for a prompt's attention over 16-bit rows (which is
        the caller's: what this package has takes packed ones)."""
        return paged_kv8_read(self.keys, self.values, self.key_scales, self.value_scales, self.table.block_table, cu_seqlens, num_tokens,
                              starts=starts, dtype=self.dtype)


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
