"""Scheduling, rotary positions, stores and attention as a serving loop runs them: one page table, layers at 16 bits and packed,
prompts, generated tokens, sequences that end and begin, and a captured step."""
from __future__ import annotations

import math

import pytest
import torch

from flashquant_amd import kernels as K
from flashquant_amd.cache import PagedKVLayer, PagedTQ4Layer, PageTable
from flashquant_amd.vllm.impl import TQ4AttentionKernels
from tests.test_gpu_paged_kv import attended

pytestmark = pytest.mark.gpu
DEV = "cuda"
HQ, HKV = 8, 8


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def qkv_of(tokens, d, dtype, g):
    return (torch.randn(tokens, HQ + 2 * HKV, d, generator=g).to(dtype).to(DEV)).split([HQ, HKV, HKV], 1)


class Told:
    """What the layers hold, kept by sequence on the side: rotated keys and values, and the packed path on pages of its own."""

    def __init__(self, seqs, d, page, dtype, freq, scale):
        self.k = [torch.empty(0, HKV, d, dtype=dtype, device=DEV) for _ in range(seqs)]
        self.v = [torch.empty_like(x) for x in self.k]
        self.page, self.freq, self.scale, self.d = page, freq, scale, d
        self.most = 40
        self.cache = torch.zeros(seqs * self.most, page, HKV * (d + 8), dtype=torch.uint8, device=DEV)
        self.table = torch.arange(seqs * self.most, dtype=torch.int32, device=DEV).view(seqs, self.most)
        self.kernels = TQ4AttentionKernels(HKV, d, 1 / math.sqrt(d), torch.device(DEV))

    def positions(self, counts):
        return torch.cat([torch.arange(len(self.k[s]), len(self.k[s]) + n, device=DEV) for s, n in enumerate(counts)])

    def add(self, counts, q, k, v):
        """The rotated queries, and the slots of the tokens on this cache."""
        q, k = K.rotary_embedding(q, k, self.positions(counts), self.freq, scale=self.scale)
        at, slots = 0, []
        for s, n in enumerate(counts):
            p = torch.arange(len(self.k[s]), len(self.k[s]) + n, device=DEV)
            slots.append(self.table[s].long()[p // self.page] * self.page + p % self.page)
            self.k[s], self.v[s] = torch.cat([self.k[s], k[at:at + n]]), torch.cat([self.v[s], v[at:at + n]])
            at += n
        return q, k, torch.cat(slots)

    def lens(self):
        return i32([len(x) for x in self.k])

    def forget(self, s):
        self.k[s], self.v[s] = self.k[s][:0], self.v[s][:0]

    def check(self, q, out):
        """One query a sequence against the definition over what was kept."""
        n = max(len(x) for x in self.k)
        kc = torch.zeros(len(self.k), n, HKV, self.d, dtype=q.dtype, device=DEV)
        vc = torch.zeros_like(kc)
        for s, (k, v) in enumerate(zip(self.k, self.v)):
            kc[s, :len(k)], vc[s, :len(v)] = k, v
        want, _, tol, _ = attended(q, kc, vc, torch.arange(len(self.k), dtype=torch.int32, device=DEV)[:, None], self.lens(), 1 / math.sqrt(self.d))
        off = (out.double() - want).abs() - tol
        assert (off <= 0).all(), float(off.max())


@pytest.mark.parametrize("d,page,dtype", [(128, 16, torch.bfloat16), (64, 32, torch.float16), (256, 8, torch.bfloat16)])
def test_a_serving_loop(d, page, dtype):
    seqs, g = 5, torch.Generator().manual_seed(d)
    freq, scale = K.rotary_frequencies(d, 10000.0, "yarn", factor=4.0, original_max_position=64)
    table = PageTable(5 * 300 // page + 7, page, seqs, 300 // page + 1)
    plain, packed = PagedKVLayer(table, HKV, d, freq, scale, dtype=dtype), PagedTQ4Layer(table, HKV, d, freq, scale)
    told = Told(seqs, d, page, dtype, freq.to(DEV), scale)
    held = [0] * seqs
    for turn, counts in enumerate([[37, 1, 100, 16, 64], [1] * 5, [1] * 5, [3, 70, 1, 16, 1], [1] * 5, "end 2", "end 0", [50, 1, 33, 1, 1], [1] * 5, [1] * 5]):
        if isinstance(counts, str):
            s = int(counts.split()[1])
            table.release(s)
            told.forget(s)
            held[s] = 0
            continue
        tokens = sum(counts)
        q, k, v = qkv_of(tokens, d, dtype, g)
        step = table.schedule(i32(counts), tokens)
        assert torch.equal(step.positions, told.positions(counts))
        qr, kr, slots = told.add(counts, q, k, v)
        lens = told.lens()
        assert torch.equal(step.seq_lens, lens) and torch.equal(table.context_lens, lens)
        # every page belongs to one sequence
        held = [h + n for h, n in zip(held, counts)]
        pages = torch.cat([table.block_table[s, :-(-h // page)] for s, h in enumerate(held)])
        assert len(pages.unique()) == len(pages) and int(pages.min()) >= 0 and int(table.free_start) == len(pages)
        if max(counts) == 1:
            told.check(qr, plain.step(q, k, v, step))
            got = packed.step(q, k, v, step)
            want = told.kernels.decode_step(qr, kr, v, told.cache, slots, told.table[:, :table.block_table.shape[1]].contiguous(), lens)
        else:
            assert torch.equal(plain.store(q, k, v, step), qr)
            got = packed.prefill(q, k, v, step, max(counts))
            told.kernels.compress_and_store(kr, v, told.cache, slots)
            want = told.kernels.prefill(qr, step.cu_seqlens, max(counts), told.cache, told.table[:, :table.block_table.shape[1]].contiguous(), lens)
        assert torch.equal(got, want), turn


def test_a_page_table_that_runs_out_and_recovers():
    table = PageTable(6, 16, 2, 10)
    step = table.schedule(i32([40, 70]), 110)              # 3 + 5 pages
    assert int(step.pages_taken) == 8 and int(table.free_start) == 6
    assert step.block_table[0].tolist()[:4] == [0, 1, 2, -1] and step.block_table[1].tolist()[:6] == [3, 4, 5, -1, -1, -1]
    assert (step.slot_mapping[40 + 48:] == -1).all() and (step.slot_mapping[:88] >= 0).all()
    table.release(1)
    assert int(table.free_start) == 3 and sorted(table.free_blocks[3:].tolist()) == [3, 4, 5]
    table.release(0)
    assert int(table.free_start) == 0 and sorted(table.free_blocks.tolist()) == list(range(6))
    table.release(0)                                        # nothing held
    assert int(table.free_start) == 0
    step = table.schedule(i32([96, 0]), 96)
    assert sorted(step.slot_mapping.tolist()) == list(range(96))


@pytest.mark.parametrize("d,first", [(128, 700), (64, 3)])
def test_a_captured_step(d, first):
    """Replays, with eager work of the same kind between them, give what the eager step gives."""
    seqs, page, dtype = 4, 16, torch.bfloat16
    freq, _ = K.rotary_frequencies(d)

    def model():
        table = PageTable(seqs * 60, page, seqs, 60)
        return table, PagedKVLayer(table, HKV, d, freq, dtype=dtype), PagedTQ4Layer(table, HKV, d, freq)

    def fill(table, plain, packed):
        g = torch.Generator().manual_seed(1)
        counts = [first, 1, first // 2 + 1, 15]
        q, k, v = qkv_of(sum(counts), d, dtype, g)
        step = table.schedule(i32(counts), sum(counts))
        plain.store(q, k, v, step)
        packed.store(q, k, v, step)

    ones = i32([1] * seqs)

    def run(m, q, k, v):
        step = m[0].schedule(ones, seqs)
        return m[1].step(q, k, v, step), m[2].step(q, k, v, step), step.slot_mapping

    eager, captured, warm = model(), model(), model()
    for m in (eager, captured, warm):
        fill(*m)
    inputs = [torch.empty(seqs, h, d, dtype=dtype, device=DEV) for h in (HQ, HKV, HKV)]
    g = torch.Generator().manual_seed(2)
    for x, y in zip(inputs, qkv_of(seqs, d, dtype, g)):
        x.copy_(y)
    run(warm, *inputs)                                      # loads what a first call loads
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(captured, *inputs)
    for turn in range(20):                                  # over the ends of pages
        for x, y in zip(inputs, qkv_of(seqs, d, dtype, g)):
            x.copy_(y)
        graph.replay()
        want = run(eager, *inputs)
        torch.cuda.synchronize()
        for got, w in zip(out, want):
            assert torch.equal(got, w), turn
    assert torch.equal(captured[0].context_lens, eager[0].context_lens)


def test_calls_on_another_stream():
    d, dtype = 128, torch.bfloat16
    freq, _ = K.rotary_frequencies(d, device=DEV)
    g = torch.Generator().manual_seed(3)
    kc, vc = (torch.randn(90, 16, HKV, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    table = torch.randperm(90, generator=g).int().view(1, 90).to(DEV)
    q, k, v = qkv_of(1, d, dtype, g)
    lens, slot = i32([1440]), table[0, -1:].long() * 16 + 15
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = kc.clone(), vc.clone()
        out = K.paged_kv_decode(K.rotary_paged_store(q, k, v, slot, slot, freq, *mine), *mine, table, lens)
        s = K.paged_schedule(i32([1439]), i32([1]), table.clone(), i32([5]), 16, 1)
    side.synchronize()
    want = K.paged_kv_decode(K.rotary_paged_store(q, k, v, slot, slot, freq, kc, vc), kc, vc, table, lens)
    assert torch.equal(out, want) and torch.equal(mine[0], kc) and torch.equal(s.slot_mapping, slot)


@pytest.mark.parametrize("padded", [True, False])
@pytest.mark.parametrize("d,page,dtype", [(128, 16, torch.bfloat16), (64, 32, torch.float16), (256, 8, torch.bfloat16)])
def test_steps_in_which_sequences_are_idle(d, page, dtype, padded):
    """Sequences without a token first, in the middle and last, ended and not: every token attends over its own sequence, rows behind the
    last token see nothing."""
    seqs, g = 5, torch.Generator().manual_seed(d + 1)
    freq, scale = K.rotary_frequencies(d)
    table = PageTable(5 * 300 // page + 7, page, seqs, 300 // page + 1)
    plain, packed = PagedKVLayer(table, HKV, d, freq, scale, dtype=dtype), PagedTQ4Layer(table, HKV, d, freq, scale)
    told = Told(seqs, d, page, dtype, freq.to(DEV), scale)
    columns = table.block_table.shape[1]
    for turn, counts in enumerate([[37, 1, 100, 16, 64], [1, 0, 1, 0, 1], [0, 1, 1, 1, 0], "end 1", [1, 0, 1, 1, 1], [0, 0, 0, 0, 1], "end 4", [0, 0, 1, 1, 0],
                                   [0, 0, 0, 0, 0], [0, 20, 0, 0, 0], [0, 1, 0, 1, 0], [1, 1, 1, 1, 1]]):
        if isinstance(counts, str):
            table.release(int(counts.split()[1]))
            told.forget(int(counts.split()[1]))
            continue
        tokens = sum(counts)
        room = max(tokens, seqs) if padded else tokens
        q, k, v = qkv_of(room, d, dtype, g)
        step = table.schedule(i32(counts), room)
        qr, kr, slots = told.add(counts, q[:tokens], k[:tokens], v[:tokens])
        assert torch.equal(step.seq_lens, told.lens()) and torch.equal(step.positions[:tokens], K.paged_schedule(told.lens() - i32(counts), i32(counts), table.block_table.clone(),
                                                                                                       table.free_blocks, page, tokens).positions)
        if max(counts) > 1:
            plain.store(q, k, v, step)
            packed.store(q, k, v, step)
            told.kernels.compress_and_store(kr, v[:tokens], told.cache, slots)
            continue
        rows = [s for s in range(seqs) if counts[s]]
        got = plain.step(q, k, v, step)
        assert got.shape == (room, HQ, d) and not got[tokens:].any()
        lens = i32([len(told.k[s]) for s in rows] + [0] * (room - tokens))
        if tokens:
            n = int(lens.max())
            kc = torch.zeros(tokens, n, HKV, d, dtype=dtype, device=DEV)
            vc = torch.zeros_like(kc)
            for i, s in enumerate(rows):
                kc[i, :len(told.k[s])], vc[i, :len(told.v[s])] = told.k[s], told.v[s]
            want, _, tol, _ = attended(qr, kc, vc, torch.arange(tokens, dtype=torch.int32, device=DEV)[:, None], lens[:tokens], 1 / math.sqrt(d))
            off = (got[:tokens].double() - want).abs() - tol
            assert (off <= 0).all(), (turn, float(off.max()))
        got = packed.step(q, k, v, step)
        # the same rows on the pages that are kept aside
        pad = [torch.cat([x, torch.zeros(room - tokens, *x.shape[1:], dtype=dtype, device=DEV)]) for x in (qr, kr, v[:tokens])]
        slots = torch.cat([slots, torch.full((room - tokens,), -1, dtype=torch.int64, device=DEV)])
        his = told.table[:, :columns][rows + [0] * (room - tokens)].contiguous()
        if room:
            want = told.kernels.decode_step(*pad, told.cache, slots, his, lens)
            assert torch.equal(got, want), turn
        assert got.shape == (room, HQ, d) and not got[tokens:].any()


def test_idle_sequences_in_a_captured_step():
    """One graph, replayed with other sequences idle each time."""
    d, seqs, page, dtype = 128, 4, 16, torch.bfloat16
    freq, _ = K.rotary_frequencies(d)

    def model():
        table = PageTable(seqs * 60, page, seqs, 60)
        m = table, PagedKVLayer(table, HKV, d, freq, dtype=dtype), PagedTQ4Layer(table, HKV, d, freq)
        q, k, v = qkv_of(200, d, dtype, torch.Generator().manual_seed(1))
        step = table.schedule(i32([100, 1, 60, 39]), 200)
        m[1].store(q, k, v, step)
        m[2].store(q, k, v, step)
        return m

    def run(m, counts, q, k, v):
        step = m[0].schedule(counts, seqs)
        return m[1].step(q, k, v, step), m[2].step(q, k, v, step), step.slot_mapping

    eager, captured, warm = model(), model(), model()
    g = torch.Generator().manual_seed(2)
    inputs, counts = [x.clone() for x in qkv_of(seqs, d, dtype, g)], i32([1] * seqs)
    run(warm, counts, *inputs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(captured, counts, *inputs)
    for turn in range(16):
        counts.copy_(i32([turn >> b & 1 for b in range(seqs)]))
        for x, y in zip(inputs, qkv_of(seqs, d, dtype, g)):
            x.copy_(y)
        graph.replay()
        want = run(eager, counts, *inputs)
        torch.cuda.synchronize()
        for got, w in zip(out, want):
            assert torch.equal(got, w), turn
        n = bin(turn).count("1")
        assert not out[0][n:].any() and not out[1][n:].any() and (n == 0 or out[0][:n].any())
    assert torch.equal(captured[0].context_lens, eager[0].context_lens)


def test_a_step_of_more_tokens_than_sequences_is_refused_before_it_stores():
    freq, _ = K.rotary_frequencies(64)
    table = PageTable(20, 16, 2, 10)
    q, k, v = qkv_of(3, 64, torch.bfloat16, torch.Generator().manual_seed(1))
    step = table.schedule(i32([2, 1]), 3)
    assert step.token_table is None and step.token_lens is None
    for layer in (PagedKVLayer(table, HKV, 64, freq), PagedTQ4Layer(table, HKV, 64, freq)):
        with pytest.raises(ValueError, match="one token of every sequence"):
            layer.step(q, k, v, step)
        assert not (layer.keys if isinstance(layer, PagedKVLayer) else layer.cache).any()


def test_rows_of_tokens_against_loops():
    """Wide tables, many sequences, more rows than tokens, rows that are full; a table without sequences."""
    g = torch.Generator().manual_seed(6)
    for seqs, blocks, page, extra in ((1, 1, 8, 0), (3, 5000, 32, 0), (700, 3, 16, 0), (2500, 40, 8, 13), (300, 2049, 8, 100)):
        table = PageTable(4 * seqs + 30, page, seqs, blocks)
        for turn in range(3):
            before = table.context_lens.tolist()
            counts = torch.randint(0, 2, (seqs,), generator=g).int().tolist() if turn else [8] * seqs
            room = min(seqs, sum(counts) + extra) if turn else sum(counts)
            step = table.schedule(i32(counts), room)
            if room > seqs:
                assert step.token_table is None
                continue
            rows = [s for s in range(seqs) if counts[s]]
            lens = [min(before[s] + 1, blocks * page) for s in rows]
            assert step.token_lens.tolist() == lens + [0] * (room - len(rows))
            assert torch.equal(step.token_table[:len(rows)], table.block_table[rows]) and (step.token_table[len(rows):] == -1).all()
            assert step.token_table.shape == (room, blocks) and torch.equal(table.context_lens, step.seq_lens)
    table = PageTable(4, 16, 0, 3)
    assert int(table.schedule(i32([]), 2).pages_taken) == 0 and int(table.free_start) == 0


def test_tokens_beyond_the_room_of_a_step_are_left_out():
    """They take no page, count in no length, and a prompt's attention does not go beyond the rows that there are."""
    table = PageTable(20, 16, 4, 10)
    step = table.schedule(i32([20, 50, 9, 0]), 40)
    assert step.cu_seqlens.tolist() == [0, 20, 40, 40, 40] and step.seq_lens.tolist() == [20, 20, 0, 0]
    assert table.context_lens.tolist() == [20, 20, 0, 0] and int(table.free_start) == 4 and int(step.pages_taken) == 4
    assert step.positions.tolist() == [*range(20), *range(20)] and (step.slot_mapping >= 0).all() and (table.block_table >= 0).sum() == 4
    step = table.schedule(i32([1, 12, 1, 1]), 14)           # the last one is left out, on the first token of a page
    assert step.cu_seqlens.tolist() == [0, 1, 13, 14, 14] and step.seq_lens.tolist() == [21, 32, 1, 0] and int(table.free_start) == 5
    step = table.schedule(i32([3, 1, 1, 1]), 0)
    assert step.cu_seqlens.tolist() == [0] * 5 and step.seq_lens.tolist() == [21, 32, 1, 0] and int(table.free_start) == 5
    for s in range(4):
        table.release(s)
    assert int(table.free_start) == 0 and sorted(table.free_blocks.tolist()) == list(range(20))
    d, g = 128, torch.Generator().manual_seed(5)
    freq, _ = K.rotary_frequencies(d)
    outs = []
    for counts in ([20, 300, 700], [20, 230, 0]):
        table = PageTable(100, 16, 3, 64)
        layer = PagedTQ4Layer(table, HKV, d, freq)
        q, k, v = qkv_of(250, d, torch.bfloat16, g.manual_seed(5))
        step = table.schedule(i32(counts), 250)
        assert int(step.cu_seqlens[-1]) == 250
        outs.append(layer.prefill(q, k, v, step, max(counts)))
    assert torch.equal(*outs)
