"""The 8-bit cache and shared prefixes as a serving loop runs them: a prompt that becomes a prefix, sequences that join it, end and begin
again, layers at 16 bits, 8 bits and packed on one table of pages, captured steps, other streams."""
from __future__ import annotations

import math

import pytest
import torch

from flashquant_amd import kernels as K
from flashquant_amd.cache import PagedKV8Layer, PagedKVLayer, PagedTQ4Layer, PageTable
from flashquant_amd.kernels._native import native
from tests.test_gpu_kv8 import BF, DEV, HF, U8, attended, check, gen, raw, stood_for
from tests.test_gpu_prefix import prefix_case, wanted, call

pytestmark = pytest.mark.gpu
HQ, HKV, D = 8, 2, 128


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def qkv_of(tokens, dtype, g):
    return (torch.randn(tokens, HQ + 2 * HKV, D, generator=g).to(dtype).to(DEV)).split([HQ, HKV, HKV], 1)


def layers_of(table, dtype):
    freq, scale = K.rotary_frequencies(D, scaling="yarn", factor=4.0, original_max_position=512, device=DEV)
    return [PagedKVLayer(table, HKV, D, freq, scale, dtype=dtype), PagedKV8Layer(table, HKV, D, freq, scale, dtype=dtype), PagedTQ4Layer(table, HKV, D, freq, scale)]


def contents(layer):
    if isinstance(layer, PagedKVLayer):
        return layer.keys.double(), layer.values.double()
    return stood_for(layer.keys, layer.key_scales), stood_for(layer.values, layer.value_scales)


def check_step(layer, q, out, step, dtype):
    """The step's rows against 64 bits over what the layer holds, row by row of the tokens."""
    q = K.rotary_embedding(q, None, step.positions, layer.inv_freq, scale=layer.rotary_scale)[0]
    keys, values = contents(layer)
    o, _, to, _ = attended(q, keys, values, step.token_table, step.token_lens, layer.sm_scale)
    size, _, _, _ = attended(q, keys, values.abs(), step.token_table, step.token_lens, layer.sm_scale)
    tol = to + (size * torch.finfo(dtype).eps / 2 + values.abs().max() * 2.0 ** -20) * 1.02       # weights over shared tokens are rounded
    assert ((out.double() - o).abs() <= tol).all()


def in_use(table):
    """Pages that sequences and prefixes hold, each once; together with the free ones they are all."""
    start = int(table.free_start)
    free = table._pages[start:table.num_blocks].tolist()
    held = set()
    for s, (row, n) in enumerate(zip(table.block_table.tolist(), table.context_lens.tolist())):
        held |= set(row[:-(-n // table.block_size)])
    for row, n in zip(table._prefix_table.tolist(), table.prefix_lens.tolist()):
        held |= set(row[:n // table.block_size])
    assert len(held) == start and not held & set(free) and held | set(free) == set(range(table.num_blocks))
    return start


@pytest.mark.parametrize("dtype", [BF, HF])
def test_serving_loop_with_prefixes(dtype):
    g, seqs, page = gen(1), 7, 16
    table = PageTable(200, page, seqs, 40, max_prefixes=2)
    layers = layers_of(table, dtype)

    def prompt(lens):
        n = sum(lens)
        step = table.schedule(i32(lens), n)
        q, k, v = qkv_of(n, dtype, g)
        for layer in layers[:2]:
            layer.store(q, k, v, step)
        layers[2].prefill(q, k, v, step, max(lens))

    def generate(lens, room=None):
        step = table.schedule(i32(lens), room or sum(lens))
        q, k, v = qkv_of(room or sum(lens), dtype, g)
        for layer in layers[:2]:
            check_step(layer, q, layer.step(q, k, v, step), step, dtype)
        packed = layers[2].step(q, k, v, step)
        assert torch.isfinite(packed).all() and (packed[sum(lens):] == 0).all()
        return step

    prompt([333, 0, 0, 0, 0, 0, 50])
    assert generate([1, 0, 0, 0, 0, 0, 1]).token_prefix is None
    table.make_prefix(0, 1)
    assert table.prefix_lens.tolist() == [0, 320] and table.context_lens.tolist()[0] == 334
    for s in (2, 3, 5):
        table.join_prefix(s, 1)
    used = in_use(table)
    assert used == 21 + 4
    step = generate([1, 0, 1, 1, 0, 1, 1])
    assert step.token_prefix.tolist() == [1, 1, 1, 1, -1] and step.token_lens.tolist() == [335, 321, 321, 321, 52]
    prompt([0, 0, 30, 7, 200, 0, 0])                                     # chunks of prompts behind the prefix, and one of its own
    table.make_prefix(4, 0)
    table.join_prefix(1, 0)
    for _ in range(4):
        generate([1, 1, 1, 1, 1, 1, 1])
    generate([1, 0, 1, 0, 1, 0, 1], room=6)                              # idle sequences, and padding behind the last
    in_use(table)
    # rows read back are what the layer holds
    cu, starts = i32([0, 5, 5, 40, 40, 40, 40, 43]), i32([320, 0, 300, 0, 0, 0, 10])
    k, v = layers[1].read(cu, 45, starts)
    keys, values = contents(layers[1])
    at = [(0, 320 + i) for i in range(5)] + [(2, 300 + i) for i in range(35)] + [(6, 10 + i) for i in range(3)]
    for got, want in ((k, keys), (v, values)):
        rows = torch.stack([want[int(table.block_table[s, t // page]), t % page] for s, t in at])
        assert torch.equal(got[:43], rows.to(dtype)) and (got[43:] == 0).all()
    # ends: pages of a prefix stay until it is dropped
    with pytest.raises(ValueError, match="still shares"):
        table.drop_prefix(1)
    for s in (0, 2, 3, 5):
        table.release(s)
        in_use(table)
    table.drop_prefix(1)
    in_use(table)
    table.join_prefix(3, 0)
    generate([0, 1, 0, 1, 1, 0, 1])
    for s in (1, 3, 4, 6):
        table.release(s)
    table.drop_prefix(0)
    assert in_use(table) == 0 and table.prefix_ids.tolist() == [-1] * seqs
    prompt([40, 3, 0, 0, 0, 0, 0])
    assert generate([1, 1, 0, 0, 0, 0, 0]).token_prefix is None


@pytest.mark.parametrize("bits", [16, 8])
def test_captured_step_over_a_prefix(bits):
    """A graph of scheduling, store and attention, replayed with other work between; every replay against the layer's contents."""
    g, seqs, page = gen(bits), 5, 16
    table = PageTable(100, page, seqs, 20, max_prefixes=1)
    layer = layers_of(table, BF)[0 if bits == 16 else 1]
    step = table.schedule(i32([100, 0, 0, 0, 9]), 109)
    layer.store(*qkv_of(109, BF, g), step)
    table.make_prefix(0, 0)
    for s in (1, 2, 3):
        table.join_prefix(s, 0)
    q, k, v = qkv_of(seqs, BF, g)
    counts = i32([1, 1, 1, 0, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step = table.schedule(counts, seqs)
        check_step(layer, q, layer.step(q, k, v, step), step, BF)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = table.schedule(counts, seqs)
        out = layer.step(q, k, v, step)
    for i in range(5):
        for t, x in zip((q, k, v), qkv_of(seqs, BF, g)):
            t.copy_(x)
        counts.copy_(i32([[1, 1, 1, 0, 1], [1, 1, 0, 1, 1], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1], [0, 0, 1, 0, 0]][i]))
        if i == 3:                                                       # a member ends and another begins, between replays
            table.release(2)
            table.join_prefix(2, 0)
        graph.replay()
        torch.cuda.synchronize()
        check_step(layer, q, out, step, BF)
        assert (out[int(counts.sum()):] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_two_calls_at_once_with_room_of_their_own(bits):
    case = [prefix_case([2000], [0] * 20, [50 + i for i in range(20)], 32, 8, 128, 16, BF, bits, seed=s) for s in range(2)]
    want = [wanted(*c, 1 / math.sqrt(128)) for c in case]
    room = native().paged_prefix_decode_workspace_bytes(20, 32, 8, 128, 1)
    rooms = [torch.empty(room, dtype=U8, device=DEV) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(call(*case[i], workspace=rooms[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for got in outs[i]:
            check(got, want[i], case[i][0])
        assert all(torch.equal(outs[i][0][0], o[0]) for o in outs[i])


def test_captured_calls_of_the_8_bit_operators():
    """Store, read and decode in one graph; replays against the same calls outside of it."""
    g = gen(4)
    blocks, page = 40, 16
    rows = torch.zeros(2, blocks, page, HKV, D, dtype=U8, device=DEV)
    scales = torch.zeros(2, blocks, HKV, page, dtype=U8, device=DEV)
    cache = (*rows.view(torch.float8_e4m3fn), *scales.view(torch.float8_e8m0fnu))
    freq = K.rotary_frequencies(D, device=DEV)[0]
    q, k, v = qkv_of(33, BF, g)
    positions, slots = torch.arange(33, device=DEV), torch.randperm(blocks * page, generator=g)[:33].to(DEV)
    table, cu, lens = torch.randperm(blocks, generator=g).int().to(DEV).view(4, 10), i32([0, 30, 30, 100, 130]), i32([160, 3, 0, 77])

    def run():
        r = K.rotary_paged_store8(q, k, v, positions, slots, freq, *cache)
        return (r, *K.paged_kv8_read(*cache, table, cu, 140), K.paged_kv8_decode(r[:4], *cache, table, lens))

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(4):
        for t, x in zip((q, k, v), qkv_of(33, BF, g)):
            t.copy_(x)
        slots.copy_(torch.randperm(blocks * page, generator=g)[:33])
        rows.zero_()
        scales.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        got, held = [o.clone() for o in outs], (rows.clone(), scales.clone())
        rows.zero_()
        scales.fill_(9)
        want = run()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(held[0], rows) and torch.equal(held[1], scales)


def test_what_a_call_writes_is_known_to_autograd():
    g = gen(6)
    q, k, v = qkv_of(5, BF, g)
    freq, at = K.rotary_frequencies(D, device=DEV)[0], torch.arange(5, device=DEV)
    kc, vc = (torch.zeros(2, 16, HKV, D, dtype=U8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros(2, HKV, 16, dtype=U8, device=DEV).view(torch.float8_e8m0fnu) for _ in range(2))
    before = [t._version for t in (kc, vc, ks, vs)]
    out = torch.empty_like(q)
    K.rotary_paged_store8(q, k, v, at, at, freq, kc, vc, ks, vs, out=out)
    assert all(t._version > b for t, b in zip((kc, vc, ks, vs), before)) and out._version > 0
    with pytest.raises(ValueError, match="gradient"):
        K.rotary_paged_store8(q, k, v, at, at, freq, kc, vc, ks, vs, out=torch.empty_like(q).requires_grad_())
    table, lens = torch.zeros(5, 2, dtype=torch.int32, device=DEV), i32([5, 3, 0, 1, 2])
    for f in (lambda o: K.paged_kv8_decode(q, kc, vc, ks, vs, table, lens, out=o),
              lambda o: K.paged_prefix_decode(q, kc, vc, table, lens, i32([0] * 5), i32([0]), key_scales=ks, value_scales=vs, out=o)):
        o = torch.empty_like(q)
        f(o)
        assert o._version > 0
        with pytest.raises(ValueError, match="gradient"):
            f(torch.empty_like(q).requires_grad_())
    rows = [torch.empty(4, HKV, D, dtype=BF, device=DEV) for _ in range(2)]
    K.paged_kv8_read(kc, vc, ks, vs, table[:1], i32([0, 4]), 4, out=tuple(rows))
    assert all(r._version > 0 for r in rows)
