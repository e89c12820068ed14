"""Prefixes that few share: a step attends to a prefix once for all only where enough sequences share it, and as before where not."""
from __future__ import annotations

import pytest
import torch

from flashquant_amd.cache import PagedKV8Layer, PagedKVLayer, PageTable
from tests.test_gpu_prefix_layers import BF, D, HKV, K, check_step, i32, qkv_of
from tests.test_gpu_kv8 import gen
from tests.test_kv8_host import taken


def test_ids_follow_the_sequences_that_share():
    """On the host: what a step is given, through joins and ends in any order."""
    g = gen(3)
    table = PageTable(400, 8, 9, 10, torch.device("cpu"), max_prefixes=3)
    of = [-1] * 9
    made = [False] * 3
    for _ in range(600):
        s, p = (int(torch.randint(0, n, (1,), generator=g)) for n in (9, 3))
        if of[s] >= 0:
            table.release(s)
            of[s] = -1
        elif not made[p]:
            taken(table, s, 20)
            table.make_prefix(s, p)
            of[s], made[p] = p, True
        elif p not in of and torch.rand(1, generator=g) < 0.3:
            table.drop_prefix(p)
            made[p] = False
        else:
            table.join_prefix(s, p)
            of[s] = p
        assert table.prefix_ids.tolist() == of
        assert table._shared_ids.tolist() == [i if i >= 0 and of.count(i) >= 3 else -1 for i in of]
        assert table._shared == {i for i in of if i >= 0 and of.count(i) >= 3}


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_a_prefix_of_few_is_attended_to_by_each(bits):
    g, seqs = gen(bits), 7
    table = PageTable(120, 16, seqs, 20, max_prefixes=2)
    freq, scale = K.rotary_frequencies(D)
    layer = (PagedKVLayer if bits == 16 else PagedKV8Layer)(table, HKV, D, freq, scale)

    def prompt(lens):
        layer.store(*qkv_of(sum(lens), BF, g), table.schedule(i32(lens), sum(lens)))

    def generate(lens):
        step = table.schedule(i32(lens), seqs)
        q, k, v = qkv_of(seqs, BF, g)
        check_step(layer, q, layer.step(q, k, v, step), step, BF)
        return None if step.token_prefix is None else step.token_prefix.tolist()

    prompt([100, 0, 0, 0, 0, 0, 70])
    table.make_prefix(0, 1)
    assert generate([1, 0, 0, 0, 0, 0, 1]) is None                       # one sequence
    table.join_prefix(1, 1)
    table.make_prefix(6, 0)
    table.join_prefix(5, 0)
    assert generate([1, 1, 0, 0, 0, 1, 1]) is None                       # two and two
    table.join_prefix(2, 1)
    assert generate([1, 1, 1, 0, 0, 1, 1]) == [1, 1, 1, -1, -1, -1, -1]  # three and two
    table.join_prefix(3, 1)
    table.join_prefix(4, 0)
    assert generate([1, 1, 1, 1, 1, 1, 1]) == [1, 1, 1, 1, 0, 0, 0]
    for s in (0, 2, 5):
        table.release(s)
    assert generate([0, 1, 0, 1, 1, 0, 1]) is None
    for s in (1, 3):
        table.release(s)
    assert generate([0, 0, 0, 0, 1, 0, 1]) is None                       # a prefix that nobody shares
    table.drop_prefix(1)
    assert generate([0, 0, 0, 0, 1, 0, 1]) is None


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("sharers", [1, 3])
def test_captured_step_while_sequences_come_and_go(sharers, bits):
    """Captured with few sequences or enough of them, replayed with none, some and all."""
    g, seqs = gen(bits + sharers), 5
    table = PageTable(100, 16, seqs, 20, max_prefixes=1)
    freq, scale = K.rotary_frequencies(D)
    layer = (PagedKVLayer if bits == 16 else PagedKV8Layer)(table, HKV, D, freq, scale)
    step = table.schedule(i32([100, 0, 0, 0, 9]), 109)
    layer.store(*qkv_of(109, BF, g), step)
    table.make_prefix(0, 0)
    for s in range(1, sharers):
        table.join_prefix(s, 0)
    q, k, v = qkv_of(seqs, BF, g)
    counts = i32([1] * sharers + [0] * (4 - sharers) + [1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(q, k, v, table.schedule(counts, seqs))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = table.schedule(counts, seqs)
        out = layer.step(q, k, v, step)
    assert (step.token_prefix is None) == (sharers < 3)
    for present in ([0, 1, 2, 3], [0, 3], [1, 2, 3], [2], [0, 1, 2, 3], []):
        for s in range(4):
            now = table._prefix_of[s] >= 0
            if now and s not in present:
                table.release(s)
            if not now and s in present:
                table.join_prefix(s, 0)
        for t, x in zip((q, k, v), qkv_of(seqs, BF, g)):
            t.copy_(x)
        counts.copy_(i32([int(s in present) for s in range(4)] + [1]))
        graph.replay()
        torch.cuda.synchronize()
        check_step(layer, q, out, step, BF)
        assert (out[int(counts.sum()):] == 0).all()
