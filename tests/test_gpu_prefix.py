"""Decode over shared prefixes against the attention of every sequence by itself in 64 bits, over 16-bit and 8-bit pages."""
from __future__ import annotations

import math

import pytest
import torch

from flashquant_amd import kernels as K
from flashquant_amd.kernels._native import native
from tests.test_gpu_kv8 import BF, DEV, E4, E8, HEADS, HF, U8, attended, caches, check, gen, raw, stood_for

pytestmark = pytest.mark.gpu
BITS = [16, 8]


def cache_of(bits, layout, blocks, page, hkv, d, dtype, g):
    """(key cache, value cache, key scales, value scales), scales None at 16 bits."""
    kc, vc, ks, vs, _ = caches(layout, blocks, page, hkv, d, g)
    if bits == 8:
        return kc, vc, ks, vs
    t = torch.randn(2, blocks, page, hkv, d, generator=g).to(dtype).to(DEV)
    if layout == "heads first":
        t = t.transpose(2, 3).contiguous().transpose(2, 3)
    return t[0], t[1], None, None


def prefix_case(prefixes, ids, own, hq, hkv, d, page, dtype, bits, seed=0, layout="apart", extra_columns=0, scale=2.0):
    """`own`: tokens of every sequence behind the whole pages of its prefix; negative: so many less than its prefix has."""
    g = gen(seed)
    pages = [n // page if n > 0 else 0 for n in prefixes]
    there = [0 <= i < len(prefixes) for i in ids]
    lens = [n + (pages[i] * page if ok else 0) for i, n, ok in zip(ids, own, there)]
    columns = max([1] + [-(-n // page) for n in lens]) + extra_columns
    blocks = sum(pages) + sum(-(-max(n, 0) // page) for n in lens) + 3
    cache = cache_of(bits, layout, blocks, page, hkv, d, dtype, g)
    order = torch.randperm(blocks, generator=g).int()
    begin = [sum(pages[:i]) for i in range(len(pages))]
    at = sum(pages)
    table = torch.full((len(ids), columns), 1 << 30, dtype=torch.int32)
    for s, (i, n, ok) in enumerate(zip(ids, lens, there)):
        used = -(-max(n, 0) // page)
        same = min(pages[i], used) if ok and n >= pages[i] * page else 0
        table[s, :same] = order[begin[i]:begin[i] + same] if same else table[s, :0]
        table[s, same:used] = order[at:at + used - same]
        at += used - same
    q = (torch.randn(len(ids), hq, d, generator=g) * scale).to(dtype).to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    return q, cache, table.to(DEV), torch.tensor(lens, **i32), torch.tensor(ids, **i32), torch.tensor(prefixes, **i32)


def wanted(q, cache, table, lens, ids, prefixes, sm):
    """`attended`, with the rounding of weights over shared tokens in the tolerance."""
    kc, vc, ks, vs = cache
    keys, values = (c.double() if s is None else stood_for(c, s) for c, s in ((kc, ks), (vc, vs)))
    o, l, to, tl = attended(q, keys, values, table, lens, sm)
    weight = torch.finfo(q.dtype).eps / 2
    # sum of weights times sizes, with the size of values as the value
    size, _, _, _ = attended(q, keys, values.abs(), table, lens, sm)
    most = values[torch.isfinite(values)].abs().max()
    return o, l, to + (size * weight + most * lens.max().clamp(min=0) * 2.0 ** -34) * (1 + 2.0 ** -6), tl


def call(q, cache, table, lens, ids, prefixes, sm=None, **more):
    kc, vc, ks, vs = cache
    return K.paged_prefix_decode(q, kc, vc, table, lens, ids, prefixes, sm, key_scales=ks, value_scales=vs, return_lse=True, **more)


def check_prefix(q, cache, table, lens, ids, prefixes, sm=None, **more):
    sm = 1.0 / math.sqrt(q.shape[-1]) if sm is None else sm
    return check(call(q, cache, table, lens, ids, prefixes, sm, **more), wanted(q, cache, table, lens, ids, prefixes, sm), q)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [8, 16, 32])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_one_prefix_of_a_batch(hq, hkv, d, page, dtype, bits):
    check_prefix(*prefix_case([333], [0] * 12, [0, 1, 7, 31, 32, 33, 64, 100, 300, 5, 2, 1], hq, hkv, d, page, dtype, bits, seed=hq + page))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
# one sequence; two; a long prefix of few; rows of several groups; several prefixes, some of them of nobody, of no page, of fewer tokens than
# a page; sequences of their own, with ids beyond the prefixes, shorter than their prefix, without tokens
@pytest.mark.parametrize("prefixes,ids,own", [([64], [0], [5]), ([1000], [0, 0], [0, 0]), ([9000], [0, 0, 0], [40, 1, 2000]), ([500], [0] * 150, [3, 40] * 75),
                                              ([100, 700, 0, 7, 2000, 64, -9], [4, 0, 1, 4, 3, 2, 1, 4, 4, 6, 0], [1, 2, 3, 700, 9, 50, 1, 0, 33, 12, 70]),
                                              ([400, 96], [-1, 0, 9, 1, 0, -(1 << 31), 1, 0, 1 << 30, 1], [50, 3, 700, 5, -1, 0, -96, -500, 1, 20]),
                                              ([], [0, -1, 3], [40, 0, 900])])
def test_mixed_batches(prefixes, ids, own, hq, hkv, d, bits):
    check_prefix(*prefix_case(prefixes, ids, own, hq, hkv, d, 16, BF, bits, seed=len(ids)))


@pytest.mark.parametrize("bits", BITS)
def test_many_sequences_and_prefixes(bits):
    g = gen(5)
    prefixes = torch.randint(0, 200, (300,), generator=g).tolist()
    ids = torch.randint(-20, 300, (1100,), generator=g).tolist()
    own = torch.randint(0, 60, (1100,), generator=g).tolist()
    check_prefix(*prefix_case(prefixes, ids, own, 4, 1, 64, 8, BF, bits))
    check_prefix(*prefix_case([120] * 1024, [i % 1024 for i in range(1030)], [3] * 1030, 2, 2, 64, 8, HF, bits))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("members,hq,hkv,d", [(200, 16, 1, 128), (70, 64, 8, 128), (40, 12, 4, 64), (90, 9, 1, 256)])
def test_groups_of_rows(members, hq, hkv, d, bits):
    """Members that fill several workgroups' rows, with others between them, over a prefix of many tiles and in dirty room."""
    ids = [0 if i % 3 else -1 for i in range(members + members // 2)]
    case = prefix_case([3100], ids, [i % 90 for i in range(len(ids))], hq, hkv, d, 32, BF, bits, extra_columns=9)
    room = native().paged_prefix_decode_workspace_bytes(len(ids), hq, hkv, d, 1)
    check_prefix(*case, workspace=torch.full((room,), 0xff, dtype=U8, device=DEV))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("hq,hkv", [(2, 1), (8, 8)])
@pytest.mark.parametrize("own", [[1] * 40 + [0] * 660, [0, 0, 33, 0, 64, 0, 0, 0, 1, 0] * 70, [5000] + [0] * 598 + [3], [0] * 598 + [2, 900], [0] * 600])
def test_shares_that_hold_little(own, hq, hkv, bits):
    """Batches too large to be kept in registers with few tokens of their own: shares smaller than what a sequence counts for, shares without
    a tile, one long sequence among many."""
    ids = [(0, 1, -1)[s % 3] for s in range(len(own))]
    check_prefix(*prefix_case([130, 700], ids, own, hq, hkv, 64, 16, BF, bits, seed=len(own) + hq))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("members,tokens", [(17, [2048]), (100, [2112]), (48, [8192, 64, 1000]), (33, [64] * 5), (9, [16384])])
def test_shares_and_groups_of_rows(members, tokens, bits):
    """Prefixes whose tiles go evenly into shares, almost so, and not at all."""
    ids = [s % len(tokens) for s in range(members)]
    check_prefix(*prefix_case(tokens, ids, [s % 5 for s in range(members)], 32, 4, 128, 32, BF, bits, seed=members))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_missing_pages_and_what_lies_beyond(d, bits):
    """Pages outside the cache in the prefix and behind it; NaN in all that is not seen, a prefix that ends inside a tile."""
    q, cache, table, lens, ids, prefixes = prefix_case([344, 80], [0, 1, 0, 0, 1, -1], [3, 40, 0, 170, 9, 33], 8, 2, d, 8, BF, bits, seed=d)
    kc, vc, ks, vs = cache
    for s, i in enumerate(ids.tolist()):
        if i == 0:
            table[s, 3], table[s, 10:15], table[s, 40] = -1, 1 << 20, kc.shape[0]
    table[1, 13] = -5
    want = wanted(q, cache, table, lens, ids, prefixes, 0.125)
    seen = torch.zeros(kc.shape[:2], dtype=torch.bool, device=DEV)
    for s, n in enumerate(lens.tolist()):
        t = torch.arange(n, device=DEV)
        b = table[s, t // 8].long()
        ok = (b >= 0) & (b < kc.shape[0])
        seen[b[ok], (t % 8)[ok]] = True
    if bits == 8:
        raw(kc)[~seen], raw(vc)[~seen] = 0x7f, 0xff
        b, t = torch.nonzero(~seen, as_tuple=True)
        raw(ks)[b, :, t], raw(vs)[b, :, t] = 255, 255
    else:
        kc[~seen], vc[~seen] = math.nan, math.inf
    check(call(q, cache, table, lens, ids, prefixes, 0.125), want, q)
    # all of a prefix missing: only what lies behind it is seen
    for s, i in enumerate(ids.tolist()):
        if i == 1:
            table[s, :10] = -1
    want = wanted(q, cache, table, lens, ids, prefixes, 0.125) if bits == 16 else None
    out, lse = call(q, cache, table, lens, ids, prefixes, 0.125)
    assert torch.isfinite(out).all()
    if want is not None:
        keys, values = (torch.where(seen[..., None, None], c, 0.0) for c in (kc, vc))
        check((out, lse), wanted(q, (keys, values, None, None), table, lens, ids, prefixes, 0.125), q)


@pytest.mark.parametrize("bits", BITS)
def test_lengths_beyond_the_table_and_below_zero(bits):
    q, cache, table, lens, ids, prefixes = prefix_case([160], [0, 0, 0, 0], [32, 32, 32, 32], 4, 4, 64, 16, BF, bits)
    check_prefix(q, cache, table, torch.tensor([1 << 30, -5, 192, 159], dtype=torch.int32, device=DEV), ids, prefixes)
    # a prefix longer than the table has nobody
    check_prefix(q, cache, table, lens, ids, torch.tensor([(1 << 31) - 1], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("layout", ["heads first", "together", "one record"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_strided_operands(d, layout, bits):
    if bits == 16 and layout != "heads first":
        pytest.skip("the layouts of 16-bit caches are those of paged_kv_decode")
    q, *rest = prefix_case([200], [0, 0, -1, 0], [70, 1, 900, 20], 8, 4, d, 16, BF, bits, seed=d, layout=layout)
    out, lse = check_prefix(q, *rest)
    wide = torch.zeros(4, 11, d + 8, dtype=BF, device=DEV)
    wide[:, 2:10, :d] = q
    assert torch.equal(call(wide[:, 2:10, :d], *rest)[0], out)
    odd = torch.zeros(4, 8, d + 3, dtype=BF, device=DEV)
    odd[..., 3:] = q
    assert torch.equal(call(odd[..., 3:], *rest)[0], out)
    cache, table, lens, ids, prefixes = rest
    padded = torch.zeros(4, table.shape[1] + 5, dtype=torch.int32, device=DEV)
    padded[:, :table.shape[1]] = table
    pairs = torch.stack([ids, ids], 1)
    big = torch.full((6, 8, d), 7.0, dtype=BF, device=DEV)
    call(q, cache, padded[:, :table.shape[1]], torch.stack([lens, lens], 1)[:, 0], pairs[:, 1], torch.stack([prefixes, prefixes], 1)[:, 0], out=big[1:5])
    assert torch.equal(big[1:5], out) and (big[0] == 7).all() and (big[5] == 7).all()


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_scores_far_apart_and_values_at_the_ends(dtype, bits):
    case = prefix_case([700, 300], [0, 1, 0, 0, 1], [300, 5, 0, 40, 1], 8, 2, 128, 16, dtype, bits, seed=9, scale=30.0)
    for sm in (None, -0.3, 0.0, 1.0):
        check_prefix(*case, sm=sm)
    q, cache, table, lens, ids, prefixes = prefix_case([700, 300], [0, 1, 0, 0, 1], [300, 5, 0, 40, 1], 8, 2, 128, 16, dtype, bits, seed=3)
    kc, vc, ks, vs = cache
    if bits == 16:
        vc.mul_(1e36 if dtype == BF else 10000).clamp_(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    else:
        raw(vs).copy_(torch.randint(240, 246, vs.shape, generator=gen(3)).to(U8) if dtype == BF else torch.randint(100, 133, vs.shape, generator=gen(3)).to(U8))
        raw(ks).copy_(torch.randint(100, 122, vs.shape, generator=gen(4)).to(U8))
    check_prefix(q, cache, table, lens, ids, prefixes)
    # NaN in a shared value and key shows in those that see them, in that coordinate
    b0 = int(table[1, 3])
    if bits == 16:
        vc[b0, 1, 0, 5], kc[b0, 2, 1, 5] = math.nan, math.nan
    else:
        raw(vc)[b0, 1, 0, 5], raw(kc)[b0, 2, 1, 5] = 0x7f, 0x7f
    o, l = call(q, cache, table, lens, ids, prefixes)
    for s in (1, 4):
        assert torch.isnan(o[s, :4, 5]).all() and torch.isfinite(o[s, :4, :5]).all() and torch.isnan(o[s, 4:]).all() and torch.isnan(l[s, 4:]).all()
        assert torch.isfinite(l[s, :4]).all()
    assert torch.isfinite(o[[0, 2, 3]]).all()


def test_rows_without_a_score_are_empty():
    q, cache, table, lens, ids, prefixes = prefix_case([320], [0, 0, -1], [40, 0, 9], 8, 2, 128, 16, BF, 16)
    q.fill_(1.0)
    cache[0][table[0, :20].long()] = -math.inf                           # all keys of the prefix
    o, l = call(q, cache, table, lens, ids, prefixes)
    assert (o[1] == 0).all() and torch.isneginf(l[1]).all() and torch.isfinite(l[0]).all() and torch.isfinite(o).all()
    want, lw = K.paged_kv_decode(q[:1], cache[0], cache[1], table[:1, 20:].contiguous(), lens[:1] - 320, return_lse=True)
    assert torch.allclose(o[:1].float(), want.float(), rtol=2.0 ** -7, atol=1e-6) and torch.allclose(l[:1], lw, rtol=1e-5)


@pytest.mark.parametrize("bits", BITS)
def test_beyond_32_bit_offsets(bits):
    """Pages at the far end of a cache of more than 2^31 elements (8 bits: 2^32 bytes)."""
    page, hkv, d = 32, 8, 128
    blocks, g = (1 << (31 if bits == 16 else 32)) // (page * hkv * d) + 40, gen(5)
    small = cache_of(bits, "apart", 39, page, hkv, d, BF, g)
    big = [torch.zeros(blocks, *t.shape[1:], dtype=U8 if bits == 8 else BF, device=DEV) if t is not None else None for t in small]
    for b, t in zip(big, small):
        if t is not None:
            b[-39:] = raw(t) if bits == 8 else t
    if bits == 8:
        big = [b.view(E4 if i < 2 else E8) for i, b in enumerate(big)]
    table = torch.arange(38, -1, -1, dtype=torch.int32, device=DEV).repeat(3, 1)
    table[1, 20:], table[2, 20:] = table[1, 20:].flip(0), table[2, 20:].roll(3)
    q = torch.randn(3, 32, d, generator=g).to(BF).to(DEV)
    lens, ids = torch.tensor([39 * 32, 30 * 32 + 9, 20 * 32], dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    prefixes = torch.tensor([20 * 32], dtype=torch.int32, device=DEV)
    want = check_prefix(q, small, table, lens, ids, prefixes)
    got = call(q, big, table + (blocks - 39), lens, ids, prefixes)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_of_nothing_and_refusals():
    q, (kc, vc, _, _), table, lens, ids, prefixes = prefix_case([64, 32], [0, 1, 0], [40, 5, 1], 8, 2, 128, 16, BF, 16)
    k8, v8, ks, vs = cache_of(8, "apart", kc.shape[0], 16, 2, 128, BF, gen(1))
    good = dict(q=q, key_cache=kc, value_cache=vc, block_table=table, seq_lens=lens, prefix_ids=ids, prefix_lens=prefixes)
    eight = dict(key_cache=k8, value_cache=v8, key_scales=ks, value_scales=vs)
    K.paged_prefix_decode(**good)
    K.paged_prefix_decode(**(good | eight))
    assert K.paged_prefix_decode(q[:0], kc, vc, table[:0], lens[:0], ids[:0], prefixes).shape == (0, 8, 128)
    for bad in (dict(q=q.float()), dict(q=q[..., :64]), dict(q=q[0]), dict(q=q[:, :7]), dict(q=q.half()), dict(key_cache=kc[:, :12], value_cache=vc[:, :12]),
                dict(value_cache=vc[:2]), dict(key_cache=kc[:0], value_cache=vc[:0]), dict(key_cache=k8, value_cache=v8), dict(key_scales=ks), dict(key_scales=ks, value_scales=vs),
                eight | dict(key_scales=raw(ks)), eight | dict(value_scales=None), dict(block_table=table.long()), dict(block_table=table[:1]), dict(block_table=table[:, :0]),
                dict(seq_lens=lens.long()), dict(seq_lens=lens[:1]), dict(prefix_ids=ids.long()), dict(prefix_ids=ids[:2]), dict(prefix_ids=ids.cpu()),
                dict(prefix_lens=prefixes.long()), dict(prefix_lens=prefixes[None]), dict(prefix_lens=prefixes.cpu()),
                dict(prefix_lens=torch.zeros(1025, dtype=torch.int32, device=DEV)), dict(out=q), dict(out=torch.empty(3, 8, 128, device=DEV)),
                dict(out=torch.empty(3, 16, 128, dtype=BF, device=DEV)[:, :8]), dict(out=kc.view(-1)[:q.numel()].view_as(q)),
                eight | dict(out=raw(v8).view(-1)[:2 * q.numel()].view(BF).view_as(q))):
        with pytest.raises(ValueError):
            K.paged_prefix_decode(**(good | bad))
    with pytest.raises(ValueError, match="workspace"):
        K.paged_prefix_decode(**good, workspace=torch.empty(256, dtype=U8, device=DEV))
    odd = torch.zeros(kc.numel() + 1, dtype=BF, device=DEV)[1:].view_as(kc)
    with pytest.raises(ValueError):
        K.paged_prefix_decode(**(good | dict(key_cache=odd)))


def test_room_does_not_shrink():
    bytes_of = native().paged_prefix_decode_workspace_bytes
    for hq, hkv, d in HEADS:
        for many in (0, 1, 5, 1024):
            got = [bytes_of(s, hq, hkv, d, many) for s in range(1, 400)]
            assert got == sorted(got)
        assert [bytes_of(60, hq, hkv, d, n) for n in range(200)] == sorted(bytes_of(60, hq, hkv, d, n) for n in range(200))
