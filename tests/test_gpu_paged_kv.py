"""Operators around a 16-bit paged cache against plain implementations in 64 bits: page scheduling, rotary positions and their
gradient, rotary store, decode; each at the sizes, strides and masks where it can go wrong, and all of them as a serving loop runs
them, over 16-bit layers and over packed ones."""
from __future__ import annotations

import math

import pytest
import torch

from flashquant_amd import kernels as K
from flashquant_amd.kernels._native import native
from flashquant_amd.vllm.impl import TQ4AttentionKernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- rotary positions ---------------------------------------------------------------------------------------------------------

def turned(x, positions, freq, interleaved=False, scale=1.0, sign=1.0):
    """The definition in 64 bits; x (..., tokens, H, D), positions (..., tokens)."""
    half, y = freq.shape[0], x.double().clone()
    a = (positions.double()[..., None] * freq.double())[..., None, :]
    c, s = scale * a.cos(), sign * scale * a.sin()
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    x0, x1 = x[..., i].double(), x[..., j].double()
    y[..., i], y[..., j] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


def turn_tolerance(x, y, positions, freq, interleaved=False, scale=1.0):
    """Rounding of the result, of cosine, sine, two products and their sum in float32, and of the angle in 64 bits."""
    half, tol = freq.shape[0], torch.zeros_like(y)
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    size = scale * (x[..., i].double().abs() + x[..., j].double().abs())
    angle = (positions.double().abs()[..., None] * freq.double())[..., None, :]
    tol[..., i] = tol[..., j] = size * (4 * 2.0 ** -24 + angle * 2.0 ** -51)
    info = torch.finfo(x.dtype)
    return tol + (y.abs() + tol) * info.eps / 2 + (0 if x.dtype == F32 else info.tiny * info.eps)


def check_turn(got, x, positions, freq, interleaved=False, scale=1.0, sign=1.0):
    want = turned(x, positions, freq, interleaved, scale, sign)
    off = (got.double() - want).abs() - turn_tolerance(x, want, positions, freq, interleaved, scale)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert (off <= 0).all(), float(off.max())
    rest = 2 * freq.shape[0]
    assert torch.equal(got[..., rest:], x[..., rest:])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
# one token; heads spread over workgroups; several tokens a workgroup and a last one with fewer; heads that are no power of two;
# part of a head; a pair a head; widths that are no multiple of 16 bytes; an odd head; more units than threads
@pytest.mark.parametrize("tokens,hq,hk,d,rot", [(1, 1, 1, 64, 64), (1, 32, 8, 128, 128), (5, 64, 8, 128, 64), (2050, 4, 1, 128, 128), (130, 7, 3, 256, 64),
                                                (33, 3, 2, 80, 80), (19, 3, 1, 96, 32), (7, 2, 2, 20, 6), (9, 1, 5, 33, 2), (3, 2, 1, 1024, 1024), (6, 5, 0, 128, 128)])
def test_rotary_against_the_formula(tokens, hq, hk, d, rot, interleaved, dtype):
    g = gen(tokens + d)
    q, k = (torch.randn(tokens, h, d, generator=g).to(dtype).to(DEV) for h in (hq, max(hk, 1)))
    k = k if hk else None
    freq, _ = K.rotary_frequencies(rot, device=DEV)
    positions = torch.randint(0, 200000, (tokens,), generator=g).to(DEV)
    positions[0] = 0
    qo, ko = K.rotary_embedding(q, k, positions, freq, interleaved=interleaved, scale=1.25)
    check_turn(qo, q, positions, freq, interleaved, 1.25)
    if hk:
        check_turn(ko, k, positions, freq, interleaved, 1.25)
    else:
        assert ko is None
    # int32 positions and the way back
    again, _ = K.rotary_embedding(q, k, positions.int(), freq, interleaved=interleaved, scale=1.25)
    assert torch.equal(again, qo)
    back, _ = K.rotary_embedding(q, k, positions, freq, interleaved=interleaved, inverse=True)
    check_turn(back, q, positions, freq, interleaved, 1.0, -1.0)


def test_rotary_at_far_and_negative_positions():
    positions = torch.tensor([0, 1, -1, 131071, 1 << 20, 16777217, -99999999, (1 << 31) - 1, 1 << 33], device=DEV)
    g = gen(1)
    q, k = (torch.randn(positions.shape[0], h, 64, generator=g).to(DEV) for h in (2, 1))
    freq, _ = K.rotary_frequencies(64, base=500000.0, device=DEV)
    qo, ko = K.rotary_embedding(q, k, positions, freq)
    check_turn(qo, q, positions, freq)
    check_turn(ko, k, positions, freq)


def test_rotary_rows_that_are_no_numbers_stay_in_their_pairs():
    freq, _ = K.rotary_frequencies(32, device=DEV)
    q = torch.ones(2, 1, 64, dtype=BF, device=DEV)
    q[0, 0, 3], q[1, 0, 40] = math.nan, math.inf
    out, _ = K.rotary_embedding(q, None, torch.tensor([0, 7], device=DEV), freq)
    bad = ~torch.isfinite(out)
    assert bad[0, 0, 3] and bad[0, 0, 19] and out[1, 0, 40] == math.inf and int(bad.sum()) == 3


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_rotary_of_strided_rows_in_batches(dtype, off):
    """Slices of one matrix product, a batch with shared and with its own positions, heads before tokens, rows at odd addresses."""
    b, n, hq, hk, d = 3, 37, 4, 2, 64
    g = gen(2)
    qkv = torch.randn(b, n, hq + 2 * hk, d + off, generator=g).to(dtype).to(DEV)
    q, k = qkv[:, :, :hq, off:], qkv[:, :, hq:hq + hk, off:]
    freq, _ = K.rotary_frequencies(d, device=DEV)
    for positions in (torch.randint(0, 5000, (b, n), generator=g).to(DEV), torch.randint(0, 5000, (n,), generator=g).to(DEV)):
        wide = positions if positions.dim() == 2 else positions.expand(b, n)
        qo, ko = K.rotary_embedding(q, k, positions, freq)
        check_turn(qo, q, wide, freq)
        check_turn(ko, k, wide, freq)
        before = q.transpose(1, 2).contiguous().transpose(1, 2)          # (b, n, h, d) with the heads before the tokens
        out = torch.empty_like(before)
        K.rotary_embedding(before, None, positions, freq, out=(out, None))
        assert torch.equal(out, qo)
        # in place, side by side in one buffer; the values stay
        whole = qkv.clone()
        K.rotary_embedding(whole[:, :, :hq, off:], whole[:, :, hq:hq + hk, off:], positions, freq,
                           out=(whole[:, :, :hq, off:], whole[:, :, hq:hq + hk, off:]))
        want = qkv.clone()
        want[:, :, :hq, off:], want[:, :, hq:hq + hk, off:] = qo, ko
        assert torch.equal(whole, want)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_has_the_same_bits_at_every_size_and_alignment(interleaved, dtype):
    """More than goes through the shared cache, a part of it, and rows at odd addresses."""
    n, h, d, rot = 9000, 40, 256 if dtype != F32 else 128, 96
    g = torch.Generator(device=DEV).manual_seed(8)
    q = torch.randn(n, h, d, generator=g, device=DEV).to(dtype)
    freq, scale = K.rotary_frequencies(rot, 500000.0, "bands", factor=8.0, original_max_position=8192, device=DEV)
    positions = torch.randint(0, 131072, (n,), generator=g, device=DEV)
    out, _ = K.rotary_embedding(q, None, positions, freq, interleaved=interleaved, scale=0.75)
    check_turn(out[-500:], q[-500:], positions[-500:], freq, interleaved, 0.75)
    part, _ = K.rotary_embedding(q[:777, :3], None, positions[:777], freq, interleaved=interleaved, scale=0.75)
    assert torch.equal(part, out[:777, :3])
    odd = torch.empty(n, h, d + 1, dtype=dtype, device=DEV)[..., 1:]
    odd.copy_(q)
    assert torch.equal(K.rotary_embedding(odd, None, positions, freq, interleaved=interleaved, scale=0.75)[0], out)


def test_rotary_of_columns_apart_and_expanded_inputs():
    g = gen(3)
    freq, _ = K.rotary_frequencies(32, device=DEV)
    positions = torch.arange(11, device=DEV)
    q = torch.randn(11, 3, 128, generator=g).to(BF).to(DEV)[:, :, ::2]
    k = torch.randn(11, 1, 64, generator=g).to(BF).to(DEV).expand(11, 4, 64)
    qo, ko = K.rotary_embedding(q, k, positions, freq)
    check_turn(qo, q, positions, freq)
    check_turn(ko, k, positions, freq)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(interleaved):
    """Against the formula, against differences of the operator itself, and of the gradient once more."""
    t, h, d, rot = 23, 3, 64, 48
    g = gen(4)
    freq, scale = K.rotary_frequencies(rot, scaling="yarn", factor=4.0, original_max_position=64, device=DEV)
    positions = torch.randint(0, 300, (t,), generator=g).to(DEV)
    q, k, dq, dk, vq, vk = (torch.randn(t, n, d, generator=g).to(DEV) for n in (h, 1, h, h, h, 1))
    q.requires_grad_()
    k.requires_grad_()
    shared = k.expand(t, h, d)                                            # a head that all others share
    qo, ko = K.rotary_embedding(q, shared, positions, freq, interleaved=interleaved, scale=scale)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk), create_graph=False, retain_graph=True)
    check_turn(gq, dq, positions, freq, interleaved, scale, -1.0)
    want = turned(dk, positions, freq, interleaved, scale, -1.0).sum(1, keepdim=True)
    assert (gk.double() - want).abs().max() <= h * 12 * 2.0 ** -24 * scale * dk.abs().max() * 2
    with torch.no_grad():                                                 # linear: a difference is the derivative, to rounding
        q1, k1 = K.rotary_embedding(q + vq, (k + vk).expand(t, h, d), positions, freq, interleaved=interleaved, scale=scale)
    left = ((q1 - qo.detach()).double() * dq).sum() + ((k1 - ko.detach()).double() * dk).sum()
    right = (gq.double() * vq).sum() + (gk.double() * vk).sum()
    size = float((q1.abs() + qo.detach().abs()).double().mul(dq.abs()).sum() + (k1.abs() + ko.detach().abs()).double().mul(dk.abs()).sum())
    assert abs(float(left - right)) <= 16 * 2.0 ** -24 * size
    # only one of the two, sums (whose gradient is expanded), and a second derivative
    only, = torch.autograd.grad(ko.sum(), (k,), retain_graph=True)
    want = turned(torch.ones_like(dk), positions, freq, interleaved, scale, -1.0).sum(1, keepdim=True)
    assert (only.double() - want).abs().max() <= h * 12 * 2.0 ** -24 * scale * 2
    dy = dq.clone().requires_grad_()
    first, = torch.autograd.grad(qo, (q,), dy, create_graph=True)
    second, = torch.autograd.grad(first, (dy,), vq)
    check_turn(second, vq, positions, freq, interleaved, scale)


def test_rotary_of_nothing_and_refusals():
    freq, _ = K.rotary_frequencies(64, device=DEV)
    q, k = torch.zeros(0, 4, 64, dtype=BF, device=DEV), torch.zeros(0, 2, 64, dtype=BF, device=DEV)
    qo, ko = K.rotary_embedding(q, k, torch.zeros(0, dtype=torch.long, device=DEV), freq)
    assert qo.shape == q.shape and ko.shape == k.shape
    q, k, p = torch.zeros(5, 4, 64, dtype=BF, device=DEV), torch.zeros(5, 2, 64, dtype=BF, device=DEV), torch.zeros(5, dtype=torch.long, device=DEV)
    for bad in (dict(q=q[0]), dict(q=q.double()), dict(k=k[:4]), dict(k=k.half()), dict(k=k[..., :32]), dict(positions=p[:4]), dict(positions=p.float()),
                dict(positions=p[None]), dict(inv_freq=freq.float()), dict(inv_freq=torch.ones(33, dtype=torch.double, device=DEV)),
                dict(inv_freq=freq[:0]), dict(inv_freq=freq.cpu()), dict(k=k.cpu()), dict(out=(torch.zeros_like(q, dtype=HF), None)),
                dict(out=(torch.zeros(5, 4, 32, dtype=BF, device=DEV), None)), dict(out=(q.flip(0).roll(1)[:, :, :1].expand(5, 4, 64), None)),
                dict(k=None, out=(torch.empty_like(q), k))):
        args = dict(q=q, k=k, positions=p, inv_freq=freq, out=None) | bad
        with pytest.raises(ValueError):
            K.rotary_embedding(args["q"], args["k"], args["positions"], args["inv_freq"], out=args["out"])
    longs = torch.zeros(5 * 4 * 64, dtype=torch.long, device=DEV)
    for out in ((longs.view(BF)[:5 * 4 * 64].view(5, 4, 64), None), (None, longs.view(BF)[:5 * 2 * 64].view(5, 2, 64))):
        with pytest.raises(ValueError):
            K.rotary_embedding(q, k, longs[:5], freq, out=out)
    buf = torch.zeros(6 * 4 * 64, dtype=BF, device=DEV)
    a, b = buf[:5 * 4 * 64].view(5, 4, 64), buf[64:64 + 5 * 4 * 64].view(5, 4, 64)
    for out in ((b, None), (torch.empty_like(a), a)):                     # memory that an input shares
        with pytest.raises(ValueError):
            K.rotary_embedding(a, None if out[1] is None else a[:, :4].clone(), p, freq, out=out)
    with pytest.raises(ValueError):
        K.rotary_embedding(q, q.clone(), p, freq, out=(a, a))
    with pytest.raises(ValueError):
        K.rotary_embedding(q.clone().requires_grad_(), k, p, freq, out=(torch.empty_like(q), torch.empty_like(k)))


def test_rotary_captured_with_its_gradient():
    g, (freq, scale) = gen(8), K.rotary_frequencies(128, 5e5, "linear", factor=4.0, device=DEV)
    q, k = (torch.randn(300, h, 128, generator=g).to(BF).to(DEV).requires_grad_() for h in (8, 2))
    dq, dk = (torch.randn(300, h, 128, generator=g).to(BF).to(DEV) for h in (8, 2))
    positions = torch.arange(300, device=DEV)

    def both_ways():
        y, z = K.rotary_embedding(q, k, positions, freq, scale=scale)
        return [*torch.autograd.grad((y, z), (q, k), (dq, dk)), y.detach(), z.detach()]      # (no record of q and k outlives it)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both_ways()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both_ways()
    for i in range(6):
        with torch.no_grad():
            for t in (q, k, dq, dk):
                t.copy_(torch.randn(t.shape, generator=g))
            positions.add_(1000 * i)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, both_ways()))


def test_what_a_call_writes_is_known_to_autograd():
    """A gradient that needs what a later call has overwritten is refused, not computed from the new values."""
    i32, (freq, _) = dict(dtype=torch.int32, device=DEV), K.rotary_frequencies(64, device=DEV)
    lens, one, table, free = torch.zeros(3, **i32), torch.ones(3, **i32), torch.full((3, 4), -1, **i32), torch.arange(12, **i32)
    s = K.paged_schedule(lens, one, table, free, 16, 3)
    q = torch.randn(3, 2, 64, device=DEV, requires_grad=True)
    y, _ = K.rotary_embedding(q, None, s.positions, freq)
    K.paged_schedule(one, one, table, free, 16, 3, out=s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    for written in ("out", "key_cache", "value_cache"):
        x = torch.randn(3, 2, 64, dtype=BF, device=DEV)
        t = dict(q=x, k=x.clone(), v=x.clone(), positions=s.positions, slot_mapping=s.slot_mapping, inv_freq=freq, out=torch.zeros_like(x),
                 key_cache=torch.zeros(2, 16, 2, 64, dtype=BF, device=DEV), value_cache=torch.zeros(2, 16, 2, 64, dtype=BF, device=DEV))
        w = torch.ones((), dtype=BF, device=DEV, requires_grad=True)
        z = t[written] * w                                                # keeps what the call overwrites
        K.rotary_paged_store(**t)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
        with pytest.raises(ValueError, match="gradient"):
            K.rotary_paged_store(**(t | {written: t[written].clone().requires_grad_()}))
        with torch.no_grad():
            K.rotary_paged_store(**(t | {written: t[written].clone().requires_grad_()}))
    with torch.inference_mode():                                          # whose tensors have no versions
        K.rotary_embedding(x, None, s.positions, freq, out=(torch.zeros_like(x), None))
        K.paged_schedule(one, one, table.clone(), free, 16, 3, out=K.paged_schedule(one, one, table.clone(), free, 16, 3))


# ---- rotary store -------------------------------------------------------------------------------------------------------------

def caches(layout, blocks, page, h, d, dtype, g):
    """(key_cache, value_cache, everything they lie in)."""
    if layout == "apart":
        t = torch.randn(2, blocks, page, h, d, generator=g).to(dtype).to(DEV)
        return t[0], t[1], t
    if layout == "together":
        t = torch.randn(blocks, 2, page, h, d, generator=g).to(dtype).to(DEV)
        return t[:, 0], t[:, 1], t
    if layout == "heads first":
        t = torch.randn(2, blocks, h, page, d, generator=g).to(dtype).to(DEV)
        return t[0].transpose(1, 2), t[1].transpose(1, 2), t
    t = torch.randn(blocks, page, h, 2 * d + 8, generator=g).to(dtype).to(DEV)          # side by side in a row with a gap
    return t[..., :d], t[..., d:2 * d], t


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout", ["apart", "together", "heads first", "one row"])
@pytest.mark.parametrize("tokens,mapped,hq,hkv,d,rot,page,interleaved", [(1, 1, 1, 1, 64, 64, 8, False), (64, 61, 32, 8, 128, 128, 16, False),
                                                                       (2300, 2290, 4, 2, 128, 64, 32, True), (9, 9, 7, 7, 80, 48, 16, False),
                                                                       (5, 0, 2, 1, 64, 32, 16, True), (40, 33, 3, 1, 36, 10, 8, True), (17, 17, 0, 2, 256, 256, 32, False)])
def test_rotary_store(tokens, mapped, hq, hkv, d, rot, page, interleaved, layout, dtype):
    g = gen(tokens + d)
    blocks = tokens // page + 3
    kc, vc, whole = caches(layout, blocks, page, hkv, d, dtype, g)
    qkv = torch.randn(tokens, hq + 2 * hkv, d, generator=g).to(dtype).to(DEV)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    positions = torch.randint(0, 100000, (tokens,), generator=g).to(DEV)
    freq, _ = K.rotary_frequencies(rot, device=DEV)
    slots = torch.randperm(blocks * page, generator=g)[:mapped]
    if mapped > 8:                                                        # not stored
        slots[3], slots[4], slots[5], slots[6] = -1, blocks * page, -(1 << 40), 1 << 40
    kk, want = K.rotary_embedding(k, None, positions, freq, interleaved=interleaved, scale=0.9)[0], whole.clone()
    kw, vw = (torch.as_strided(want, t.shape, t.stride(), t.storage_offset()) for t in (kc, vc))
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < blocks * page:
            kw[s // page, s % page], vw[s // page, s % page] = kk[i], v[i]
    got = K.rotary_paged_store(q, k, v, positions, slots.to(DEV), freq, kc, vc, interleaved=interleaved, scale=0.9)
    assert torch.equal(whole, want)                                       # the rows, and nothing beside them
    assert got.shape == q.shape
    if hq:
        assert torch.equal(got, K.rotary_embedding(q, None, positions, freq, interleaved=interleaved, scale=0.9)[0])
        K.rotary_paged_store(q, k, v, positions, slots.to(DEV), freq, kc, vc, interleaved=interleaved, scale=0.9, out=q)
        assert torch.equal(q, got) and torch.equal(whole, want)


def test_rotary_store_refusals():
    freq, _ = K.rotary_frequencies(64, device=DEV)
    t = dict(q=torch.zeros(5, 4, 64, dtype=BF, device=DEV), k=torch.zeros(5, 2, 64, dtype=BF, device=DEV), v=torch.zeros(5, 2, 64, dtype=BF, device=DEV),
             positions=torch.zeros(5, dtype=torch.long, device=DEV), slot_mapping=torch.arange(5, device=DEV), inv_freq=freq,
             key_cache=torch.zeros(2, 16, 2, 64, dtype=BF, device=DEV), value_cache=torch.zeros(2, 16, 2, 64, dtype=BF, device=DEV))
    K.rotary_paged_store(**t)
    for name, bad in (("q", t["q"].float()), ("q", t["q"][:4]), ("k", t["k"][:, :1]), ("v", t["v"].half()), ("v", t["v"][:, :1]), ("positions", t["positions"][:3]),
                      ("slot_mapping", t["slot_mapping"].int()), ("slot_mapping", torch.arange(6, device=DEV)), ("slot_mapping", t["slot_mapping"].cpu()),
                      ("key_cache", t["key_cache"].half()), ("key_cache", t["key_cache"][:, :, :1]), ("value_cache", t["value_cache"][:1]),
                      ("key_cache", t["key_cache"][:, :12]), ("key_cache", t["key_cache"][:1].expand(2, 16, 2, 64)), ("key_cache", t["key_cache"].cpu()),
                      ("out", torch.zeros(5, 4, 64, device=DEV)), ("out", t["k"].expand(5, 2, 64)), ("q", t["q"].cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            K.rotary_paged_store(**(t | {name: bad}))
    with pytest.raises(ValueError):                                       # pages of 12 tokens
        K.rotary_paged_store(**(t | dict(key_cache=t["key_cache"][:, :12], value_cache=t["value_cache"][:, :12])))
    # memory that two operands share
    both = torch.zeros(5 * 4 * 64 + 2 * 16 * 2 * 64, dtype=BF, device=DEV)
    cache = both[4 * 64:4 * 64 + 2 * 16 * 2 * 64].view(2, 16, 2, 64)
    longs = torch.zeros(5 * 4 * 64, dtype=torch.long, device=DEV)
    for bad in (dict(value_cache=t["key_cache"]), dict(q=both[:5 * 4 * 64].view(5, 4, 64), key_cache=cache), dict(out=both[:5 * 4 * 64].view(5, 4, 64), value_cache=cache),
                dict(v=cache[0, :5], key_cache=cache), dict(k=cache[1, :5], value_cache=cache), dict(out=longs.view(BF)[:5 * 4 * 64].view(5, 4, 64), positions=longs[:5]),
                dict(out=longs.view(BF)[:5 * 4 * 64].view(5, 4, 64), slot_mapping=longs[:5])):
        with pytest.raises(ValueError):
            K.rotary_paged_store(**(t | bad))
    # no pages at all: nothing is stored, the queries are rotated
    got = K.rotary_paged_store(**(t | dict(q=torch.ones_like(t["q"]), key_cache=t["key_cache"][:0], value_cache=t["value_cache"][:0])))
    assert (got[:, :, :32] == 1).all()


def test_rotary_and_store_beyond_32_bit_offsets():
    """The last tokens of 2.4 10^9 elements, and the last pages of as many, against the same rows by themselves."""
    freq, _ = K.rotary_frequencies(128, device=DEV)
    tokens, blocks = 590_000, 147_000
    q = torch.empty(tokens, 32, 128, dtype=BF, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    q[-40:] = torch.randn(40, 32, 128, generator=g, device=DEV).to(BF)
    q[:40] = q[-40:]
    positions = torch.arange(tokens, device=DEV) % 1000
    alone, _ = K.rotary_embedding(q[-40:].clone(), None, positions[-40:].clone(), freq)
    keys, values = (torch.zeros(blocks, 16, 8, 128, dtype=BF, device=DEV) for _ in range(2))
    got, _ = K.rotary_embedding(q, None, positions, freq)
    assert got.numel() > 2 ** 31 and keys.numel() > 2 ** 31 and torch.equal(got[-40:], alone)
    del got
    k, v, slots = alone[:, :8].contiguous(), alone[:, 8:16].contiguous(), torch.arange(blocks * 16 - 40, blocks * 16, device=DEV)
    K.rotary_paged_store(q[:40], k, v, torch.zeros(40, dtype=torch.long, device=DEV), slots, freq, keys, values)   # (position 0: as they are)
    assert torch.equal(keys.view(-1, 8, 128)[-40:], k) and torch.equal(values.view(-1, 8, 128)[-40:], v)
    assert not keys.view(-1, 8, 128)[:-40].any() and not values.view(-1, 8, 128)[:-40].any()


# ---- pages, slots and positions -------------------------------------------------------------------------------------------------

def scheduled(context, query, table, free, start, page, room):
    """(table, slots, positions, lens, cu, end) by loops."""
    table, cap = [row[:] for row in table], len(table[0]) * page if table else 0
    at, slots, positions, lens, cu = start, [], [], [], [0]
    for r, (c, n) in enumerate(zip(context, query)):
        c, n = max(c, 0), max(n, 0)
        held = -(-min(c, cap) // page)
        wanted = -(-min(c + n, cap) // page) - held
        for i in range(wanted):
            block = free[at + i] if 0 <= at + i < len(free) else -1
            first = cu[-1] + (held + i) * page - c                       # of its tokens, among the step's
            if first < room:
                table[r][held + i] = block
        for p in range(c, c + n):
            block = -1
            if p < cap:
                b = p // page
                block = table[r][b] if b < held else (free[at + b - held] if 0 <= at + b - held < len(free) else -1)
            slots.append(block * page + p % page if block >= 0 else -1)
            positions.append(p)
        at += wanted
        lens.append(min(c + n, cap))
        cu.append(cu[-1] + n)
    pad = max(0, room - len(slots))
    return table, (slots + [-1] * pad)[:room], (positions + [0] * pad)[:room], lens, cu, at


def run_schedule(context, query, blocks, free, start, page, room, gap=0, seed=0, use_start=True):
    g = gen(seed)
    n = len(context)
    buf = torch.randint(0, 1000, (n, blocks + gap), dtype=torch.int32, generator=g)
    table = buf[:, :blocks]
    want = scheduled(context, query, table.tolist(), free, start, page, room)
    dev = buf.to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    got = K.paged_schedule(torch.tensor(context, **i32), torch.tensor(query, **i32), dev[:, :blocks], torch.tensor(free, **i32), page, room,
                           free_start=torch.tensor([start], **i32) if use_start else None)
    whole = buf.clone()
    whole[:, :blocks] = torch.tensor(want[0], dtype=torch.int32).view(n, blocks)
    assert torch.equal(dev.cpu(), whole)                                  # entries of new pages, and nothing beside them
    for name, mine, his, t in zip(got._fields, got, want[1:5] + ([want[5]],), (torch.int64, torch.int64, torch.int32, torch.int32, torch.int32)):
        assert mine.dtype == t and mine.tolist() == his, name


@pytest.mark.parametrize("page", [8, 16, 32])
@pytest.mark.parametrize("reqs,most,chunk,extra,gap", [(1, 0, 1, 0, 0), (1, 500, 1, 0, 0), (3, 100, 900, 0, 3), (64, 70, 1, 0, 0), (256, 300, 1, 7, 0), (257, 40, 3, 0, 1),
                                                       (700, 33, 40, 300, 0), (5, 10, 3000, 1, 0)])
def test_schedule_against_loops(page, reqs, most, chunk, extra, gap):
    g = gen(reqs + page)
    context = torch.randint(0, most + 1, (reqs,), generator=g).tolist()
    query = torch.randint(0 if reqs > 2 else 1, chunk + 1, (reqs,), generator=g).tolist()
    blocks = max(-(-(c + n) // page) for c, n in zip(context, query))
    free = torch.randperm(sum(query) + 50, generator=g).tolist()
    run_schedule(context, query, max(1, blocks), free, 5, page, sum(query) + extra, gap)


def test_schedule_at_its_edges():
    run_schedule([16, 32, 0, 15], [1, 0, 16, 1], 3, list(range(9, 20)), 0, 16, 18, use_start=False)      # full pages, no new token, a page's last
    run_schedule([0, 5, 30], [40, 1, 40], 5, [7, 8, 9], 1, 16, 100)                                     # too few pages
    run_schedule([0, 5], [40, 30], 5, [], 0, 16, 70)                                                    # none
    run_schedule([0, 5], [40, 30], 5, [1, 2, 3, 4], -2, 16, 70)                                         # a start before the list
    run_schedule([20, 100, 31, 0], [30, 4, 2, 100], 2, list(range(50)), 0, 16, 140)                     # rows that are full
    run_schedule([-3, 4, -1], [2, -5, 3], 2, list(range(8)), 0, 8, 9)                                   # negative lengths
    run_schedule([3, 9, 12], [700, 2, 600], 50, list(range(100)), 0, 32, 777)                           # less room than tokens
    run_schedule([3, 9], [0, 0], 4, [1], 0, 8, 0)
    run_schedule([3, 9], [1, 1], 4, [1], 0, 8, 0)                                                       # no room at all
    run_schedule([0] * 300 + [40], [0] * 300 + [600], 30, list(range(100)), 0, 32, 600)
    # requests that the threads share out unevenly, and more than they take at a time
    for n in (255, 256, 257, 511, 513, 1500, 2047, 2048, 2049, 5000):
        run_schedule([i % 37 for i in range(n)], [i % 3 for i in range(n)], 6, list(range(n)), 2, 8, n + 1)
    # many requests of one token, and one request over many workgroups
    run_schedule(list(range(3000)), [1] * 3000, 400, list(range(3000)), 0, 8, 3000)
    run_schedule([1], [5000], 700, list(range(3000)), 0, 8, 5100)
    empty = torch.zeros(0, dtype=torch.int32, device=DEV)
    got = K.paged_schedule(empty, empty, torch.zeros(0, 4, dtype=torch.int32, device=DEV), empty, 16, 3)
    assert got.slot_mapping.tolist() == [-1] * 3 and got.positions.tolist() == [0] * 3 and got.cu_seqlens.tolist() == [0] and got.free_end.tolist() == [0]


def test_schedule_writes_given_outputs_and_refuses():
    i32 = dict(dtype=torch.int32, device=DEV)
    context, query, free = torch.tensor([3, 20], **i32), torch.tensor([2, 13], **i32), torch.arange(10, **i32)
    table = torch.zeros(2, 5, **i32)
    a = K.paged_schedule(context, query, table, free, 16, 15)
    kept = [t.clone() for t in a]
    for t in a:
        t.fill_(77)
    b = K.paged_schedule(context, query, table, free, 16, 15, out=a)
    assert all(x.data_ptr() == y.data_ptr() and torch.equal(x, z) for x, y, z in zip(a, b, kept))
    for bad in (dict(context_lens=context.long()), dict(query_lens=query[:1]), dict(block_table=table.long()), dict(block_table=table[:1]),
                dict(block_table=table[0].expand(2, 5)), dict(block_table=table.t().contiguous().t()), dict(free_blocks=free.long()), dict(free_blocks=free[::2]), dict(block_size=12),
                dict(num_tokens=-1), dict(num_tokens=14, out=a), dict(free_start=torch.zeros(2, **i32)), dict(free_start=a.free_end, out=a),
                dict(query_lens=query.cpu()), dict(out=a._replace(seq_lens=context)), dict(out=a._replace(seq_lens=table[0, :2])),
                dict(out=a._replace(positions=a.slot_mapping)), dict(context_lens=table[0, :2]), dict(query_lens=table[1, 2:4]), dict(free_blocks=table[1]),
                dict(free_start=table[0, :1])):
        args = dict(context_lens=context, query_lens=query, block_table=table, free_blocks=free, block_size=16, num_tokens=15) | bad
        with pytest.raises(ValueError):
            K.paged_schedule(**args)


# ---- attention of one new token ---------------------------------------------------------------------------------------------------

def attended(q, kc, vc, table, lens, sm, window=0):
    """(out, lse, tolerance of out, tolerance of lse) from the definition in 64 bits, sequence by sequence."""
    page, hkv, d = kc.shape[1], kc.shape[2], kc.shape[3]
    outs = []
    for s, (row, n) in enumerate(zip(table, lens.tolist())):
        n = min(max(n, 0), table.shape[1] * page)
        token = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        block = row[token // page].long()
        token, block = token[(block >= 0) & (block < kc.shape[0])], block[(block >= 0) & (block < kc.shape[0])]
        k, v = (c[block, token % page].double().transpose(0, 1).contiguous() for c in (kc, vc))           # (hkv, n, d)
        x = q[s].double().view(hkv, -1, d)
        if token.numel() == 0:
            zero = torch.zeros_like(x)
            outs.append([zero, torch.full_like(x[..., 0], -math.inf), zero, torch.zeros_like(x[..., 0])])
            continue
        score = (k @ x.transpose(1, 2).contiguous()).transpose(1, 2).contiguous() * sm                  # (hkv, g, n)
        p = torch.softmax(score, -1)
        o, size = p @ v, p @ v.abs()
        # the score's float32 sum of d products and its scaling
        off = (((k.abs() @ x.abs().transpose(1, 2).contiguous()).amax(1) * abs(sm)) * (d + 4) * 2.0 ** -24)[..., None]
        # a weight's two terms, the exponential, the sums over keys and parts; twice the scores' part: weights and their sum
        tol = size * (2.0 ** -16 + 2 * off + (token.numel() + 64) * 2.0 ** -23)
        info = torch.finfo(q.dtype)
        lse = torch.logsumexp(score, -1)
        outs.append([o, lse, tol + (o.abs() + tol) * info.eps / 2 + info.tiny * info.eps,
                     off[..., 0] + (token.numel() + 64) * 2.0 ** -23 + lse.abs() * 2.0 ** -21 + 2.0 ** -20])
    return [torch.stack([t[i].reshape(-1, d) if i in (0, 2) else t[i].reshape(-1) for t in outs]) for i in range(4)]


def check_decode(q, kc, vc, table, lens, sm=None, window=0, **more):
    sm = 1.0 / math.sqrt(q.shape[-1]) if sm is None else sm
    out, lse = K.paged_kv_decode(q, kc, vc, table, lens, sm, window=window, return_lse=True, **more)
    o, l, to, tl = attended(q, kc, vc, table, lens, sm, window)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == q.shape[:2] and lse.dtype == F32
    off = (out.double() - o).abs() - to
    assert (off <= 0).all(), float(off.max())
    none = torch.isneginf(l)
    assert torch.equal(torch.isneginf(lse), none) and (out[none] == 0).all()
    assert ((lse.double() - l).abs()[~none] <= tl[~none]).all()
    return out, lse


def decode_case(lens, hq, hkv, d, page, dtype, seed=0, layout="apart", extra_columns=0, scale=2.0):
    g = gen(seed)
    columns = max(1, max(-(-n // page) for n in lens)) + extra_columns
    blocks = sum(-(-n // page) for n in lens) + 3
    kc, vc, _ = caches(layout, blocks, page, hkv, d, dtype, g)
    order, at = torch.randperm(blocks, generator=g).int(), 0
    table = torch.full((len(lens), columns), 1 << 30, dtype=torch.int32)   # no page of the cache
    for s, n in enumerate(lens):
        used = -(-n // page)
        table[s, :used] = order[at:at + used]
        at += used
    q = (torch.randn(len(lens), hq, d, generator=g) * scale).to(dtype).to(DEV)
    return q, kc, vc, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)


HEADS = [(1, 1, 128), (8, 8, 64), (32, 8, 128), (16, 1, 256), (12, 4, 64), (5, 1, 128), (32, 2, 128), (6, 2, 256)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [8, 16, 32])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_decode_of_ragged_lengths(hq, hkv, d, page, dtype):
    # no token, one, the edges of a page and of a tile, several tiles a wavefront, parts
    check_decode(*decode_case([0, 1, 7, 8, 31, 32, 33, 64, 255, 256, 257, 1000, 0, 2100], hq, hkv, d, page, dtype, seed=hq + d))


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lens", [[1], [40], [513], [5000], [20011], [3000, 1], [9000, 0, 20, 4000, 77]])
def test_decode_of_few_sequences(lens, hq, hkv, d):
    check_decode(*decode_case(lens, hq, hkv, d, 16, BF, seed=len(lens) + d))


@pytest.mark.parametrize("lens", [list(range(0, 300)), [33] * 257, [1] * 70 + [6000] + [0] * 60 + [2500, 9]])
def test_decode_of_many_sequences(lens):
    q, kc, vc, table, sl = decode_case(lens, 8, 2, 128, 16, HF, seed=7, extra_columns=3)
    out, lse = check_decode(q, kc, vc, table, sl)
    again, lse2 = K.paged_kv_decode(q, kc, vc, table, sl, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)              # the same call, the same bits


# rows of no tokens before, between and after those that have some, by the tens and the hundreds; and so many sequences that their
# lengths are read in several parts
@pytest.mark.parametrize("lens", [[0] * 600 + [2100] + [0] * 130 + [5, 3000] + [0] * 700, [1700, 40] + [0] * 254, [0] * 63 + [4000] + [0] * 64 + [3000, 0],
                                  [900] * 20 + [0] * 500 + [1200] * 30, [n % 97 for n in range(1130)], [0] * 1100, [0] * 1023 + [5000]])
def test_decode_of_padded_batches(lens):
    q, kc, vc, table, sl = decode_case(lens, 8, 2, 64, 32, BF, seed=len(lens), extra_columns=80)
    ws = torch.full((native().paged_kv_decode_workspace_bytes(len(lens), 8, 2, 64, 32, table.shape[1]),), 0xff, dtype=torch.uint8, device=DEV)
    check_decode(q, kc, vc, table, sl, workspace=ws)
    check_decode(q, kc, vc, table, sl, window=100, workspace=ws)


# so many sequences that a workgroup takes four heads of one; so many tokens that a wavefront looks its pages up more than once
@pytest.mark.parametrize("lens,hq,hkv,d,page", [([0, 1, 30, 33, 65, 300, 200] * 40, 16, 8, 64, 16), ([5, 0, 129, 40] * 130, 8, 4, 256, 8), ([70000], 16, 16, 64, 8),
                                                ([40000, 3, 50000], 32, 16, 64, 32), ([38000, 0, 1], 16, 16, 256, 16)])
def test_decode_of_full_workgroups(lens, hq, hkv, d, page):
    check_decode(*decode_case(lens, hq, hkv, d, page, BF, seed=len(lens)))


@pytest.mark.parametrize("layout", ["together", "heads first", "one row"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_of_strided_operands(layout, d):
    q, kc, vc, table, sl = decode_case([70, 1, 900, 2048], 8, 4, d, 16, BF, seed=d, layout=layout)
    out, _ = check_decode(q, kc, vc, table, sl)
    wide = torch.zeros(4, 11, d + 8, dtype=BF, device=DEV)
    wide[:, 2:10, :d] = q
    assert torch.equal(K.paged_kv_decode(wide[:, 2:10, :d], kc, vc, table, sl), out)
    odd = torch.zeros(4, 8, d + 3, dtype=BF, device=DEV)                   # rows at odd addresses, columns apart
    odd[..., 3:] = q
    assert torch.equal(K.paged_kv_decode(odd[..., 3:], kc, vc, table, sl), out)
    apart = torch.zeros(4, 8, 2 * d, dtype=BF, device=DEV)
    apart[..., ::2] = q
    assert torch.equal(K.paged_kv_decode(apart[..., ::2], kc, vc, table, sl), out)
    padded = torch.zeros(4, table.shape[1] + 5, dtype=torch.int32, device=DEV)
    padded[:, :table.shape[1]] = table
    assert torch.equal(K.paged_kv_decode(q, kc, vc, padded[:, :table.shape[1]], sl), out)
    # given memory: its neighbours stay
    big = torch.full((6, 8, d), 7.0, dtype=BF, device=DEV)
    K.paged_kv_decode(q, kc, vc, table, sl, out=big[1:5])
    assert torch.equal(big[1:5], out) and (big[0] == 7).all() and (big[5] == 7).all()


@pytest.mark.parametrize("window", [1, 31, 32, 100, 1000, 5000])
def test_decode_of_a_window(window):
    q, kc, vc, table, sl = decode_case([0, 1, 30, 32, 33, 100, 131, 1500, 4096], 8, 2, 128, 16, BF, seed=window)
    # what lies before the window is not looked at
    for s, n in enumerate(sl.tolist()):
        for t in range(0, max(0, n - window)):
            b = int(table[s, t // 16])
            kc[b, t % 16], vc[b, t % 16] = math.nan, math.inf
    check_decode(q, kc, vc, table, sl, window=window)


def test_decode_looks_at_no_token_behind_the_last_and_at_no_missing_page():
    lens = [5, 33, 640, 1000, 50, 2000]
    q, kc, vc, table, sl = decode_case(lens, 8, 2, 64, 8, HF, seed=3)
    seen = torch.zeros(kc.shape[:2], dtype=torch.bool, device=DEV)
    table[2, 3], table[2, 40:44], table[3, :] = -1, 1 << 20, -7            # pages inside, a run of them, all of a row
    table[5, 100:] = kc.shape[0]
    for s, n in enumerate(lens):
        for t in range(n):
            b = int(table[s, t // 8])
            if 0 <= b < kc.shape[0]:
                seen[b, t % 8] = True
    kc[~seen], vc[~seen] = math.nan, math.nan
    kc[:, :, :, 0][~seen], vc[:, :, :, 1][~seen] = math.inf, -math.inf
    check_decode(q, kc, vc, table, sl)


def test_decode_lengths_beyond_the_table_and_below_zero():
    q, kc, vc, table, _ = decode_case([64, 64, 64], 4, 4, 64, 16, BF)
    check_decode(q, kc, vc, table, torch.tensor([1 << 30, -5, 65], dtype=torch.int32, device=DEV))


def test_decode_of_extreme_values():
    """One key that takes all weight, scores far apart, values at the types' ends; rows of -inf scores are empty, NaN stays."""
    q, kc, vc, table, sl = decode_case([300, 700, 1300], 8, 2, 128, 16, HF, seed=9, scale=30.0)
    check_decode(q, kc, vc, table, sl)
    check_decode(q, kc, vc, table, sl, sm=-0.3)
    check_decode(q, kc, vc, table, sl, sm=0.0)
    vc.mul_(10000).clamp_(-65504, 65504)
    check_decode(q, kc, vc, table, sl, sm=1.0)
    q, kc, vc, table, sl = decode_case([300, 700, 1300], 8, 2, 128, 16, BF, seed=9)
    check_decode(q, kc * 1e-3, vc * 1e30, table, sl)
    q.fill_(1.0)
    kc[int(table[1, 20]), 3, 1] = -math.inf                                # one key of sequence 1 is out
    o, l = K.paged_kv_decode(q, kc, vc, table, sl, return_lse=True)
    k2 = kc.clone()
    k2[int(table[1, 20]), 3, 1] = 0
    k2[int(table[1, 20]), 3, 1, 0] = -60000.0
    want, lw = K.paged_kv_decode(q, k2, vc, table, sl, return_lse=True)
    assert torch.equal(o, want) and torch.equal(l, lw)
    kc[table[2, :82].long()] = -math.inf                                   # all scores of sequence 2: an empty row
    o, l = K.paged_kv_decode(q, kc, vc, table, sl, return_lse=True)
    assert (o[2] == 0).all() and torch.isneginf(l[2]).all() and torch.isfinite(o[:2]).all()
    vc[int(table[0, 3]), 1, 0, 5] = math.nan
    kc[int(table[0, 3]), 2, 1, 5] = math.nan
    o, l = K.paged_kv_decode(q, kc, vc, table, sl, return_lse=True)
    assert torch.isnan(o[0, :4, 5]).all() and torch.isfinite(o[0, :4, :5]).all() and torch.isnan(o[0, 4:]).all() and torch.isnan(l[0, 4:]).all()
    assert torch.isfinite(l[0, :4]).all()


def test_decode_beyond_32_bit_offsets():
    """A cache of more than 2^31 elements, its pages at the far end."""
    page, hkv, d = 32, 8, 128
    blocks = (1 << 31) // (page * hkv * d) + 40
    kc = torch.zeros(blocks, page, hkv, d, dtype=BF, device=DEV)
    vc = torch.zeros_like(kc)
    g = torch.Generator(device=DEV).manual_seed(5)
    kc[-39:], vc[-39:] = (torch.randn(39, page, hkv, d, generator=g, device=DEV).to(BF) for _ in range(2))
    table = torch.arange(blocks - 1, blocks - 39, -1, dtype=torch.int32, device=DEV)[None]
    q = torch.randn(1, 32, d, generator=g, device=DEV).to(BF)
    check_decode(q, kc, vc, table, torch.tensor([37 * 32 + 9], dtype=torch.int32, device=DEV))


def test_decode_of_nothing_and_refusals():
    q, kc, vc, table, sl = decode_case([40, 5], 8, 2, 128, 16, BF)
    assert K.paged_kv_decode(q[:0], kc, vc, table[:0], sl[:0]).shape == (0, 8, 128)
    for bad in (dict(q=q.float()), dict(q=q[..., :64]), dict(q=q[0]), dict(q=q[:, :7]), dict(q=torch.zeros(2, 40, 128, dtype=BF, device=DEV)), dict(q=q.half()),
                dict(key_cache=kc[:, :12], value_cache=vc[:, :12]), dict(value_cache=vc[:2]), dict(key_cache=kc.half()), dict(key_cache=kc[:0], value_cache=vc[:0]),
                dict(key_cache=kc[..., 1:], value_cache=vc[..., 1:]), dict(block_table=table.long()), dict(block_table=table[:1]), dict(block_table=table[:, :0]),
                dict(seq_lens=sl.long()), dict(seq_lens=sl[:1]), dict(seq_lens=sl.cpu()), dict(key_cache=kc.cpu()), dict(window=-1), dict(out=q),
                dict(out=torch.empty(2, 8, 128, device=DEV)), dict(out=torch.empty(2, 16, 128, dtype=BF, device=DEV)[:, :8])):
        args = dict(q=q, key_cache=kc, value_cache=vc, block_table=table, seq_lens=sl) | bad
        with pytest.raises(ValueError):
            K.paged_kv_decode(**args)
    room = torch.zeros(2 * 4000 * 16 * 128, dtype=BF, device=DEV)               # results and workspaces in the operands' memory
    cache, big = room[:kc.numel()].view_as(kc), torch.zeros(2, 4000, dtype=torch.int32, device=DEV)
    for bad in (dict(key_cache=cache, out=room[:q.numel()].view_as(q)), dict(value_cache=cache, out=room[:q.numel()].view_as(q)),
                dict(block_table=big, out=big.view(BF).view(-1)[:q.numel()].view_as(q)), dict(seq_lens=big[0, :2], out=big.view(BF).view(-1)[:q.numel()].view_as(q)),
                dict(key_cache=cache, block_table=big, workspace=room.view(torch.uint8)),
                dict(out=room[:q.numel()].view_as(q), block_table=big, workspace=room.view(torch.uint8)),
                dict(q=room[:q.numel()].view_as(q), block_table=big, workspace=room.view(torch.uint8))):
        with pytest.raises(ValueError, match="share no memory"):
            K.paged_kv_decode(**(dict(q=q, key_cache=kc, value_cache=vc, block_table=table, seq_lens=sl) | bad))
    wide = torch.zeros(kc.numel() + 1, dtype=BF, device=DEV)[1:].view_as(kc)  # a cache at an odd address
    with pytest.raises(ValueError):
        K.paged_kv_decode(q, wide, vc, table, sl)
    long = torch.zeros(2, 4000, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="workspace"):
        K.paged_kv_decode(q, kc, vc, long, sl, workspace=torch.empty(256, dtype=torch.uint8, device=DEV))


@pytest.mark.parametrize("seqs", [1, 5, 40, 300])
@pytest.mark.parametrize("columns", [10, 33, 60, 130, 700])
def test_decode_has_room_for_every_window(seqs, columns):
    """What a call without a window needs suffices with one, however the work is divided then."""
    g = gen(columns)
    kc, vc, _ = caches("apart", 50, 16, 4, 64, BF, g)
    table = torch.randint(0, 50, (seqs, columns), dtype=torch.int32, generator=g).to(DEV)
    lens = torch.randint(0, 16 * columns + 1, (seqs,), dtype=torch.int32, generator=g).to(DEV)
    q = torch.randn(seqs, 4, 64, generator=g).to(BF).to(DEV)
    outs = [K.paged_kv_decode(q, kc, vc, table, lens, window=w).float() for w in (0, 1, 300, 900, 3000, 1 << 20)]
    assert torch.equal(outs[5], outs[0]) and all(torch.isfinite(o).all() for o in outs)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads", [1, 2, 8])
def test_decode_has_room_for_windows_of_every_length(heads, d):
    """The same where the lines between the ways to divide the work lie: tables and windows of 8 to 90 tiles, 1 to 600 sequences."""
    g = gen(heads + d)
    kc, vc, _ = caches("apart", 50, 32, heads, d, BF, g)
    for seqs in (1, 4, 13, 16, 40, 130, 270, 600):
        q, lens = torch.randn(seqs, heads, d, generator=g).to(BF).to(DEV), torch.full((seqs,), 5, dtype=torch.int32, device=DEV)
        for columns in (9, 11, 13, 15, 20, 25, 26, 64, 65, 80, 90):
            table = torch.zeros(seqs, columns, dtype=torch.int32, device=DEV)
            want = K.paged_kv_decode(q, kc, vc, table, lens)
            for tiles in (1, 7, 10, 12, 14, 18, 24, 30, 60, 79):
                assert torch.allclose(K.paged_kv_decode(q, kc, vc, table, lens, window=32 * tiles), want)


def test_decode_joins_two_caches_by_their_normalisers():
    q, kc, vc, table, sl = decode_case([1500], 8, 2, 128, 16, HF, seed=4)
    first = torch.tensor([800], dtype=torch.int32, device=DEV)
    a, la = K.paged_kv_decode(q, kc, vc, table, first, return_lse=True)
    b, lb = K.paged_kv_decode(q, kc, vc, table, sl, window=700, return_lse=True)
    top = torch.maximum(la, lb)
    wa, wb = (la - top).exp()[..., None], (lb - top).exp()[..., None]
    joined = (a.float() * wa + b.float() * wb) / (wa + wb)
    o, _, tol, _ = attended(q, kc, vc, table, sl, 1 / math.sqrt(128))
    # each part is rounded once more, its share of the result
    more = (a.float().abs() * wa + b.float().abs() * wb) / (wa + wb) * torch.finfo(HF).eps
    assert ((joined.double() - o).abs() <= tol * 2 + more).all()


@pytest.mark.parametrize("reqs", [1, 2, 5, 200, 256, 257, 700, 3000])
def test_capped_schedule_is_that_of_the_tokens_with_room(reqs):
    g = gen(reqs)
    i32 = dict(dtype=torch.int32, device=DEV)
    for page, blocks, chunk in ((8, 60, 3), (16, 4, 100), (32, 20, 1)):
        context = torch.randint(0, 30, (reqs,), generator=g)
        query = torch.randint(0, chunk + 1, (reqs,), generator=g)
        free, total = torch.randperm(max(1, int(query.sum())), generator=g).to(**i32), int(query.sum())
        for room in sorted({0, 1, total // 3, total - 1, total, total + 9} - {-1}):
            before = torch.cumsum(query, 0) - query
            with_room = (room - before).clamp(min=0).minimum(query)
            outs = []
            for q, capped in ((query, True), (with_room, False)):
                table = torch.full((reqs, blocks), -1, **i32)
                s = K.paged_schedule(context.to(**i32), q.to(**i32), table, free, page, room, free_start=torch.tensor([2], **i32), capped=capped)
                outs.append([table, *s])
            for name, a, b in zip(("table",) + s._fields, *outs):
                assert torch.equal(a, b), (name, room, total)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_in_forward_mode(interleaved, dtype):
    """The map is linear: the tangent is the operator on the tangent; also of a gradient, and beside one."""
    import torch.autograd.forward_ad as fwAD
    t, h, d, rot = 19, 3, 64, 48
    g = gen(11)
    freq, _ = K.rotary_frequencies(rot, device=DEV)
    positions = torch.randint(0, 300, (t,), generator=g).to(DEV)
    q, k, vq, vk, dy, vy = (torch.randn(t, n, d, generator=g).to(dtype).to(DEV) for n in (h, 1, h, 1, h, h))
    args = dict(interleaved=interleaved, scale=1.5)
    want = K.rotary_embedding(q, k, positions, freq, **args)
    for tq, tk, inverse in ((vq, vk, False), (vq, None, False), (None, vk, False), (vq, vk, True)):
        with fwAD.dual_level():
            a, b = (x if v is None else fwAD.make_dual(x, v) for x, v in ((q, tq), (k, tk)))
            outs = K.rotary_embedding(a, b, positions, freq, inverse=inverse, **args)
            for y, v, w in zip(outs, (tq, tk), want):
                primal, tangent = fwAD.unpack_dual(y)
                assert inverse or torch.equal(primal, w)
                if v is not None:
                    check_turn(tangent, v, positions, freq, interleaved, 1.5, -1.0 if inverse else 1.0)
                else:
                    assert tangent is None or not tangent.any()
            with pytest.raises(ValueError, match="gradient"):
                K.rotary_embedding(a, b, positions, freq, out=(torch.empty_like(q), torch.empty_like(k)))
    with fwAD.dual_level():                                               # alone, of strided rows
        y, none = K.rotary_embedding(fwAD.make_dual(q[:, 1:], vq[:, 1:]), None, positions, freq, **args)
        check_turn(fwAD.unpack_dual(y).tangent, vq[:, 1:], positions, freq, interleaved, 1.5)
        assert none is None
    # where a gradient is recorded as well: of the result, of its tangent, and the tangent of the gradient
    leaf, vleaf = q.clone().requires_grad_(), vq.clone().requires_grad_()
    with fwAD.dual_level():
        y, _ = K.rotary_embedding(fwAD.make_dual(leaf, vleaf), None, positions, freq, **args)
        primal, tangent = fwAD.unpack_dual(y)
        first, = torch.autograd.grad(primal, (leaf,), dy, retain_graph=True)
        second, = torch.autograd.grad(tangent, (vleaf,), dy, retain_graph=True)
        check_turn(first, dy, positions, freq, interleaved, 1.5, -1.0)
        check_turn(second, dy, positions, freq, interleaved, 1.5, -1.0)
        over, = torch.autograd.grad(primal, (leaf,), fwAD.make_dual(dy, vy))
        check_turn(fwAD.unpack_dual(over).tangent, vy, positions, freq, interleaved, 1.5, -1.0)


def test_rotary_under_function_transforms_is_right_or_refused():
    g, (freq, _) = gen(12), K.rotary_frequencies(64, device=DEV)
    q, v = (torch.randn(5, 2, 64, generator=g).to(DEV) for _ in range(2))
    positions = torch.arange(5, device=DEV)

    def f(x):
        return K.rotary_embedding(x, None, positions, freq)[0]

    for call, want in ((lambda: torch.func.jvp(f, (q,), (v,))[1], lambda: f(v)), (lambda: torch.func.vmap(f)(torch.stack([q, v])), lambda: torch.stack([f(q), f(v)])),
                       (lambda: torch.func.grad(lambda x: (f(x) * v).sum())(q), lambda: K.rotary_embedding(v, None, positions, freq, inverse=True)[0])):
        try:
            got = call()
        except RuntimeError:
            continue
        assert torch.equal(got, want())


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (32, 8, 64), (16, 16, 256), (8, 1, 128)])
@pytest.mark.parametrize("lens", [[1], [40, 3], [700, 300], [5000], [9000, 20, 4000], [300] * 70])
def test_decode_of_values_at_the_end_of_bfloat16(lens, hq, hkv, d):
    """One key has all the weight (the others e^-40 of it) and values go to 2^127: the average is finite, on every path."""
    q, kc, vc, table, sl = decode_case(lens, hq, hkv, d, 16, BF, seed=d)
    vc.copy_((vc * 1e38).clamp(-3e38, 3e38))
    q.fill_(1.0)
    kc.zero_()
    for s, n in enumerate(lens):
        at = (7 * s + n // 3) % n
        kc[int(table[s, at // 16]), at % 16] = 1.0
    out, _ = check_decode(q, kc, vc, table, sl, sm=40.0 / d)
    assert torch.isfinite(out).all() and out.abs().max() > 1e38


@pytest.mark.parametrize("lens", [[1], [700, 300], [5000], [9000, 20, 4000], [300] * 70])
def test_decode_of_equal_weights_over_very_large_and_very_small_values(lens):
    """All keys weigh the same and all values lie near 2^128: the sum does not overflow where the average does not."""
    q, kc, vc, table, sl = decode_case(lens, 8, 2, 128, 16, BF, seed=len(lens))
    vc.fill_(3.2e38)
    check_decode(q, kc, vc, table, sl, sm=0.0)
    vc[:, ::3] = -3.2e38
    check_decode(q, kc, vc, table, sl)
    vc.copy_(torch.randn(vc.shape, generator=gen(1)) * 1e-30)
    out, _ = check_decode(q, kc, vc, table, sl)
    assert out.any()


def test_rotary_store_into_caches_that_share_rows():
    """Refused; caches whose rows only lie among each other are not."""
    freq, _ = K.rotary_frequencies(64, device=DEV)
    x = torch.randn(5, 2, 64, generator=gen(5)).to(BF).to(DEV)
    t = dict(q=x, k=x.clone(), v=x.clone(), positions=torch.arange(5, device=DEV), slot_mapping=torch.arange(5, device=DEV), inv_freq=freq)
    buf = torch.zeros(5, 16, 2, 64, dtype=BF, device=DEV)
    wide = torch.zeros(4, 16, 4, 128, dtype=BF, device=DEV)
    flat = torch.zeros(8 * 16 * 2 * 64, dtype=BF, device=DEV)
    for kc, vc in ((buf[:-1], buf[1:]), (buf[1:], buf[:-1]), (wide[:, :, :2, :64], wide[:, :, 1:3, :64]), (wide[..., :2, :64], wide[..., :2, 32:96]),
                   (flat[:4 * 2048].view(4, 16, 2, 64), flat[1024:1024 + 4 * 2048].view(4, 16, 2, 64)),
                   (flat[:4 * 2048].view(4, 16, 2, 64), flat[64:64 + 4 * 2048].view(4, 2, 16, 64).transpose(1, 2)),
                   (flat.view(4, 2, 16, 2, 64)[:, 0], flat[2048:2048 * 5].view(4, 16, 2, 64)), (buf, buf)):
        with pytest.raises(ValueError, match="share no memory|cache each"):
            K.rotary_paged_store(**t, key_cache=kc, value_cache=vc)
    blocks = torch.zeros(4, 2, 16 * 2 * 64, dtype=BF, device=DEV)
    for whole, kc, vc in ((blocks, blocks[:, 0].view(4, 16, 2, 64), blocks[:, 1].view(4, 2, 16, 64).transpose(1, 2)),        # heads first in one of them
                          (wide, wide[:, :, :2, :64], wide[:, :, 2:, :64]), (wide, wide[..., :2, :64], wide[..., :2, 64:]),
                          (wide, wide[:2, :, :2, :64], wide[2:, :, :2, :64]), (wide, wide[::2, :, :2, 64:], wide[1::2, :, :2, :64]),
                          (flat, flat.view(4, 2, 16, 2, 64)[:, 1], flat.view(4, 2, 16, 2, 64)[:, 0])):
        whole.zero_()
        K.rotary_paged_store(**t, key_cache=kc, value_cache=vc)
        assert torch.equal(kc[0, :5], K.rotary_embedding(t["k"], None, t["positions"], freq)[0]) and torch.equal(vc[0, :5], t["v"])
        assert int((whole != 0).sum()) == int((kc != 0).sum()) + int((vc != 0).sum())


def test_outputs_whose_own_rows_share_memory_are_refused():
    freq, _ = K.rotary_frequencies(64, device=DEV)
    x = torch.randn(5, 2, 64, generator=gen(5)).to(BF).to(DEV)
    t = dict(q=x, k=x.clone(), v=x.clone(), positions=torch.arange(5, device=DEV), slot_mapping=torch.arange(5, device=DEV), inv_freq=freq,
             key_cache=torch.zeros(3, 16, 2, 64, dtype=BF, device=DEV), value_cache=torch.zeros(3, 16, 2, 64, dtype=BF, device=DEV))
    buf = torch.zeros(3 * 16 * 2 * 64, dtype=BF, device=DEV)
    for sizes, strides in (((5, 2, 64), (64, 64, 1)), ((5, 2, 64), (0, 64, 1)), ((5, 2, 64), (128, 32, 1)), ((5, 2, 64), (96, 64, 1)), ((5, 2, 64), (1, 512, 1))):
        bad = buf.as_strided(sizes, strides)
        with pytest.raises(ValueError, match="share memory"):
            K.rotary_embedding(x, None, t["positions"], freq, out=(bad, None))
        with pytest.raises(ValueError, match="share memory"):
            K.rotary_paged_store(**t, out=bad)
    for strides in ((1024, 128, 64, 1), (2048, 64, 64, 1), (0, 128, 64, 1)):
        for name in ("key_cache", "value_cache"):
            with pytest.raises(ValueError, match="share memory"):
                K.rotary_paged_store(**(t | {name: buf.as_strided((3, 16, 2, 64), strides)}))
    want = K.rotary_embedding(x, None, t["positions"], freq)[0]
    for strides in ((128, 64, 1), (64, 320, 1), (200, 64, 1), (64, 777, 1)):  # and these do not
        out = buf.as_strided((5, 2, 64), strides)
        K.rotary_embedding(x, None, t["positions"], freq, out=(out, None))
        assert torch.equal(out, want)


def test_results_have_memory_of_their_own():
    """One may be resized, kept or dropped without the others."""
    freq, _ = K.rotary_frequencies(64, device=DEV)
    q, k = (torch.randn(8, 4, 64, generator=gen(s)).to(BF).to(DEV) for s in (1, 2))
    qo, ko = K.rotary_embedding(q, k, torch.arange(8, device=DEV), freq)
    kept = ko.clone()
    torch.full((9, 4, 64), 7.0, dtype=BF, device=DEV, out=qo.resize_(0))
    assert torch.equal(ko, kept)
    i32 = dict(dtype=torch.int32, device=DEV)
    lens = torch.arange(64, **i32)
    s = K.paged_schedule(lens, torch.ones(64, **i32), torch.full((64, 8), -1, **i32), torch.arange(64, **i32), 16, 64)
    for name in s._fields:
        kept = {n: t.clone() for n, t in s._asdict().items() if n != name}
        t = getattr(s, name)
        t.resize_(t.numel() + 3).fill_(-9)
        assert all(torch.equal(getattr(s, n), x) for n, x in kept.items()), name


def test_decode_in_the_room_of_the_largest_call():
    """One workspace, of the size that the largest batch asks for, serves all of them."""
    g = gen(7)
    kc, vc, _ = caches("apart", 60, 16, 8, 128, BF, g)
    room = native().paged_kv_decode_workspace_bytes(63, 32, 8, 128, 16, 128)
    ws = torch.full((room,), 0xff, dtype=torch.uint8, device=DEV)
    for seqs in (1, 2, 15, 16, 32, 63):
        for columns in (3, 28, 30, 51, 128):
            table = torch.randint(0, 60, (seqs, columns), dtype=torch.int32, generator=g).to(DEV)
            lens = torch.randint(0, 16 * columns + 1, (seqs,), dtype=torch.int32, generator=g).to(DEV)
            q = torch.randn(seqs, 32, 128, generator=g).to(BF).to(DEV)
            for window in (0, 200):
                assert torch.equal(K.paged_kv_decode(q, kc, vc, table, lens, window=window, workspace=ws), K.paged_kv_decode(q, kc, vc, table, lens, window=window))


def test_outputs_in_the_memory_of_transposed_inputs_are_refused():
    freq, _ = K.rotary_frequencies(64, device=DEV)
    buf = torch.zeros(5, 512, dtype=BF, device=DEV)
    x = buf[:, :256].view(5, 64, 4).transpose(1, 2)                        # a row's values lie four apart, over 256
    positions, apart = torch.arange(5, device=DEV), torch.ones(5, 4, 64, dtype=BF, device=DEV)
    for at in (0, 128, 255):
        out = buf.as_strided((5, 4, 64), (512, 64, 1), at)
        with pytest.raises(ValueError, match="share no memory"):
            K.rotary_embedding(x, None, positions, freq, out=(out, None))
        with pytest.raises(ValueError, match="share no memory"):
            K.rotary_embedding(apart, x, positions, freq, out=(out, torch.empty_like(apart)))
    K.rotary_embedding(x, None, positions, freq, out=(buf[:, 256:].view(5, 4, 64), None))
