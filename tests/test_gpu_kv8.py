"""The 8-bit paged cache against plain implementations in 64 bits: rotary store, read and decode, at the sizes, strides and masks where
each can go wrong."""
from __future__ import annotations

import math

import pytest
import torch

from flashquant_amd import kernels as K
from flashquant_amd.kernels._native import native

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
E4, E8, U8 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.uint8
HEADS = [(1, 1, 128), (8, 8, 64), (32, 8, 128), (16, 1, 256), (12, 4, 64), (5, 1, 128), (32, 2, 128), (6, 2, 256)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def raw(t):
    return t.view(U8)


def quantised(x):
    """Codes (as float64) and powers of two of rows, from the definition in 64 bits."""
    size = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    power = torch.where(size > 0, torch.ceil(torch.log2(size.clamp(min=1e-300) / 448.0)), -1000.0).clamp(-118, 120)
    y = x * torch.exp2(-power)[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(x.isfinite(), torch.round(y / step) * step, math.nan), power


def caches(layout, blocks, page, h, d, g, scale=1.0):
    """(key_cache, value_cache, key_scales, value_scales, what they lie in): rows of normal values, quantised."""
    x = torch.randn(2, blocks, page, h, d, generator=g).double() * scale
    codes, power = quantised(x)
    codes, power = raw(codes.float().to(E4)), (power + 127).to(U8).transpose(2, 3).contiguous()
    if layout == "apart":
        c, p = codes.to(DEV), power.to(DEV)
        k, v, ks, vs, whole = c[0], c[1], p[0], p[1], [c, p]
    elif layout == "together":
        c, p = codes.transpose(0, 1).contiguous().to(DEV), power.transpose(0, 1).contiguous().to(DEV)
        k, v, ks, vs, whole = c[:, 0], c[:, 1], p[:, 0], p[:, 1], [c, p]
    elif layout == "heads first":
        c, p = codes.transpose(2, 3).contiguous().to(DEV), power.transpose(1, 2).contiguous().to(DEV)
        k, v, ks, vs, whole = c[0].transpose(1, 2), c[1].transpose(1, 2), p[0].transpose(0, 1), p[1].transpose(0, 1), [c, p]
    else:                                                                # one record a page: codes side by side, then the scales
        record = page * h * (2 * d + 16) + 2 * h * 32
        c = torch.full((blocks, record), 0x55, dtype=U8, device=DEV)
        rows = c[:, :page * h * (2 * d + 16)].view(blocks, page, h, 2 * d + 16)
        tail = c[:, page * h * (2 * d + 16):].view(blocks, 2, h, 32)
        rows[..., :d], rows[..., d:2 * d] = codes[0].to(DEV), codes[1].to(DEV)
        tail[:, 0, :, :page], tail[:, 1, :, :page] = power[0].to(DEV), power[1].to(DEV)
        k, v, ks, vs, whole = rows[..., :d], rows[..., d:2 * d], tail[:, 0, :, :page], tail[:, 1, :, :page], [c]
    return k.view(E4), v.view(E4), ks.view(E8), vs.view(E8), whole


LAYOUTS = ["apart", "together", "heads first", "one record"]


def stood_for(cache, scales):
    """The values (blocks, page, heads, d), float64."""
    power = raw(scales).double().transpose(1, 2)[..., None] - 127
    return raw(cache.contiguous() if not cache.is_contiguous() else cache).view(E4).float().double() * torch.exp2(power)


# ---- store ------------------------------------------------------------------------------------------------------------------------

def turned(x, positions, freq, interleaved=False, scale=1.0):
    """(rotated values, their float32 error), 64 bits."""
    half, y, tol = freq.shape[0], x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    a = (positions.double()[:, None] * freq.double())[:, None]
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    x0, x1 = x[..., i].double(), x[..., j].double()
    y[..., i], y[..., j] = scale * (x0 * a.cos() - x1 * a.sin()), scale * (x1 * a.cos() + x0 * a.sin())
    # cosine, sine, two products and their sum in float32, and the angle in 64 bits
    tol[..., i] = tol[..., j] = scale * (x0.abs() + x1.abs()) * (4 * 2.0 ** -24 + a.abs() * 2.0 ** -51)
    return y, tol


def check_rows(codes, power, y, tol):
    """Codes (float) and power bytes of rows against values `y` known to `tol`: half a step of e4m3, 2^-4 of the value or 2^-10 of the unit."""
    size = y.abs().amax(-1)
    low, high = (torch.ceil(torch.log2((size * s).clamp(min=1e-300) / 448.0)).clamp(-118, 120) for s in (1 - 1e-6, 1 + 1e-6))
    assert ((power >= low) & (power <= high)).all()
    unit = torch.exp2(power)[..., None]
    half_step = torch.exp2(torch.floor(torch.log2(((y.abs() + tol) / unit).clamp(min=2.0 ** -6))) - 4) * unit
    assert ((codes.double() * unit - y).abs() <= half_step + tol).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout", LAYOUTS)
# one token; a padded step; interleaved part of a head over several workgroups; odd heads; a rotation of odd pairs; none mapped; no queries
@pytest.mark.parametrize("tokens,mapped,hq,hkv,d,rot,page,interleaved", [(1, 1, 1, 1, 64, 64, 8, False), (64, 61, 32, 8, 128, 128, 16, False),
                                                                       (1100, 1090, 4, 2, 128, 64, 32, True), (9, 9, 7, 7, 64, 48, 16, False),
                                                                       (40, 33, 3, 1, 256, 10, 8, True), (33, 30, 5, 3, 128, 100, 16, False),
                                                                       (5, 0, 2, 1, 64, 32, 16, True), (17, 17, 0, 2, 256, 256, 32, False)])
def test_store(tokens, mapped, hq, hkv, d, rot, page, interleaved, layout, dtype):
    g = gen(tokens + d)
    blocks = tokens // page + 3
    kc, vc, ks, vs, whole = caches(layout, blocks, page, hkv, d, g)
    qkv = (torch.randn(tokens, hq + 2 * hkv, d, generator=g) * torch.exp2(torch.randint(-9, 9, (tokens, 1, 1), generator=g))).to(dtype).to(DEV)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    positions = torch.randint(0, 100000, (tokens,), generator=g).to(DEV)
    freq, _ = K.rotary_frequencies(rot, device=DEV)
    slots = torch.randperm(blocks * page, generator=g)[:mapped]
    if mapped > 8:                                                       # not stored
        slots[3], slots[4], slots[5], slots[6] = -1, blocks * page, -(1 << 40), 1 << 40
    stored = [i for i, s in enumerate(slots.tolist()) if 0 <= s < blocks * page]
    before = [w.clone() for w in whole]
    got = K.rotary_paged_store8(q, k, v, positions, slots.to(DEV), freq, kc, vc, ks, vs, interleaved=interleaved, scale=0.9)
    assert got.shape == q.shape and got.dtype == dtype
    if hq:                                                               # queries: half a step of their type
        y, tol = turned(q, positions, freq, interleaved, 0.9)
        info = torch.finfo(dtype)
        assert ((got.double() - y).abs() <= tol + (y.abs() + tol) * info.eps / 2 + info.tiny * info.eps / 2).all()
    at = slots[stored].to(DEV)
    block, inside = at // page, at % page
    y, tol = turned(k, positions, freq, interleaved, 0.9)
    check_rows(raw(kc)[block, inside].view(E4).float(), raw(ks)[block, :, inside].double() - 127, y[stored], tol[stored])
    codes, power = quantised(v[stored].double())                         # values: bit for bit
    assert torch.equal(raw(vc)[block, inside].view(E4).double(), codes) and torch.equal(raw(vs)[block, :, inside].double() - 127, power)
    # nothing beside these rows
    after = [w.clone() for w in whole]
    raw(kc)[block, inside], raw(vc)[block, inside], raw(ks)[block, :, inside], raw(vs)[block, :, inside] = 0, 0, 0, 0
    left = [w.clone() for w in whole]
    for w, b in zip(whole, before):
        w.copy_(b)
    raw(kc)[block, inside], raw(vc)[block, inside], raw(ks)[block, :, inside], raw(vs)[block, :, inside] = 0, 0, 0, 0
    assert all(torch.equal(a, b) for a, b in zip(left, whole))
    if hq:                                                               # in place
        K.rotary_paged_store8(q, k, v, positions, slots.to(DEV), freq, kc, vc, ks, vs, interleaved=interleaved, scale=0.9, out=q)
        assert torch.equal(q, got) and all(torch.equal(a, b) for a, b in zip(whole, after))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq", [0, 1])
def test_store_of_the_fewest_heads(hq, d):
    """A workgroup's rows reach into the most tokens, all of each turned."""
    test_store(150, 150, hq, 1, d, d, 16, False, "apart", BF)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_store_has_the_same_bits_at_every_alignment(off, d):
    """Rows at odd addresses, columns apart, int32 positions: the kernel for any row gives what the wide one does."""
    g = gen(d)
    kc, vc, ks, vs, whole = caches("apart", 9, 16, 3, d, g)
    x = torch.randn(70, 11, d + 8, generator=g).to(BF).to(DEV)
    q, k, v = (t.contiguous() for t in (x[:, :5, :d], x[:, 5:8, :d], x[:, 8:, :d]))
    positions, slots = torch.randint(0, 5000, (70,), generator=g).to(DEV), torch.randperm(140, generator=g)[:70].to(DEV)
    freq, _ = K.rotary_frequencies(d // 2, device=DEV)
    for interleaved in (False, True):
        want_q = K.rotary_paged_store8(q, k, v, positions, slots, freq, kc, vc, ks, vs, interleaved=interleaved)
        want = [w.clone() for w in whole]
        for w in whole:
            w.zero_()
        moved = torch.zeros(70, 11, d + 8, dtype=BF, device=DEV)
        moved[..., off:off + d] = x[..., :d]
        m = moved[..., off:off + d]
        got = K.rotary_paged_store8(m[:, :5], m[:, 5:8], m[:, 8:], positions.int(), slots, freq, kc, vc, ks, vs, interleaved=interleaved)
        assert torch.equal(got, want_q)
        at = slots.cpu()
        for a, b in ((whole[0].view(2, -1, 3, d)[:, at], want[0].view(2, -1, 3, d)[:, at]),):
            assert torch.equal(a, b)
        assert torch.equal(whole[1][:, at // 16, :, at % 16], want[1][:, at // 16, :, at % 16])
        apart = torch.zeros(70, 11, 2 * d, dtype=BF, device=DEV)
        apart[..., ::2] = x[..., :d]
        a = apart[..., ::2]
        assert torch.equal(K.rotary_paged_store8(a[:, :5], a[:, 5:8], a[:, 8:], positions, slots, freq, kc, vc, ks, vs, interleaved=interleaved), want_q)


def test_store_of_rows_at_their_ends():
    """Zeros, infinities and NaN, rows at the powers' limits and at 1.75 of a binade, values that round to zero or up to the next binade."""
    d, page = 128, 16
    rows = torch.zeros(12, d, dtype=F32)
    rows[1, 0], rows[1, 5] = math.inf, 3.0
    rows[2, 0], rows[2, 1], rows[2, 2] = math.nan, -math.inf, -1e-3
    rows[3, :] = math.nan
    rows[4, 0] = 448.0
    rows[5, 0], rows[5, 1] = 450.0, 449.0
    rows[6, 0], rows[6, 1] = 3.3e38, 1.0
    rows[7, 0] = 2.0 ** -126
    rows[8, 0], rows[8, 1], rows[8, 2] = 2.0 ** -110, 2.0 ** -127, 2.0 ** -128
    rows[9] = torch.linspace(-1, 1, d)
    rows[10, 0], rows[10, 1:] = 1.0, 2.0 ** torch.linspace(-20, -8, d - 1)
    rows[11, 0], rows[11, 1] = 1.7578125, -1.75
    x = rows.to(BF).to(DEV)[:, None]
    kc, vc, ks, vs, _ = caches("apart", 1, page, 1, d, gen(0))
    freq, _ = K.rotary_frequencies(d, device=DEV)
    slots = torch.arange(12, device=DEV)
    K.rotary_paged_store8(x, x, x, torch.zeros(12, dtype=torch.long, device=DEV), slots, freq, kc, vc, ks, vs)
    codes, power = quantised(x[:, 0].double())
    assert torch.equal(raw(vs)[0, 0, :12].double() - 127, power)
    got = vc[0, :12, 0].double()
    assert torch.equal(got.isnan(), codes.isnan()) and torch.equal(got.nan_to_num(), codes.nan_to_num())
    assert float(power[0]) == -118 and float(power[4]) == 0 and float(power[5]) == 1 and float(power[6]) == 120 and int(raw(vs).min()) >= 9
    # at position 0 keys are values, but in rows where 0 times an infinity is added
    same = [0, 4, 5, 6, 7, 8, 9, 10, 11]
    assert torch.equal(raw(kc)[0, same], raw(vc)[0, same]) and torch.equal(raw(ks)[0, :, same], raw(vs)[0, :, same])


def test_store_beyond_32_bit_offsets():
    page, h, d = 32, 8, 128
    blocks = (1 << 32) // (page * h * d) + 9
    cache = torch.zeros(2, blocks, page, h, d, dtype=U8, device=DEV)
    scales = torch.zeros(2, blocks, h, page, dtype=U8, device=DEV)
    g = gen(1)
    x = torch.randn(40, 3 * h, d, generator=g).to(BF).to(DEV)
    slots = blocks * page - 1 - torch.arange(40, device=DEV) * 5
    freq, _ = K.rotary_frequencies(d, device=DEV)
    args = x[:, :h], x[:, h:2 * h], x[:, 2 * h:], torch.arange(40, device=DEV)
    K.rotary_paged_store8(*args, slots, freq, cache[0].view(E4), cache[1].view(E4), scales[0].view(E8), scales[1].view(E8))
    small, small_scales = torch.zeros(2, 8, page, h, d, dtype=U8, device=DEV), torch.zeros(2, 8, h, page, dtype=U8, device=DEV)
    K.rotary_paged_store8(*args, slots - (blocks - 8) * page, freq, small[0].view(E4), small[1].view(E4), small_scales[0].view(E8), small_scales[1].view(E8))
    assert torch.equal(cache[:, -8:], small) and torch.equal(scales[:, -8:], small_scales)
    table = torch.arange(blocks - 8, blocks, dtype=torch.int32, device=DEV)[None]
    cu = torch.tensor([0, 8 * page], dtype=torch.int32, device=DEV)
    for got, c, s in zip(K.paged_kv8_read(cache[0].view(E4), cache[1].view(E4), scales[0].view(E8), scales[1].view(E8), table, cu, 8 * page), small, small_scales):
        assert torch.equal(got.double(), stood_for(c.view(E4), s.view(E8)).view(-1, h, d))
    q = torch.randn(1, 4 * h, d, generator=g).to(BF).to(DEV)
    lens = torch.tensor([8 * page - 3], dtype=torch.int32, device=DEV)
    assert torch.equal(K.paged_kv8_decode(q, cache[0].view(E4), cache[1].view(E4), scales[0].view(E8), scales[1].view(E8), table, lens),
                       K.paged_kv8_decode(q, small[0].view(E4), small[1].view(E4), small_scales[0].view(E8), small_scales[1].view(E8), table - (blocks - 8), lens))


def test_store_refusals():
    g = gen(2)
    kc, vc, ks, vs, whole = caches("apart", 4, 16, 2, 128, g)
    x = torch.randn(5, 8, 128, generator=g).to(BF).to(DEV)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    positions, slots, freq = torch.arange(5, device=DEV), torch.arange(5, device=DEV), K.rotary_frequencies(128, device=DEV)[0]
    good = dict(q=q, k=k, v=v, positions=positions, slot_mapping=slots, inv_freq=freq, key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs)
    K.rotary_paged_store8(**good)
    room = torch.zeros(1 << 16, dtype=U8, device=DEV)
    for bad in (dict(q=q.float()), dict(k=k[:3]), dict(k=k.half()), dict(v=v[:, :1]), dict(q=q[..., :64], k=k[..., :64], v=v[..., :64]), dict(positions=positions[:4]),
                dict(positions=positions.float()), dict(slot_mapping=slots.int()), dict(slot_mapping=torch.arange(6, device=DEV)), dict(inv_freq=freq.float()),
                dict(inv_freq=K.rotary_frequencies(256, device=DEV)[0]), dict(key_cache=raw(kc)), dict(key_scales=raw(ks)), dict(key_scales=ks[:3]),
                dict(key_scales=ks[..., :8]), dict(value_scales=vs.cpu()), dict(key_cache=kc[:3]), dict(key_cache=kc[:, :8]), dict(key_cache=kc.cpu()),
                dict(key_cache=kc[:, :12], value_cache=vc[:, :12], key_scales=ks[..., :12], value_scales=vs[..., :12]), dict(value_cache=kc), dict(value_scales=ks),
                dict(key_cache=kc[:1].expand(4, -1, -1, -1)), dict(key_scales=ks[:1].expand(4, -1, -1)), dict(out=q[:, :2]), dict(out=q.float()), dict(out=k),
                dict(out=room[:q.numel() * 2].view(BF).view(5, 4, 128), key_cache=room[:kc.numel()].view(E4).view_as(kc)),
                dict(key_scales=room[:ks.numel()].view(E8).view_as(ks), value_cache=room[:vc.numel()].view(E4).view_as(vc)),
                dict(key_cache=kc.transpose(2, 3))):
        with pytest.raises(ValueError):
            K.rotary_paged_store8(**(good | bad))
    with pytest.raises(ValueError):                                      # no kernel of that width
        c = torch.zeros(4, 16, 2, 96, dtype=U8, device=DEV).view(E4)
        K.rotary_paged_store8(q[..., :96], k[..., :96], v[..., :96], positions, slots, K.rotary_frequencies(96, device=DEV)[0], c, c.clone(), ks, vs)
    assert K.rotary_paged_store8(q[:0], k[:0], v[:0], positions[:0], slots[:0], freq, kc, vc, ks, vs).shape == (0, 4, 128)


# ---- read -------------------------------------------------------------------------------------------------------------------------

def gathered(kc, vc, ks, vs, table, cu, starts, room, fill):
    """Rows by the definition; `fill`: what is behind the last sequence."""
    page, out = kc.shape[1], []
    for cache, scales in ((kc, ks), (vc, vs)):
        values, rows = stood_for(cache, scales), fill.clone().double()
        for s in range(table.shape[0]):
            for i in range(cu[s], min(cu[s + 1], room)):
                t = starts[s] + i - cu[s]
                block = int(table[s, t // page]) if 0 <= t < table.shape[1] * page else -1
                rows[i] = values[block, t % page] if 0 <= block < kc.shape[0] else 0.0
        out.append(rows)
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("lens,h,d,page,extra", [([1], 1, 64, 8, 0), ([0, 5, 0, 0, 70, 1], 8, 128, 16, 3), ([33], 3, 256, 32, 0), ([2, 0, 9] * 70, 2, 64, 8, 40),
                                                 ([0], 2, 128, 16, 5), ([40, 200], 1, 256, 16, -30)])
def test_read(lens, h, d, page, extra, layout, dtype):
    g = gen(len(lens) + d)
    starts = [int(torch.randint(0, 60, (1,), generator=g)) for _ in lens]
    columns = max(-(-(n + s) // page) for n, s in zip(lens, starts)) + 1
    blocks = 40
    kc, vc, ks, vs, _ = caches(layout, blocks, page, h, d, g)
    table = torch.randint(0, blocks, (len(lens), columns), generator=g).int().to(DEV)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    room = max(cu[-1] + extra, 0)
    args = kc, vc, ks, vs, table, torch.tensor(cu, dtype=torch.int32, device=DEV), room
    first = torch.tensor(starts, dtype=torch.int32, device=DEV)
    want = gathered(kc, vc, ks, vs, table, cu, starts, room, torch.zeros(room, h, d, device=DEV))
    got = K.paged_kv8_read(*args, starts=first, dtype=dtype)
    for a, b in zip(got, want):
        assert a.dtype == dtype and torch.equal(a, b.to(dtype))
    out = torch.full((2, room + 2, h, d), 7.0, dtype=dtype, device=DEV)
    want = gathered(kc, vc, ks, vs, table, cu, starts, room, torch.full((room, h, d), 7.0, device=DEV))
    K.paged_kv8_read(*args, starts=first, dtype=dtype, out=(out[0, 1:-1], out[1, 1:-1]))
    for a, b in zip(out, want):
        assert torch.equal(a[1:-1], b.to(dtype)) and (a[0] == 7).all() and (a[-1] == 7).all()
    if min(starts) == 0 and max(starts) == 0 or len(lens) == 1:
        plain = K.paged_kv8_read(*args, dtype=dtype)
        for a, b in zip(plain, gathered(kc, vc, ks, vs, table, cu, [0] * len(lens), room, torch.zeros(room, h, d, device=DEV))):
            assert torch.equal(a, b.to(dtype))


def test_read_of_many_sequences_and_of_missing_pages():
    g = gen(7)
    kc, vc, ks, vs, _ = caches("apart", 50, 8, 1, 64, g)
    lens = torch.randint(0, 3, (5000,), generator=g).tolist()
    cu = torch.tensor([0] + lens).cumsum(0)
    table = torch.randint(-2, 53, (5000, 3), generator=g).int().to(DEV)
    starts = torch.randint(-3, 28, (5000,), generator=g)
    got = K.paged_kv8_read(kc, vc, ks, vs, table, cu.int().to(DEV), int(cu[-1]), starts=starts.int().to(DEV))
    for a, b in zip(got, gathered(kc, vc, ks, vs, table.cpu(), cu.tolist(), starts.tolist(), int(cu[-1]), torch.zeros(int(cu[-1]), 1, 64, device=DEV))):
        assert torch.equal(a.double(), b)


def test_read_of_extreme_rows():
    """NaN codes stay; in float16 what is beyond its range is infinite and what is below is rounded."""
    kc, vc, ks, vs, _ = caches("apart", 2, 8, 1, 64, gen(3))
    raw(kc)[0, 0, 0, 3], raw(kc)[0, 0, 0, 4] = 0x7f, 0xff
    raw(ks)[0, 0] = torch.tensor([9, 30, 100, 110, 127, 135, 136, 247], dtype=U8, device=DEV)
    table, cu = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    want = stood_for(kc, ks)[0].float()
    for dtype in (BF, HF):
        got = K.paged_kv8_read(kc, vc, ks, vs, table, cu, 8, dtype=dtype)[0]
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=5.0), want.to(dtype).nan_to_num(nan=5.0))


def test_read_refusals():
    kc, vc, ks, vs, whole = caches("apart", 4, 16, 2, 128, gen(2))
    table, cu = torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.tensor([0, 5, 9], dtype=torch.int32, device=DEV)
    out = torch.empty(2, 9, 2, 128, dtype=BF, device=DEV)
    good = dict(key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs, block_table=table, cu_seqlens=cu, num_tokens=9)
    K.paged_kv8_read(**good, out=(out[0], out[1]))
    for bad in (dict(key_cache=raw(kc)), dict(value_cache=vc[:2]), dict(value_scales=raw(vs)), dict(key_scales=ks.transpose(1, 2)), dict(block_table=table.long()),
                dict(block_table=table[0]), dict(block_table=table[:, :0]), dict(cu_seqlens=cu[:2]), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu.cpu()), dict(num_tokens=-1),
                dict(starts=cu), dict(starts=cu[:2].long()), dict(dtype=F32), dict(out=(out[0], out[0])), dict(out=(out[0, :8], out[1, :8])), dict(out=(out[0].half(), out[1].half())),
                dict(out=(out[0].transpose(0, 1), out[1])), dict(key_cache=kc[:, :12], value_cache=vc[:, :12], key_scales=ks[..., :12], value_scales=vs[..., :12]),
                dict(out=(whole[0].view(-1)[:9 * 2 * 128 * 2].view(BF).view(9, 2, 128), out[1]))):
        with pytest.raises(ValueError):
            K.paged_kv8_read(**(good | bad))
    odd = torch.zeros(kc.numel() + 8, dtype=U8, device=DEV)[8:].view(E4).view_as(kc)    # a cache at an odd address
    with pytest.raises(ValueError):
        K.paged_kv8_read(**(good | dict(key_cache=odd)))
    assert K.paged_kv8_read(**(good | dict(num_tokens=0)))[0].shape == (0, 2, 128)
    none = K.paged_kv8_read(kc, vc, ks, vs, table[:0], cu[:1], 3)
    assert (none[0] == 0).all() and none[0].shape == (3, 2, 128)


# ---- decode -----------------------------------------------------------------------------------------------------------------------

def attended(q, keys, values, table, lens, sm, window=0):
    """(out, lse, tolerance of out, tolerance of lse) from the definition in 64 bits, sequence by sequence; keys, values float64."""
    page, hkv, d = keys.shape[1], keys.shape[2], keys.shape[3]
    outs = []
    for s, (row, n) in enumerate(zip(table, lens.tolist())):
        n = min(max(n, 0), table.shape[1] * page)
        token = torch.arange(max(0, n - window) if window else 0, n, device=q.device)
        block = row[token // page].long()
        there = (block >= 0) & (block < keys.shape[0])
        token, block = token[there], block[there]
        k, v = (c[block, token % page].transpose(0, 1).contiguous() for c in (keys, values))             # (hkv, n, d)
        x = q[s].double().view(hkv, -1, d)
        if token.numel() == 0:
            zero = torch.zeros_like(x)
            outs.append([zero, torch.full_like(x[..., 0], -math.inf), zero, torch.zeros_like(x[..., 0])])
            continue
        score = (k @ x.transpose(1, 2).contiguous()).transpose(1, 2).contiguous() * sm                  # (hkv, g, n)
        p = torch.softmax(score, -1)
        o, size = p @ v, p @ v.abs()
        # the score's float32 sum of d products and its scaling
        off = (((k.abs() @ x.abs().transpose(1, 2).contiguous()).amax(1) * abs(sm)) * (d + 5) * 2.0 ** -24)[..., None]
        # a weight's two terms, the exponential, the sums over keys and parts; twice the scores' part: weights and their sum
        tol = size * (2.0 ** -16 + 2 * off + (token.numel() + 64) * 2.0 ** -23)
        info = torch.finfo(q.dtype)
        lse = torch.logsumexp(score, -1)
        outs.append([o, lse, tol + (o.abs() + tol) * info.eps / 2 + info.tiny * info.eps,
                     off[..., 0] + (token.numel() + 64) * 2.0 ** -23 + lse.abs() * 2.0 ** -21 + 2.0 ** -20])
    return [torch.stack([t[i].reshape(-1, d) if i in (0, 2) else t[i].reshape(-1) for t in outs]) for i in range(4)]


def check(got, want, q):
    out, lse = got
    o, l, to, tl = want
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == q.shape[:2] and lse.dtype == F32
    off = (out.double() - o).abs() - to
    assert (off <= 0).all(), float(off.max())
    none = torch.isneginf(l)
    assert torch.equal(torch.isneginf(lse), none) and (out[none] == 0).all()
    assert ((lse.double() - l).abs()[~none] <= tl[~none]).all()
    return out, lse


def check_decode(q, kc, vc, ks, vs, table, lens, sm=None, window=0, **more):
    sm = 1.0 / math.sqrt(q.shape[-1]) if sm is None else sm
    got = K.paged_kv8_decode(q, kc, vc, ks, vs, table, lens, sm, window=window, return_lse=True, **more)
    return check(got, attended(q, stood_for(kc, ks), stood_for(vc, vs), table, lens, sm, window), q)


def decode_case(lens, hq, hkv, d, page, dtype, seed=0, layout="apart", extra_columns=0, scale=2.0):
    g = gen(seed)
    columns = max(1, max(-(-n // page) for n in lens)) + extra_columns
    blocks = sum(-(-n // page) for n in lens) + 3
    kc, vc, ks, vs, _ = caches(layout, blocks, page, hkv, d, g)
    order, at = torch.randperm(blocks, generator=g).int(), 0
    table = torch.full((len(lens), columns), 1 << 30, dtype=torch.int32)  # no page of the cache
    for s, n in enumerate(lens):
        used = -(-n // page)
        table[s, :used] = order[at:at + used]
        at += used
    q = (torch.randn(len(lens), hq, d, generator=g) * scale).to(dtype).to(DEV)
    return q, kc, vc, ks, vs, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [8, 16, 32])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_decode_of_ragged_lengths(hq, hkv, d, page, dtype):
    check_decode(*decode_case([1, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 500, 1000, 0, 2], hq, hkv, d, page, dtype, seed=hq + page))


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lens", [[1], [40], [513], [5000], [20011], [3000, 1], [9000, 0, 20, 4000, 77]])
def test_decode_of_few_sequences(lens, hq, hkv, d):
    check_decode(*decode_case(lens, hq, hkv, d, 16, BF, seed=len(lens)))


@pytest.mark.parametrize("lens", [list(range(0, 300)), [33] * 257, [1] * 70 + [6000] + [0] * 60 + [2500, 9], [0] * 600 + [2100] + [0] * 130 + [5, 3000] + [0] * 700])
def test_decode_of_many_sequences(lens):
    case = decode_case(lens, 8, 2, 64, 32, BF, seed=len(lens), extra_columns=80)
    ws = torch.full((native().paged_kv8_decode_workspace_bytes(len(lens), 8, 2, 64, 32, case[5].shape[1]),), 0xff, dtype=U8, device=DEV)
    check_decode(*case, workspace=ws)
    check_decode(*case, window=100, workspace=ws)


# so many sequences that a workgroup takes four heads of one; so many tokens that a wavefront looks its pages up more than once
@pytest.mark.parametrize("lens,hq,hkv,d,page", [([0, 1, 30, 33, 65, 300, 200] * 40, 16, 8, 64, 16), ([5, 0, 129, 40] * 130, 8, 4, 256, 8), ([40000, 3, 20000], 32, 16, 64, 32),
                                                ([38000, 0, 1], 16, 16, 128, 16)])
def test_decode_of_full_workgroups(lens, hq, hkv, d, page):
    check_decode(*decode_case(lens, hq, hkv, d, page, BF, seed=len(lens)))


@pytest.mark.parametrize("layout", LAYOUTS[1:])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_of_strided_operands(layout, d):
    q, *rest = decode_case([70, 1, 900, 2048], 8, 4, d, 16, BF, seed=d, layout=layout)
    out, _ = check_decode(q, *rest)
    wide = torch.zeros(4, 11, d + 8, dtype=BF, device=DEV)
    wide[:, 2:10, :d] = q
    assert torch.equal(K.paged_kv8_decode(wide[:, 2:10, :d], *rest), out)
    odd = torch.zeros(4, 8, d + 3, dtype=BF, device=DEV)                 # rows at odd addresses
    odd[..., 3:] = q
    assert torch.equal(K.paged_kv8_decode(odd[..., 3:], *rest), out)
    big = torch.full((6, 8, d), 7.0, dtype=BF, device=DEV)               # given memory: its neighbours stay
    K.paged_kv8_decode(q, *rest, out=big[1:5])
    assert torch.equal(big[1:5], out) and (big[0] == 7).all() and (big[5] == 7).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [1, 31, 32, 100, 1000, 5000])
def test_decode_of_a_window(window, d):
    q, kc, vc, ks, vs, table, sl = decode_case([0, 1, 30, 32, 33, 100, 131, 1500, 4096], 8, 2, d, 16, BF, seed=window)
    want = attended(q, stood_for(kc, ks), stood_for(vc, vs), table, sl, 0.1, window)
    for s, n in enumerate(sl.tolist()):                                  # what lies before the window is not looked at
        t = torch.arange(0, max(0, n - window), device=DEV)
        b = table[s, t // 16].long()
        raw(kc)[b, t % 16], raw(vc)[b, t % 16] = 0x7f, 0x7f
        raw(ks)[b, :, t % 16], raw(vs)[b, :, t % 16] = 255, 255
    check(K.paged_kv8_decode(q, kc, vc, ks, vs, table, sl, 0.1, window=window, return_lse=True), want, q)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_looks_at_no_token_behind_the_last_and_at_no_missing_page(d):
    lens = [5, 33, 640, 1000, 50, 2000]
    q, kc, vc, ks, vs, table, sl = decode_case(lens, 8, 2, d, 8, HF, seed=3)
    seen = torch.zeros(kc.shape[:2], dtype=torch.bool, device=DEV)
    table[2, 3], table[2, 40:44], table[3, :] = -1, 1 << 20, -7          # pages inside, a run of them, all of a row
    table[5, 100:] = kc.shape[0]
    for s, n in enumerate(lens):
        t = torch.arange(n, device=DEV)
        b = table[s, t // 8].long()
        ok = (b >= 0) & (b < kc.shape[0])
        seen[b[ok], (t % 8)[ok]] = True
    want = attended(q, stood_for(kc, ks), stood_for(vc, vs), table, sl, 0.125)
    raw(kc)[~seen], raw(vc)[~seen] = 0x7f, 0xff
    b, t = torch.nonzero(~seen, as_tuple=True)
    raw(ks)[b, :, t], raw(vs)[b, :, t] = 255, 255
    check(K.paged_kv8_decode(q, kc, vc, ks, vs, table, sl, 0.125, return_lse=True), want, q)
    q, kc, vc, ks, vs, table, _ = decode_case([64, 64, 64], 4, 4, d, 16, BF)
    check_decode(q, kc, vc, ks, vs, table, torch.tensor([1 << 30, -5, 65], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_of_extreme_rows(d):
    """Rows many binades apart, at the types' ends, scores far apart; NaN codes stay in what they belong to."""
    q, kc, vc, ks, vs, table, sl = decode_case([300, 700, 1300], 8, 2, d, 16, HF, seed=9, scale=30.0)
    check_decode(q, kc, vc, ks, vs, table, sl)
    check_decode(q, kc, vc, ks, vs, table, sl, sm=-0.3)
    check_decode(q, kc, vc, ks, vs, table, sl, sm=0.0)
    raw(ks).copy_(torch.randint(100, 122, ks.shape, generator=gen(1)).to(U8))
    raw(vs).copy_(torch.randint(100, 130, ks.shape, generator=gen(2)).to(U8))
    check_decode(q, kc, vc, ks, vs, table, sl)
    raw(vs)[:] = 9
    q, kc, vc, ks, vs, table, sl = decode_case([300, 700, 1300, 9000], 8, 2, d, 16, BF, seed=9)
    raw(vs).copy_(torch.randint(240, 246, vs.shape, generator=gen(3)).to(U8))          # values up to 2^127
    check_decode(q, kc, vc, ks, vs, table, sl)
    raw(vs).copy_(torch.randint(20, 40, vs.shape, generator=gen(3)).to(U8))
    check_decode(q, kc, vc, ks, vs, table, sl)
    raw(vc)[int(table[0, 3]), 1, 0, 5] = 0x7f
    raw(kc)[int(table[0, 3]), 2, 1, 5] = 0x7f
    o, l = K.paged_kv8_decode(q, kc, vc, ks, vs, table, sl, return_lse=True)
    assert torch.isnan(o[0, :4, 5]).all() and torch.isfinite(o[0, :4, :5]).all() and torch.isnan(o[0, 4:]).all() and torch.isnan(l[0, 4:]).all()
    assert torch.isfinite(l[0, :4]).all() and torch.isfinite(o[1:]).all()


@pytest.mark.parametrize("lens", [[700], [50] * 40, [4000, 300, 0]])
def test_decode_equals_16_bit_decode_of_the_rows_read_back(lens):
    """The same keys and values in 16-bit pages give the same within the rounding of both."""
    q, kc, vc, ks, vs, table, sl = decode_case(lens, 8, 2, 128, 16, BF, seed=5)
    blocks = kc.shape[0]
    every = torch.arange(blocks, dtype=torch.int32, device=DEV)[None]
    k, v = K.paged_kv8_read(kc, vc, ks, vs, every, torch.tensor([0, blocks * 16], dtype=torch.int32, device=DEV), blocks * 16)
    a, la = K.paged_kv8_decode(q, kc, vc, ks, vs, table, sl, return_lse=True)
    b, lb = K.paged_kv_decode(q, k.view(kc.shape), v.view(kc.shape), table, sl, return_lse=True)
    _, _, tol, tl = attended(q, k.view(kc.shape).double(), v.view(kc.shape).double(), table, sl, 1 / math.sqrt(128))
    assert ((a.double() - b.double()).abs() <= 2 * tol).all() and ((la.double() - lb.double()).abs().nan_to_num() <= 2 * tl).all()


def test_decode_of_nothing_and_refusals():
    q, kc, vc, ks, vs, table, sl = decode_case([40, 5], 8, 2, 128, 16, BF)
    assert K.paged_kv8_decode(q[:0], kc, vc, ks, vs, table[:0], sl[:0]).shape == (0, 8, 128)
    good = dict(q=q, key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs, block_table=table, seq_lens=sl)
    for bad in (dict(q=q.float()), dict(q=q[..., :64]), dict(q=q[0]), dict(q=q[:, :7]), dict(q=torch.zeros(2, 40, 128, dtype=BF, device=DEV)),
                dict(key_cache=raw(kc)), dict(key_scales=raw(ks)), dict(key_scales=ks[:2]), dict(value_scales=vs.transpose(1, 2)), dict(value_cache=vc[:2], value_scales=vs[:2]),
                dict(key_cache=kc[:, :12], value_cache=vc[:, :12], key_scales=ks[..., :12], value_scales=vs[..., :12]), dict(key_scales=ks.cpu()),
                dict(key_cache=kc[:0], value_cache=vc[:0], key_scales=ks[:0], value_scales=vs[:0]), dict(block_table=table.long()), dict(block_table=table[:1]),
                dict(block_table=table[:, :0]), dict(seq_lens=sl.long()), dict(seq_lens=sl[:1]), dict(seq_lens=sl.cpu()), dict(window=-1), dict(out=q),
                dict(out=torch.empty(2, 8, 128, device=DEV)), dict(out=torch.empty(2, 16, 128, dtype=BF, device=DEV)[:, :8]),
                dict(out=raw(kc).view(-1)[:q.numel() * 2].view(BF).view_as(q))):
        with pytest.raises(ValueError):
            K.paged_kv8_decode(**(good | bad))
    odd = torch.zeros(kc.numel() + 8, dtype=U8, device=DEV)[8:].view(E4).view_as(kc)
    odd_scales = torch.zeros(ks.numel() + 1, dtype=U8, device=DEV)[1:].view(E8).view_as(ks)
    for bad in (dict(key_cache=odd), dict(value_scales=odd_scales)):     # at addresses that are not read
        with pytest.raises(ValueError):
            K.paged_kv8_decode(**(good | bad))
    long = torch.zeros(2, 4000, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="workspace"):
        K.paged_kv8_decode(q, kc, vc, ks, vs, long, sl, workspace=torch.empty(256, dtype=U8, device=DEV))
