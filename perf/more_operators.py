"""Operators of the 8-bit paged cache and of shared prefixes, and what is measured of them.

Each case is a dict of plain values; its ``op`` names the operator:

  store   ``kernels.rotary_paged_store8``: rotary positions on queries and keys; keys and values, at 8 bits, into their slots
  read    ``kernels.paged_kv8_read``: tokens of an 8-bit cache back as 16-bit rows
  decode  ``kernels.paged_kv8_decode``: attention of one new token per sequence over 8-bit pages
  prefix  ``kernels.paged_prefix_decode``: the same over 16-bit or 8-bit pages, where sequences begin with the same pages

A row (the ``d`` values of a token and KV head) at 8 bits is e4m3 times a power of two of its own.  ``run`` computes them in
elementary torch operations, or calls the framework where ``own`` is true.  Ragged lengths come from the case's own ``mix`` number,
values from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
LOWEST, HIGHEST = -118, 120     # powers of two of a row


def listed():
    return [
        # a step of 45 sequences, padded to 48 rows; interleaved pairs in the first quarter of wide heads
        dict(name="store_step_48", op="store", tokens=48, mapped=45, hq=16, hkv=4, d=256, rot=64, inter=True, far=60000, page=16, type="fp16"),
        # the tokens of a prefill batch
        dict(name="store_9001", op="store", tokens=9001, mapped=9001, hq=32, hkv=8, d=128, rot=128, inter=False, far=16384, page=32, type="bf16"),
        # what three requests have in the cache, for the attention of their next chunks
        dict(name="read_3_short", op="read", seqs=3, lo=90, hi=700, first=0, hkv=8, d=128, page=16, type="bf16", mix=1),
        # a batch of longer contexts, from a token of its own on
        dict(name="read_13_long", op="read", seqs=13, lo=1500, hi=6000, first=900, hkv=8, d=128, page=16, type="fp16", mix=2),
        # one user, short context: latency
        dict(name="decode_1x900", op="decode", seqs=1, lo=900, hi=900, hq=32, hkv=8, d=128, page=16, window=0, lse=False, type="bf16", mix=1),
        # a batch of 32 at 4096 tokens
        dict(name="decode_32x4096", op="decode", seqs=32, lo=4096, hi=4096, hq=32, hkv=8, d=128, page=16, window=0, lse=False, type="bf16",
             mix=1),
        # a larger ragged batch over long contexts, with the normaliser that joins it to another cache
        dict(name="decode_57_ragged", op="decode", seqs=57, lo=400, hi=15000, hq=64, hkv=8, d=128, page=32, window=0, lse=True, type="fp16",
             mix=3),
        # heads of 64 that see the last 1500 tokens
        dict(name="decode_20_d64_window", op="decode", seqs=20, lo=200, hi=5000, hq=32, hkv=8, d=64, page=16, window=1500, lse=False,
             type="fp16", mix=5),
        # a few requests behind one system prompt
        dict(name="prefix_6_of_2000", op="prefix", seqs=6, prefixes=1, plo=2000, phi=2000, alone=0, lo=1, hi=150, hq=32, hkv=8, d=128, page=16,
             bits=16, lse=False, type="bf16", mix=1),
        # a full batch behind a long system prompt
        dict(name="prefix_96_of_6000", op="prefix", seqs=96, prefixes=1, plo=6000, phi=6000, alone=0, lo=50, hi=1200, hq=32, hkv=8, d=128,
             page=16, bits=16, lse=False, type="bf16", mix=2),
        # three prompts and requests of their own kind, over 8 bits
        dict(name="prefix_150_mixed_8", op="prefix", seqs=150, prefixes=3, plo=900, phi=6000, alone=14, lo=1, hi=900, hq=64, hkv=8, d=128, page=32,
             bits=8, lse=True, type="fp16", mix=3),
        # many answers to one long document, one rank of eight
        dict(name="prefix_40_of_32768_shard", op="prefix", seqs=40, prefixes=1, plo=32768, phi=32768, alone=0, lo=1, hi=500, hq=8, hkv=1, d=128,
             page=16, bits=8, lse=False, type="bf16", mix=4),
    ]


# (query heads, KV heads, dimension): whole models and their tensor-parallel shards
HEADS = ((32, 8, 128), (64, 8, 128), (32, 4, 128), (16, 2, 128), (8, 1, 128), (32, 32, 128), (32, 8, 64), (16, 4, 64), (32, 8, 256),
         (16, 4, 256), (8, 1, 256))
MAX_VALUES = 450 << 20           # keys that one drawn decode gathers, in values, padded


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("store", "read", "decode", "decode", "prefix", "prefix", "prefix"))
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice((8, 16, 16, 32))
    mix = rng.randrange(1, 1 << 20)
    ty = rng.choice(("bf16", "bf16", "fp16"))
    if op == "store":
        rot = d if rng.random() < 0.5 else max(16, d // rng.choice((2, 4)))
        tokens = _log(rng, 1, 9001 * 48 * 128 // ((hq + 2 * hkv) * d))
        return dict(op=op, tokens=tokens, mapped=tokens - rng.randint(0, tokens // 8), hq=hq, hkv=hkv, d=d, rot=rot, inter=rng.random() < 0.4,
                    far=_log(rng, 100, 1000000), page=page, type=ty)
    if op == "read":
        hi = _log(rng, 1, 12000)
        seqs = _log(rng, 1, max(1, min(200, 48000 * 1024 // (hi * hkv * d))))
        return dict(op=op, seqs=seqs, lo=rng.randint(1, hi), hi=hi, first=rng.choice((0, rng.randint(0, 3000))), hkv=hkv, d=d, page=page, type=ty,
                    mix=mix)
    if op == "decode":
        hi = _log(rng, 16, 50000)
        seqs = _log(rng, 1, min(256, max(1, MAX_VALUES // (hi * hkv * d))))
        return dict(op=op, seqs=seqs, lo=max(1, hi // rng.choice((1, 4, 20))), hi=hi, hq=hq, hkv=hkv, d=d, page=page,
                    window=rng.choice((0, 0, 0, _log(rng, 16, 4096))), lse=rng.random() < 0.3, type=ty, mix=mix)
    phi = _log(rng, 64, 32768)
    hi = _log(rng, 1, 1200)
    seqs = _log(rng, 2, min(200, max(2, MAX_VALUES // ((phi + hi) * hkv * d))))
    return dict(op=op, seqs=seqs, prefixes=rng.randint(1, 1 + min(4, seqs // 8)), plo=max(1, phi // rng.choice((1, 1, 3))), phi=phi,
                alone=rng.choice((0, 0, seqs // 10)), lo=rng.randint(1, hi), hi=hi, hq=hq, hkv=hkv, d=d, page=page, bits=rng.choice((16, 8)),
                lse=rng.random() < 0.3, type=ty, mix=mix)


# ---- sizes ------------------------------------------------------------------------------------------------

def _lens(case):
    r = random.Random(case["mix"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]


def _shared(case):
    """(tokens of every prefix, prefix of every sequence or -1, tokens of a sequence behind it).  Shared are whole pages."""
    r = random.Random(case["mix"])
    prefixes = [r.randint(case["plo"], case["phi"]) // case["page"] * case["page"] for _ in range(case["prefixes"])]
    ids = [r.randrange(case["prefixes"]) for _ in range(case["seqs"])]
    for s in r.sample(range(case["seqs"]), case["alone"]):
        ids[s] = -1
    return prefixes, ids, [r.randint(case["lo"], case["hi"]) for _ in ids]


def work(case):
    hkv, d = case["hkv"], case["d"]
    row = d + 1                                                          # bytes of a row at 8 bits
    if case["op"] == "read":
        n = sum(_lens(case))
        return {"bytes": 2 * n * hkv * (row + 2 * d) + 4 * n // case["page"], "flops": 2.0 * n * hkv * d}
    hq = case["hq"]
    if case["op"] == "store":
        t, m = case["tokens"], case["mapped"]
        return {"bytes": 4 * t * hq * d + 2 * m * hkv * (2 * d + row) + 8 * (t + m),
                "flops": 3.0 * (t * hq + m * hkv) * case["rot"] + 4.0 * m * hkv * d}
    rows = case["seqs"] * hq
    outer = 4 * rows * d + 4 * rows * case["lse"]
    if case["op"] == "decode":
        tokens = sum(min(n, case["window"] or n) for n in _lens(case))
        return {"bytes": 2 * tokens * hkv * row + outer + 4 * tokens // case["page"], "flops": 4.0 * tokens * hq * d}
    prefixes, ids, lens = _shared(case)
    read = sum(n for p, n in enumerate(prefixes) if p in ids) + sum(lens)
    seen = sum(lens) + sum(prefixes[p] for p in ids if p >= 0)
    return {"bytes": 2 * read * hkv * (row if case["bits"] == 8 else 2 * d) + outer + 4 * read // case["page"], "flops": 4.0 * seen * hq * d}


# ---- inputs -----------------------------------------------------------------------------------------------

def _normal(g, *shape, type="fp32", scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(TYPES[type])


def _quantised(x):
    """Rows of float32 values as e4m3 and the power of two of each row, both as bytes: the largest magnitude goes to (224, 448]."""
    finite = torch.where(x.isfinite(), x.abs(), 0.0)
    part, power = torch.frexp(finite.amax(-1))
    power = (power - 9 + (part > 0.875)).clamp(LOWEST, HIGHEST)
    return torch.ldexp(x, -power[..., None]).to(E4M3).view(torch.uint8), (power + 127).to(torch.uint8)


def _cache(g, blocks, case):
    """Keys or values (blocks, page, heads, d) at 8 bits and their powers (blocks, heads, page)."""
    codes, powers = _quantised(_normal(g, blocks, case["page"], case["hkv"], case["d"]))
    return codes.view(E4M3), powers.transpose(1, 2).contiguous().view(E8M0)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(case)
    hkv, d, page, ty = case["hkv"], case["d"], case["page"], case["type"]
    if case["op"] == "store":
        t, hq, half = case["tokens"], case["hq"], case["rot"] // 2
        # one matrix product of a model gives queries, keys and values side by side
        qkv = _normal(g, t, (hq + 2 * hkv), d, type=ty)
        blocks = t // page + 5
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], scale=1.0,
                     positions=torch.randint(0, case["far"], (t,), generator=g, device=DEV),
                     freq=500000.0 ** -(torch.arange(half, dtype=torch.float64, device=DEV) / half),
                     slots=torch.randperm(blocks * page, generator=g, device=DEV)[:case["mapped"]])
        (state["kc"], state["ks"]), (state["vc"], state["vs"]) = _cache(g, blocks, case), _cache(g, blocks, case)
        return state
    shared = []                                                          # pages of every prefix
    if case["op"] == "prefix":
        prefixes, ids, lens = _shared(case)
        shared = [n // page for n in prefixes]
        lens = [n + (prefixes[p] if p >= 0 else 0) for p, n in zip(ids, lens)]
    else:
        ids, lens = [-1] * case["seqs"], _lens(case)
    first = [random.Random(case["mix"] + s).randint(0, case["first"]) for s in range(len(lens))] if case["op"] == "read" else [0] * len(lens)
    ends = [n + f for n, f in zip(lens, first)]
    most = max(1, -(-max(ends) // page))
    mine = [-(-n // page) - (shared[p] if p >= 0 else 0) for p, n in zip(ids, ends)]
    blocks = sum(shared) + sum(mine) + 3
    order = torch.randperm(blocks, generator=g, device=DEV, dtype=torch.int32).cpu()
    table, at = torch.zeros(len(ends), most, dtype=torch.int32), sum(shared)
    for s, (p, n) in enumerate(zip(ids, mine)):
        skip = shared[p] if p >= 0 else 0
        begin = sum(shared[:p]) if p >= 0 else 0
        table[s, :skip] = order[begin:begin + skip]
        table[s, skip:skip + n] = order[at:at + n]
        at += n
    state.update(table=table.to(DEV), lens=torch.tensor(ends, dtype=torch.int32, device=DEV), ks=None, vs=None)
    if case["op"] == "prefix" and case["bits"] == 16:
        state["kc"], state["vc"] = (_normal(g, blocks, page, hkv, d, type=ty) for _ in range(2))
    else:
        (state["kc"], state["ks"]), (state["vc"], state["vs"]) = _cache(g, blocks, case), _cache(g, blocks, case)
    if case["op"] == "read":
        cu = torch.tensor([0] + lens).cumsum(0)
        state.update(cu=cu.int().to(DEV), first=torch.tensor(first, dtype=torch.int32, device=DEV), tokens=sum(lens))
        return state
    state.update(q=_normal(g, case["seqs"], case["hq"], d, type=ty, scale=2.0), sm=1.0 / math.sqrt(d))
    if case["op"] == "prefix":
        state.update(ids=torch.tensor(ids, dtype=torch.int32, device=DEV), shared=torch.tensor(prefixes, dtype=torch.int32, device=DEV))
    return state


# ---- one pass ---------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else {"store": _store, "read": _read, "decode": _decode, "prefix": _decode}[state["op"]](state)


def _own(s):
    from flashquant_amd import kernels as K
    if s["op"] == "store":
        q = K.rotary_paged_store8(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["freq"], s["kc"], s["vc"], s["ks"], s["vs"],
                                  interleaved=s["inter"], scale=s["scale"])
        return q, s["kc"], s["vc"], s["ks"], s["vs"]
    if s["op"] == "read":
        return K.paged_kv8_read(s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["cu"], s["tokens"], starts=s["first"], dtype=TYPES[s["type"]])
    if s["op"] == "decode":
        return K.paged_kv8_decode(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"], s["sm"], window=s["window"],
                                  return_lse=s["lse"])
    return K.paged_prefix_decode(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["ids"], s["shared"], s["sm"], key_scales=s["ks"],
                                 value_scales=s["vs"], return_lse=s["lse"])


def _turned(x, positions, freq, inter, scale):
    """Rotary positions, in float32."""
    half = freq.shape[0]
    angle = positions.double()[:, None] * freq
    cos, sin = (scale * angle.cos()).float()[:, None], (scale * angle.sin()).float()[:, None]
    y = x.float().clone()
    if inter:
        a, b = x[..., 0:2 * half:2].float(), x[..., 1:2 * half:2].float()
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :half].float(), x[..., half:2 * half].float()
        y[..., :half], y[..., half:2 * half] = a * cos - b * sin, a * sin + b * cos
    return y


def _store(s):
    q, k = (_turned(s[n], s["positions"], s["freq"], s["inter"], s["scale"]) for n in ("q", "k"))
    n, slots, page = s["mapped"], s["slots"], s["page"]
    for cache, scales, rows in ((s["kc"], s["ks"], k[:n]), (s["vc"], s["vs"], s["v"][:n].float())):
        codes, powers = _quantised(rows)
        cache.view(torch.uint8).view(-1, s["hkv"], s["d"])[slots] = codes
        scales.view(torch.uint8)[slots // page, :, slots % page] = powers
    return q.to(s["q"].dtype), s["kc"], s["vc"], s["ks"], s["vs"]


def _values(cache, scales, at):
    """Rows (.., page, heads, d) of the pages `at`, in float32."""
    if scales is None:
        return cache[at].float()
    rows = cache.view(torch.uint8)[at].view(E4M3).float()
    return rows * torch.exp2(scales.view(torch.uint8)[at].float() - 127.0).transpose(-1, -2)[..., None]


def _read(s):
    token = torch.arange(s["tokens"], device=DEV)
    cu = s["cu"].long()
    seq = torch.searchsorted(cu, token, right=True) - 1
    place = token - cu[seq] + s["first"].long()[seq]
    block, inside = s["table"][seq, place // s["page"]].long(), place % s["page"]
    rows = []
    for cache, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        codes = cache.view(torch.uint8)[block, inside].view(E4M3).float()
        power = torch.exp2(scales.view(torch.uint8)[block, :, inside].float() - 127.0)
        rows.append((codes * power[..., None]).to(TYPES[s["type"]]))
    return tuple(rows)


def _decode(s):
    seqs, hq, hkv, d, page = s["seqs"], s["hq"], s["hkv"], s["d"], s["page"]
    lens, n = s["lens"], s["table"].shape[1] * page
    token = torch.arange(n, device=DEV)
    seen = token < lens[:, None]
    if s.get("window"):
        seen &= token >= lens[:, None] - s["window"]
    keys = _values(s["kc"], s["ks"], s["table"]).view(seqs, n, hkv, d).permute(0, 2, 3, 1)
    scores = torch.matmul(s["q"].float().view(seqs, hkv, hq // hkv, d), keys) * s["sm"]
    del keys
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top)
    del scores
    total = weights.sum(-1, keepdim=True)
    values = torch.where(seen[:, :, None, None], _values(s["vc"], s["vs"], s["table"]).view(seqs, n, hkv, d), 0.0).permute(0, 2, 1, 3)
    out = (torch.matmul(weights, values) / total).view(seqs, hq, d).to(s["q"].dtype)
    return (out, (top + torch.log(total)).view(seqs, hq)) if s["lse"] else out


# ---- the definition, in 64 bits ------------------------------------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        return {"store": _exact_store, "read": _exact_read, "decode": _exact_decode, "prefix": _exact_decode}[case["op"]](prepare(case, seed))


def _exact_turn(x, s):
    """The pairs of a row as complex numbers, each times scale * e^(i position frequency)."""
    half, x = s["freq"].shape[0], x.double()
    pairs = x[..., :2 * half].unflatten(-1, (half, 2) if s["inter"] else (2, half))
    z = torch.view_as_complex(pairs.contiguous() if s["inter"] else pairs.transpose(-1, -2).contiguous())
    unit = torch.polar(torch.full_like(s["freq"], s["scale"]).expand(x.shape[0], half), s["positions"][:, None].double() * s["freq"])[:, None]
    y = torch.view_as_real(z * unit)
    return torch.cat([(y if s["inter"] else y.transpose(-1, -2)).flatten(-2), x[..., 2 * half:]], -1)


def _exact_store(s):
    n, out = s["mapped"], [_exact_turn(s["q"], s)]
    scales = []
    for cache, kept, rows in ((s["kc"], s["ks"], _exact_turn(s["k"], s)), (s["vc"], s["vs"], s["v"].double())):
        rows = rows[:n]
        # the smallest power of two that leaves nothing above the largest e4m3, then four significant bits down to 2^-9
        power = torch.ceil(torch.log2(rows.abs().amax(-1) / 448.0)).clamp(LOWEST, HIGHEST)
        x = rows * torch.exp2(-power)[..., None]
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        codes = torch.round(x / step) * step
        out.append(cache.float().double().view(-1, s["hkv"], s["d"]).index_copy(0, s["slots"], codes).view(cache.shape))
        all_scales = torch.exp2(kept.view(torch.uint8).double() - 127).transpose(1, 2).reshape(-1, s["hkv"])
        all_scales = all_scales.index_copy(0, s["slots"], torch.exp2(power))
        scales.append(all_scales.view(kept.shape[0], s["page"], s["hkv"]).transpose(1, 2))
    return (*out, *scales)


def _exact_rows(s, row, first, last):
    """Keys and values (heads, tokens, d) of tokens [first, last) on the pages of `row`."""
    token = torch.arange(first, last, device=DEV)
    at = row[token // s["page"]].long(), token % s["page"]
    rows = []
    for cache, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        if scales is None:
            x = cache[at].double()
        else:
            power = scales.view(torch.uint8).transpose(1, 2)[at].double() - 127
            x = cache.view(torch.uint8)[at].view(E4M3).double() * torch.exp2(power)[..., None]
        rows.append(x.transpose(0, 1))
    return rows


def _exact_read(s):
    cu, parts = s["cu"].tolist(), ([], [])
    for i, (row, first) in enumerate(zip(s["table"], s["first"].tolist())):
        for part, x in zip(parts, _exact_rows(s, row, first, first + cu[i + 1] - cu[i])):
            part.append(x.transpose(0, 1))
    return tuple(torch.cat(p) for p in parts)


def _exact_decode(s):
    outs, norms = [], []
    for q, row, n in zip(s["q"].double(), s["table"], s["lens"].tolist()):
        k, v = _exact_rows(s, row, max(0, n - s["window"]) if s.get("window") else 0, n)    # (KV heads, tokens, d)
        x = (k @ q.view(s["hkv"], -1, s["d"]).transpose(1, 2).contiguous()) * s["sm"]       # (KV heads, tokens, group)
        norms.append(torch.logsumexp(x, 1).flatten())
        outs.append((torch.softmax(x, 1).transpose(1, 2).contiguous() @ v).flatten(0, 1))
    return (torch.stack(outs), torch.stack(norms)) if s["lse"] else torch.stack(outs)
