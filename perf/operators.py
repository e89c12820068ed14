"""Operators around the 16-bit paged cache, and what is measured of them.

Each case is a dict of plain values; its ``op`` names the operator:

  schedule  ``kernels.paged_schedule``: pages for a step's new tokens from the list of free ones, block tables, slots, positions
  rotary    ``kernels.rotary_embedding``: rotary positions on queries and keys; ``train``: forward and backward
  store     ``kernels.rotary_paged_store``: rotary positions on queries and keys, keys and values into their cache slots
  decode    ``kernels.paged_kv_decode``: attention of one new token per sequence over 16-bit pages

``run`` computes them in elementary torch operations, or calls the framework where ``own`` is true.  Ragged lengths come from
the case's own ``mix`` number, values from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the batch of a serving loop that generates: one token a request
        dict(name="schedule_256", op="schedule", reqs=256, lo=1, hi=4096, prompts=0, chunk=0, page=16, mix=1),
        # many requests, some of them with a chunk of their prompt
        dict(name="schedule_1500_prompts", op="schedule", reqs=1500, lo=0, hi=16000, prompts=100, chunk=700, page=32, mix=2),
        # queries and keys of one step of 32 sequences, far positions
        dict(name="rotary_step_32", op="rotary", tokens=32, hq=32, hkv=8, d=128, rot=128, inter=False, far=1000000, type="bf16",
             train=False),
        # a chunk of prompts, interleaved pairs in the first quarter of wide heads, an odd number of tokens
        dict(name="rotary_part_3001", op="rotary", tokens=3001, hq=16, hkv=4, d=256, rot=64, inter=True, far=40000, type="fp16",
             train=False),
        # a training batch of 4 x 4096 tokens, forward and backward
        dict(name="rotary_train_16384", op="rotary", tokens=16384, hq=32, hkv=8, d=128, rot=128, inter=False, far=4096, type="bf16",
             train=True),
        # a step of 61 sequences, padded to 64 rows of which only the first 61 have a slot
        dict(name="store_step_61", op="store", tokens=64, mapped=61, hq=64, hkv=8, d=128, rot=128, inter=False, far=30000, page=16,
             type="fp16"),
        # the tokens of a large prefill batch
        dict(name="store_12000", op="store", tokens=12000, mapped=12000, hq=32, hkv=8, d=128, rot=128, inter=False, far=8192, page=16,
             type="bf16"),
        # one user, short context: latency
        dict(name="decode_1x777", op="decode", seqs=1, lo=777, hi=777, hq=32, hkv=8, d=128, page=16, window=0, lse=False, type="bf16",
             mix=1),
        # a batch of 32 at 4096 tokens
        dict(name="decode_32x4096", op="decode", seqs=32, lo=4096, hi=4096, hq=32, hkv=8, d=128, page=16, window=0, lse=False,
             type="bf16", mix=1),
        # a larger ragged batch over long contexts, with the normaliser that joins it to another cache
        dict(name="decode_61_ragged", op="decode", seqs=61, lo=500, hi=16000, hq=64, hkv=8, d=128, page=32, window=0, lse=True,
             type="fp16", mix=3),
        # one rank of eight under tensor parallelism: one KV head, long contexts
        dict(name="decode_3x65536_shard", op="decode", seqs=3, lo=40000, hi=65536, hq=8, hkv=1, d=128, page=16, window=0, lse=False,
             type="bf16", mix=4),
        # heads of 64 that see the last 1024 tokens
        dict(name="decode_24_d64_window", op="decode", seqs=24, lo=200, hi=4000, hq=32, hkv=8, d=64, page=16, window=1024, lse=False,
             type="fp16", mix=5),
    ]


# (query heads, KV heads, dimension): whole models and their tensor-parallel shards
HEADS = ((32, 8, 128), (64, 8, 128), (32, 4, 128), (16, 2, 128), (8, 1, 128), (32, 32, 128), (32, 8, 64), (16, 4, 64), (32, 8, 256),
         (16, 4, 256), (8, 1, 256))
MAX_CACHE = 1600 << 20          # bytes of cache behind one drawn decode


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("schedule", "rotary", "store", "decode", "decode", "decode"))
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice((8, 16, 16, 32))
    mix = rng.randrange(1, 1 << 20)
    ty = rng.choice(("bf16", "bf16", "fp16"))
    if op == "schedule":
        reqs = _log(rng, 1, 1500)
        prompts = rng.choice((0, rng.randint(0, min(reqs, 100))))
        return dict(op=op, reqs=reqs, lo=rng.randint(0, 5), hi=_log(rng, 16, 16000), prompts=prompts, chunk=_log(rng, 2, 700), page=page,
                    mix=mix)
    if op in ("rotary", "store"):
        rot = d if rng.random() < 0.5 else max(16, d // rng.choice((2, 4)))
        tokens = _log(rng, 1, 12000 * 4096 // ((hq + hkv) * d))
        case = dict(op=op, tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, inter=rng.random() < 0.4, far=_log(rng, 100, 1000000), type=ty)
        if op == "rotary":
            return dict(case, type=rng.choice((ty, ty, "fp32")), train=rng.random() < 0.4)
        return dict(case, mapped=tokens - rng.randint(0, tokens // 8), page=page)
    hi = _log(rng, 16, 65536)
    seqs = _log(rng, 1, min(256, max(1, MAX_CACHE // (hi * hkv * d * 4))))
    return dict(op=op, seqs=seqs, lo=max(1, hi // rng.choice((1, 4, 20))), hi=hi, hq=hq, hkv=hkv, d=d, page=page,
                window=rng.choice((0, 0, 0, _log(rng, 16, 4096))), lse=rng.random() < 0.3, type=ty, mix=mix)


# ---- sizes ------------------------------------------------------------------------------------------------

def _lens(case):
    r = random.Random(case["mix"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]


def _requests(case):
    """(tokens in the cache, new tokens) per request: one new token, or a chunk of a prompt for some of them."""
    r = random.Random(case["mix"])
    chunked = set(r.sample(range(case["reqs"]), case["prompts"]))
    return [(r.randint(case["lo"], case["hi"]), r.randint(1, case["chunk"]) if i in chunked else 1) for i in range(case["reqs"])]


def work(case):
    if case["op"] == "schedule":
        reqs, page = _requests(case), case["page"]
        new = sum(n for _, n in reqs)
        pages = sum(-(-(c + n) // page) - -(-c // page) for c, n in reqs)
        # lengths in and out, a page read and written for each new one, the open page of a request, a slot and a position per token
        return {"bytes": 8 * len(reqs) + 8 * len(reqs) + 4 + 8 * pages + 4 * len(reqs) + 16 * new, "flops": 0}
    size = 4 if case["type"] == "fp32" else 2
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "rotary":
        n = case["tokens"] * (hq + hkv)
        both = 2 if case["train"] else 1
        return {"bytes": both * (2 * n * d * size + 8 * case["tokens"]), "flops": both * 3.0 * n * case["rot"]}
    if case["op"] == "store":
        t, m = case["tokens"], case["mapped"]
        return {"bytes": 2 * (t * hq + 2 * m * hkv) * d * size + 8 * (t + m), "flops": 3.0 * (t * hq + m * hkv) * case["rot"]}
    tokens = sum(min(n, case["window"] or n) for n in _lens(case))
    rows = case["seqs"] * hq
    return {"bytes": 2 * tokens * hkv * d * size + 2 * rows * d * size + 4 * rows * case["lse"] + 4 * tokens // case["page"],
            "flops": 4.0 * tokens * hq * d}


# ---- inputs -----------------------------------------------------------------------------------------------

def _normal(g, *shape, type="fp32", scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(TYPES[type])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = dict(case)
    if case["op"] == "schedule":
        reqs, page = _requests(case), case["page"]
        most = max(-(-(c + n) // page) for c, n in reqs)
        held = sum(-(-c // page) for c, _ in reqs)
        wanted = sum(-(-(c + n) // page) - -(-c // page) for c, n in reqs)
        pool = torch.randperm(held + 2 * wanted + 7, generator=g, device=DEV, dtype=torch.int32)
        context = torch.tensor([c for c, _ in reqs], dtype=torch.int32, device=DEV)
        table = torch.full((len(reqs), most), -1, dtype=torch.int32, device=DEV)
        mine = torch.arange(most, device=DEV) < ((context + page - 1) // page)[:, None]
        table[mine] = pool[:held]
        state.update(context=context, query=torch.tensor([n for _, n in reqs], dtype=torch.int32, device=DEV), table=table,
                     free=pool[held:].clone(), start=torch.tensor([3], dtype=torch.int32, device=DEV), tokens=sum(n for _, n in reqs))
        return state
    hq, hkv, d, ty = case["hq"], case["hkv"], case["d"], case["type"]
    if case["op"] in ("rotary", "store"):
        t = case["tokens"]
        # one matrix product of a model gives queries, keys and values side by side
        qkv = _normal(g, t, (hq + 2 * hkv), d, type=ty)
        half = case["rot"] // 2
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:],
                     positions=torch.randint(0, case["far"], (t,), generator=g, device=DEV),
                     freq=500000.0 ** -(torch.arange(half, dtype=torch.float64, device=DEV) / half), scale=1.0)
        if case["op"] == "rotary":
            if case["train"]:
                state["q"], state["k"] = state["q"].detach().requires_grad_(), state["k"].detach().requires_grad_()
                state["dq"], state["dk"] = _normal(g, t, hq, d, type=ty), _normal(g, t, hkv, d, type=ty)
            return state
        blocks = t // case["page"] + 5
        state.update(slots=torch.randperm(blocks * case["page"], generator=g, device=DEV)[:case["mapped"]],
                     kc=_normal(g, blocks, case["page"], hkv, d, type=ty), vc=_normal(g, blocks, case["page"], hkv, d, type=ty))
        return state
    lens, page = _lens(case), case["page"]
    most = -(-max(lens) // page)
    held = sum(-(-n // page) for n in lens)
    order = torch.randperm(held + 3, generator=g, device=DEV, dtype=torch.int32)
    lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    table = torch.zeros(case["seqs"], most, dtype=torch.int32, device=DEV)
    table[torch.arange(most, device=DEV) < ((lens + page - 1) // page)[:, None]] = order[:held]
    state.update(q=_normal(g, case["seqs"], hq, d, type=ty, scale=2.0), lens=lens, table=table, sm=1.0 / math.sqrt(d),
                 kc=_normal(g, held + 3, page, hkv, d, type=ty), vc=_normal(g, held + 3, page, hkv, d, type=ty))
    return state


# ---- one pass ---------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else {"schedule": _schedule, "rotary": _rotary, "store": _store, "decode": _decode}[state["op"]](state)


def _own(s):
    from flashquant_amd import kernels as K
    if s["op"] == "schedule":
        step = K.paged_schedule(s["context"], s["query"], s["table"], s["free"], s["page"], s["tokens"], free_start=s["start"])
        return s["table"], step.slot_mapping, step.positions, step.seq_lens, step.cu_seqlens, step.free_end
    if s["op"] == "rotary":
        q, k = K.rotary_embedding(s["q"], s["k"], s["positions"], s["freq"], interleaved=s["inter"], scale=s["scale"])
        if not s["train"]:
            return q, k
        return (q, k, *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    if s["op"] == "store":
        q = K.rotary_paged_store(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["freq"], s["kc"], s["vc"], interleaved=s["inter"],
                                 scale=s["scale"])
        return q, s["kc"], s["vc"]
    return K.paged_kv_decode(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["sm"], window=s["window"], return_lse=s["lse"])


def _schedule(s):
    context, query, table, page = s["context"].long(), s["query"].long(), s["table"], s["page"]
    total = context + query
    old, after = (context + page - 1) // page, (total + page - 1) // page
    first = s["start"].long() + torch.cumsum(after - old, 0) - (after - old)
    column = torch.arange(table.shape[1], device=DEV)
    wanted = first[:, None] + column - old[:, None]
    new = (column >= old[:, None]) & (column < after[:, None])
    page_of = torch.where(wanted < s["free"].shape[0], s["free"][wanted.clamp(0, s["free"].shape[0] - 1)], -1)
    table.copy_(torch.where(new, page_of, table))
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(query, 0)])
    request = torch.repeat_interleave(torch.arange(query.shape[0], device=DEV), query, output_size=s["tokens"])
    positions = torch.arange(s["tokens"], device=DEV) - cu[request] + context[request]
    block = table[request, positions // page].long()
    slots = torch.where(block >= 0, block * page + positions % page, -1)
    return table, slots, positions, total.int(), cu.int(), s["start"] + (after - old).sum().int()


def _turned(x, positions, freq, inter, scale, sign=1.0):
    half = freq.shape[0]
    angle = positions.double()[:, None] * freq
    cos, sin = (scale * angle.cos()).float()[:, None], (sign * scale * angle.sin()).float()[:, None]
    y = x.float().clone()
    if inter:
        a, b = x[..., 0:2 * half:2].float(), x[..., 1:2 * half:2].float()
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :half].float(), x[..., half:2 * half].float()
        y[..., :half], y[..., half:2 * half] = a * cos - b * sin, a * sin + b * cos
    return y.to(x.dtype)


def _rotary(s):
    with torch.no_grad():
        out = [_turned(s[n], s["positions"], s["freq"], s["inter"], s["scale"]) for n in ("q", "k")]
        if s["train"]:
            out += [_turned(s[n], s["positions"], s["freq"], s["inter"], s["scale"], -1.0) for n in ("dq", "dk")]
    return tuple(out)


def _store(s):
    q, k = (_turned(s[n], s["positions"], s["freq"], s["inter"], s["scale"]) for n in ("q", "k"))
    n = s["mapped"]
    s["kc"].view(-1, s["hkv"], s["d"])[s["slots"]] = k[:n]
    s["vc"].view(-1, s["hkv"], s["d"])[s["slots"]] = s["v"][:n]
    return q, s["kc"], s["vc"]


def _decode(s):
    seqs, hq, hkv, d, page = s["seqs"], s["hq"], s["hkv"], s["d"], s["page"]
    lens, n = s["lens"], s["table"].shape[1] * page
    token = torch.arange(n, device=DEV)
    seen = token < lens[:, None]
    if s["window"]:
        seen &= token >= lens[:, None] - s["window"]
    keys = s["kc"][s["table"]].view(seqs, n, hkv, d).permute(0, 2, 3, 1).float()
    scores = torch.matmul(s["q"].float().view(seqs, hkv, hq // hkv, d), keys) * s["sm"]
    del keys
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top)
    del scores
    total = weights.sum(-1, keepdim=True)
    values = torch.where(seen[:, :, None, None], s["vc"][s["table"]].view(seqs, n, hkv, d).float(), 0.0).permute(0, 2, 1, 3)
    out = (torch.matmul(weights, values) / total).view(seqs, hq, d).to(s["q"].dtype)
    return (out, (top + torch.log(total)).view(seqs, hq)) if s["lse"] else out


# ---- the definition, in 64 bits ------------------------------------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        return {"schedule": _exact_schedule, "rotary": _exact_rotary, "store": _exact_store, "decode": _exact_decode}[case["op"]](
            prepare(case, seed))


def _exact_schedule(s):
    table, free, page = s["table"].tolist(), s["free"].tolist(), s["page"]
    at, slots, positions, lens, cu = s["start"].item(), [], [], [], [0]
    for row, (context, new) in zip(table, zip(s["context"].tolist(), s["query"].tolist())):
        for block in range(-(-context // page), -(-(context + new) // page)):
            row[block] = free[at] if at < len(free) else -1
            at += 1
        for p in range(context, context + new):
            positions.append(p)
            slots.append(row[p // page] * page + p % page if row[p // page] >= 0 else -1)
        lens.append(context + new)
        cu.append(cu[-1] + new)
    whole = (table, slots, positions, lens, cu, [at])
    return tuple(torch.tensor(v, dtype=t) for v, t in zip(whole, (torch.int32, torch.int64, torch.int64, torch.int32, torch.int32, torch.int32)))


def _exact_turn(x, s, conjugate=False):
    """The pairs of a row as complex numbers, each times scale * e^(i position frequency)."""
    half, x = s["freq"].shape[0], x.double()
    pairs = x[..., :2 * half].unflatten(-1, (half, 2) if s["inter"] else (2, half))
    z = torch.view_as_complex(pairs.contiguous() if s["inter"] else pairs.transpose(-1, -2).contiguous())
    unit = torch.polar(torch.full_like(s["freq"], s["scale"]).expand(x.shape[0], half), s["positions"][:, None].double() * s["freq"])[:, None]
    y = torch.view_as_real(z * (unit.conj() if conjugate else unit))
    return torch.cat([(y if s["inter"] else y.transpose(-1, -2)).flatten(-2), x[..., 2 * half:]], -1)


def _exact_rotary(s):
    return tuple(_exact_turn(s[n], s, n in ("dq", "dk")) for n in (("q", "k", "dq", "dk") if s["train"] else ("q", "k")))


def _exact_store(s):
    n = s["mapped"]
    caches = []
    for cache, rows in ((s["kc"], _exact_turn(s["k"], s)), (s["vc"], s["v"].double())):
        caches.append(cache.double().view(-1, s["hkv"], s["d"]).index_copy(0, s["slots"], rows[:n]).view(cache.shape))
    return (_exact_turn(s["q"], s), *caches)


def _exact_decode(s):
    outs, norms = [], []
    for q, row, n in zip(s["q"].double(), s["table"], s["lens"].tolist()):
        first = max(0, n - s["window"]) if s["window"] else 0
        token = torch.arange(first, n, device=DEV)
        at = row[token // s["page"]].long(), token % s["page"]
        k, v = (s[c][at].double().transpose(0, 1) for c in ("kc", "vc"))                   # (KV heads, tokens, d)
        x = (k @ q.view(s["hkv"], -1, s["d"]).transpose(1, 2).contiguous()) * s["sm"]      # (KV heads, tokens, group)
        norms.append(torch.logsumexp(x, 1).flatten())
        outs.append((torch.softmax(x, 1).transpose(1, 2).contiguous() @ v).flatten(0, 1))
    return (torch.stack(outs), torch.stack(norms)) if s["lse"] else torch.stack(outs)
