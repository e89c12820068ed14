"""What attention over shared pages rounds: no more than that of a sequence by itself, over 16-bit and 8-bit pages."""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_kv8 import BF, DEV, E4, HF, attended, check, raw, stood_for
from tests.test_gpu_prefix import BITS, call, prefix_case

pytestmark = pytest.mark.gpu


def alone(q, cache, table, lens, sm):
    """``attended``, with the tolerance of a decode: weights have 16 significant bits."""
    kc, vc, ks, vs = cache
    return attended(q, *(c.double() if s is None else stood_for(c, s) for c, s in ((kc, ks), (vc, vs))), table, lens, sm)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (32, 8, 128), (12, 1, 128), (6, 2, 256)])
def test_weights_over_shared_tokens_are_those_of_a_sequence_by_itself(hq, hkv, d, dtype, bits):
    sm = 0.5 / math.sqrt(d)                                              # (many tokens count, and their values cancel)
    q, cache, table, lens, ids, prefixes = prefix_case([1500, 640], [0, 1, 0, 0, 1, 0, 0], [0, 5, 300, 1, 0, 40, 2], hq, hkv, d, 16, dtype, bits, seed=d + hq, scale=1.0)
    check(call(q, cache, table, lens, ids, prefixes, sm), alone(q, cache, table, lens, sm), q)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (8, 2, 128), (4, 1, 256)])
def test_small_rows_beside_large_ones(hq, hkv, d, dtype):
    """Each row's power is its own: tokens of small values that have all the weight, beside tokens of large values that have none."""
    q, cache, table, lens, ids, prefixes = prefix_case([640], [0] * 5, [0, 3, 50, 0, 17], hq, hkv, d, 16, dtype, 8, seed=d)
    kc, vc, ks, vs = cache
    q.fill_(1.0)
    unit = 6.0 * math.sqrt(128 / d)                                      # of keys: scores of 68 and -68 round ones of 1
    raw(vs).fill_(127 - 21)                                              # values up to 2^-12
    for t in (2, 38, 303, 639):
        page, at = int(table[0, t // 16]), t % 16
        kc[page, at], kc[page, at ^ 1], kc[page, at ^ 2] = (torch.tensor(x, device=DEV).to(E4) for x in (unit, -unit, -unit))
        raw(ks)[page, :, [at, at ^ 1, at ^ 2]] = 127
        raw(vs)[page, :, at ^ 1], raw(vs)[page, :, at ^ 2] = 127 + 7, 127 + 3     # up to 57344, nearly the most that float16 holds
    check(call(q, cache, table, lens, ids, prefixes), alone(q, cache, table, lens, 1.0 / math.sqrt(d)), q)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prefix_without_a_page_of_the_cache(d, dtype, bits):
    """Nothing of the prefix is there, with NaN in all that is not seen: results and normalisers are those of the tokens behind it."""
    q, cache, table, lens, ids, prefixes = prefix_case([344, 80], [0, 1, 0, 0, 1, -1], [3, 40, 0, 170, 9, 33], 8, 2, d, 8, dtype, bits, seed=d)
    kc, vc, ks, vs = cache
    for s, i in enumerate(ids.tolist()):
        if i == 0:
            table[s, :43] = torch.tensor([-1, kc.shape[0], 1 << 30] * 15, dtype=torch.int32, device=DEV)[:43]
        if i == 1:
            table[s, 2], table[s, 9] = -1, -7
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
        keys, values = stood_for(kc, ks), stood_for(vc, vs)
    else:
        kc[~seen], vc[~seen] = math.nan, math.inf
        keys, values = kc.double(), vc.double()
    keys, values = (torch.where(seen[..., None, None], c, 0.0) for c in (keys, values))
    out, lse = check(call(q, cache, table, lens, ids, prefixes, 0.125), attended(q, keys, values, table, lens, 0.125), q)
    assert (out[2] == 0).all() and torch.isneginf(lse[2]).all()          # no token of its own
