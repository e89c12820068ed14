"""Values at the ends of their types in an 8-bit cache: what is finite on the way in is finite on the way out, within a code's error."""
from __future__ import annotations

import math

import pytest
import torch

from flashquant_amd import kernels as K
from tests.test_gpu_kv8 import BF, DEV, E4, E8, HF, U8, attended, check, gen, raw, stood_for

pytestmark = pytest.mark.gpu
PAGE, HKV, HQ = 16, 2, 8
# the largest of the type, and down to where codes end at 1.75 of the last binade; from 1.9375 of it on the nearest code is a binade further
ENDS = {BF: [3.3895313892515355e38, 3.3e38, 3.297e38, 3.19e38], HF: [65504.0, 64000.0, 63488.0, 61440.0]}


def stored(d, dtype, keys_too):
    """(q, caches, values): 48 tokens whose values reach the ends of ``dtype``; with ``keys_too`` their keys do as well."""
    g = gen(d)
    ends = torch.tensor(ENDS[dtype], dtype=torch.float64)
    v = torch.randn(48, HKV, d, generator=g).double() * (ends[0] / 8)
    v[:, :, ::7] = (ends[torch.randint(0, 4, v[:, :, ::7].shape, generator=g)] * (2 * torch.randint(0, 2, v[:, :, ::7].shape, generator=g) - 1))
    v = v.clamp(-float(ends[0]), float(ends[0])).to(dtype).to(DEV)
    k = v.flip(0).contiguous() if keys_too else torch.randn(48, HKV, d, generator=g).to(dtype).to(DEV)
    assert torch.isfinite(v).all()
    rows, scales = torch.zeros(2, 4, PAGE, HKV, d, dtype=U8, device=DEV), torch.zeros(2, 4, HKV, PAGE, dtype=U8, device=DEV)
    cache = (*rows.view(E4), *scales.view(E8))
    K.rotary_paged_store8(v[:, :0].expand(-1, 0, -1), k, v, torch.zeros(48, dtype=torch.long, device=DEV), torch.arange(48, device=DEV),
                          K.rotary_frequencies(d, device=DEV)[0], *cache)
    # scores of a few units
    q = torch.randn(4, HQ, d, generator=g) * (2.0 ** (-122 if dtype == BF else -10) if keys_too else 1.0)
    return q.to(dtype).to(DEV), cache, v


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_read_of_what_reaches_the_end_of_its_type(d, dtype):
    _, cache, v = stored(d, dtype, False)
    table, cu = torch.arange(3, dtype=torch.int32, device=DEV)[None], torch.tensor([0, 48], dtype=torch.int32, device=DEV)
    got = K.paged_kv8_read(*cache, table, cu, 48, dtype=dtype)[1]
    assert (raw(cache[1])[:3] & 0x7f == 0x78).any()                      # codes of 256 are among them
    assert torch.isfinite(got).all()
    assert ((got.double() - v.double()).abs() <= v.double().abs() * 2.0 ** -4 + v.double().abs().amax(-1, keepdim=True) * 2.0 ** -17).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("columns", [3, 200])
@pytest.mark.parametrize("keys_too", [False, True])
def test_attention_over_what_reaches_the_end_of_its_type(keys_too, columns, d, dtype):
    q, cache, v = stored(d, dtype, keys_too)
    kc, vc, ks, vs = cache
    table = torch.full((4, columns), -1, dtype=torch.int32, device=DEV)
    table[:, :3] = torch.arange(3, device=DEV)
    lens = torch.tensor([33, 48, 32, 1], dtype=torch.int32, device=DEV)
    sm = 1.0 / math.sqrt(d)
    want = attended(q, stood_for(kc, ks), stood_for(vc, vs), table, lens, sm)
    ids, prefixes = torch.tensor([0, 0, 0, -1], dtype=torch.int32, device=DEV), torch.tensor([32], dtype=torch.int32, device=DEV)
    for got in (K.paged_kv8_decode(q, kc, vc, ks, vs, table, lens, sm, return_lse=True),
                K.paged_prefix_decode(q, kc, vc, table, lens, ids, prefixes, sm, key_scales=ks, value_scales=vs, return_lse=True)):
        assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()
        check(got, want, q)
        assert ((got[0][3].double().view(HKV, -1, d) - v[0].double()[:, None]).abs() <= v[0].double().abs()[:, None] * 2.0 ** -4 + float(v[0].double().abs().max()) * 2.0 ** -17).all()
