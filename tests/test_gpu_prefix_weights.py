"""What attention over shared pages rounds: no more than that of a sequence by itself, over 16-bit and 8-bit pages."""
from __future__ import annotations

import math

import pytest
import torch

from flashquant_amd import kernels as K
from tests.test_gpu_kv8 import BF, DEV, HF, attended, check, stood_for
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
