"""CPU-only checks of the operators around a 16-bit paged cache: the rotary frequencies against their formulas, refusals of the
Python layer, status codes of the C ABI before anything touches the GPU."""
from __future__ import annotations

import ctypes
import math
import os

import pytest
import torch

from flashquant_amd import kernels as K

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashquant_amd", "libfq_hip.so")
FQ_OK, FQ_NULL, FQ_DIM, FQ_BLOCK, FQ_DTYPE, FQ_SHAPE, FQ_ALIGN, FQ_WS, FQ_LAUNCH = range(9)


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(LIB)


# ---- frequencies ------------------------------------------------------------------------------------------------------------

def test_plain_linear_and_ntk_frequencies():
    f, scale = K.rotary_frequencies(8, base=10000.0)
    assert f.dtype == torch.float64 and scale == 1.0
    assert f.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    assert torch.equal(K.rotary_frequencies(8, scaling="linear", factor=4.0)[0], f / 4.0)
    ntk, scale = K.rotary_frequencies(64, scaling="ntk", factor=8.0)
    plain = K.rotary_frequencies(64)[0]
    assert scale == 1.0 and ntk[0] == 1.0 and float(ntk[-1] * 8.0) == pytest.approx(float(plain[-1]), rel=1e-12)
    assert K.rotary_frequencies(2)[0].tolist() == [1.0]


def test_yarn_frequencies_by_the_turns_of_a_pair():
    dim, base, factor, original = 128, 10000.0, 16.0, 4096
    f, scale = K.rotary_frequencies(dim, base, "yarn", factor=factor, original_max_position=original)
    plain = K.rotary_frequencies(dim, base)[0]
    turns = original * plain / (2 * math.pi)
    share = f / plain
    assert scale == pytest.approx(0.1 * math.log(16.0) + 1.0)
    assert (share[turns > 40] == 1.0).all() and (share[turns < 0.8] - 1 / factor).abs().max() < 1e-12
    assert (share[1:] <= share[:-1]).all()
    # the ramp runs over the pairs between those that turn 32 times and once
    low, high = math.floor(64 * math.log(original / 32 / 2 / math.pi) / math.log(base)), math.ceil(64 * math.log(original / 2 / math.pi) / math.log(base))
    i = (low + high) // 2
    r = (i - low) / (high - low)
    assert float(share[i]) == pytest.approx(1 - r + r / factor, rel=1e-12)


def test_band_frequencies_by_wavelength():
    f, scale = K.rotary_frequencies(128, 500000.0, "bands", factor=8.0, original_max_position=8192, low_freq_factor=1.0, high_freq_factor=4.0)
    plain = K.rotary_frequencies(128, 500000.0)[0]
    assert scale == 1.0
    for got, w in zip(f.tolist(), plain.tolist()):
        length = 2 * math.pi / w
        if length < 8192 / 4.0:
            want = w
        elif length > 8192 / 1.0:
            want = w / 8.0
        else:
            smooth = (8192 / length - 1.0) / 3.0
            want = (1 - smooth) * w / 8.0 + smooth * w
        assert got == pytest.approx(want, rel=1e-12)


def test_factor_frequencies_and_refusals():
    f, scale = K.rotary_frequencies(4, scaling="factors", factors=[2.0, 5.0], factor=4.0, original_max_position=256)
    assert f.tolist() == pytest.approx([0.5, 0.002], rel=1e-12) and scale == pytest.approx(math.sqrt(1.25))
    for args, more in (((7,), {}), ((0,), {}), ((8, 0.0), {}), ((8, 1e4, "linear"), dict(factor=0.0)), ((8, 1e4, "yarn"), dict(factor=2.0)), ((8, 1e4, "bands"), {}),
                       ((2, 1e4, "ntk"), {}), ((8, 1e4, "what"), {}), ((8, 1e4, "factors"), {}), ((8, 1e4, "factors"), dict(factors=[1.0])),
                       ((8, 1e4, "factors"), dict(factors=[1.0] * 4, factor=2.0)), ((8, 1.0, "yarn"), dict(original_max_position=100)),
                       ((8, 1e4, "bands"), dict(original_max_position=100, low_freq_factor=4.0))):
        with pytest.raises(ValueError):
            K.rotary_frequencies(*args, **more)


# ---- the Python layer ---------------------------------------------------------------------------------------------------------

def test_no_cpu_fallback():
    q, p, f = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.long), K.rotary_frequencies(64)[0]
    cache, ints = torch.zeros(1, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: K.rotary_embedding(q, q, p, f), lambda: K.rotary_embedding(q.clone().requires_grad_(), None, p, f),
                 lambda: K.rotary_paged_store(q, q, q, p, p, f, cache, cache), lambda: K.paged_schedule(ints, ints, ints[None], ints, 16, 1),
                 lambda: K.paged_kv_decode(q, cache, cache, ints[None], ints)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


# ---- the C ABI ------------------------------------------------------------------------------------------------------------------

def _p(v):
    return ctypes.c_void_p(v)


def _strides(*v):
    return (ctypes.c_int64 * len(v))(*v)


I, L, F, P, Z = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t


def test_rotary_argument_errors(lib):
    f = lib.fq_rotary_embedding
    f.argtypes = [P, P, P, P, I, P, P, P, P, I, P, I, L, P, I, I, F, I, L, L, I, I, P]
    s = _strides(0, 512, 64)

    def call(q=64, hq=8, k=64, hk=2, positions=64, pb=8, freq=64, half=32, batch=1, tokens=3, d=64, dtype=1):
        return f(_p(q), s, _p(q), s, hq, _p(k), s, _p(k), s, hk, _p(positions), pb, 0, _p(freq), half, 0, 1.0, 0, batch, tokens, d, dtype, _p(0))

    assert call(tokens=0) == FQ_OK and call(batch=0) == FQ_OK
    for bad in (dict(tokens=-1), dict(batch=-1), dict(hq=-1), dict(hq=0, hk=0), dict(hq=5000), dict(half=0), dict(half=33), dict(d=1026, half=2), dict(batch=1 << 30, tokens=1 << 30)):
        assert call(**bad) == FQ_SHAPE, bad
    assert call(pb=2) == FQ_DTYPE and call(dtype=7) == FQ_DTYPE
    for name in ("q", "k", "positions", "freq"):
        assert call(**{name: 0}) == FQ_NULL, name


def test_rotary_store_argument_errors(lib):
    f = lib.fq_rotary_paged_store
    f.argtypes = [P, P, P, P, I, P, P, P, P, I, P, I, P, I, I, F, P, L, P, P, P, P, I, L, L, I, I, P]
    s, c = _strides(512, 64), _strides(2048, 128, 64)

    def call(q=64, hq=8, k=64, v=64, hkv=2, positions=64, pb=8, freq=64, half=32, slots=64, mapped=3, cache=64, page=16, blocks=4, tokens=3, d=64, dtype=1):
        return f(_p(q), s, _p(q), s, hq, _p(k), s, _p(v), s, hkv, _p(positions), pb, _p(freq), half, 0, 1.0, _p(slots), mapped, _p(cache), c, _p(cache), c,
                 page, blocks, tokens, d, dtype, _p(0))

    assert call(tokens=0, mapped=0) == FQ_OK
    for bad in (dict(tokens=-1), dict(hkv=0), dict(mapped=4), dict(mapped=-1), dict(blocks=-1), dict(blocks=1 << 31), dict(half=33), dict(hq=5000)):
        assert call(**bad) == FQ_SHAPE, bad
    assert call(page=12) == FQ_BLOCK and call(dtype=2) == FQ_DTYPE and call(pb=1) == FQ_DTYPE
    for name in ("q", "k", "v", "positions", "freq", "slots", "cache"):
        assert call(**{name: 0}) == FQ_NULL, name


def test_schedule_argument_errors(lib):
    f = lib.fq_paged_schedule
    f.argtypes = [P, P, P, L, P, L, P, P, P, P, P, P, I, L, I, I, P]

    def call(context=64, table=64, stride=4, free=64, num_free=5, start=0, end=128, slots=64, lens=64, cu=64, reqs=2, tokens=3, blocks=4, page=16):
        return f(_p(context), _p(64), _p(table), stride, _p(free), num_free, _p(start), _p(end), _p(slots), _p(64), _p(lens), _p(cu), reqs, tokens, blocks, page, _p(0))

    for bad in (dict(reqs=-1), dict(tokens=-1), dict(tokens=1 << 31), dict(blocks=0), dict(num_free=-1), dict(stride=3), dict(blocks=1 << 28, stride=1 << 28), dict(start=128)):
        assert call(**bad) == FQ_SHAPE, bad
    assert call(page=24) == FQ_BLOCK
    for name in ("context", "table", "free", "end", "slots", "lens", "cu"):
        assert call(**{name: 0}) == FQ_NULL, name


def test_decode_argument_errors_and_sizes(lib):
    f, need = lib.fq_paged_kv_decode, lib.fq_paged_kv_decode_workspace_bytes
    f.argtypes = [P, P, P, P, P, P, P, L, P, P, P, I, I, I, I, I, I, L, F, I, I, P, Z, P]
    need.argtypes, need.restype = [I] * 6, Z

    def call(q=64, cache=64, table=64, lens=64, out=64, seqs=2, hq=8, hkv=2, d=128, page=16, columns=4, blocks=9, window=0, dtype=1, ws=0, room=0,
             qs=(1024, 128), cs=(4096, 256, 128), row=4):
        return f(_p(q), _strides(*qs), _p(cache), _strides(*cs), _p(cache), _strides(*cs), _p(table), row, _p(lens), _p(out), _p(0), seqs, hq, hkv, d, page, columns,
                 blocks, 0.1, window, dtype, _p(ws), room, _p(0))

    assert call(seqs=0) == FQ_OK
    for bad in (dict(seqs=-1), dict(hq=9), dict(hq=34), dict(hkv=0), dict(columns=0), dict(blocks=0), dict(blocks=1 << 31), dict(columns=1 << 27), dict(window=-1), dict(row=-1)):
        assert call(**bad) == FQ_SHAPE, bad
    assert call(d=96) == FQ_DIM and call(page=64) == FQ_BLOCK and call(dtype=2) == FQ_DTYPE
    for name in ("q", "cache", "table", "lens", "out"):
        assert call(**{name: 0}) == FQ_NULL, name
    for bad in (dict(q=72), dict(cache=72), dict(out=72), dict(qs=(1020, 128)), dict(cs=(4096, 252, 128))):
        assert call(**bad) == FQ_ALIGN, bad
    bytes_ = need(2, 8, 2, 128, 16, 4000)
    assert bytes_ > 0 and call(columns=4000) == FQ_WS and call(columns=4000, ws=256, room=bytes_ - 1) == FQ_WS
    assert call(columns=4000, ws=320, room=bytes_) == FQ_ALIGN
    assert need(2, 8, 2, 96, 16, 4000) == 0 and need(0, 8, 2, 128, 16, 4000) == 0
    assert need(1, 8, 2, 128, 16, 4) == 0                                  # a context of one part
    assert need(70000, 8, 8, 64, 32, 1 << 16) > 0                          # more tiles than are counted, fewer with a window


def test_advance_argument_errors(lib):
    f = lib.fq_paged_advance
    f.argtypes = [P, P, I, P, P, P, P, P, L, P, P, I, L, I, I, P]

    def call(lens=64, end=64, num_blocks=9, context=64, start=64, cu=64, positions=64, table=64, stride=4, rows=64, row_lens=64, reqs=2, tokens=3, blocks=4, page=16):
        return f(_p(lens), _p(end), num_blocks, _p(context), _p(start), _p(cu), _p(positions), _p(table), stride, _p(rows), _p(row_lens), reqs, tokens, blocks, page, _p(0))

    for bad in (dict(reqs=-1), dict(reqs=0), dict(tokens=-1), dict(tokens=1 << 31), dict(blocks=0), dict(num_blocks=-1), dict(stride=3),
                dict(blocks=1 << 28, stride=1 << 28), dict(tokens=1 << 30, blocks=1 << 20, stride=1 << 20)):
        assert call(**bad) == FQ_SHAPE, bad
    assert call(page=24) == FQ_BLOCK
    for name in ("lens", "end", "context", "start", "cu", "positions", "table", "rows", "row_lens"):
        assert call(**{name: 0}) == FQ_NULL, name


def test_decode_room_does_not_shrink_with_larger_calls(lib):
    """A workspace for the largest batch and table serves every smaller one, whatever line between the ways to divide lies between."""
    need = lib.fq_paged_kv_decode_workspace_bytes
    need.argtypes, need.restype = [I] * 6, Z
    for hq, hkv, d in ((32, 8, 128), (8, 1, 128), (32, 32, 128), (16, 2, 64), (32, 8, 256), (128, 128, 64)):
        for page in (8, 16, 32):
            columns = [1, 2, 5, 9, 10, 14, 15, 24, 25, 26, 40, 64, 65, 80, 81, 128, 200, 512, 5000, 60000]
            table = [[need(s, hq, hkv, d, page, c) for c in columns] for s in (*range(1, 140), 200, 255, 256, 257, 511, 512, 513, 1000, 2047, 2048, 5000, 70000)]
            for smaller, larger in zip(table, table[1:]):
                assert all(a <= b for a, b in zip(smaller, larger)), (hq, hkv, d, page)
            for row in table:
                assert row == sorted(row), (hq, hkv, d, page)
    must = lib.fq_paged_kv_decode_workspace_needed
    must.argtypes, must.restype = [I] * 7, Z
    for s in (1, 15, 16, 63, 64, 255, 256, 257, 3000, 70000):
        for c in (1, 14, 30, 31, 52, 60, 130, 700, 1 << 16):
            for window in (0, 1, 33, 500, 900, 3000, 1 << 30):
                assert must(s, 32, 8, 128, 16, c, window) in (0, need(s, 32, 8, 128, 16, c))
    assert must(0, 32, 8, 128, 16, 9, 0) == 0 and must(1, 32, 8, 96, 16, 9, 0) == 0 and must(1, 32, 8, 128, 16, 9, -1) == 0
