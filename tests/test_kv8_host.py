"""CPU-only checks of the 8-bit paged cache and of shared prefixes: refusals of the Python layer, page accounting of prefixes, status
codes of the C ABI before anything touches the GPU."""
from __future__ import annotations

import ctypes
import os

import pytest
import torch

from flashquant_amd import kernels as K
from flashquant_amd.cache import PageTable

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashquant_amd", "libfq_hip.so")
FQ_OK, FQ_NULL, FQ_DIM, FQ_BLOCK, FQ_DTYPE, FQ_SHAPE, FQ_ALIGN, FQ_WS, FQ_LAUNCH = range(9)


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(LIB)


def test_no_cpu_fallback():
    q, p, f = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.long), K.rotary_frequencies(64)[0]
    c, s = torch.zeros(1, 16, 2, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(1, 2, 16, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    ints = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: K.rotary_paged_store8(q, q, q, p, p, f, c, c, s, s), lambda: K.paged_kv8_read(c, c, s, s, ints[None], ints, 1),
                 lambda: K.paged_kv8_decode(q, c, c, s, s, ints[None], ints), lambda: K.paged_prefix_decode(q, c, c, ints[None], ints, ints, ints)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


# ---- prefixes of a table of pages -------------------------------------------------------------------------------------------------

def taken(table, seq, tokens):
    """What a schedule leaves: ``tokens`` of sequence ``seq`` on free pages."""
    n = -(-tokens // table.block_size)
    start = int(table.free_start)
    table.block_table[seq, :n] = table.free_blocks[start:start + n]
    table.free_start += n
    table.context_lens[seq] = tokens


def test_prefixes_own_their_pages():
    table = PageTable(20, 8, 4, 10, torch.device("cpu"), max_prefixes=2)
    taken(table, 1, 29)
    pages = table.block_table[1, :4].tolist()
    table.make_prefix(1, 0)
    assert table.prefix_lens.tolist() == [24, 0] and table.prefix_ids.tolist() == [-1, 0, -1, -1]
    table.join_prefix(3, 0)
    assert table.block_table[3].tolist() == pages[:3] + [-1] * 7 and int(table.context_lens[3]) == 24 and int(table.free_start) == 4
    table.release(1)                                                     # its own page is the next to be taken
    assert int(table.free_start) == 3 and int(table._pages[3]) == pages[3] and table.prefix_ids.tolist() == [-1, -1, -1, 0]
    with pytest.raises(ValueError, match="still shares"):
        table.drop_prefix(0)
    table.release(3)
    assert int(table.free_start) == 3
    table.drop_prefix(0)
    assert int(table.free_start) == 0 and sorted(table._pages[:20].tolist()) == list(range(20)) and table.prefix_lens.tolist() == [0, 0]
    taken(table, 0, 5)                                                   # fewer tokens than a page: nothing is shared
    table.make_prefix(0, 1)
    table.join_prefix(2, 1)
    assert table.prefix_lens.tolist() == [0, 0] and int(table.context_lens[2]) == 0
    table.release(0)
    table.release(2)
    table.drop_prefix(1)
    assert int(table.free_start) == 0


def test_refusals_of_prefixes():
    table = PageTable(20, 8, 3, 10, torch.device("cpu"), max_prefixes=2)
    taken(table, 0, 16)
    for call in (lambda: table.join_prefix(1, 0), lambda: table.drop_prefix(0), lambda: table.make_prefix(0, 2), lambda: table.make_prefix(3, 0), lambda: table.make_prefix(-1, 0),
                 lambda: PageTable(20, 8, 3, 10, torch.device("cpu"), max_prefixes=1025), lambda: PageTable(20, 8, 3, 10, torch.device("cpu"), max_prefixes=-1)):
        with pytest.raises(ValueError):
            call()
    table.make_prefix(0, 0)
    for call in (lambda: table.make_prefix(0, 1), lambda: table.join_prefix(0, 0), lambda: table.make_prefix(1, 0), lambda: table.drop_prefix(1)):
        with pytest.raises(ValueError):
            call()
    plain = PageTable(20, 8, 3, 10, torch.device("cpu"))
    with pytest.raises(ValueError):
        plain.make_prefix(0, 0)


def test_a_prefix_that_does_not_exist_is_not_dropped():
    """-1 is no prefix, whatever a list makes of it, and the last one keeps its pages."""
    table = PageTable(20, 8, 1, 10, torch.device("cpu"), max_prefixes=2)
    taken(table, 0, 16)
    table.make_prefix(0, 1)
    for prefix in (-1, -2, 2):
        with pytest.raises(ValueError):
            table.drop_prefix(prefix)
    assert table.prefix_lens.tolist() == [0, 16] and int(table.free_start) == 2


# ---- the C ABI ------------------------------------------------------------------------------------------------------------------

def _p(v):
    return ctypes.c_void_p(v)


def _strides(*v):
    return (ctypes.c_int64 * len(v))(*v)


C, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
ROWS, CODES, SCALES = _strides(1024, 128, 0), _strides(4096, 256, 128), _strides(32, 16)


def test_store8_status_codes(lib):
    f = lib.fq_rotary_paged_store8
    f.argtypes = [C, C, C, C, I, C, C, C, C, I, C, I, C, I, I, F, C, L, C, C, C, C, C, C, C, C, I, L, L, I, I, C]
    good = dict(q=_p(4096), qs=ROWS, qo=_p(8192), qos=ROWS, HQ=8, k=_p(4096), ks=ROWS, v=_p(4096), vs=ROWS, HKV=2, pos=_p(4096), pb=8, freq=_p(4096), half=64, inter=0, scale=1.0,
                slots=_p(4096), mapped=3, kc=_p(4096), kcs=CODES, vc=_p(4096), vcs=CODES, ksc=_p(4096), kscs=SCALES, vsc=_p(4096), vscs=SCALES, bs=16, nb=10, tokens=3, D=128, dt=1, st=_p(0))

    def status(**bad):
        return f(*(good | bad).values())

    assert status(tokens=0, mapped=0) == FQ_OK
    assert status(D=96, half=48) == FQ_DIM
    assert status(bs=12) == FQ_BLOCK
    assert status(dt=2) == FQ_DTYPE and status(pb=3) == FQ_DTYPE
    for bad in (dict(tokens=-1), dict(mapped=4), dict(mapped=-1), dict(HKV=0), dict(HQ=-1), dict(HQ=5000), dict(half=0), dict(half=65), dict(nb=-1), dict(nb=1 << 31),
                dict(ks=_strides(8, 1 << 31)), dict(kcs=_strides(4096, 1 << 31, 128)), dict(kscs=_strides(32, 1 << 31))):
        assert status(**bad) == FQ_SHAPE, bad
    for name in ("q", "qs", "qo", "k", "v", "pos", "freq", "slots", "kc", "kcs", "vc", "ksc", "kscs", "vsc", "vscs"):
        assert status(**{name: _p(0)}) == FQ_NULL, name


def test_read8_status_codes(lib):
    f = lib.fq_paged_kv8_read
    f.argtypes = [C] * 8 + [C, L, C, C, C, C, I, I, L, I, I, I, I, L, I, C]
    good = dict(kc=_p(4096), kcs=CODES, vc=_p(4096), vcs=CODES, ksc=_p(4096), kscs=SCALES, vsc=_p(4096), vscs=SCALES, table=_p(4096), row=4, cu=_p(4096), starts=_p(0), keys=_p(4096),
                values=_p(8192), fill=1, S=2, tokens=9, H=2, D=128, bs=16, mb=4, nb=10, dt=1, st=_p(0))

    def status(**bad):
        return f(*(good | bad).values())

    assert status(tokens=0) == FQ_OK
    assert status(D=96) == FQ_DIM and status(bs=12) == FQ_BLOCK and status(dt=2) == FQ_DTYPE
    for bad in (dict(S=-1), dict(tokens=-1), dict(H=0), dict(H=5000), dict(mb=0), dict(nb=-1), dict(row=-1)):
        assert status(**bad) == FQ_SHAPE, bad
    for name in ("kc", "kcs", "vsc", "vscs", "table", "cu", "keys", "values"):
        assert status(**{name: _p(0)}) == FQ_NULL, name
    for bad in (dict(kc=_p(4104)), dict(vcs=_strides(4096, 264, 128)), dict(keys=_p(4100))):
        assert status(**bad) == FQ_ALIGN, bad


def test_decode8_status_codes(lib):
    f = lib.fq_paged_kv8_decode
    f.argtypes = [C] * 10 + [C, L, C, C, C] + [I] * 6 + [L, F, I, I, C, ctypes.c_size_t, C]
    good = dict(q=_p(4096), qs=_strides(1024, 128), kc=_p(4096), kcs=CODES, vc=_p(4096), vcs=CODES, ksc=_p(4096), kscs=SCALES, vsc=_p(4096), vscs=SCALES, table=_p(4096), row=400, lens=_p(4096),
                out=_p(4096), lse=_p(0), S=2, HQ=8, HKV=2, D=128, bs=16, mb=400, nb=10, sm=0.1, window=0, dt=1, ws=_p(0), wb=0, st=_p(0))

    def status(**bad):
        return f(*(good | bad).values())

    assert status(S=0) == FQ_OK
    assert status(D=96) == FQ_DIM and status(bs=12) == FQ_BLOCK and status(dt=2) == FQ_DTYPE
    for bad in (dict(S=-1), dict(HQ=7), dict(HQ=34), dict(mb=0), dict(nb=0), dict(window=-1), dict(row=-1)):
        assert status(**bad) == FQ_SHAPE, bad
    for name in ("q", "qs", "kc", "kcs", "vc", "vcs", "ksc", "kscs", "vsc", "vscs", "table", "lens", "out"):
        assert status(**{name: _p(0)}) == FQ_NULL, name
    for bad in (dict(q=_p(4104)), dict(kc=_p(4104)), dict(kcs=_strides(4096, 264, 128)), dict(ksc=_p(4097)), dict(kscs=_strides(36, 16)), dict(out=_p(4104)), dict(qs=_strides(1020, 128))):
        assert status(**bad) == FQ_ALIGN, bad
    assert status() == FQ_WS


def test_prefix_status_codes(lib):
    f = lib.fq_paged_prefix_decode
    f.argtypes = [C] * 10 + [C, L, C, C, C, I, C, C] + [I] * 6 + [L, F, I, C, ctypes.c_size_t, C]
    room = lib.fq_paged_prefix_decode_workspace_bytes
    room.restype = ctypes.c_size_t
    good = dict(q=_p(4096), qs=_strides(1024, 128), kc=_p(4096), kcs=CODES, vc=_p(4096), vcs=CODES, ksc=_p(0), kscs=None, vsc=_p(0), vscs=None, table=_p(4096), row=400, lens=_p(4096),
                ids=_p(4096), plens=_p(4096), P=3, out=_p(4096), lse=_p(0), S=2, HQ=8, HKV=2, D=128, bs=16, mb=400, nb=10, sm=0.1, dt=1, ws=_p(4096), wb=0, st=_p(0))

    def status(**bad):
        return f(*(good | bad).values())

    eight = dict(ksc=_p(4096), kscs=SCALES, vsc=_p(4096), vscs=SCALES)
    assert status(S=0) == FQ_OK
    assert status(D=96) == FQ_DIM and status(bs=12) == FQ_BLOCK and status(dt=2) == FQ_DTYPE
    for bad in (dict(S=-1), dict(HQ=7), dict(HQ=34), dict(mb=0), dict(nb=0), dict(P=-1), dict(P=1025), dict(row=-1)):
        assert status(**bad) == FQ_SHAPE, bad
    # more units of work than are counted
    assert status(S=1 << 20, mb=(1 << 27) - 4, P=1000, wb=1 << 62) == FQ_SHAPE
    # tiles are asked for ahead, and their tokens are counted in 32 bits
    assert status(S=1, mb=(1 << 27) - 4096, P=1, wb=0) == FQ_WS and status(S=1, mb=(1 << 27) - 4095, P=1, wb=0) == FQ_SHAPE
    for name in ("q", "qs", "kc", "kcs", "vc", "vcs", "table", "lens", "ids", "plens", "out", "ws"):
        assert status(**{name: _p(0)}) == FQ_NULL, name
    for name in eight:
        assert status(**(eight | {name: _p(0)})) == FQ_NULL, name
    for bad in (dict(q=_p(4104)), dict(kc=_p(4104)), dict(kcs=_strides(4096, 260, 128)), eight | dict(ksc=_p(4097)), eight | dict(kcs=_strides(4096, 264, 128)), dict(out=_p(4104)),
                dict(ws=_p(4097), wb=1 << 40)):
        assert status(**bad) == FQ_ALIGN, bad
    assert status() == FQ_WS and status(**eight) == FQ_WS
    assert room(2, 7, 2, 128, 1) == 0 and room(2, 8, 2, 96, 1) == 0 and room(2, 8, 2, 128, 1025) == 0 and room(2, 8, 2, 128, 0) > 0


def test_advance_prefix_status_codes(lib):
    f = lib.fq_paged_advance_prefix
    f.argtypes = [C, C, I, C, C, C, C, C, L, C, C, C, C, I, L, I, I, C]
    p = _p(4096)
    assert f(p, p, 10, p, p, p, p, p, 4, None, p, p, p, 2, 3, 4, 16, None) == FQ_NULL       # a prefix for every token, and none for the sequences
    assert f(p, p, 10, p, p, p, p, p, 4, p, p, p, p, 2, 3, 4, 12, None) == FQ_BLOCK
    assert f(p, p, 10, p, p, p, p, p, 3, p, p, p, p, 2, 3, 4, 16, None) == FQ_SHAPE
