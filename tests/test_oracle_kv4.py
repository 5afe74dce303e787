"""The 4-bit cache's oracle against counts done by hand, and what the entry points refuse (before anything is launched: no GPU)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from btb_amd import mxfp4, native
from oracle import kv4

P = ctypes.c_void_p(0x1000)  # an address that no refused call follows
OFF = ctypes.c_void_p(0x1004)
FAR = ctypes.c_void_p(0x10000000)  # far from it
F = ctypes.c_float


def test_codes_are_the_nearest_and_ties_are_even():
    a = [0.0, 0.25, 0.2500001, 0.75, 0.7499999, 1.25, 1.75, 2.5, 2.5000001, 3.5, 5.0, 5.0000001, 6.0, 7.0, 1e30]
    assert kv4.codes(a).tolist() == [0, 0, 1, 2, 1, 2, 4, 4, 5, 6, 6, 7, 7, 7, 7]


def test_keys_keep_the_smallest_power_that_holds_seven_of_them():
    k = np.zeros((6, 32))
    k[0, 3], k[1, 3], k[2, 3], k[3, 3], k[4, 3], k[5, 31] = 7.0, 7.03125, -4.0, 2.0**-130, np.inf, np.nan
    v, e = kv4.held_k(k)
    assert e[:, 0].tolist() == [127, 128, 127, 0, 255, 255]
    assert v[0, 3] == 6.0 and v[1, 3] == 8.0 and v[2, 3] == -4.0 and v[3, 3] == 0.0
    assert np.isnan(v[4]).all() and np.isnan(v[5]).all()


def test_values_keep_a_sixth_of_their_largest():
    v = np.zeros((3, 64))
    v[0, 5], v[0, 6], v[1, 0] = 3.0, -0.3, np.nan
    x, s = kv4.held_v(v)
    assert s[0] == 0.5 and x[0, 5] == 3.0 and x[0, 6] == -0.25 and np.isnan(x[1]).all() and s[2] == 0.0 and not x[2].any()


def test_a_key_reads_as_mxfp4_reads_it():
    import torch

    k = np.random.default_rng(0).standard_normal((5, 64)).astype(np.float32)
    v, e = kv4.held_k(k)
    blocks, scales = mxfp4.quantize(torch.from_numpy(v.astype(np.float32)))
    assert np.array_equal(mxfp4.dequantize(blocks, scales).numpy(), v)


def test_tiles_of_bytes():
    raw = np.zeros(4288, np.uint8)
    raw[4096:4096 + 128] = 127
    raw[1024 + 16 * (32 + 7) + 3] = 0x52  # token 7, step 1, half 1, byte 3: dims 64 + 32 + 6 and + 7
    # token 13: half 1, index 5; dim 100 = 64 + 32 + 4: part 1, d 1, c 4, dword 2, nibble 5
    raw[2048 + 1024 + 16 * (32 + 4) + 8 + 2] = 0xF0
    raw[4224:].view(np.uint16)[16 + 5] = 0x4000
    K, V = kv4.tile(raw, 128)
    assert K[7, 102] == 1.0 and K[7, 103] == 3.0 and np.abs(K).sum() == 4.0
    assert V[13, 100] == -12.0 and np.abs(V).sum() == 12.0


def test_pages_that_are_not_there_and_lengths_past_the_table():
    tables = np.array([[0, 9], [3, -1], [-1, -1]], np.int32)
    pool = np.arange(5, dtype=np.int64)[None, :, None].copy()
    out, used = kv4.compact(pool, tables, np.array([900, 3, -4]), 32)
    assert used == 2 and out.tolist() == [[0, -1], [1, -1], [-1, -1]] and pool[0, :, 0].tolist() == [0, 3, 2, 3, 4]
    tables, lens = np.array([[0, 9], [3, -1], [-1, -1]], np.int32), np.array([40, 3, 0], np.int32)
    kv4.fork(pool, tables, lens, [0, 1, 1, 2], [2, 1, 7, 0], [4, 2, 2, 8], 32)
    assert tables.tolist() == [[0, 9], [3, -1], [0, -1]] and lens.tolist() == [40, 3, 40]  # (pages 9 and 8 are none of five)


def test_sizes():
    lib = native.load_library()
    assert [lib.btb_hip_kv4_tile_bytes(d) for d in (64, 128, 256, 0)] == [2176, 4288, 0, 0]
    assert lib.btb_hip_pages_compact_words(0) == 0 and lib.btb_hip_pages_compact_words((1 << 19) + 1) == 0
    assert lib.btb_hip_pages_compact_words(5) == 4 + 5 + 4
    floats = lib.btb_hip_attn_kv4_floats
    assert floats(1, 1, 32, 8, 128, 100) > 0
    for bad in ((0, 1, 32, 8, 128, 100), (1, 0, 32, 8, 128, 100), (1, 1, 33, 8, 128, 100), (1, 1, 32, 0, 128, 100), (1, 1, 0, 8, 128, 100),
                (1, 1, 520, 8, 128, 100), (1, 1, 32, 8, 96, 100), (1, 1, 32, 8, 128, 0), (1, 1, 32, 8, 128, (1 << 30) + 1)):
        assert floats(*bad) == 0, bad


ROWS = dict(k=P, v=FAR, cache=P, tables=P, lens=P, first=None, B=2, W=4, pages=9, page=64, stride=8 * 2 * 4288, T=6, Hk=8, D=128, kr=1024,
            kh=128, vr=1024, vh=128)
# what every operator over such a cache refuses
SEQS = [dict(B=0), dict(B=65537, first=P), dict(W=0), dict(pages=0), dict(page=0), dict(page=48), dict(page=1 << 21, W=1),
        dict(W=1 << 25), dict(stride=8 * 2 * 4288 - 16), dict(stride=8 * 2 * 4288 + 8), dict(T=0), dict(T=7), dict(T=(1 << 24) + 2, first=P),
        dict(Hk=0), dict(Hk=1025), dict(D=96), dict(D=256), dict(cache=OFF)]


def _write(lib, **other):
    a = {**ROWS, **other}
    return lib.btb_hip_kv4_write(a["k"], a["v"], a["cache"], a["tables"], a["lens"], a["first"], a["B"], a["W"], a["pages"], a["page"],
                                 a["stride"], a["T"], a["Hk"], a["D"], a["kr"], a["kh"], a["vr"], a["vh"], None)


def _read(lib, **other):
    a = {**ROWS, **other}
    return lib.btb_hip_kv4_read(a["cache"], a["tables"], a["lens"], a["first"], a["B"], a["W"], a["pages"], a["page"], a["stride"], a["T"],
                                a["Hk"], a["D"], a["k"], a["v"], 1, a["kr"], a["kh"], a["vr"], a["vh"], None)


def _attn(lib, **other):
    a = dict(q=P, cache=P, tables=P, lens=P, first=None, att=FAR, lse=P, B=2, W=4, pages=9, page=64, stride=8 * 2 * 4288, T=6, Hq=32, Hk=8, D=128,
             scale=0.1, keys=200, ws=P)
    a.update(other)
    return lib.btb_hip_attn_kv4(a["q"], a["cache"], a["tables"], a["lens"], a["first"], a["att"], a["lse"], a["B"], a["W"], a["pages"],
                                a["page"], a["stride"], a["T"], a["Hq"], a["Hk"], a["D"], F(a["scale"]), a["keys"], a["ws"], None)


@pytest.mark.parametrize("other", SEQS + [dict(k=OFF), dict(v=OFF), dict(kr=1023), dict(kh=4), dict(vr=-8), dict(vh=12)])
def test_rows_refused(other):
    lib = native.load_library()
    assert _write(lib, **other) == native.ERR_DOMAIN and b"kv4_write" in lib.btb_hip_last_error()
    assert _read(lib, **other) == native.ERR_DOMAIN and b"kv4_read" in lib.btb_hip_last_error()


@pytest.mark.parametrize("other", [dict(kr=0), dict(kh=0), dict(vr=120), dict(vh=64), dict(kr=512), dict(vr=128, vh=512)])
def test_read_refuses_outputs_that_share_memory(other):
    assert _read(native.load_library(), **other) == native.ERR_DOMAIN


@pytest.mark.parametrize("other", SEQS + [dict(q=OFF), dict(att=OFF), dict(ws=OFF), dict(Hq=33), dict(Hq=0), dict(Hq=520), dict(scale=0.0),
                                          dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(keys=0),
                                          dict(T=1 << 20, Hq=32)])
def test_attention_refused(other):
    lib = native.load_library()
    assert _attn(lib, **other) == native.ERR_DOMAIN and b"attn_kv4" in lib.btb_hip_last_error()


def _fork(lib, **other):
    a = dict(pool=P, L=3, pages=9, bytes=4096, layer=9 * 4096, stride=4096, tables=P, lens=P, B=4, W=5, page=64, src=P, dst=P, fresh=P, F=2)
    a.update(other)
    return lib.btb_hip_pages_fork(a["pool"], a["L"], a["pages"], a["bytes"], a["layer"], a["stride"], a["tables"], a["lens"], a["B"], a["W"],
                                  a["page"], a["src"], a["dst"], a["fresh"], a["F"], None)


def _compact(lib, **other):
    a = dict(pool=P, L=3, pages=9, bytes=4096, layer=9 * 4096, stride=4096, tables=P, lens=P, B=4, W=5, page=64, out=P, used=P, ws=P)
    a.update(other)
    return lib.btb_hip_pages_compact(a["pool"], a["L"], a["pages"], a["bytes"], a["layer"], a["stride"], a["tables"], a["lens"], a["B"],
                                     a["W"], a["page"], a["out"], a["used"], a["ws"], None)


@pytest.mark.parametrize("other", [dict(L=0), dict(pages=0), dict(bytes=0), dict(bytes=24), dict(stride=4080), dict(stride=4104), dict(layer=4088),
                                   dict(layer=8 * 4096), dict(layer=0), dict(layer=-4096), dict(stride=2 * 4096, layer=4096), dict(B=0), dict(B=65537),
                                   dict(W=0), dict(page=0), dict(page=1 << 28, W=8), dict(pool=OFF)])
def test_pages_refused(other):
    lib = native.load_library()
    assert _fork(lib, **other) == native.ERR_DOMAIN and b"pages_fork" in lib.btb_hip_last_error()
    assert _compact(lib, **other) == native.ERR_DOMAIN and b"pages_compact" in lib.btb_hip_last_error()


def test_more_refusals():
    lib = native.load_library()
    assert _fork(lib, F=0) == native.ERR_DOMAIN and _fork(lib, F=65537) == native.ERR_DOMAIN
    assert _compact(lib, tables=ctypes.c_void_p(0x1000), out=ctypes.c_void_p(0x1010)) == native.ERR_DOMAIN  # four entries on
    assert _compact(lib, pages=(1 << 19) + 1, layer=((1 << 19) + 1) * 4096) == native.ERR_DOMAIN
    for name in ("k", "v", "cache", "tables", "lens"):
        assert _write(lib, **{name: None}) == native.ERR_NULL and _read(lib, **{name: None}) == native.ERR_NULL
    for name in ("q", "cache", "tables", "lens", "att", "ws"):
        assert _attn(lib, **{name: None, "D": 96}) == native.ERR_NULL  # (before the sizes)
    for name in ("pool", "tables", "lens", "src", "dst", "fresh"):
        assert _fork(lib, **{name: None}) == native.ERR_NULL
    for name in ("pool", "tables", "lens", "out", "used", "ws"):
        assert _compact(lib, **{name: None}) == native.ERR_NULL


@pytest.mark.parametrize("first", [None, P])
def test_more_workgroups_than_a_launch_has(first):
    """a launch's threads are counted in 32 bits: 2^24 workgroups of 256 are one too many"""
    lib = native.load_library()
    heads = dict(Hk=1024, stride=1024 * 2 * 4288)
    for T in (1 << 24, 1 << 20):  # 2^19 and 2^15 tiles, 1024 heads
        assert _write(lib, T=T, first=first, **heads) == native.ERR_DOMAIN
        assert _read(lib, T=T, first=first, kr=1 << 17, vr=1 << 17, **heads) == native.ERR_DOMAIN
    assert _attn(lib, B=1 << 16, T=1 << 14, first=P, Hq=1024, **heads) == native.ERR_DOMAIN
    assert _attn(lib, B=1 << 14, T=1 << 14, Hq=1024, **heads) == native.ERR_DOMAIN
    assert _fork(lib, F=65536, L=64, bytes=1 << 16, stride=1 << 16, layer=9 << 16) == native.ERR_DOMAIN


def test_outputs_over_each_other_or_the_input():
    lib = native.load_library()
    assert _read(lib, v=P) == native.ERR_DOMAIN and b"share memory" in lib.btb_hip_last_error()
    for at in (0x1010, 0x1000 + 6 * 32 * 128 * 2 - 16, 0x1000 - 16):  # all but the first 16 bytes, the last, all but the last
        assert _attn(lib, q=P, att=ctypes.c_void_p(at)) == native.ERR_DOMAIN and b"across q" in lib.btb_hip_last_error()


@pytest.mark.parametrize("other", [dict(Hk=1025, Hq=1025), dict(Hq=1 << 62, Hk=1 << 62), dict(B=2, Hq=1 << 63, Hk=1 << 63), dict(T=1 << 20, Hq=32),
                                   dict(B=8, Hq=1 << 63, Hk=1 << 61), dict(T=(1 << 24) + 1), dict(B=65537), dict(keys=1 << 63)])
def test_a_workspace_is_refused_where_the_call_is(other):
    """sizes whose product wraps to zero would end the process in a division by it"""
    a = dict(T=1, B=1, Hq=32, Hk=8, D=128, keys=100)
    a.update(other)
    lib = native.load_library()
    assert lib.btb_hip_attn_kv4_floats(*a.values()) == 0
    assert lib.btb_hip_attn_kv4_floats(1, 1, 1024, 1024, 128, 100) > 0 and lib.btb_hip_attn_kv4_floats(1 << 18, 1, 64, 1, 64, 1 << 30) > 0


@pytest.mark.parametrize("f32", [0, 1])
def test_read_refuses_outputs_that_lie_across_each_other(f32):
    lib, size, at = native.load_library(), 4 if f32 else 2, 0x10000000

    def read(apart, **other):
        """the second output so many values behind the first; strides as given, for both"""
        a = {**ROWS, **other}
        return lib.btb_hip_kv4_read(a["cache"], a["tables"], a["lens"], a["first"], a["B"], a["W"], a["pages"], a["page"], a["stride"], a["T"],
                                    a["Hk"], a["D"], ctypes.c_void_p(at), ctypes.c_void_p(at + apart * size), f32, a["kr"], a["kh"], a["vr"],
                                    a["vh"], None)

    whole = 6 * 1024  # rows one after another: any place inside the other's
    for apart in (8, 128, 1024, 1024 + 8, whole - 8, -8, -128, -1024, 8 - whole):
        assert read(apart) == native.ERR_DOMAIN and b"share memory" in lib.btb_hip_last_error(), apart
    fused = dict(kr=2048, vr=2048)  # room for the other between the rows: 1024 values in, and only there
    for apart in (1024 - 8, 1024 + 8, 2048, 4096 - 8, -8, 8 - 1024, 2048 * 5 + 8):
        assert read(apart, **fused) == native.ERR_DOMAIN, apart
    heads = dict(kr=128, vr=128, kh=6 * 256, vh=6 * 256)  # head after head, with room between them
    for apart in (6 * 128 - 8, 8, -8, 6 * 256, 7 * 6 * 256 + 8):
        assert read(apart, **heads) == native.ERR_DOMAIN, apart
    one = dict(B=1, T=1, kr=0, vr=0, kh=256, vh=256)  # a row alone, and a head alone
    for apart in (8, -8, 120, 256, 256 * 7 + 120):
        assert read(apart, **one) == native.ERR_DOMAIN, apart
    alone = dict(Hk=1, kr=256, vr=256, kh=0, vh=0, stride=2 * 4288)
    for apart in (8, -8, 120, 256, 256 * 5 + 120):
        assert read(apart, **alone) == native.ERR_DOMAIN, apart
    for other in (dict(kr=2048, vr=1024), dict(vr=2048), dict(kr=128, kh=1024)):  # unlike strides, inside each other's range
        assert read(1024, **other) == native.ERR_DOMAIN, other


@pytest.mark.parametrize("other", [dict(kr=1 << 60), dict(kh=1 << 60), dict(vr=(1 << 63) - 8), dict(vh=1 << 44)])
def test_strides_past_any_memory(other):
    lib = native.load_library()
    assert _write(lib, **other) == native.ERR_DOMAIN and _read(lib, **other) == native.ERR_DOMAIN


@pytest.mark.parametrize("T,B,Hq,D,keys", [(1, 1, 3, 128, 9000), (1, 1, 1, 64, 1400), (7, 7, 5, 128, 3001), (3, 3, 3, 64, 2500)])
def test_spans_outputs_lie_in_whole_pieces(T, B, Hq, D, keys):
    """an odd number of maxima and sums is filled up to 16 bytes: the outputs behind them are written 16 bytes at a time"""
    n = native.load_library().btb_hip_attn_kv4_floats(T, B, Hq, 1, D, keys)
    assert n > 4 and n % 4 == 0  # (outputs are a multiple of four floats themselves)


@pytest.mark.parametrize("scale", [2.359e38, 2.4e38, 3.4e38])
def test_a_scale_whose_exponent_overflows(scale):
    """scores go through exp2: scale log2(e) is an f32 number too"""
    lib = native.load_library()
    assert _attn(lib, scale=scale) == native.ERR_DOMAIN and b"scale" in lib.btb_hip_last_error()
