"""A paged cache held in 4 bits, on the GPU against oracle/kv4.py in 64 bits.

Bars, from the arithmetic; u = 2^-24 is half an f32 step, h = 2^-11 half an f16 step and w = 2^-8 half a bf16 step, each relative.
  write, read, fork, compact   equal (a quotient of two bf16 numbers, or a tie of one, is told apart by f32; K's and V's values are exact
          in f32: a code's two bits times eight; read as bf16 they are rounded once)
  scores  D products, exact, added in f32: e = D u scale sum |q_i k_i| at worst, the same relative error in exp(s); exp2's argument
          in f32 adds u log2(e) |s| and the exponential 2 u
  att     a weight times its scale rounded to f16: h times the weighted mean of |v|, and 2^-36 of the largest |v| where a product is
          below f16's normal numbers; sums, spans and scales: (e + 64 u) of the mean; the output's rounding: w |att|
  lse     e and 8 u (1 + |lse|)
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from btb_amd.decode import recording
from btb_amd.native import HipError
from oracle import kv4

from .helpers import gen

pytestmark = pytest.mark.gpu

U, H, W = 2.0**-24, 2.0**-11, 2.0**-8
NAN, INF = float("nan"), float("inf")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _first(rows):
    return _i32(np.concatenate([[0], np.cumsum(rows)]).tolist())


def _tables(g, lens, page, spare=2, width=0):
    """pages in any order: (int32 [B, W] on the GPU, the pool's pages)"""
    counts = [-(-n // page) for n in lens]
    W_, total = max(1, width, *counts), sum(counts)
    order = torch.randperm(total + spare, generator=g)[:total].tolist()
    out = torch.full((len(lens), W_), -1, dtype=torch.int32)
    for b, c in enumerate(counts):
        out[b, :c] = torch.tensor(order[:c], dtype=torch.int32)
        order = order[c:]
    return out.cuda(), total + spare


def _rows(g, *shape, wide=False):
    x = torch.randn(*shape, generator=g)
    if wide:
        x = x * torch.exp2(torch.randint(-20, 20, shape[:-1] + (1,), generator=g).float())
    return x.to(torch.bfloat16).cuda()


def _filled(card, pages, Hk, D, page, byte=0xFF):
    pool = card.kv4_pool(pages, Hk, D, page)
    pool.fill_(byte)
    return pool


def _put(card, g, lens, Hk, D, page, wide=False, byte=0xFF):
    """sequences of these lengths written at once: (pool, tables, k, v)"""
    tables, pages = _tables(g, lens, page)
    pool = _filled(card, pages, Hk, D, page, byte)
    k, v = _rows(g, sum(lens), Hk, D, wide=wide), _rows(g, sum(lens), Hk, D, wide=wide)
    if sum(lens):
        card.kv4_write(k, v, pool, tables, _i32(lens), first=_first(lens))
    return pool, tables, k, v


def _same(got, want):
    got = got.double().cpu().numpy() if isinstance(got, torch.Tensor) else got
    return np.array_equal(got, want, equal_nan=True)


# ---- rows in and back ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("lens,rows,Hk,D,page", [
    ([1], [1], 1, 64, 32),
    ([33, 64, 7], [33, 64, 7], 2, 128, 64),
    ([100, 31, 32, 65], [1, 1, 1, 1], 8, 128, 32),
    ([500, 0, 97, 3], [77, 0, 96, 3], 3, 64, 96),
    ([1025, 256], [1000, 2], 2, 128, 256),
    ([40] * 70, [2] * 70, 1, 128, 64),
])
def test_write_and_read(card, lens, rows, Hk, D, page):
    g = gen(9000 + sum(lens) + D)
    T = sum(rows)
    tables, pages = _tables(g, lens, page, width=3)
    pool = _filled(card, pages, Hk, D, page, 0x5A)
    before = pool.cpu().numpy().copy()
    k, v = _rows(g, T, Hk, D, wide=True), _rows(g, T, Hk, D, wide=True)
    first = _first(rows) if len(set(rows)) > 1 else None
    card.kv4_write(k, v, pool, tables, _i32(lens), first=first)
    out = [torch.full((T, Hk, D), 7.0, dtype=t, device="cuda") for t in (torch.float32, torch.float32, torch.bfloat16, torch.bfloat16)]
    card.kv4_read(pool, tables, _i32(lens), out[0], out[1], first=first)
    card.kv4_read(pool, tables, _i32(lens), out[2], out[3], first=first)
    torch.cuda.synchronize()
    wk, wv = kv4.held_k(k.double().cpu().numpy())[0], kv4.held_v(v.double().cpu().numpy())[0]
    assert _same(out[0], wk) and _same(out[1], wv)
    assert torch.equal(out[2], out[0].to(torch.bfloat16)) and torch.equal(out[3], out[1].to(torch.bfloat16))
    # where the tiles keep them, and everything else as it was
    after, tab, row = pool.cpu().numpy(), tables.cpu().numpy(), 0
    seen = np.zeros(after.shape[0] * page, bool).reshape(after.shape[0], page)
    for b, (n, r) in enumerate(zip(lens, rows)):
        for i in range(n - r, n):
            seen[tab[b, i // page], i % page] = True
        for hk in range(Hk):
            K, V, there = kv4.tokens(after, tab[b], n, page, hk, D)
            assert there.all() and _same(K[n - r:], wk[row:row + r, hk]) and _same(V[n - r:], wv[row:row + r, hk])
        row += r
    for p in range(after.shape[0]):
        for j in range(page // 32):
            untouched = ~seen[p, 32 * j:32 * j + 32]
            if untouched.all():
                assert np.array_equal(after[p, :, j], before[p, :, j])
            elif untouched.any():
                for hk in range(Hk):
                    old, new = kv4.tile(before[p, hk, j], D), kv4.tile(after[p, hk, j], D)
                    assert _same(new[0][untouched], old[0][untouched]) and _same(new[1][untouched], old[1][untouched])


@pytest.mark.parametrize("D", [64, 128])
def test_numbers_at_borders(card, D):
    """ties, powers, the largest and smallest numbers, zeros, infinities and NaN"""
    g = gen(9100 + D)
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 6.96875, 7.03125]
    T = 64
    k, v = torch.randn(T, 1, D, generator=g) * 0.3, torch.randn(T, 1, D, generator=g) * 0.3
    for t in range(16):  # scales of 2^e exactly: every tie of the grid, both signs
        for x in (k, v):
            x[t, 0, :11] = torch.tensor(mids) * 2.0 ** (t - 8)
            x[t, 0, 11:22] = -torch.tensor(mids) * 2.0 ** (t - 8)
        v[t, 0, :22] = v[t, 0, :22].clamp(-6.0 * 2.0 ** (t - 8), 6.0 * 2.0 ** (t - 8))
    for t in range(16, 32):  # a scale of eight bits, and its ties
        s = torch.tensor(1.0 + t / 128.0).to(torch.bfloat16).float()
        v[t, 0] = torch.tensor(([6.0] + mids[:7] * 40)[:D]) * s
    k[32], v[32] = 0.0, 0.0
    k[33], v[33] = -0.0, -0.0
    big = float(torch.finfo(torch.bfloat16).max)
    k[34], v[34] = big, -big
    k[35, 0, 1], v[35, 0, 1] = big, big
    tiny = 2.0**-133  # bf16's smallest
    k[36], v[36] = tiny, -tiny
    k[37], v[37] = tiny * 5, tiny * 97
    k[38, 0, 7], v[38, 0, 9] = INF, -INF
    k[39, 0, 40], v[39, 0, 63] = NAN, NAN
    k[40], v[40] = 2.0**-120, 2.0**-120
    k, v = k.to(torch.bfloat16).cuda(), v.to(torch.bfloat16).cuda()
    tables, pages = _tables(g, [T], 64)
    pool = _filled(card, pages, 1, D, 64)
    card.kv4_write(k, v, pool, tables, _i32([T]))
    a, b = torch.zeros(T, 1, D, device="cuda"), torch.zeros(T, 1, D, device="cuda")
    card.kv4_read(pool, tables, _i32([T]), a, b)
    assert _same(a, kv4.held_k(k.double().cpu().numpy())[0])
    assert _same(b, kv4.held_v(v.double().cpu().numpy())[0])


def test_one_by_one_is_all_at_once(card):
    g = gen(9200)
    Hk, D, page, n = 2, 128, 64, 150
    tables, pages = _tables(g, [n, n], page)
    k, v = _rows(g, 2 * n, Hk, D), _rows(g, 2 * n, Hk, D)
    one, all_ = _filled(card, pages, Hk, D, page), _filled(card, pages, Hk, D, page)
    card.kv4_write(k, v, all_, tables, _i32([n, n]))
    for i in range(n):
        rows = torch.stack([k[i], k[n + i]]), torch.stack([v[i], v[n + i]])
        card.kv4_write(*rows, one, tables, _i32([i + 1, i + 1]))
    assert torch.equal(one, all_)


def test_strides(card):
    """rows out of a fused row of qkv and out of a cache's layout, back into both; a layer of a pool, pages apart"""
    g = gen(9300)
    T, Hq, Hk, D, page, L = 45, 4, 2, 64, 32, 3
    qkv = _rows(g, T, (Hq + 2 * Hk) * D)
    k, v = (qkv.view(T, Hq + 2 * Hk, D)[:, Hq + i * Hk:Hq + (i + 1) * Hk] for i in range(2))
    tables, pages = _tables(g, [T], page)
    pools = card.kv4_pool(pages, Hk, D, page, layers=L).transpose(0, 1).contiguous().transpose(0, 1)  # a page's layers together
    assert not pools[1].is_contiguous()
    card.kv4_write(k, v, pools[1], tables, _i32([T]))
    want = kv4.held_k(k.double().cpu().numpy())[0], kv4.held_v(v.double().cpu().numpy())[0]
    a, b = (torch.zeros(Hk, T + 3, D, device="cuda").transpose(0, 1)[:T] for _ in range(2))
    card.kv4_read(pools[1], tables, _i32([T]), a, b)
    assert _same(a, want[0]) and _same(b, want[1])
    assert not pools[0].any() and not pools[2].any()
    card.kv4_write(k.transpose(0, 1).contiguous().transpose(0, 1), v, pools[2], tables, _i32([T]))
    assert torch.equal(pools[1], pools[2])


def test_one_row_or_head_of_any_stride(card):
    """the stride from the only row, or head, to a next one that is not there"""
    g = gen(9350)
    D, page = 64, 32
    for T, Hk in ((1, 2), (2, 1), (1, 1)):
        pool, tables = card.kv4_pool(1, Hk, D, page), _i32([[0]])
        k, v = (_rows(g, T, Hk, D) for _ in range(2))
        strides = 3 if T == 1 else Hk * D, 5 if Hk == 1 else D, 1
        card.kv4_write(k.as_strided(k.shape, strides), v.as_strided(v.shape, strides), pool, tables, _i32([T]))
        a, b = torch.zeros_like(k), torch.zeros_like(v)
        card.kv4_read(pool, tables, _i32([T]), a.as_strided(a.shape, strides), b.as_strided(b.shape, strides))
        assert _same(a, kv4.held_k(k.double().cpu().numpy())[0])
        want = kv4.held_v(v.double().cpu().numpy())[0]
        assert _same(b, torch.from_numpy(want).bfloat16().double().numpy())


@pytest.mark.parametrize("T,Hk", [(45, 2), (1, 3), (7, 1), (1, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_read_into_one_fused_tensor(card, T, Hk, dtype):
    """outputs between each other's rows and heads: a row's keys before its values, a head's, a sequence's, a layer's"""
    g = gen(9370 + T)
    D, page = 64, 32
    tables, pages = _tables(g, [T], page)
    pool, k, v = _filled(card, pages, Hk, D, page), _rows(g, T, Hk, D), _rows(g, T, Hk, D)
    card.kv4_write(k, v, pool, tables, _i32([T]))
    want = [torch.from_numpy(x).to(dtype) for x in (kv4.held_k(k.double().cpu().numpy())[0], kv4.held_v(v.double().cpu().numpy())[0])]
    for shape, split in (((T, 2 * Hk, D), lambda t: (t[:, :Hk], t[:, Hk:])), ((T, Hk, 2, D), lambda t: (t[:, :, 0], t[:, :, 1])),
                         ((2, T, Hk, D), lambda t: (t[0], t[1])), ((Hk, 2, T, D), lambda t: (t[:, 0].transpose(0, 1), t[:, 1].transpose(0, 1))),
                         ((Hk, T, 2, D), lambda t: (t[:, :, 1].transpose(0, 1), t[:, :, 0].transpose(0, 1))),
                         ((2, Hk, T + 1, D), lambda t: (t[1, :, 1:].transpose(0, 1), t[0, :, :T].transpose(0, 1)))):
        t = torch.full(shape, 9.0, dtype=dtype, device="cuda")
        a, b = split(t)
        card.kv4_read(pool, tables, _i32([T]), a, b)
        assert torch.equal(a.cpu(), want[0]) and torch.equal(b.cpu(), want[1]), shape


def test_rows_that_are_nobodys_and_pages_that_are_not_there(card):
    g = gen(9400)
    Hk, D, page, T = 1, 64, 32, 40
    k, v = _rows(g, T, Hk, D), _rows(g, T, Hk, D)
    # 5 rows of a sequence of 3 (two stand below 0), one of length 0, one whose second page is none, rows behind the last
    lens, rows = [3, 0, 50, -7], [5, 2, 20, 1]
    tables = _i32([[0, 1], [2, 3], [4, 99], [5, 6]])
    pool = _filled(card, 8, Hk, D, page, 0)
    card.kv4_write(k, v, pool, tables, _i32(lens), first=_first(rows))
    a, b = (torch.full((T, Hk, D), 9.0, device="cuda") for _ in range(2))
    card.kv4_read(pool, tables, _i32(lens), a, b, first=_first(rows))
    wk, wv = kv4.held_k(k.double().cpu().numpy())[0], kv4.held_v(v.double().cpu().numpy())[0]
    a, b = a.cpu().double().numpy(), b.cpu().double().numpy()
    for x, want in ((a, wk), (b, wv)):
        assert (x[:2] == 9.0).all() and _same(x[2:5], want[2:5]) and (x[5:7] == 9.0).all()  # below 0: left alone
        assert _same(x[7:9], want[7:9]) and (x[9:27] == 0.0).all()                            # 30 and 31, then the missing page
        assert (x[27:] == 9.0).all()
    assert not pool[1:4].any() and not pool[5:].any()
    # what `first` says is cut to the rows there are
    card.kv4_write(k, v, pool, tables, _i32([3, 3, 3, 3]), first=_i32([0, 3, 2, 100, 7]))
    torch.cuda.synchronize()


def test_a_full_table(card):
    """a sequence longer than its table: rows past it are not written, what stands there stays, attention is over what is held"""
    g = gen(9450)
    Hk, G, D, page = 1, 2, 64, 32
    tables = _i32([[2, 0]])
    pool = _filled(card, 3, Hk, D, page)
    k, v = _rows(g, 66, Hk, D), _rows(g, 66, Hk, D)
    card.kv4_write(k[:64], v[:64], pool, tables, _i32([64]))
    full = pool.clone()
    card.kv4_write(k[64:65], v[64:65], pool, tables, _i32([65]))
    card.kv4_write(k[:1], v[:1], pool, tables, _i32([(1 << 31) - 1]))
    assert torch.equal(pool, full)
    card.kv4_write(k[60:66], v[60:66], pool, tables, _i32([66]))  # the first four of them are the last that fit, and the same
    assert torch.equal(pool, full)
    a, b = (torch.full((6, Hk, D), 9.0, device="cuda") for _ in range(2))
    card.kv4_read(pool, tables, _i32([66]), a, b)
    assert _same(a[:4], kv4.held_k(k[60:64].double().cpu().numpy())[0]) and bool((a[4:] == 9.0).all()) and bool((b[4:] == 9.0).all())
    q = _rows(g, 3, G, D)
    att, lse = _attend(card, q, pool, tables, [66], [3], G, page, check=False)  # at 63, 64 and 65
    _check(q, pool, _i32([[2, 0, -1]]), [66], [3], att, lse, 1.0 / math.sqrt(D), G, page)


# ---- attention -----------------------------------------------------------------------------------------------------------------


def _check(q, pool, tables, lens, rows, att, lse, scale, G, page, hk_of=None):
    """each row against the oracle, within the bars"""
    T, Hq, D = q.shape
    qf, cache, tab = q.double().cpu().numpy(), pool.cpu().numpy(), tables.cpu().numpy()
    got, z = att.double().cpu().numpy().reshape(T, Hq, D), lse.double().cpu().numpy()
    row = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        n = max(min(n, tab.shape[1] * page), 0)
        for hk in range(Hq // G):
            K, V, there = kv4.tokens(cache, tab[b], n, page, hk, D)
            for i in range(r):
                sees = max(n - r + i + 1, 0)
                for h in range(hk * G, hk * G + G):
                    want, wz, spread, most = kv4.attention(qf[row + i, h], K[:sees], V[:sees], there[:sees], scale)
                    at = (b, i, h)
                    if wz == -np.inf:
                        assert (got[row + i, h] == 0.0).all() and z[row + i, h] == -np.inf, at
                        continue
                    if not np.isfinite(wz):
                        assert np.isnan(got[row + i, h]).all() and np.isnan(z[row + i, h]), at
                        continue
                    size = (np.abs(K[:sees][there[:sees]]) @ np.abs(qf[row + i, h])).max() * scale
                    e = D * U * size + U * 1.5 * size + 2 * U
                    bar = W * np.abs(want) + (H + e + 64 * U) * spread + 2.0**-36 * most
                    off = np.abs(got[row + i, h] - want)
                    if np.isfinite(want).all():
                        assert (off <= bar).all(), (at, (off / bar).max())
                    else:
                        assert np.array_equal(np.isnan(got[row + i, h]), np.isnan(want)), at
                    assert abs(z[row + i, h] - wz) <= e + 8 * U * (1 + abs(wz)), (at, z[row + i, h], wz)
        row += r


def _attend(card, q, pool, tables, lens, rows, G, page, first=True, cap=0, check=True):
    T, Hq, D = q.shape
    att, lse = torch.full((T, Hq * D), 5.0, dtype=torch.bfloat16, device="cuda"), torch.full((T, Hq), 5.0, device="cuda")
    scale = 1.0 / math.sqrt(D)
    scratch = card.attn_kv4_scratch(T, len(lens), Hq, Hq // G, D, cap or tables.shape[1] * page)
    scratch.fill_(NAN)
    card.attn_kv4(q.view(T, -1), pool, tables, _i32(lens), att, Hq, Hq // G, D, scale, scratch, first=_first(rows) if first else None, lse=lse,
                  keys_cap=cap)
    torch.cuda.synchronize()
    if check:
        _check(q, pool, tables, lens, rows, att, lse, scale, G, page)
    return att, lse


@pytest.mark.parametrize("lens,rows,Hk,G,D,page,cap", [
    ([1], [1], 1, 1, 64, 32, 0),
    ([1, 2, 31, 32, 33], [1] * 5, 2, 4, 128, 32, 0),
    ([700], [1], 2, 4, 128, 64, 0),
    ([700], [1], 1, 3, 64, 96, 0),
    ([2500], [1], 1, 8, 128, 128, 0),
    ([2500], [1], 1, 8, 128, 128, 64),          # longer than the bound that sized the launch
    ([9000], [1], 1, 2, 64, 256, 0),            # many spans
    ([300, 40, 1001], [8, 8, 8], 2, 5, 64, 32, 0),
    ([300, 40, 1001], [8, 8, 8], 1, 4, 128, 64, 0),
    ([129, 64, 77], [100, 64, 1], 1, 4, 128, 64, 0),   # a prompt from its first token on beside single ones
    ([200], [200], 2, 1, 128, 32, 0),
    ([90, 5], [33, 5], 1, 16, 64, 32, 0),
    ([40], [3], 1, 64, 128, 32, 0),
    ([512] * 3, [1] * 3, 1, 17, 128, 64, 0),
])
def test_attention(card, lens, rows, Hk, G, D, page, cap):
    g = gen(9500 + sum(lens) + D + G)
    pool, tables, _, _ = _put(card, g, lens, Hk, D, page)
    q = _rows(g, sum(rows), Hk * G, D) * 1.5
    a = _attend(card, q, pool, tables, lens, rows, G, page, cap=cap)
    if len(set(rows)) == 1:
        b = _attend(card, q, pool, tables, lens, rows, G, page, first=False, cap=cap, check=False)
        _check(q, pool, tables, lens, rows, *b, 1.0 / math.sqrt(D), G, page)
    again = _attend(card, q, pool, tables, lens, rows, G, page, cap=cap, check=False)
    assert torch.equal(a[0], again[0]) and torch.equal(a[1], again[1])


@pytest.mark.parametrize("lens,rows,G,D,cap", [
    # one span of more than 256 tiles, and of more than 512: a wave looks its next 64 places up on the way
    ([17000], [1], 4, 64, 64), ([17000], [1], 4, 128, 64),                    # four and two tiles at a time, past the caches
    ([9000, 8300], [9, 1], 8, 64, 64), ([9000, 8300], [9, 1], 8, 128, 64),    # a tile at a time, and what is left of it by four and two
    ([16500], [40], 2, 64, 64), ([8192 + 33], [33], 1, 128, 64),
    # more spans than a join asks for at once: 64 at head_dim 128, 128 at 64
    ([34000], [1], 3, 128, 34000), ([36000], [1], 1, 64, 36000), ([66000], [1], 4, 64, 66000),
])
def test_long_walks_and_joins(card, lens, rows, G, D, cap):
    g = gen(9540 + sum(lens) + D)
    pool, tables, _, _ = _put(card, g, lens, 1, D, 64)
    floats, q = card.attn_kv4_scratch(sum(rows), len(lens), G, 1, D, cap).numel(), _rows(g, sum(rows), G, D)
    spans = floats // (sum(rows) * G * (D + 2)) if floats > 4 else 1
    assert spans == 1 if cap == 64 else spans > (64 if D == 128 else 128), spans
    _attend(card, q, pool, tables, lens, rows, G, 64, cap=cap)


@pytest.mark.parametrize("lens,rows,Hk,G,D", [([9000], [1], 1, 2, 64), ([1500, 40], [1, 1], 2, 4, 128), ([129, 64, 0, 2000], [100, 64, 2, 1], 2, 5, 128)])
def test_in_the_place_of_its_rows(card, lens, rows, Hk, G, D):
    """att is q: many spans, few, none"""
    g = gen(9550 + D + G)
    page, scale = 64, 0.1
    pool, tables, _, _ = _put(card, g, lens, Hk, D, page)
    q = _rows(g, sum(rows), Hk * G * D)
    att = torch.zeros_like(q)
    scratch = card.attn_kv4_scratch(sum(rows), len(lens), Hk * G, Hk, D, max(lens))
    for out in (att, q):
        card.attn_kv4(q, pool, tables, _i32(lens), out, Hk * G, Hk, D, scale, scratch, first=_first(rows), keys_cap=max(lens))
    torch.cuda.synchronize()
    assert torch.equal(att, q) and bool(att.any())


@pytest.mark.parametrize("size", [2.0**4, 2.0**9, 2.0**12, 2.0**30])
@pytest.mark.parametrize("G,rows,n", [(4, 40, 240), (4, 1, 240), (2, 3, 9000), (8, 200, 240)])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_of_any_size(card, D, G, rows, n, size):
    """one key is far above the others a row sees: its value is the output, whatever the scores' own rounding"""
    g = gen(9560 + D + G)
    page, scale = 64, 0.1
    held = torch.full((n,), 0.5)
    held[37], held[n - 30], held[n - 10] = 4.0, 6.0, -6.0
    tables, pages = _tables(g, [n], page)
    pool = _filled(card, pages, 1, D, page)
    k = (held * size).cuda()[:, None, None].expand(n, 1, D).to(torch.bfloat16).contiguous()
    v = _rows(g, n, 1, D)
    card.kv4_write(k, v, pool, tables, _i32([n]))
    q = torch.full((rows, G * D), size, dtype=torch.bfloat16, device="cuda")
    att, lse = torch.zeros_like(q), torch.zeros(rows, G, device="cuda")
    scratch = card.attn_kv4_scratch(rows, 1, G, 1, D, n)
    card.attn_kv4(q, pool, tables, _i32([n]), att, G, 1, D, scale, scratch, first=_first([rows]), lse=lse)
    torch.cuda.synchronize()
    V = torch.from_numpy(kv4.held_v(v.double().cpu().numpy())[0][:, 0])
    scale = float(np.float32(scale))
    for i in range(rows):
        sees = n - rows + i + 1
        best = n - 30 if sees > n - 30 else 37
        if sees > 37:
            off = (att[i].view(G, D).double().cpu() - V[best]).abs()
            assert bool((off <= (W + H) * V[best].abs()).all()), i
            s = scale * D * size * size * float(held[best])
            assert np.allclose(lse[i].cpu().numpy(), s, rtol=4 * 2.0**-23, atol=0), i


@pytest.mark.parametrize("size,scale", [(2.0**58, 1.0), (1.0, 2.0**115), (2.0**58, 2.0**-116), (2.0**-40, 2.0**83), (2.0**-60, 2.0**127)])
@pytest.mark.parametrize("G,rows,n", [(4, 40, 240), (4, 1, 240), (2, 3, 9000)])
@pytest.mark.parametrize("D", [64, 128])
def test_products_and_scales_at_their_ends(card, D, G, rows, n, size, scale):
    """products of q and k, and scales, near f32's largest and smallest: the key far above the others gives its value. D 6 size^2 is up to
    2^125.6, and that times scale log2(e) up to 2^126.2; the best of them is 128 or more above the next
    (D 2 size^2 scale)"""
    g = gen(9570 + D + G)
    page = 64
    held = torch.full((n,), 0.5)
    held[37], held[n - 30], held[n - 10] = 4.0, 6.0, -6.0
    tables, pages = _tables(g, [n], page)
    pool = _filled(card, pages, 1, D, page)
    k = (held * size).cuda()[:, None, None].expand(n, 1, D).to(torch.bfloat16).contiguous()
    v = _rows(g, n, 1, D)
    card.kv4_write(k, v, pool, tables, _i32([n]))
    q = torch.full((rows, G * D), size, dtype=torch.bfloat16, device="cuda")
    att, lse = torch.zeros_like(q), torch.zeros(rows, G, device="cuda")
    scratch = card.attn_kv4_scratch(rows, 1, G, 1, D, n)
    card.attn_kv4(q, pool, tables, _i32([n]), att, G, 1, D, scale, scratch, first=_first([rows]), lse=lse)
    torch.cuda.synchronize()
    V = torch.from_numpy(kv4.held_v(v.double().cpu().numpy())[0][:, 0])
    least = D * 2.0 * size * size * scale
    for i in range(rows):
        sees = n - rows + i + 1
        best = n - 30 if sees > n - 30 else 37
        assert sees > 37 and least >= 128
        off = (att[i].view(G, D).double().cpu() - V[best]).abs()
        assert bool((off <= (W + H) * V[best].abs()).all()), i
        s = scale * D * size * size * float(held[best])
        assert np.allclose(lse[i].cpu().numpy(), s, rtol=4 * 2.0**-23, atol=0), i


@pytest.mark.parametrize("D", [64, 128])
def test_many_ragged_sequences(card, D):
    """more sequences than are looked through at a time, some without rows where the looking goes on; long ones in spans"""
    g = gen(9580 + D)
    B, Hk, G, page = 150, 1, 4, 64
    rows = [(3 * b) % 5 for b in range(B)]
    rows[62:67], rows[127:129], rows[149], rows[100], rows[140] = [0] * 5, [0, 9], 0, 40, 33
    lens = [r + (7 * b) % 50 for b, r in enumerate(rows)]
    lens[3], lens[70], lens[128], lens[140], lens[148] = 1500, 900, 1200, 700, 600
    tables, pages = _tables(g, lens, page)
    T, n = sum(rows), sum(lens)
    pool = _filled(card, pages, Hk, D, page)
    k, v = _rows(g, n, Hk, D), _rows(g, n, Hk, D)
    card.kv4_write(k, v, pool, tables, _i32(lens), first=_first(lens))
    at = torch.cat([torch.arange(e - r, e) for e, r in zip(np.cumsum(lens).tolist(), rows)]).cuda()
    new_k, new_v = _rows(g, T, Hk, D), _rows(g, T, Hk, D)
    card.kv4_write(new_k, new_v, pool, tables, _i32(lens), first=_first(rows))  # the last rows once more, others
    k[at], v[at] = new_k, new_v
    for what, want, count in (("the pass's", (new_k, new_v), rows), ("all", (k, v), lens)):
        a, b = (torch.zeros(sum(count), Hk, D, device="cuda") for _ in range(2))
        card.kv4_read(pool, tables, _i32(lens), a, b, first=_first(count))
        assert _same(a, kv4.held_k(want[0].double().cpu().numpy())[0]), what
        assert _same(b, kv4.held_v(want[1].double().cpu().numpy())[0]), what
    _attend(card, _rows(g, T, Hk * G, D), pool, tables, lens, rows, G, page, cap=1500)


def test_attention_without_anything_to_see(card):
    """lengths of zero and below, rows before the first token, sequences without rows, rows behind the last sequence"""
    g = gen(9600)
    lens, rows = [0, 3, -5, 40, 70], [1, 5, 2, 0, 1]
    Hk, G, D, page, T = 2, 2, 128, 64, 12
    pool = _filled(card, 6, Hk, D, page)
    tables = _i32([[0, 5], [1, -1], [2, -1], [3, -1], [4, 5]])
    k, v = _rows(g, 113, Hk, D), _rows(g, 113, Hk, D)
    card.kv4_write(k, v, pool, tables, _i32(lens), first=_first([0, 3, 0, 40, 70]))
    q = _rows(g, T, Hk * G, D)
    att, lse = _attend(card, q, pool, tables, lens, rows, G, page, check=False)
    _check(q[:9], pool, tables, lens, rows, att[:9], lse[:9], 1.0 / math.sqrt(D), G, page)
    assert bool((att[9:] == 5.0).all()) and bool((lse[9:] == 5.0).all())


@pytest.mark.parametrize("G,rows", [(4, 1), (4, 8), (8, 5)])
def test_pages_that_are_not_the_pools(card, G, rows):
    g = gen(9700 + G)
    Hk, D, page, lens = 1, 128, 64, [300, 1000]
    pool, tables, _, _ = _put(card, g, lens, Hk, D, page)
    tables[0, 1], tables[0, 4], tables[1, 0], tables[1, 15] = -1, 1 << 30, -(1 << 31), pool.shape[0]
    q = _rows(g, 2 * rows, G, D)
    _attend(card, q, pool, tables, lens, [rows] * 2, G, page)
    tables.fill_(-7)
    _attend(card, q, pool, tables, lens, [rows] * 2, G, page)


@pytest.mark.parametrize("G,rows", [(2, 1), (4, 9)])
@pytest.mark.parametrize("D", [64, 128])
def test_nan_and_infinities(card, G, rows, D):
    """a key or value that is NaN reaches the rows that see it and no other; what lies behind a sequence's end reaches nobody"""
    g = gen(9800 + G + D)
    Hk, page, n = 1, 32, 200
    tables, pages = _tables(g, [n, n, n], page)
    pool = _filled(card, pages, Hk, D, page, 0xFF)  # every scale NaN
    k, v = _rows(g, 3 * n, Hk, D), _rows(g, 3 * n, Hk, D)
    k[n - 2, 0, 3] = NAN            # sequence 0: a key the last two rows see
    v[2 * n - 3, 0, 5] = INF        # sequence 1: a value the last three rows see
    card.kv4_write(k, v, pool, tables, _i32([n] * 3))
    q = _rows(g, 3 * rows, G, D)
    q[2 * rows, 0, 1] = NAN         # sequence 2: one row's query
    att, lse = _attend(card, q, pool, tables, [n] * 3, [rows] * 3, G, page, check=False)
    att = att.float().view(3, rows, G, D).cpu().numpy()
    lse = lse.view(3, rows, G).cpu().numpy()
    sees = min(rows, 2)
    assert np.isnan(att[0, rows - sees:]).all() and np.isfinite(att[0, :rows - sees]).all() and np.isnan(lse[0, rows - sees:]).all()
    sees = min(rows, 3)
    assert np.isnan(att[1, rows - sees:]).all() and np.isfinite(att[1, :rows - sees]).all() and np.isfinite(lse[1]).all()
    assert np.isnan(att[2, 0, 0]).all() and np.isfinite(att[2, 1:]).all() and np.isfinite(att[2, 0, 1:]).all()
    # the rows that see nothing of it are those of a cache without it
    k2, v2 = k.clone(), v.clone()
    k2[n - 2:n], v2[2 * n - 3:2 * n] = 0.0, 0.0
    pool2 = _filled(card, pages, Hk, D, page, 0)
    card.kv4_write(k2, v2, pool2, tables, _i32([n] * 3))
    _check(q[:rows - min(rows, 2)], pool2, tables[:1], [n - 2], [max(rows - 2, 0)], torch.from_numpy(att[0, :max(rows - 2, 0)]),
           torch.from_numpy(lse[0, :max(rows - 2, 0)]), 1.0 / math.sqrt(D), G, page)


@pytest.mark.parametrize("D", [64, 128])
def test_values_of_unlike_size(card, D):
    """scales that grow and shrink by powers along a sequence, and scores that keep passing the maximum"""
    g = gen(9900 + D)
    Hk, G, page, n = 1, 4, 64, 1500
    tables, pages = _tables(g, [n], page)
    pool = _filled(card, pages, Hk, D, page)
    k, v = _rows(g, n, Hk, D), _rows(g, n, Hk, D)
    size = torch.exp2(torch.linspace(-14, 14, n) * torch.where(torch.arange(n) % 2 == 0, 1.0, -1.0)).cuda()
    v = (v.float() * size[:, None, None]).to(torch.bfloat16)
    k = (k.float() * torch.linspace(0.1, 6.0, n).cuda()[:, None, None]).to(torch.bfloat16)
    card.kv4_write(k, v, pool, tables, _i32([n]))
    _attend(card, _rows(g, 3, G, D) * 3.0, pool, tables, [n], [3], G, page)
    _attend(card, _rows(g, 40, G, D) * 3.0, pool, tables, [n], [40], G, page)


@pytest.mark.parametrize("byte", [0xFF, 0x7F, 0x00])
@pytest.mark.parametrize("G,rows", [(4, 40), (8, 3), (1, 90)])
@pytest.mark.parametrize("D", [64, 128])
def test_a_large_value_that_not_every_row_sees(card, D, G, rows, byte):
    """rows before it keep their own precision; so do all where what lies behind the last token has the largest scale there is"""
    g = gen(9950 + D + G)
    page, n, at = 32, 300, 300 - rows // 2
    tables, pages = _tables(g, [n], page)
    pool = _filled(card, pages, 1, D, page, byte)
    k, v = _rows(g, n, 1, D), _rows(g, n, 1, D) * 2.0**-9
    v[at] *= 2.0**60
    v[at + 1:] *= 2.0**20
    card.kv4_write(k, v, pool, tables, _i32([n]))
    _attend(card, _rows(g, rows, G, D), pool, tables, [n], [rows], G, page)


def test_far_pages(card):
    """pages whose bytes start past 2^32, in a pool with a row of layers a page"""
    g = gen(9950)
    Hk, G, D, page = 1, 2, 128, 32
    stride = 4288 * 1024
    pages = (5 << 30) // stride
    big = torch.empty(pages * stride, dtype=torch.uint8, device="cuda")
    pool = big.as_strided((pages, 1, 1, 4288), (stride, 4288, 4288, 1), 4288 * 7)
    lens = [90, 33]
    tables = _i32([[pages - 1, pages - 3, 0], [pages - 2, 1, -1]])
    k, v = _rows(g, 123, Hk, D), _rows(g, 123, Hk, D)
    card.kv4_write(k, v, pool, tables, _i32(lens), first=_first(lens))
    a, b = torch.zeros(123, 1, D, device="cuda"), torch.zeros(123, 1, D, device="cuda")
    card.kv4_read(pool, tables, _i32(lens), a, b, first=_first(lens))
    assert _same(a, kv4.held_k(k.double().cpu().numpy())[0]) and _same(b, kv4.held_v(v.double().cpu().numpy())[0])
    q = _rows(g, 2, G, D)
    att, lse = _attend(card, q, pool, tables, lens, [1, 1], G, page, check=False)
    near = pool[torch.tensor([pages - 1, pages - 3, 0, pages - 2, 1], device="cuda")].contiguous()
    _check(q, near, _i32([[0, 1, 2], [3, 4, -1]]), lens, [1, 1], att, lse, 1.0 / math.sqrt(D), G, page)


def test_recorded_and_replayed_as_sequences_grow(card):
    """write and attention recorded once; tokens, lengths, tables and rows change between replays. Two recordings have a workspace each."""
    g = gen(9960)
    Hk, G, D, page, B, cap = 2, 4, 128, 32, 3, 400
    tables, pages = _tables(g, [cap] * B, page)
    pool = _filled(card, pages, Hk, D, page)
    lens = [40, 7, 300]
    k, v = _rows(g, sum(lens), Hk, D), _rows(g, sum(lens), Hk, D)
    dlens = _i32(lens)
    card.kv4_write(k, v, pool, tables, dlens, first=_first(lens))
    shapes = ((B, None), (8, _i32([0, 1, 3, 6])))
    graphs = []
    for T, first in shapes:
        s = dict(k=_rows(g, T, Hk, D), v=_rows(g, T, Hk, D), q=_rows(g, T, Hk * G, D), att=torch.zeros(T, Hk * G * D, dtype=torch.bfloat16, device="cuda"),
                 lse=torch.zeros(T, Hk * G, device="cuda"), ws=card.attn_kv4_scratch(T, B, Hk * G, Hk, D, cap), first=first)

        def body(s=s, T=T):
            card.kv4_write(s["k"], s["v"], pool, tables, dlens, first=s["first"])
            card.attn_kv4(s["q"].view(T, -1), pool, tables, dlens, s["att"], Hk * G, Hk, D, 0.1, s["ws"], first=s["first"], lse=s["lse"], keys_cap=cap)

        graph = torch.cuda.CUDAGraph()
        with recording(graph):
            body()
        graphs.append((s, graph, body))
    for n in range(5):
        for i, (s, graph, body) in enumerate(graphs):
            rows = [1, 1, 1] if i == 0 else [[1, 2, 3], [0, 4, 1], [8, 0, 0], [2, 2, 2], [1, 1, 6]][n]
            lens = [a + r for a, r in zip(lens, rows)]
            dlens.copy_(_i32(lens))
            if s["first"] is not None:
                s["first"].copy_(_first(rows))
            for name in ("k", "v", "q"):
                s[name].copy_(_rows(g, *s[name].shape))
            was, kept = pool.clone(), [s["att"].clone(), s["lse"].clone()]
            graph.replay()
            torch.cuda.synchronize()
            got = [s["att"].clone(), s["lse"].clone(), pool.clone()]
            pool.copy_(was)
            s["att"].copy_(kept[0])
            s["lse"].copy_(kept[1])
            s["ws"].fill_(NAN)
            body()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, (s["att"], s["lse"], pool))), (n, i)


def test_another_stream(card):
    g = gen(9970)
    pool, tables, _, _ = _put(card, g, [500], 1, 64, 32)
    q = _rows(g, 1, 4, 64)
    want = _attend(card, q, pool, tables, [500], [1], 4, 32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _attend(card, q, pool, tables, [500], [1], 4, 32, check=False)
    side.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


# ---- pages ---------------------------------------------------------------------------------------------------------------------------


def _pool(g, L, pages, nb, dtype, by_page):
    raw = torch.randint(0, 256, (L, pages, nb), generator=g, dtype=torch.uint8)
    t = raw.view(dtype).cuda()
    return t.transpose(0, 1).contiguous().transpose(0, 1) if by_page else t


@pytest.mark.parametrize("L,nb,dtype,by_page,page", [
    (1, 16, torch.uint8, False, 32), (3, 4288 * 2, torch.uint8, False, 64), (2, 16384 + 48, torch.bfloat16, True, 1), (5, 1024, torch.int32, True, 100),
])
def test_fork(card, L, nb, dtype, by_page, page):
    g = gen(10000 + nb)
    B, W_, pages = 9, 5, 40
    pool = _pool(g, L, pages, nb, dtype, by_page)
    lens = [0, 1, page, 3 * page, 2 * page + page // 2, W_ * page, W_ * page + 7, -3, 2]
    tables = torch.randperm(pages, generator=g)[:27].to(torch.int32)
    tables = torch.cat([tables, torch.full((18,), -1, dtype=torch.int32)]).view(B, W_)
    tables[4, 2] = 10
    src = [4, 4, 1, 3, 5, 2, 0, 7, 4, 9, -1, 4]
    dst = [6, 8, -1, 9, 7, 2, 2, 2, 4, 0, 0, 20]
    fresh = [39, 38, 0, 0, 99, 1, -1, 5, 3, 4, 4, 4]
    src, dst, fresh = src[:6] + src[8:], dst[:6] + dst[8:], fresh[:6] + fresh[8:]
    want, wt, wl = pool.cpu().view(torch.uint8).numpy().copy(), tables.numpy().copy(), np.array(lens)
    kv4.fork(want, wt, wl, src, dst, fresh, page)
    dt, dl = tables.cuda(), _i32(lens)
    card.pages_fork(pool, dt, dl, _i32(src), _i32(dst), _i32(fresh), page)
    torch.cuda.synchronize()
    assert np.array_equal(dt.cpu().numpy(), wt) and np.array_equal(dl.cpu().numpy(), wl)
    assert np.array_equal(pool.cpu().contiguous().view(torch.uint8).numpy(), want)


def test_fork_of_a_page_that_is_not_there(card):
    g = gen(10050)
    pool = _pool(g, 2, 6, 64, torch.uint8, False)
    was = pool.clone()
    tables, lens = _i32([[0, 77], [-1, -1], [1, -1], [-1, -1]]), _i32([40, 0, 5, 0])
    card.pages_fork(pool, tables, lens, _i32([0, 2]), _i32([1, 3]), _i32([3, 6]), 32)  # the second's fresh page is none
    assert tables.tolist() == [[0, 77], [0, -1], [1, -1], [-1, -1]] and lens.tolist() == [40, 40, 5, 0] and torch.equal(pool, was)


@pytest.mark.parametrize("L,nb,dtype,by_page,pages,B,W_,live", [
    (1, 16, torch.uint8, False, 1, 1, 1, 1.0), (3, 4288, torch.uint8, False, 70, 5, 30, 0.6), (2, 16384 + 48, torch.bfloat16, True, 33, 3, 20, 0.3),
    (1, 64, torch.int32, False, 5000, 40, 130, 0.8), (2, 32, torch.uint8, True, 300000, 64, 3000, 0.4), (4, 4288, torch.uint8, False, 64, 4, 16, 0.0),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(card, L, nb, dtype, by_page, pages, B, W_, live, in_place):
    g = gen(10100 + pages)
    page = 32
    pool = _pool(g, L, pages, nb, dtype, by_page)
    held = min(int(pages * live), B * W_)
    order = torch.randperm(pages, generator=g)[:held].tolist()
    tables, lens = np.full((B, W_), -1, np.int32), np.zeros(B, np.int64)
    at = 0
    for b in range(B):
        k = min(W_, (held - at) // (B - b) + (1 if b % 2 else 0), held - at)
        tables[b, :k] = order[at:at + k]
        lens[b] = k * page - (b * 7) % page if k else -b
        at += k
    if held > 12:
        tables[1, 0], tables[2, 1] = tables[0, 0], tables[0, 0]  # shared
        tables[B - 1, 0] = pages + 5                                # none of the pool's
        tables[0, W_ - 1] = 3                                       # behind the sequence's end: named by nobody (unless it is as long)
        lens[0] = min(lens[0], (W_ - 1) * page)
    dt, dl = torch.from_numpy(tables).cuda(), _i32(lens.tolist())
    want = pool.cpu().contiguous().view(torch.uint8).numpy().copy()
    wt, used = kv4.compact(want, tables, lens, page)
    out = dt if in_place else torch.full_like(dt, 77)
    got = card.pages_compact(pool, dt, dl, page, None if in_place else out)
    torch.cuda.synchronize()
    assert got.tolist() == [used] and np.array_equal(out.cpu().numpy(), wt)
    after = pool.cpu().contiguous().view(torch.uint8).numpy()
    assert np.array_equal(after, want)
    if not in_place:
        assert np.array_equal(dt.cpu().numpy(), tables)
    # closed up already: nothing moves
    again = card.pages_compact(pool, out, dl, page)
    assert again.tolist() == [used] and np.array_equal(out.cpu().numpy(), wt)
    assert np.array_equal(pool.cpu().contiguous().view(torch.uint8).numpy(), want)


def test_pages_recorded(card):
    """a fork and a compaction recorded, and replayed over other tables"""
    g = gen(10200)
    L, pages, page, B, W_ = 2, 20, 32, 4, 4
    pool = _pool(g, L, pages, 64, torch.uint8, False)
    tables, lens = torch.full((B, W_), -1, dtype=torch.int32, device="cuda"), _i32([0] * B)
    src, dst, fresh = _i32([0]), _i32([3]), _i32([0])
    out = torch.empty_like(tables)

    def body():
        card.pages_fork(pool, tables, lens, src, dst, fresh, page)
        return card.pages_compact(pool, tables, lens, page, out)

    graph = torch.cuda.CUDAGraph()
    with recording(graph):
        used = body()
    for n in range(4):
        order = torch.randperm(pages, generator=g).tolist()
        table = np.full((B, W_), -1, np.int32)
        table[0, :3], table[1, :2], table[2, :1] = order[:3], order[3:5], order[5:6]
        size = [70 + n, 64, 0 if n % 2 else 9, 0]
        tables.copy_(torch.from_numpy(table))
        lens.copy_(_i32(size))
        fresh.fill_(order[6])
        want, wl = pool.cpu().numpy().copy(), np.array(size)
        kv4.fork(want, table, wl, [0], [3], [order[6]], page)
        wt, wu = kv4.compact(want, table, wl, page)
        graph.replay()
        torch.cuda.synchronize()
        assert used.tolist() == [wu] and np.array_equal(out.cpu().numpy(), wt) and np.array_equal(pool.cpu().numpy(), want)


# ---- all of them --------------------------------------------------------------------------------------------------------------------


def test_a_batch_over_its_life(card):
    """two prompts go in, one branches, all step, one ends, the pool is closed up, the rest step on: outputs as over whole caches of
    their own, equal before and after pages have moved"""
    g = gen(10300)
    L, Hk, G, D, page, B, pages = 2, 2, 4, 128, 64, 4, 24
    pool = card.kv4_pool(pages, Hk, D, page, layers=L)
    tables = torch.full((B, 6), -1, dtype=torch.int32, device="cuda")
    lens = [150, 0, 90, 0]
    tables[0, :3], tables[2, :2] = _i32([20, 3, 11]), _i32([7, 23])
    history = [[_rows(g, 150, Hk, D) for _ in range(2 * L)], None, [_rows(g, 90, Hk, D) for _ in range(2 * L)], None]
    for layer in range(L):
        k = torch.cat([history[0][2 * layer], history[2][2 * layer]])
        v = torch.cat([history[0][2 * layer + 1], history[2][2 * layer + 1]])
        card.kv4_write(k, v, pool[layer], tables, _i32(lens), first=_first(lens))
    dl = _i32(lens)
    card.pages_fork(pool, tables, dl, _i32([0]), _i32([1]), _i32([5]), page)
    history[1] = [t.clone() for t in history[0]]
    lens = dl.tolist()
    assert lens == [150, 150, 90, 0]

    def step(alive):
        outs = []
        for b in alive:
            lens[b] += 1
            if (lens[b] - 1) % page == 0:
                free = sorted(set(range(pages)) - {p for c in alive for p in tables[c].tolist()})
                tables[b, (lens[b] - 1) // page] = free[0]
        rows = [1 if b in alive else 0 for b in range(B)]
        for layer in range(L):
            k, v, q = _rows(g, len(alive), Hk, D), _rows(g, len(alive), Hk, D), _rows(g, len(alive), Hk * G, D)
            card.kv4_write(k, v, pool[layer], tables, _i32(lens), first=_first(rows))
            for i, b in enumerate(alive):
                history[b][2 * layer] = torch.cat([history[b][2 * layer], k[i:i + 1]])
                history[b][2 * layer + 1] = torch.cat([history[b][2 * layer + 1], v[i:i + 1]])
            outs.append((q, *_attend(card, q, pool[layer], tables, lens, rows, G, page)))
        return outs

    for _ in range(3):
        step([0, 1, 2])
    lens[0] = 0  # the first one ends
    moved = _i32(lens)
    q = _rows(g, 2, Hk * G, D)
    before = [_attend(card, q, pool[layer], tables, lens, [0, 1, 1, 0], G, page) for layer in range(L)]
    used = card.pages_compact(pool, tables, moved, page)
    assert used.item() == 5 and sorted(p for p in tables.flatten().tolist() if p >= 0) == [0, 1, 2, 3, 4]
    after = [_attend(card, q, pool[layer], tables, lens, [0, 1, 1, 0], G, page) for layer in range(L)]
    assert all(torch.equal(x, y) for a, b in zip(before, after) for x, y in zip(a, b))
    for _ in range(40):
        step([1, 2])
    for b in (1, 2):
        for layer in range(L):
            k, v = history[b][2 * layer], history[b][2 * layer + 1]
            for hk in range(Hk):
                K, V, there = kv4.tokens(pool[layer].cpu().numpy(), tables[b].cpu().numpy(), lens[b], page, hk, D)
                assert there.all() and _same(K, kv4.held_k(k[:, hk].double().cpu().numpy())[0])
                assert _same(V, kv4.held_v(v[:, hk].double().cpu().numpy())[0])


def test_refusals(card):
    g = gen(10400)
    Hk, G, D, page = 2, 2, 128, 64
    pool, tables, k, v = _put(card, g, [100, 40], Hk, D, page)
    lens, first = _i32([100, 40]), _first([100, 40])
    T = 140
    write = dict(k=k, v=v, cache=pool, tables=tables, lens=lens, first=first)
    for name, bad in [("k", k.float()), ("k", k.cpu()), ("v", v[:, :1]), ("k", k.view(T, -1)), ("v", v.transpose(1, 2)), ("cache", pool[:, :1]),
                      ("cache", pool.view(torch.int8)), ("cache", pool[..., :4096]), ("cache", pool.transpose(1, 2)), ("cache", pool.cpu()),
                      ("tables", tables.long()), ("tables", tables.flatten()), ("tables", tables.t()), ("tables", tables[:1]), ("lens", lens[:1]),
                      ("lens", lens.cpu()), ("first", first[:2]), ("first", first.long()), ("first", first.cpu())]:
        with pytest.raises(ValueError):
            card.kv4_write(**{**write, name: bad})
    with pytest.raises(ValueError):
        card.kv4_write(k[:3], v[:3], pool, tables, lens)  # three rows for two sequences
    with pytest.raises(ValueError):
        card.kv4_write(k, v, pool, tables[:0], lens[:0])
    f = torch.zeros(T, Hk, D, device="cuda")
    with pytest.raises(ValueError):
        card.kv4_read(pool, tables, lens, f, f.bfloat16(), first=first)
    with pytest.raises(ValueError):
        card.kv4_read(pool, tables, lens, f.half(), f.half(), first=first)
    with pytest.raises(HipError):
        card.kv4_read(pool, tables, lens, f[:1].expand(T, Hk, D), f, first=first)
    with pytest.raises(HipError):
        card.kv4_write(torch.zeros(2, Hk, D + 4, dtype=torch.bfloat16, device="cuda")[:, :, 4:], v[:2], pool, tables, lens)  # 8 bytes off
    q = _rows(g, 2, Hk * G * D)
    att = torch.zeros_like(q)
    ws = card.attn_kv4_scratch(2, 2, Hk * G, Hk, D, 128)
    attn = dict(q=q, cache=pool, tables=tables, lens=lens, att=att, Hq=Hk * G, Hk=Hk, D=D, scale=0.1, scratch=ws, keys_cap=128)
    card.attn_kv4(**attn)
    for name, bad in [("q", q.float()), ("q", q[:, :-1]), ("att", att[:1]), ("lse", torch.zeros(3, device="cuda")), ("scratch", ws[:3]), ("scratch", ws.half()),
                      ("D", 64), ("Hk", 4), ("Hq", 7), ("lens", lens.float()), ("first", first)]:
        if name == "first":
            card.attn_kv4(**{**attn, name: bad})
            continue
        with pytest.raises(ValueError):
            card.attn_kv4(**{**attn, name: bad})
    for bad in (0.0, -1.0, NAN, INF):
        with pytest.raises(HipError):
            card.attn_kv4(**{**attn, "scale": bad})
    for bad in (96, 256):
        with pytest.raises(ValueError):
            card.kv4_pool(4, 2, bad)
        with pytest.raises(ValueError):
            card.attn_kv4_scratch(1, 1, 4, 2, bad, 100)
    for bad in (0, 48):
        with pytest.raises(ValueError):
            card.kv4_pool(4, 2, 128, bad)
    pools = pool[None]
    with pytest.raises(ValueError):
        card.pages_fork(pool.view(-1, 4288), tables, lens, _i32([0]), _i32([1]), _i32([0]), page)
    with pytest.raises(ValueError):
        card.pages_fork(pools, tables, lens, _i32([0]), _i32([1]), _i32([0, 1]), page)
    with pytest.raises(ValueError):
        card.pages_fork(pools, tables, lens, _i32([0]).long(), _i32([1]), _i32([0]), page)
    with pytest.raises(HipError):
        card.pages_fork(pools[..., :8].contiguous(), tables, lens, _i32([0]), _i32([1]), _i32([0]), 0)
    with pytest.raises(ValueError):
        card.pages_compact(pools, tables, lens, page, tables_out=tables[:1])
    with pytest.raises(ValueError):
        card.pages_compact(pools, tables, lens[:1], page)
    with pytest.raises(HipError):
        card.pages_compact(torch.zeros(2, 9, 6, dtype=torch.uint8, device="cuda"), tables, lens, page)  # pages of six bytes
    torch.cuda.synchronize()
