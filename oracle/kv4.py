"""TEST INFRASTRUCTURE: a paged cache held in 4 bits, in 64 bits and written from the definitions: what rows are held as, where a tile
keeps them, attention over what is held, and the operators on whole pages."""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def bf16(x):
    """the bf16 number nearest to each of x (f64, within f32's range), ties to even, as f64"""
    f = np.asarray(x, np.float64).astype(np.float32)  # (what is rounded here has few bits, or a period: no tie is made)
    b = f.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(f), np.nan, r.astype(np.float64))


def codes(a):
    """the e2m1 code nearest to each magnitude: the closest of eight, of two as close the even one; past 6: 6"""
    a = np.asarray(a, np.float64)
    d = np.abs(np.minimum(a, 8.0)[..., None] - GRID)
    best = d.min(-1, keepdims=True)
    near = d == best
    first = near.argmax(-1)
    return np.where((first % 2 == 1) & (near.sum(-1) > 1), first + 1, first)


def held_k(k):
    """keys [..., D] as they are held: (values, the blocks' exponent bytes [..., D / 32])"""
    k = np.asarray(k, np.float64)
    x = k.reshape(*k.shape[:-1], -1, 32)
    top = np.abs(x).max(-1)
    lost = ~np.isfinite(top)
    safe = np.where(lost | (top == 0.0), 1.0, top)
    e = np.floor(np.log2(safe)).astype(np.int64) - 4
    for _ in range(3):
        e = np.where(safe > 7.0 * 2.0**e, e + 1, e)  # the smallest with top <= 7 2^e (the start is below it, by three at most)
    e = np.where(top == 0.0, -127, np.clip(e, -127, 125))
    unit = 2.0 ** e[..., None].astype(np.float64)
    with np.errstate(invalid="ignore"):
        v = np.copysign(GRID[codes(np.where(lost[..., None], 0.0, np.abs(x) / unit))] * unit, np.where(lost[..., None], 1.0, x))
    v = np.where(lost[..., None], np.nan, v)
    return v.reshape(k.shape), np.where(lost, 255, e + 127).astype(np.uint8)


def held_v(v):
    """values [..., D] as they are held: (values, the scales [...])"""
    v = np.asarray(v, np.float64)
    top = np.abs(v).max(-1)
    lost = ~np.isfinite(top)
    s = bf16(np.where(lost, 0.0, top) / 6.0)
    a = np.abs(np.where(lost[..., None], 0.0, v)) / np.where(s == 0.0, 1.0, s)[..., None]
    x = np.where((s == 0.0)[..., None], 0.0, GRID[codes(a)] * s[..., None])
    x = np.copysign(x, np.where(lost[..., None], 1.0, v))
    return np.where(lost[..., None], np.nan, x), np.where(lost, np.nan, s)


def tile(raw, D):
    """a tile's bytes (32 tokens of one head) as (K [32, D], V [32, D])"""
    raw = np.asarray(raw, np.uint8)
    steps = D // 64
    v0, ks = 1024 * steps, 2048 * steps
    vs = ks + 64 * steps
    sign = lambda c: np.where(c & 8, -1.0, 1.0) * GRID[c & 7]
    K, V = np.empty((32, D)), np.empty((32, D))
    scales = raw[vs:vs + 64].copy().view(np.uint16).astype(np.uint32) << 16
    scales = scales.view(np.float32).astype(np.float64)
    for token in range(32):
        for step in range(steps):
            for h in range(2):
                lane = 32 * h + token
                b = raw[1024 * step + 16 * lane:1024 * step + 16 * lane + 16]
                c = np.stack([b & 15, b >> 4], -1).reshape(-1)
                e = int(raw[ks + lane * steps + step])
                K[token, 64 * step + 32 * h:64 * step + 32 * h + 32] = sign(c) * (np.nan if e == 255 else 2.0 ** (e - 127))
        h, i = (token >> 2) & 1, (token >> 3) * 4 + (token & 3)
        for d in range(D):
            at = v0 + 1024 * (d // 64) + 16 * (32 * h + d % 32) + 8 * (d // 32 % 2) + 4 * (i // 8) + (i % 8) // 2
            V[token, d] = sign((raw[at] >> (4 * (i % 2))) & 15) * scales[16 * h + i]
    return K, V


def tokens(cache, table, n, page, hk, D):
    """the first n tokens of a sequence's head out of a pool [pages, Hk, page / 32, tile bytes]: (K, V [n, D], whether each is there)"""
    K, V, there = np.zeros((n, D)), np.zeros((n, D)), np.zeros(n, bool)
    for j in range((n + 31) // 32):
        p = int(table[j * 32 // page])
        if 0 <= p < cache.shape[0]:
            m = min(32, n - 32 * j)
            k, v = tile(cache[p, hk, j * 32 % page // 32], D)
            K[32 * j:32 * j + m], V[32 * j:32 * j + m], there[32 * j:32 * j + m] = k[:m], v[:m], True
    return K, V, there


def attention(q, K, V, there, scale):
    """one query [D] over tokens [n, D], of which only those that are there count: (att [D], lse, sum of |weight value| [D], the largest
    |weight value|)"""
    K, V = K[there], V[there]
    if len(K) == 0:
        return np.zeros(len(q)), -np.inf, np.zeros(len(q)), 0.0
    s = K @ q * scale
    top = s.max()
    w = np.exp(s - top)
    z = w.sum()
    return w @ V / z, top + np.log(z), w @ np.abs(V) / z, np.abs(V).max()


def fork(pool, tables, lens, src, dst, fresh, page):
    """pool [L, pages, ...], tables [B, W] and lens [B], changed in place"""
    B, W = tables.shape
    for s, d, f in zip(src, dst, fresh):
        if not (0 <= s < B and 0 <= d < B and s != d):
            continue
        n = min(max(int(lens[s]), 0), W * page)
        whole, rest = divmod(n, page)
        if rest and not 0 <= f < pool.shape[1]:
            continue
        tables[d] = -1
        tables[d, :whole] = tables[s, :whole]
        if rest and 0 <= tables[s, whole] < pool.shape[1]:
            pool[:, f] = pool[:, tables[s, whole]]
            tables[d, whole] = f
        lens[d] = n


def compact(pool, tables, lens, page):
    """pool changed in place; (the tables as they are then, the pages in use)"""
    B, W = tables.shape
    pages = pool.shape[1]
    named = [[int(p) for p in tables[b, :-(-min(max(int(lens[b]), 0), W * page) // page)]] for b in range(B)]
    live = sorted({p for row in named for p in row if 0 <= p < pages})
    used, alive = len(live), set(live)
    holes = [p for p in range(used) if p not in alive]
    goes = {p: p for p in live}
    goes.update(zip([p for p in live if p >= used], holes))
    for a, b in goes.items():
        if a != b:
            pool[:, b] = pool[:, a]
    out = np.full((B, W), -1, tables.dtype)
    for b, row in enumerate(named):
        for j, p in enumerate(row):
            out[b, j] = goes.get(p, -1)
    return out, used
