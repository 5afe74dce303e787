"""TEST INFRASTRUCTURE: a batch over one shared, bounded cache in 64 bits, written from the formulas: rotation by several
axes, attention over a shared prefix and rows' own keys, the weight keys received, eviction."""

from __future__ import annotations

import numpy as np


def norm_rope_axes(x, w, eps, cos, sin, pos, axes, centered=False):
    """x [T, heads, D], w [D] or None, cos / sin [positions, >= D / 2], pos [A, T], axes [D / 2] -> [T, heads, D]"""
    x = np.asarray(x, np.float64)
    half = x.shape[-1] // 2
    if w is not None:
        rms = np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        x = x / rms * (np.asarray(w, np.float64) + (1.0 if centered else 0.0))
    where = np.asarray(pos)[np.asarray(axes), :].T  # [T, D / 2]
    c = np.asarray(cos, np.float64)[where, np.arange(half)][:, None, :]
    s = np.asarray(sin, np.float64)[where, np.arange(half)][:, None, :]
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def attention(q, keys, values, scale):
    """q [G, D], keys / values [n, D] of one kv head -> (att [G, D], lse [G]); no keys: zeros and -inf"""
    q, keys, values = (np.asarray(a, np.float64) for a in (q, keys, values))
    if len(keys) == 0:
        return np.zeros_like(q), np.full(q.shape[0], -np.inf)
    s = q @ keys.T * scale
    top = s.max(-1, keepdims=True)
    e = np.exp(s - top)
    z = e.sum(-1, keepdims=True)
    return e @ values / z, (top + np.log(z))[:, 0]


def attn_shared(q, K, V, off, n, own, scale):
    """q [T, Hq, D], K / V [Hk, cap, D], own [(off, n)] a row (n < 0: padding) -> (att, lse, the largest sum of |weight value|)"""
    T, Hq, D = q.shape
    Hk = K.shape[0]
    G = Hq // Hk
    att, lse, spread = np.zeros((T, Hq, D)), np.full((T, Hq), -np.inf), np.zeros((T, Hq, D))
    for t, (o, m) in enumerate(own):
        if m < 0:
            continue
        at = np.r_[off:off + n, o:o + m]
        for g in range(Hk):
            h = slice(g * G, (g + 1) * G)
            att[t, h], lse[t, h] = attention(q[t, h], K[g, at], V[g, at], scale)
            spread[t, h] = attention(q[t, h], K[g, at], np.abs(V[g, at]), scale)[0]
    return att, lse, spread


def attn_mass(q, K, lse, seen, mass, scale, n):
    """q [T, Hq, D], K [Hk, cap, D], lse [T, Hq], seen [T], mass [Hk, >= n] or None -> [Hk, n]"""
    T, Hq, _ = q.shape
    Hk = K.shape[0]
    G = Hq // Hk
    out = np.zeros((Hk, n)) if mass is None else np.asarray(mass, np.float64)[:, :n].copy()
    for t in range(T):
        m = min(int(seen[t]), n)
        for h in range(Hq):
            if m > 0 and lse[t, h] != -np.inf:
                out[h // G, :m] += np.exp(np.asarray(q[t, h], np.float64) @ np.asarray(K[h // G, :m], np.float64).T * scale - lse[t, h])
    return out


def evict(mass, pos, n, budget, sinks=0, recent_from=0x7FFFFFFF):
    """mass / pos [heads, >= n] -> idx [heads, min(n, budget)]: the slot each kept slot's key comes from"""
    kept = min(n, budget)
    idx = np.empty((len(mass), kept), np.int64)
    for r in range(len(mass)):
        order = []
        for j in range(n):
            m = float(mass[r][j])
            m = -np.inf if np.isnan(m) else m
            if pos[r][j] < sinks or pos[r][j] >= recent_from:
                m = np.inf
            order.append((-m, j))
        stay = {j for _, j in sorted(order)[:kept]}
        late = iter(sorted(j for j in stay if j >= kept))
        idx[r] = [j if j in stay else next(late) for j in range(kept)]
    return idx
