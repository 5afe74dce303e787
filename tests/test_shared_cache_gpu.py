"""A batch over one shared, bounded cache, on the GPU against oracle/shared.py in 64 bits.

Bars, from the arithmetic. Inputs are bf16 and exact in f32 and f64 alike; u = 2^-24 is f32's rounding and
w = 2^-8 bf16's (eight significant bits: 1 + 2^-8 lies midway between two of them).
  rope    one rounding of the result, w |out|, and the f32 steps before it: at most 16 u (|y_i| + |y_j|) with the norm's
  scores  D products added in f32: e = D u scale sum |q_i k_i| at worst, the same relative error in exp(s); exp2's argument
          in f32 adds u log2(e) |s| and the exponential 2 u
  shared  a weight rounded to bf16 for the product: w times the weighted mean of |v|; the sums and the fold: (e + 64 u) of
          the same; the output's rounding: w |att|. lse: e and 8 u (1 + |lse|)
  mass    sum of the weights times (e + 16 u (1 + max |s|)), and (T + 8) u of the total
  evict   equal
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from btb_amd.decode import StackConfig, recording, rope_axes, rope_tables
from btb_amd.native import HipError
from oracle import shared

from .helpers import gen

pytestmark = pytest.mark.gpu

U, W = 2.0**-24, 2.0**-8
NAN, INF = float("nan"), float("inf")


def _f64(t):
    return t.detach().double().cpu().numpy()


def _cache(g, Hk, cap, D, slot_major=False):
    t = torch.randn(Hk, cap, D, generator=g).to(torch.bfloat16)
    return t.transpose(0, 1).contiguous().cuda().transpose(0, 1) if slot_major else t.cuda()


# ---- norm and rotation ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("T,Hq,Hk,D,A,table,norm,centered,slot_major", [
    (1, 32, 8, 128, 1, "bf16", True, False, False),
    (1, 1, 1, 64, 4, "f32", True, True, True),
    (7, 14, 2, 64, 3, "f32", True, False, True),
    (33, 5, 5, 128, 3, "bf16", False, False, False),
    (130, 9, 3, 256, 2, "f32", True, True, False),
    (301, 16, 4, 128, 3, "bf16", True, False, True),
])
def test_rope_axes(card, T, Hq, Hk, D, A, table, norm, centered, slot_major):
    g = gen(5000 + T + D)
    positions, cap = 500, T + 9
    cos, sin = rope_tables(StackConfig(head_dim=D), positions, "cuda")
    if table == "f32":
        ang = torch.rand(positions, D // 2, generator=g) * 6.0
        cos, sin = ang.cos().cuda(), ang.sin().cuda()
    pos = torch.randint(0, positions, (A, T), generator=g, dtype=torch.int32).cuda()
    runs = [D // 2 // A] * (A - 1)
    axes = rope_axes(runs + [D // 2 - sum(runs)], "cuda", interleaved=T % 2 == 1)
    slots = torch.randperm(cap, generator=g)[:T].to(torch.int32)
    if T > 4:
        slots[1], slots[3] = -1, cap  # outside the cache: not written
    qkv = (torch.randn(T, Hq + 2 * Hk, D, generator=g) * 3.0).to(torch.bfloat16).cuda()
    wq, wk = ((1.0 + 0.3 * torch.randn(D, generator=g)).to(torch.bfloat16).cuda() if norm else None for _ in range(2))
    K, V = _cache(g, Hk, cap, D, slot_major), _cache(g, Hk, cap, D, slot_major)
    K0, V0 = K.clone(), V.clone()
    q = torch.full((T, Hq * D), NAN, dtype=torch.bfloat16, device="cuda")
    card.norm_rope_axes(qkv.view(T, -1), wq, wk, 1e-6, cos, sin, pos, axes, slots.cuda(), K, V, q, Hq, Hk, D, centered=centered)
    torch.cuda.synchronize()
    x, c, s = _f64(qkv), _f64(cos)[:, :D // 2], _f64(sin)[:, :D // 2]
    args = (1e-6, c, s, pos.cpu().numpy(), axes.cpu().numpy(), centered)

    def held(got, heads, w):
        want = shared.norm_rope_axes(x[:, heads], None if w is None else _f64(w), *args)
        size = np.abs(shared.norm_rope_axes(x[:, heads], None if w is None else _f64(w), 1e-6, np.ones_like(c), np.zeros_like(s),
                                            *args[3:]))
        pair = size + np.roll(size, D // 2, -1)
        assert (np.abs(got - want) <= W * np.abs(want) * (1 + W) + 16 * U * pair).all()

    held(_f64(q).reshape(T, Hq, D), slice(0, Hq), wq)
    on = ((slots >= 0) & (slots < cap)).numpy()
    at = slots.long()[torch.from_numpy(on)]
    got = np.full((T, Hk, D), np.nan)
    got[on] = _f64(K[:, at.cuda()]).transpose(1, 0, 2)
    want = shared.norm_rope_axes(x[:, Hq:Hq + Hk], None if wk is None else _f64(wk), *args)
    got[~on] = want[~on]
    held(got, slice(Hq, Hq + Hk), wk)
    assert torch.equal(V[:, at.cuda()].transpose(0, 1), qkv[torch.from_numpy(on).cuda(), Hq + Hk:])
    rest = torch.ones(cap, dtype=torch.bool)
    rest[at] = False
    assert torch.equal(K[:, rest.cuda()], K0[:, rest.cuda()]) and torch.equal(V[:, rest.cuda()], V0[:, rest.cuda()])


def test_rope_positions_outside_the_tables_stay_inside(card):
    """a place before the first or past the last row of the tables is that row; an axis past the last is the last"""
    g = gen(5100)
    T, D = 3, 128
    cos, sin = rope_tables(StackConfig(), 16, "cuda")
    qkv = torch.randn(T, 3 * D, generator=g).to(torch.bfloat16).cuda()
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    outs = []
    for pos, axes in (([[-5, 99, 7]], [9] * 64), ([[0, 15, 7]], [0] * 64)):
        K, V, q = torch.zeros(1, T, D, dtype=torch.bfloat16, device="cuda"), _cache(g, 1, T, D), torch.empty(
            T, D, dtype=torch.bfloat16, device="cuda")
        card.norm_rope_axes(qkv, None, None, 1e-6, cos, sin, torch.tensor(pos, dtype=torch.int32, device="cuda"),
                            torch.tensor(axes, dtype=torch.uint8, device="cuda"), slots, K, V, q, 1, 1, D)
        torch.cuda.synchronize()
        outs.append((q, K))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


# ---- attention ------------------------------------------------------------------------------------------------------


def _score_error(q, K, scale):
    """the largest e of the bars above, over all rows and keys"""
    top = np.abs(q).max(axis=tuple(range(q.ndim - 1))) @ np.nan_to_num(np.abs(K), nan=0.0, posinf=0.0).reshape(-1, K.shape[-1]).max(0)
    return K.shape[-1] * U * scale * top


def _shared_case(g, T, Hq, Hk, D, P, lens, slot_major=False, std=1.5):
    """prefix and rows' own stretches with unused slots, full of NaN, between them"""
    offs, at = [], 2
    for t, n in enumerate(lens):
        if t == len(lens) // 2:
            off, at = at, at + P + 3
        offs.append(at)
        at += max(n, 0) + 1
    K, V = _cache(g, Hk, at, D, slot_major), _cache(g, Hk, at, D, slot_major)
    used = torch.zeros(at, dtype=torch.bool)
    used[off:off + P] = True
    for o, n in zip(offs, lens):
        used[o:o + max(n, 0)] = True
    K[:, ~used.cuda()], V[:, ~used.cuda()] = NAN, NAN
    q = (torch.randn(T, Hq, D, generator=g) * std).to(torch.bfloat16).cuda()
    return q, K, V, off, offs


def _run_shared(card, q, K, V, off, P, own, scale, prefix_cap, own_cap, **kw):
    T, Hq, D = q.shape
    Hk = K.shape[0]
    lay = card.shared_layout(off, P, own)
    att = torch.full((T, Hq * D), 9.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((T, Hq), 9.0, dtype=torch.float32, device="cuda")
    scratch = torch.full_like(card.attn_shared_scratch(T, Hq, Hk, D, prefix_cap, own_cap), NAN)
    card.attn_shared(q.view(T, -1), K, V, att, lay, Hq, Hk, D, scale, prefix_cap, own_cap, scratch, lse=lse)
    torch.cuda.synchronize()
    return att.view(T, Hq, D), lse


def _hold_shared(att, lse, q, K, V, off, P, own, scale):
    qd, Kd, Vd = _f64(q), _f64(K), _f64(V)
    want, z, spread = shared.attn_shared(qd, Kd, Vd, off, P, own, scale)
    e = _score_error(qd, Kd, scale)
    live = np.array([n >= 0 for _, n in own])
    a, l = _f64(att), _f64(lse)
    assert (a[~live] == 9.0).all() and (l[~live] == 9.0).all()
    bar = (W + e + 64 * U) * spread + W * np.abs(want)
    assert (np.abs(a - want)[live] <= bar[live]).all(), float((np.abs(a - want) / np.maximum(bar, 1e-30))[live].max())
    empty = z == -np.inf
    assert (l[empty & live[:, None]] == -np.inf).all()
    some = ~empty & live[:, None]
    assert (np.abs(l - z)[some] <= (e + 8 * U * (1 + np.abs(z)))[some]).all()


SHARED = [  # T, Hq, Hk, D, P, own lengths (repeated), slot-major
    (1, 1, 1, 64, 1, [0], False),
    (1, 8, 8, 128, 0, [1], False),
    (1, 32, 8, 128, 31, [33], True),
    (2, 6, 2, 64, 32, [0, 129], False),
    (3, 5, 1, 128, 33, [1, 0, 40], False),
    (4, 32, 8, 128, 700, [5, 6, 7, 8], False),
    (5, 16, 1, 64, 129, [128, -1, 0, 1, 300], True),
    (7, 64, 2, 128, 500, [3], False),
    (9, 12, 3, 64, 1000, [17, 0, 65], False),
    (17, 14, 2, 128, 2049, [100, 1], True),
    (33, 32, 8, 128, 257, [0], False),
    (40, 28, 4, 64, 4100, [31, 32, 33, -1], False),
    (65, 16, 8, 128, 0, [64, 2, 0], False),
    (130, 4, 1, 128, 3000, [0, 5], False),
]


@pytest.mark.parametrize("T,Hq,Hk,D,P,lens,slot_major", SHARED)
def test_attn_shared(card, T, Hq, Hk, D, P, lens, slot_major):
    g = gen(5200 + T + P)
    lens = (lens * T)[:T]
    q, K, V, off, offs = _shared_case(g, T, Hq, Hk, D, P, lens, slot_major)
    own, scale = list(zip(offs, lens)), 1.0 / math.sqrt(D)
    att, lse = _run_shared(card, q, K, V, off, P, own, scale, P, max(max(lens), 0))
    _hold_shared(att, lse, q, K, V, off, P, own, scale)
    # launches sized for far more keys than there are: the same answer to the same bars
    att2, lse2 = _run_shared(card, q, K, V, off, P, own, scale, K.shape[1], K.shape[1])
    _hold_shared(att2, lse2, q, K, V, off, P, own, scale)


@pytest.mark.parametrize("D,T", [(64, 3), (128, 50)])
def test_attn_shared_bounds_past_the_cache(card, D, T):
    """rows of unlike lengths in a cache that holds no more than they need: the longest may be more than all of its rows"""
    g = gen(5215 + T)
    q, K, V, off, offs = _shared_case(g, T, 8, 2, D, 4, [2] * T)
    own = [(o, 2) for o in offs]
    for prefix_cap, own_cap in ((4, 4 * K.shape[1]), (4 * K.shape[1], 2), (1 << 20, 1 << 20)):
        att, lse = _run_shared(card, q, K, V, off, 4, own, 0.1, prefix_cap, own_cap)
        _hold_shared(att, lse, q, K, V, off, 4, own, 0.1)
    # lengths that run past the cache are cut at its last row
    K, V = K.nan_to_num(nan=0.5), V.nan_to_num(nan=0.5)
    lay = card.shared_layout(off, 1 << 20, [(o, -1) for o in offs[1:]] + [(offs[0], 2)])
    att, lse = torch.zeros(T, 8 * D, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, 8, device="cuda")
    card.attn_shared(q.view(T, -1), K, V, att, lay, 8, 2, D, 0.1, 1 << 20, 1 << 20, card.attn_shared_scratch(T, 8, 2, D, 1 << 20, 1 << 20), lse=lse)
    torch.cuda.synchronize()
    _hold_shared(att.view(T, 8, D)[-1:], lse[-1:], q[-1:], K, V, off, K.shape[1] - off, [(offs[0], 2)], 0.1)


def test_attn_shared_scores_far_apart(card):
    """maxima that grow along the keys, by hundreds, and keys whose weight underflows"""
    g = gen(5300)
    T, Hq, Hk, D, P = 6, 8, 2, 128, 900
    q, K, V, off, offs = _shared_case(g, T, Hq, Hk, D, P, [40] * T, std=1.0)
    ramp = torch.linspace(0.0, 12.0, P).to(torch.bfloat16).cuda()[None, :, None]
    K[:, off:off + P] = (ramp * torch.sign(q[0, :1].mean(0)).to(torch.bfloat16)[None, None, :] + K[:, off:off + P]).to(torch.bfloat16)
    own, scale = [(o, 40) for o in offs], 0.5
    att, lse = _run_shared(card, q, K, V, off, P, own, scale, P, 40)
    _hold_shared(att, lse, q, K, V, off, P, own, scale)


def test_attn_shared_values_that_are_not_finite(card):
    """an infinite value in a row's own keys reaches that row alone; a NaN in q its own head alone; a stretch cut at the
    cache's end and one with a negative start are read no further"""
    g = gen(5310)
    T, Hq, Hk, D, P = 4, 4, 2, 64, 100
    q, K, V, off, offs = _shared_case(g, T, Hq, Hk, D, P, [10] * T)
    own, scale = [(o, 10) for o in offs], 0.125
    clean, z = _run_shared(card, q, K, V, off, P, own, scale, P, 10)
    V[0, offs[1] + 9, 3] = INF
    q[2, 3, 0] = NAN
    att, lse = _run_shared(card, q, K, V, off, P, own, scale, P, 10)
    assert torch.equal(att[0], clean[0]) and torch.equal(att[3], clean[3]) and torch.equal(lse[0], z[0])
    assert bool((att[1, :2, 3] == INF).all())
    keep = torch.ones(D, dtype=torch.bool, device="cuda")
    keep[3] = False
    assert torch.equal(att[1, :, keep], clean[1, :, keep]) and torch.equal(att[1, 2:], clean[1, 2:])
    assert torch.equal(att[2, :3], clean[2, :3]) and bool(att[2, 3].isnan().all()) and bool(lse[2, 3].isnan())
    # past the end, and from before the start: no keys of theirs
    cap = K.shape[1]
    att, lse = _run_shared(card, q[:2], K, V, off, P, [(cap + 7, 5), (-3, 5)], scale, P, 10)
    base, zb = _run_shared(card, q[:2], K, V, off, P, [(0, 0), (0, 0)], scale, P, 10)
    assert torch.equal(att, base) and torch.equal(lse, zb)


def test_attn_shared_far_into_a_large_cache(card):
    """slots whose values lie past 2^31 values and 2^32 bytes from the cache's start"""
    g = gen(5320)
    T, Hq, Hk, D, P = 3, 8, 2, 128, 300
    cap = (1 << 24) + 2048
    K = torch.empty(Hk, cap, D, dtype=torch.bfloat16, device="cuda")
    V = torch.empty(Hk, cap, D, dtype=torch.bfloat16, device="cuda")
    off, first = (1 << 24) - 100, (1 << 24) + 500
    for t in (K, V):
        t[:, off:] = torch.randn(Hk, cap - off, D, generator=g).to(torch.bfloat16).cuda()
    q = torch.randn(T, Hq, D, generator=g).to(torch.bfloat16).cuda()
    own = [(first + 200 * t, 50 + t) for t in range(T)]
    lay = card.shared_layout(off, P, own)
    att, lse = torch.empty(T, Hq * D, dtype=torch.bfloat16, device="cuda"), torch.empty(T, Hq, device="cuda")
    card.attn_shared(q.view(T, -1), K, V, att, lay, Hq, Hk, D, 0.1, P, 60, card.attn_shared_scratch(T, Hq, Hk, D, P, 60), lse=lse)
    torch.cuda.synchronize()
    back = [(o - off, n) for o, n in own]
    _hold_shared(att.view(T, Hq, D), lse, q, K[:, off:], V[:, off:], 0, P, back, 0.1)


def test_attn_shared_recorded_while_the_rows_grow(card):
    """one recorded launch, replayed as the layout on the device moves on: every replay is the eager call's bits; on a stream
    of its own"""
    g = gen(5330)
    T, Hq, Hk, D, P = 5, 16, 4, 128, 600
    q, K, V, off, offs = _shared_case(g, T, Hq, Hk, D, P, [200] * T)
    lay = card.shared_layout(off, P, [(o, 0) for o in offs])
    scratch = card.attn_shared_scratch(T, Hq, Hk, D, P, 200)
    att, lse = torch.zeros(T, Hq * D, dtype=torch.bfloat16, device="cuda"), torch.zeros(T, Hq, device="cuda")
    call = lambda: card.attn_shared(q.view(T, -1), K, V, att, lay, Hq, Hk, D, 0.09, P, 200, scratch, lse=lse)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with recording(graph):
        call()
    for n in (0, 1, 127, 128, 129, 200):
        lay[3::2] = n
        att.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = att.clone(), lse.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        assert torch.equal(att, got[0]) and torch.equal(lse, got[1])
        _hold_shared(att.view(T, Hq, D), lse, q, K, V, off, P, [(o, n) for o in offs], 0.09)


# ---- the weight keys received ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("T,Hq,Hk,D,n,chain,slot_major", [
    (1, 1, 1, 64, 1, True, False),
    (1, 32, 8, 128, 515, True, False),
    (3, 6, 2, 64, 33, False, True),
    (11, 5, 1, 128, 128, True, False),
    (16, 64, 2, 64, 129, True, False),
    (40, 12, 3, 128, 700, False, True),
    (65, 8, 8, 128, 64, True, False),
    (200, 4, 2, 64, 1100, True, False),
    (150, 32, 8, 128, 90, True, False),
    (500, 12, 4, 128, 31, False, False),
])
def test_attn_mass(card, T, Hq, Hk, D, n, chain, slot_major):
    g = gen(5400 + T + n)
    cap = n + 6
    K = _cache(g, Hk, cap, D, slot_major)
    K[:, n:] = NAN
    q = (torch.randn(T, Hq, D, generator=g) * 1.5).to(torch.bfloat16).cuda()
    scale = 1.0 / math.sqrt(D)
    seen = [min(n, max(0, n - T + 1 + t)) for t in range(T)] if chain else [(37 * t) % (n + 2) for t in range(T)]
    qd, Kd = _f64(q), _f64(K)
    s = np.stack([qd[:, h] @ Kd[h // (Hq // Hk), :n].T * scale for h in range(Hq)], 1)
    lse = np.stack([[np.log(np.exp(s[t, h, :seen[t]]).sum()) if seen[t] else -np.inf for h in range(Hq)] for t in range(T)])
    lse32 = torch.from_numpy(lse.astype(np.float32)).cuda()
    mass = torch.rand(Hk, cap, generator=g).cuda()
    out = torch.full((Hk, cap), 7.0, device="cuda")
    seen_t = torch.tensor(seen, dtype=torch.int32, device="cuda")
    card.attn_mass(q.view(T, -1), K, lse32, seen_t, mass, Hq, Hk, D, scale, n, out=out)
    alone = card.attn_mass(q.view(T, -1), K, lse32, seen_t, None, Hq, Hk, D, scale, n)
    kept = mass.clone()
    card.attn_mass(q.view(T, -1), K, lse32, seen_t, mass, Hq, Hk, D, scale, n)
    torch.cuda.synchronize()
    want = shared.attn_mass(qd, Kd, _f64(lse32), seen, None, scale, n)
    e = _score_error(qd, Kd[:, :n], scale) + 16 * U * (1 + np.abs(s).max())
    assert (np.abs(_f64(alone) - want) <= want * (e + (T + 8) * U) + 1e-37).all()
    total = want + _f64(kept[:, :n])
    assert (np.abs(_f64(out[:, :n]) - total) <= want * e + (T + 8) * U * total + 1e-37).all()
    assert torch.equal(out[:, :n], mass[:, :n]) and bool((out[:, n:] == 7.0).all()) and torch.equal(mass[:, n:], kept[:, n:])


@pytest.mark.parametrize("T,Hq,Hk,D,n", [(5, 3, 3, 128, 70), (9, 8, 2, 64, 300), (90, 6, 6, 128, 400), (70, 12, 3, 64, 257)])
def test_attn_mass_log_sums_of_any_strides(card, T, Hq, Hk, D, n):
    """the log-sums head by head, in a wider array, or one for all rows: the bits of the dense ones"""
    g = gen(5440 + T)
    q, K = torch.randn(T, Hq * D, generator=g).to(torch.bfloat16).cuda(), _cache(g, Hk, n, D, False)
    seen = torch.randint(0, n + 1, (T,), generator=g).to(torch.int32).cuda()
    lse = torch.rand(T, Hq, generator=g).cuda() * 4
    wide = torch.full((T, 2 * Hq + 3), NAN, device="cuda")
    wide[:, 1:2 * Hq:2] = lse
    call = lambda z: card.attn_mass(q, K, z, seen, None, Hq, Hk, D, 0.1, n)
    want = call(lse)
    for z in (lse.t().contiguous().t(), wide[:, 1:2 * Hq:2]):
        assert z.shape == (T, Hq) and (T == 1 or not z.is_contiguous()) and torch.equal(call(z), want)
    assert torch.equal(call(lse[:1].expand(T, Hq)), call(lse[:1].repeat(T, 1)))


def test_attn_mass_takes_attentions_own_log_sums(card):
    """after attn_shared, the weights over prefix and own keys come to one a head"""
    g = gen(5450)
    T, Hq, Hk, D, P = 9, 24, 3, 128, 400
    q, K, V, off, offs = _shared_case(g, T, Hq, Hk, D, P, [0] * T)
    _, lse = _run_shared(card, q, K, V, off, P, [(o, 0) for o in offs], 0.09, P, 1)
    seen = torch.full((T,), P, dtype=torch.int32, device="cuda")
    out = card.attn_mass(q.view(T, -1), K[:, off:off + P], lse, seen, None, Hq, Hk, D, 0.09, P)
    assert torch.allclose(out.sum(-1), torch.full((Hk,), T * Hq / Hk, device="cuda"), rtol=1e-4)


# ---- eviction -------------------------------------------------------------------------------------------------------


def _evict_case(g, L, Hk, n, cap, kind):
    mass = torch.exp(2.0 * torch.randn(L, Hk, cap, generator=g))
    if kind == "ties":
        mass = torch.floor(mass * 2.0)
    elif kind == "equal":
        mass = torch.zeros(L, Hk, cap)
    elif kind == "odd":
        pick = torch.randint(0, 7, (L, Hk, cap), generator=g)
        mass = torch.tensor([0.0, -0.0, NAN, INF, -INF, 1.0, -2.0])[pick]
    pos = torch.stack([torch.randperm(cap, generator=g) for _ in range(L * Hk)]).view(L, Hk, cap).to(torch.int32)
    return mass.cuda(), pos.cuda()


EVICT = [  # L, Hk, D, n, budget, sinks, recent_from, kind
    (1, 1, 64, 1, 1, 0, 1 << 30, "free"),
    (1, 2, 128, 7, 3, 1, 6, "free"),
    (2, 3, 64, 100, 1, 0, 1 << 30, "ties"),
    (1, 8, 128, 700, 512, 4, 636, "free"),
    (3, 2, 128, 1024, 1023, 0, 1 << 30, "ties"),
    (2, 2, 64, 1025, 1024, 4, 1000, "equal"),
    (1, 4, 128, 3000, 1000, 0, 0, "free"),
    (1, 4, 128, 5001, 2049, 5, 4000, "odd"),
    (2, 1, 64, 5000, 5000, 0, 1 << 30, "free"),
    (1, 2, 128, 900, 1200, 0, 1 << 30, "ties"),
    (1, 1, 128, 40000, 9000, 4, 39000, "ties"),
    (1, 2, 64, 70001, 33000, 0, 1 << 30, "odd"),
    (36, 8, 64, 300, 256, 2, 290, "ties"),
]


@pytest.mark.parametrize("L,Hk,D,n,budget,sinks,recent,kind", EVICT)
def test_evict(card, L, Hk, D, n, budget, sinks, recent, kind):
    g = gen(5500 + n)
    cap, kept = n + 5, min(n, budget)
    mass, pos = _evict_case(g, L, Hk, n, cap, kind)
    kv = torch.randn(L, 2, Hk, cap, D, generator=g).to(torch.bfloat16).cuda()  # as the decode step lays its caches out
    K, V = kv[:, 0], kv[:, 1]
    K_out = torch.full((L, kept + 2, Hk, D), 3.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2)  # slot-major
    V_out, M_out, P_out = K_out.clone(), torch.full((L, Hk, kept + 1), 3.0, device="cuda"), torch.full(
        (L, Hk, kept + 3), 3, dtype=torch.int32, device="cuda")
    V_out = torch.full((L, kept + 2, Hk, D), 3.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    idx = torch.full((L, Hk, kept), -1, dtype=torch.int32, device="cuda")
    got = card.kv_evict(mass, pos, K, V, n, budget, K_out, V_out, M_out, P_out, idx, sinks=sinks, recent_from=recent)
    torch.cuda.synchronize()
    want = shared.evict(mass.cpu().view(-1, cap).numpy(), pos.cpu().view(-1, cap).numpy(), n, budget, sinks, recent)
    assert got == kept and np.array_equal(idx.cpu().view(L * Hk, kept).numpy(), want)
    rows = torch.from_numpy(want).view(L, Hk, kept).cuda()
    wide = rows[..., None].expand(-1, -1, -1, D)
    same = lambda a, b: torch.equal(a.contiguous().view(torch.int32 if a.element_size() == 4 else torch.int16),
                                    b.contiguous().view(torch.int32 if b.element_size() == 4 else torch.int16))
    assert same(K_out[:, :, :kept], K.gather(2, wide)) and same(V_out[:, :, :kept], V.gather(2, wide))
    assert same(M_out[..., :kept], mass.gather(2, rows)) and same(P_out[..., :kept], pos.gather(2, rows))
    assert bool((K_out[:, :, kept:] == 3.0).all()) and bool((M_out[..., kept:] == 3.0).all())
    # in place: the same keys in the same slots, everything past them as it was
    before = kv.clone(), mass.clone(), pos.clone()
    idx2 = torch.full_like(idx, -1)
    card.kv_evict(mass, pos, K, V, n, budget, K, V, mass, pos, idx2, sinks=sinks, recent_from=recent)
    torch.cuda.synchronize()
    assert torch.equal(idx, idx2)
    assert same(K[:, :, :kept], K_out[:, :, :kept]) and same(V[:, :, :kept], V_out[:, :, :kept])
    assert same(mass[..., :kept], M_out[..., :kept]) and same(pos[..., :kept], P_out[..., :kept])
    assert same(kv[:, :, :, kept:], before[0][:, :, :, kept:]) and same(mass[..., kept:], before[1][..., kept:])
    assert same(pos[..., kept:], before[2][..., kept:])


def test_attention_over_a_cut_cache_is_attention_over_the_kept_keys(card):
    g = gen(5600)
    Hq, Hk, D, n, budget = 8, 2, 128, 900, 300
    K, V = _cache(g, Hk, n, D), _cache(g, Hk, n, D)
    mass, pos = _evict_case(g, 1, Hk, n, n, "free")
    K0, V0 = _f64(K), _f64(V)
    idx = torch.empty(1, Hk, budget, dtype=torch.int32, device="cuda")
    card.kv_evict(mass[0], pos[0], K, V, n, budget, K, V, mass[0], pos[0], idx)
    q = torch.randn(3, Hq, D, generator=g).to(torch.bfloat16).cuda()
    att, lse = _run_shared(card, q, K, V, 0, budget, [(0, 0)] * 3, 0.09, budget, 1)
    at = idx[0].cpu().numpy()
    kept = np.stack([K0[h, np.sort(at[h])] for h in range(Hk)]), np.stack([V0[h, np.sort(at[h])] for h in range(Hk)])
    _hold_shared(att, lse, q, torch.from_numpy(kept[0]), torch.from_numpy(kept[1]), 0, budget, [(0, 0)] * 3, 0.09)


# ---- refusals -------------------------------------------------------------------------------------------------------


def test_refusals(card):
    Hq, Hk, D, T, cap = 8, 2, 128, 2, 64
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")
    i32, f32 = torch.int32, torch.float32
    K, V, q, att = z(Hk, cap, D), z(Hk, cap, D), z(T, Hq * D), z(T, Hq * D)
    qkv, cos = z(T, (Hq + 2 * Hk) * D), z(16, D)
    pos, axes, slots = z(3, T, dt=i32), z(D // 2, dt=torch.uint8), torch.arange(T, dtype=i32, device="cuda")
    rope = lambda **k: card.norm_rope_axes(*[k.get(n, v) for n, v in dict(
        qkv=qkv, wq=None, wk=None, eps=1e-6, cos=cos, sin=cos, pos=pos, axes=axes, slots=slots, K=K, V=V, q=q, Hq=Hq, Hk=Hk, D=D).items()])
    rope()
    for bad in (dict(cos=z(16, D).half(), sin=z(16, D).half()), dict(cos=z(16, D + 8), sin=z(16, D + 8)), dict(sin=z(8, D)), dict(axes=z(D, dt=torch.uint8)),
                dict(pos=z(3, T + 1, dt=i32)), dict(slots=slots[:1].contiguous()), dict(wq=z(D + 1)), dict(K=z(Hk, cap, D).float()),
                dict(K=z(Hk + 1, cap, D)), dict(q=z(T, Hq * D + 8)), dict(pos=pos.float()), dict(V=z(Hk, cap + 1, D))):
        with pytest.raises(ValueError):
            rope(**bad)
    with pytest.raises(HipError):  # keys that do not start on 16 bytes
        off = z(Hk * cap * D + 1)[1:].view(Hk, cap, D)
        rope(K=off, V=off)
    lay, scratch = card.shared_layout(0, 10, [(10, 1), (11, 1)]), card.attn_shared_scratch(T, Hq, Hk, D, 20, 4)
    shared_ = lambda **k: card.attn_shared(*[k.get(n, v) for n, v in dict(
        q=q, K=K, V=V, att=att, lay=lay, Hq=Hq, Hk=Hk, D=D, scale=0.1, prefix_cap=20, own_cap=4, scratch=scratch, lse=None).items()])
    shared_()
    for bad in (dict(own_cap=-1), dict(scratch=scratch[:-1]), dict(lay=lay[:5].contiguous()),
                dict(lse=z(T, Hq + 1, dt=f32)), dict(q=q.float()), dict(K=K.transpose(1, 2)), dict(att=z(T, D))):
        with pytest.raises(ValueError):
            shared_(**bad)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=INF), dict(scale=NAN)):
        with pytest.raises(HipError):
            shared_(**bad)
    with pytest.raises(ValueError):
        card.attn_shared_scratch(T, 66, 2, D, 20, 4)  # 33 query heads a kv head
    with pytest.raises(ValueError):
        card.attn_shared_scratch(T, Hq, Hk, 256, 20, 4)
    lse, seen = z(T, Hq, dt=f32), z(T, dt=i32)
    for bad in (dict(n=0), dict(n=cap + 1), dict(lse=z(T, 1, dt=f32)), dict(mass=z(Hk, 9, dt=f32)), dict(mass=z(Hk + 1, 10, dt=f32))):
        k = dict(lse=lse, mass=None, n=10) | bad
        with pytest.raises(ValueError):
            card.attn_mass(q, K, k["lse"], seen, k["mass"], Hq, Hk, D, 0.1, k["n"])
    with pytest.raises(HipError):
        card.attn_mass(q, K, lse, seen, None, Hq, Hk, D, 0.0, 10)
    mass, p32, idx = z(Hk, cap, dt=f32), z(Hk, cap, dt=i32), z(Hk, 8, dt=i32)
    ev = lambda **k: card.kv_evict(*[k.get(n, v) for n, v in dict(
        mass=mass, pos=p32, K=K, V=V, n=16, budget=8, K_out=K, V_out=V, mass_out=mass, pos_out=p32, idx=idx).items()])
    assert ev() == 8
    for bad in (dict(n=cap + 1), dict(n=0), dict(budget=0), dict(idx=z(Hk, 9, dt=i32)), dict(mass=mass.half()), dict(K_out=z(Hk, 7, D), V_out=z(Hk, 7, D)),
                dict(pos=p32.float()), dict(V=z(Hk, cap + 1, D))):
        with pytest.raises(ValueError):
            ev(**bad)
    with pytest.raises(HipError):  # some in place and some not
        ev(mass_out=z(Hk, cap, dt=f32))
    lib, p = card.lib, lambda t: None if t is None else ctypes.c_void_p(t.data_ptr())
    assert lib.btb_hip_attn_shared(None, p(K), p(V), p(att), None, p(lay), T, Hq, Hk, D, cap, 1, 1, 0.1, 20, 4, p(scratch), None) == -1
    assert lib.btb_hip_attn_shared(p(q), p(K), p(V), p(att), None, p(lay), T, 7, 2, D, cap, 8, 8, 0.1, 20, 4, p(scratch), None) == -6
    assert lib.btb_hip_attn_mass(p(q), p(K), p(lse), None, None, p(lse), T, Hq, Hk, D, 10, 8, 8, 0, 0, Hq, 1, 0.1, None, None) == -1
    assert lib.btb_hip_kv_evict(p(mass), 1, None, 1, p(K), p(V), 0, 8, 8, 1, Hk, D, 16, 8, 0, 0, p(K), p(V), 0, 8, 8, p(mass), 1, p(p32), 1,
                                p(idx), None, None) == -1
    assert lib.btb_hip_norm_rope_axes(p(qkv), None, None, 1e-6, p(cos), p(cos), 0, 16, D, p(pos), 3, p(axes), None, p(K), p(V), p(q), T, Hq,
                                      Hk, D, cap, 8, 8, 0, None) == -1
    torch.cuda.synchronize()
