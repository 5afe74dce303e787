"""The operators over one shared cache on the paths that long passes and full caches take: loops that go round more than once, buffers
written again, tables refilled, the wide forms of the kernels. Small tests seldom get there, so each test says by which numbers
of the launch - worked out from the workspaces' sizes and the chip's compute units - its sizes do. Against oracle/shared.py in
64 bits, with the bars of test_shared_cache_gpu.py and, in the 2-norm (u = 2^-24):
  att, lse  as in test_shared_cache_bits_gpu.py
  mass      weights apart by u scale |q| |k| (a score's partial sums wander, so that their roundings come to less than one of
            its largest possible value), 2 u (1 + |score| + |log-sum|) for the exponent, and sqrt(pairs) u for their sum"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from btb_amd.decode import StackConfig, rope_axes, rope_tables
from btb_amd.native import HipError
from oracle import shared

from . import test_shared_cache_gpu as base
from .helpers import gen
from .test_guard_gpu import Fenced, fin
from .test_shared_cache_bits_gpu import _norm, _score_rms
from .test_shared_cache_gpu import U, _f64

pytestmark = pytest.mark.gpu


def _cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


# ---- rotation: several groups of heads a wave -------------------------------------------------------------------------


@pytest.mark.parametrize("T,Hq,Hk,D,A,table,norm,centered,slot_major", [
    (1500, 32, 8, 128, 3, "bf16", True, False, False),
    (2100, 40, 8, 128, 2, "f32", False, False, True),
    (2050, 64, 4, 64, 3, "f32", True, True, False),
    (1101, 9, 3, 256, 2, "bf16", True, False, True),
])
def test_rope_waves_with_several_groups_of_heads(card, T, Hq, Hk, D, A, table, norm, centered, slot_major):
    groups = -(-(Hq + 2 * Hk) // (1024 // D))
    assert min(groups, -(-8 * _cus() // T)) < groups  # waves a row
    base.test_rope_axes(card, T, Hq, Hk, D, A, table, norm, centered, slot_major)


# ---- attention: several stages a workgroup ----------------------------------------------------------------------------


def _spans(card, T, Hq, Hk, D, prefix_cap, own_cap):
    """(spans of the prefix, spans of a row's own keys): a (row, head) has D + 2 floats of scratch a span"""
    states = lambda p, o: card.lib.btb_hip_attn_shared_floats(T, Hq, Hk, D, p, o) // (D + 2) // (T * Hq)
    own = states(0, own_cap) if own_cap else 0
    return states(prefix_cap, own_cap) - own, own


def _stages(n, spans):
    return -(-(-(-n // spans)) // 128)


def _hold(att, lse, q, K, V, off, P, own, scale):
    base._hold_shared(att, lse, q, K, V, off, P, own, scale)
    qd, Kd, Vd = _f64(q), _f64(K), _f64(V)
    want, z, spread = shared.attn_shared(qd, Kd, Vd, off, P, own, scale)
    e = _score_rms(qd, Kd, scale)
    rounding = _norm(torch.from_numpy(want).to(torch.bfloat16).double().numpy() - want)
    assert _norm(_f64(att) - want) <= 1.02 * rounding + (2.0**-15 + e) * _norm(spread)
    assert _norm(_f64(lse) - z) <= (e + 4 * U * (1 + np.abs(z).max())) * math.sqrt(z.size)


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,stages,own", [
    (2, 32, 16, 128, 4, 0),     # up to 32 pairs a kv head: a wave's own tiles
    (4, 16, 16, 64, 3, 0),
    (12, 64, 16, 128, 5, 0),    # up to 64
    (9, 80, 16, 64, 6, 0),
    (30, 48, 8, 128, 3, 0),     # more
    (20, 64, 8, 64, 5, 0),
    (16, 32, 16, 128, 0, 450),  # a row's own keys
    (32, 16, 8, 64, 0, 700),
    (16, 64, 16, 128, 3, 300),  # both
    (26, 80, 10, 64, 3, 261),
])
def test_attn_shared_several_stages_a_workgroup(card, T, Hq, Hk, D, stages, own, rising):
    """rising: scores a stage above the last one's by 9 log 2, so that every state moves to a new maximum at every stage"""
    g = gen(5800 + T + D + stages)
    P = 0
    if stages:
        P = stages * 128 * _spans(card, T, Hq, Hk, D, 1 << 20, own)[0] - 77
    spans, own_spans = _spans(card, T, Hq, Hk, D, P, own)
    assert (not P or _stages(P, spans) >= 3) and (not own or _stages(own, own_spans) >= 3)
    q, K, V, off, offs = base._shared_case(g, T, Hq, Hk, D, P, [own] * T, std=1.0 if rising else 3.0)
    scale, rows = 1.0 / math.sqrt(D), [(o, own) for o in offs]
    if rising:
        q[..., 0] = 4.0
        for o, n, s in [(off, P, spans)] + [(o, own, own_spans) for o in offs]:
            level = torch.arange(n, device="cuda") // 128 % max(1, _stages(n, s) if n else 1)
            K[:, o:o + n, 0] = (level * (9.0 * math.log(2.0) / (4.0 * scale))).to(torch.bfloat16)
    att, lse = base._run_shared(card, q, K, V, off, P, rows, scale, P, own)
    _hold(att, lse, q, K, V, off, P, rows, scale)


@pytest.mark.parametrize("D,P", [(64, 13000), (128, 33000)])
def test_attn_shared_wide_batches_over_long_prefixes(card, D, P):
    """two prefix workgroups a CU, and states of 2048 heads folded a wave a head"""
    T, Hq, Hk, own = 64, 32, 2, 3
    assert T * Hq >= 2048
    assert _spans(card, T, Hq, Hk, D, P, own)[0] == -(-2 * _cus() // (Hk * -(-T * Hq // Hk // 128)))
    g = gen(5850 + D)
    q, K, V, off, offs = base._shared_case(g, T, Hq, Hk, D, P, [own] * T, std=3.0)
    scale, rows = 1.0 / math.sqrt(D), [(o, own) for o in offs]
    att, lse = base._run_shared(card, q, K, V, off, P, rows, scale, P, own)
    _hold(att, lse, q, K, V, off, P, rows, scale)


# ---- the weight keys received -----------------------------------------------------------------------------------------


def _mass_parts(card, T, Hq, Hk, D, n):
    """(workgroups the pairs are cut over, their stages)"""
    parts = max(1, card.lib.btb_hip_attn_mass_floats(T, Hq, Hk, D, n) // (Hk * n))
    return parts, -(-T * (Hq // Hk) // (16384 // D))


@pytest.mark.parametrize("D", [64, 128])
def test_attn_mass_no_workgroup_without_a_stage(card, D):
    for T in list(range(1, 140, 7)) + [200, 331, 500, 1000]:
        for Hq, Hk in ((32, 8), (12, 4), (5, 1), (48, 2)):
            for n in (31, 512, 700, 2000, 4000, 16384):
                parts, stages = _mass_parts(card, T, Hq, Hk, D, n)
                assert parts == 1 or (parts - 1) * -(-stages // parts) < stages, (T, Hq, Hk, n, parts, stages)


def _mass_case(card, T, Hq, Hk, D, n, chain):
    """the operator's sums and the formula's, both with and without what the keys had; the bar relative to the 2-norm"""
    g = gen(5900 + T + n)
    q = (torch.randn(T, Hq, D, generator=g) * 1.5).to(torch.bfloat16).cuda()
    K, scale = base._cache(g, Hk, n, D), 1.0 / math.sqrt(D)
    seen = (n - T + 1 + torch.arange(T)).clamp(min=0) if chain else (torch.arange(T) * 37) % (n + 2)
    seen = seen.to(torch.int32).cuda()
    hidden = torch.arange(n, device="cuda")[None, :] >= seen[:, None]
    lse, want, top = torch.empty(T, Hq, device="cuda"), torch.zeros(Hk, n, dtype=torch.float64, device="cuda"), 0.0
    for h in range(Hq):
        s = q[:, h].double() @ K[h // (Hq // Hk)].double().T * scale
        s.masked_fill_(hidden, -math.inf)
        lse[:, h] = torch.logsumexp(s, -1).float()
        w = torch.exp(s - lse[:, h].double()[:, None])
        w[lse[:, h] == -math.inf] = 0.0
        want[h // (Hq // Hk)] += w.sum(0)
        top = max(top, float(s.masked_fill(hidden, 0.0).abs().max()) + float(lse[:, h].nan_to_num(neginf=0.0).abs().max()))
    mass = torch.rand(Hk, n, generator=g).cuda()
    alone = card.attn_mass(q.view(T, -1), K, lse, seen, None, Hq, Hk, D, scale, n)
    both = card.attn_mass(q.view(T, -1), K, lse, seen, mass, Hq, Hk, D, scale, n, out=torch.empty_like(mass))
    torch.cuda.synchronize()
    qn, kn = (float(t.double().norm(dim=-1).max()) for t in (q, K))
    bar = U * scale * qn * kn + 2 * U * (1 + top) + math.sqrt(T * Hq / Hk) * U
    print(f"relative 2-norm {float((alone.double() - want).norm() / want.norm()):.2e}, bar {bar:.2e}")
    assert float((alone.double() - want).norm()) <= bar * float(want.norm())
    total = want + mass.double()
    assert float((both.double() - total).norm()) <= bar * float(want.norm()) + U * float(total.norm())


@pytest.mark.parametrize("T,Hq,Hk,D", [(3, 32, 16, 128), (7, 64, 16, 64), (16, 64, 16, 128), (15, 48, 16, 64)])
def test_attn_mass_few_pairs_many_tiles_a_wave(card, T, Hq, Hk, D):
    """a wave's two buffers in turn, and its sums written eight tiles at a time more than once"""
    pairs, n = T * Hq // Hk, 256 * 9 * -(-_cus() // Hk) + 45
    assert pairs <= 64 and n > 2 * 8 * 32 * -(-_cus() // Hk) * 4
    _mass_case(card, T, Hq, Hk, D, n, chain=T != 7)


@pytest.mark.parametrize("T,Hq,Hk,D,chain", [(1300, 64, 64, 128, False), (1300, 64, 64, 64, True), (650, 128, 64, 128, True)])
def test_attn_mass_many_pairs_many_stages(card, T, Hq, Hk, D, chain):
    """both buffers written again, and the tables of 1024 pairs' log-sums and limits filled again"""
    n = 256 * (2 * _cus() // 2 // Hk) + 1
    parts, stages = _mass_parts(card, T, Hq, Hk, D, n)
    assert parts == 1 and stages >= 5 and T * Hq // Hk > 1024
    _mass_case(card, T, Hq, Hk, D, n, chain)


@pytest.mark.parametrize("T,Hq,Hk,D,n", [(400, 16, 2, 128, 6000), (400, 32, 2, 64, 5000)])
def test_attn_mass_pairs_cut_over_workgroups_of_several_stages(card, T, Hq, Hk, D, n):
    parts, stages = _mass_parts(card, T, Hq, Hk, D, n)
    assert parts > 1 and stages > 2 * parts
    _mass_case(card, T, Hq, Hk, D, n, chain=True)


@pytest.mark.parametrize("T,Hq,Hk,D,n", [(5, 32, 8, 128, 300), (90, 8, 4, 64, 500), (90, 8, 4, 128, 700)])
def test_attn_mass_holds_its_weights_in_32_bits(card, T, Hq, Hk, D, n):
    _mass_case(card, T, Hq, Hk, D, n, chain=True)


# ---- eviction ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("L,Hk,D,n,budget,sinks,recent,kind", [
    (2, 2, 256, 700, 300, 1, 690, "ties"),
    (1, 2, 256, 9000, 5000, 0, 1 << 30, "free"),
    (1, 2, 64, 8192, 4096, 4, 8000, "ties"),       # the last length a workgroup takes alone
    (1, 2, 128, 8192, 8191, 0, 1 << 30, "odd"),
    (1, 2, 64, 8193, 4096, 4, 8000, "ties"),       # the first over two
    (1, 2, 128, 8193, 8192, 0, 1 << 30, "free"),
    (1, 1, 64, 540000, 530000, 3, 539000, "odd"),  # more than 64 workgroups: their counts are added up in several trips
    (1, 1, 64, 600001, 70001, 0, 1 << 30, "ties"),
])
def test_evict_lengths_and_widths(card, L, Hk, D, n, budget, sinks, recent, kind):
    assert (card.lib.btb_hip_kv_evict_words(L, Hk, n) > 0) == (n > 8192)
    base.test_evict(card, L, Hk, D, n, budget, sinks, recent, kind)


# ---- writes stay inside their buffers ---------------------------------------------------------------------------------


@pytest.mark.parametrize("T,Hq,Hk,D", [(1, 4, 2, 64), (7, 9, 3, 256), (1300, 24, 4, 128)])
def test_rope_outputs_stay_inside(card, T, Hq, Hk, D):
    g, cap, bf = gen(5950 + T), T + 3, torch.bfloat16
    cos, sin = (fin(t) for t in rope_tables(StackConfig(head_dim=D), 40, "cpu"))
    qkv = fin(torch.randn(T, (Hq + 2 * Hk) * D, generator=g).to(bf))
    pos, slots = fin(torch.randint(0, 40, (2, T), generator=g, dtype=torch.int32)), torch.randperm(cap, generator=g)[:T].to(torch.int32)
    axes = rope_axes([D // 4, D // 4], "cuda")
    outs = [Fenced((Hk, cap, D), bf, torch.zeros(Hk, cap, D)) for _ in range(2)] + [Fenced((T, Hq * D), bf)]
    w = fin(torch.ones(D, dtype=bf))
    card.norm_rope_axes(qkv, w, w, 1e-6, cos, sin, pos, axes, fin(slots), *(o.t for o in outs), Hq, Hk, D)
    for o in outs:
        o.check("norm_rope_axes")
    plain = [torch.zeros_like(outs[0].t), torch.zeros_like(outs[1].t), torch.empty_like(outs[2].t)]
    card.norm_rope_axes(qkv.clone(), w.clone(), w.clone(), 1e-6, cos.clone(), sin.clone(), pos.clone(), axes, slots.cuda(), *plain, Hq, Hk, D)
    assert all(torch.equal(o.t, p) for o, p in zip(outs, plain))


@pytest.mark.parametrize("T,Hq,Hk,D,P,own", [(1, 4, 2, 64, 0, 1), (3, 5, 1, 128, 70, 9), (15, 16, 4, 128, 300, 40), (70, 32, 4, 64, 600, 130)])
def test_attn_shared_outputs_stay_inside(card, T, Hq, Hk, D, P, own):
    g, f32 = gen(5960 + T), torch.float32
    cap, bf = P + T * own, torch.bfloat16
    q, K, V = (fin(torch.randn(*s, generator=g).to(bf)) for s in ((T, Hq * D), (Hk, cap, D), (Hk, cap, D)))
    lay = fin(card.shared_layout(0, P, [(P + t * own, own) for t in range(T)]))
    n = card.attn_shared_scratch(T, Hq, Hk, D, P, own).numel()
    att, lse, scratch = Fenced((T, Hq * D), bf), Fenced((T, Hq), f32), Fenced((n,), f32)
    card.attn_shared(q, K, V, att.t, lay, Hq, Hk, D, 0.1, P, own, scratch.t, lse=lse.t)
    for o in (att, lse, scratch):
        o.check("attn_shared")
    att2, lse2 = torch.empty_like(att.t), torch.empty_like(lse.t)
    card.attn_shared(q.clone(), K.clone(), V.clone(), att2, lay.clone(), Hq, Hk, D, 0.1, P, own, torch.empty_like(scratch.t), lse=lse2)
    assert torch.equal(att.t, att2) and torch.equal(lse.t, lse2) and bool(att2.isfinite().all())


@pytest.mark.parametrize("T,Hq,Hk,D,n", [(1, 4, 2, 64, 1), (6, 40, 8, 128, 1000), (90, 6, 2, 128, 333), (300, 8, 2, 64, 257)])
def test_attn_mass_outputs_stay_inside(card, T, Hq, Hk, D, n):
    g = gen(5970 + T)
    q, K = (fin(torch.randn(*s, generator=g).to(torch.bfloat16)) for s in ((T, Hq * D), (Hk, n, D)))
    lse, seen = fin(torch.rand(T, Hq, generator=g) + 3.0), fin(torch.randint(0, n + 1, (T,), generator=g, dtype=torch.int32))
    mass, out = fin(torch.rand(Hk, n, generator=g)), Fenced((Hk, n), torch.float32)
    card.attn_mass(q, K, lse, seen, mass, Hq, Hk, D, 0.1, n, out=out.t)
    out.check("attn_mass")
    again = card.attn_mass(q.clone(), K.clone(), lse.clone(), seen.clone(), mass.clone(), Hq, Hk, D, 0.1, n)
    assert torch.equal(out.t, again) and bool(again.isfinite().all())


@pytest.mark.parametrize("L,Hk,D,n,budget", [(1, 1, 64, 2, 1), (3, 2, 256, 200, 77), (1, 2, 128, 9000, 4100)])
def test_evict_outputs_stay_inside(card, L, Hk, D, n, budget):
    g, bf, i32, f32 = gen(5980 + n), torch.bfloat16, torch.int32, torch.float32
    K, V = (fin(torch.randn(L, Hk, n, D, generator=g).to(bf)) for _ in range(2))
    mass, pos = fin(torch.rand(L, Hk, n, generator=g)), fin(torch.arange(n, dtype=i32).expand(L, Hk, n).contiguous())
    make = lambda: [Fenced((L, Hk, budget, D), bf), Fenced((L, Hk, budget, D), bf), Fenced((L, Hk, budget), f32), Fenced((L, Hk, budget), i32),
                    Fenced((L, Hk, budget), i32)]
    outs = make()
    card.kv_evict(mass, pos, K, V, n, budget, *(o.t for o in outs), sinks=1)
    for o in outs:
        o.check("kv_evict")
    # in place
    inside = [Fenced(tuple(t.shape), t.dtype, t) for t in (K, V, mass, pos)] + [Fenced((L, Hk, budget), i32)]
    k, v, m, p, idx = (o.t for o in inside)
    card.kv_evict(m, p, k, v, n, budget, k, v, m, p, idx, sinks=1)
    for o in inside:
        o.check("kv_evict in place")
    assert torch.equal(idx, outs[4].t) and torch.equal(k[:, :, :budget], outs[0].t) and torch.equal(m[..., :budget], outs[2].t)


# ---- refusals ---------------------------------------------------------------------------------------------------------


def test_outputs_whose_heads_share_memory(card):
    """one mass for all heads may be read, and not written: their workgroups would race for it"""
    T, Hq, Hk, D, n = 2, 8, 4, 64, 40
    g = gen(5990)
    q, K = (torch.randn(*s, generator=g).to(torch.bfloat16).cuda() for s in ((T, Hq * D), (Hk, n, D)))
    lse, seen = torch.full((T, Hq), 3.0, device="cuda"), torch.full((T,), n, dtype=torch.int32, device="cuda")
    one = torch.rand(1, n, generator=g).cuda().expand(Hk, n)
    call = lambda mass, out: card.attn_mass(q, K, lse, seen, mass, Hq, Hk, D, 0.1, n, out=out)
    assert torch.equal(call(one, torch.empty(Hk, n, device="cuda")), call(one.contiguous(), None))
    half = torch.zeros(Hk * n, device="cuda").as_strided((Hk, n), (n // 2, 1))
    for mass, out in ((one, None), (None, one), (None, half)):
        with pytest.raises(ValueError):
            call(mass, out)
    pos, i32 = torch.arange(n, dtype=torch.int32, device="cuda"), torch.int32
    kept = 8
    outs = lambda **k: [k.get(a, v) for a, v in dict(
        K=torch.empty(Hk, kept, D, dtype=torch.bfloat16, device="cuda"), V=torch.empty(Hk, kept, D, dtype=torch.bfloat16, device="cuda"),
        mass=torch.empty(Hk, kept, device="cuda"), pos=torch.empty(Hk, kept, dtype=i32, device="cuda"),
        idx=torch.empty(Hk, kept, dtype=i32, device="cuda")).items()]
    assert card.kv_evict(one, pos.expand(Hk, n), K, K, n, kept, *outs()) == kept
    for bad in (dict(mass=torch.empty(1, kept, device="cuda").expand(Hk, kept)), dict(pos=torch.empty(1, kept, dtype=i32, device="cuda").expand(Hk, kept))):
        with pytest.raises(ValueError):
            card.kv_evict(one, pos.expand(Hk, n), K, K, n, kept, *outs(**bad))
    # one head has no other to share with
    assert card.kv_evict(one[:1], pos[None], K[:1], K[:1], n, kept, *(t[:1].contiguous() for t in outs())) == kept
    torch.cuda.synchronize()


def test_caches_whose_rows_share_memory_are_not_written(card):
    """an expanded cache may be read; written, its heads or slots would race for one place"""
    T, Hq, Hk, D, cap, kept = 2, 4, 2, 64, 16, 8
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")
    i32 = torch.int32
    cos, axes = z(8, D), z(D // 2, dt=torch.uint8)
    heads, slots = z(1, cap, D).expand(Hk, cap, D), z(Hk, 1, D).expand(Hk, cap, D)
    rope = lambda K, V, hq, hk: card.norm_rope_axes(z(T, (hq + 2 * hk) * D), None, None, 1e-6, cos, cos, z(1, T, dt=i32), axes,
                                                 torch.arange(T, dtype=i32, device="cuda"), K, V, z(T, hq * D), hq, hk, D)
    rope(z(Hk, cap, D), z(Hk, cap, D), Hq, Hk)
    rope(heads[:1], z(1, cap, D).expand(Hk, cap, D)[:1], Hq, 1)  # one head: no other to share with
    for K in (heads, slots):
        with pytest.raises(HipError):
            rope(K, K, Hq, Hk)
    K, mass, pos = z(2, Hk, cap, D), z(2, Hk, cap, dt=torch.float32), z(2, Hk, cap, dt=i32)
    evict = lambda K_out, V_out: card.kv_evict(mass, pos, K, K, cap, kept, K_out, V_out, z(2, Hk, kept, dt=torch.float32), z(2, Hk, kept, dt=i32),
                                        z(2, Hk, kept, dt=i32))
    for bad in (z(1, Hk, kept, D).expand(2, Hk, kept, D), z(2, 1, kept, D).expand(2, Hk, kept, D), z(2, Hk, 1, D).expand(2, Hk, kept, D)):
        with pytest.raises(HipError):
            evict(bad, bad)
    assert evict(z(2, Hk, kept, D), z(2, Hk, kept, D)) == kept
    lib, p = card.lib, lambda t: t.data_ptr()
    q, f = z(T, Hq * D), z(64, dt=torch.float32)
    assert lib.btb_hip_attn_mass(p(q), p(K), p(f), p(pos), None, p(f), T, Hq, Hk, D, 8, cap * D, D, 0, 7, Hq, 1, 0.1, None, None) == -6
    torch.cuda.synchronize()
