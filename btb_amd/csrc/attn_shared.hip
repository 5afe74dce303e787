// Attention of rows that share one long prefix: the prefix's keys are read once for all the rows, each row's own keys
// once for itself.
//
//   s_j = scale q . k_j over the prefix's and the row's own keys;  lse = log sum_j exp s_j;  att = sum_j exp(s_j - lse) v_j
//
// in one pass over the keys with a running maximum and sum. A workgroup is four waves and one of two kinds of work:
//   prefix: one kv head, one span of the prefix, a tile of 32, 64 or 128 (row, query head) pairs, of which a wave takes 32 - with
//           128 pairs every key, else the half or the quarter of the keys that the waves of the same pairs share out
//   own:    one row, one kv head, one span of the row's own keys; a wave a quarter of them
// and leaves states (maximum, sum, output) in the scratch, which a second launch folds in a fixed order. The spans are
// cut from the keys there are (the layout lies on the device), so a recorded launch holds while the rows grow.
//
// Sums and outputs are f32; a weight goes to the matrix cores as two bf16 terms, since one leaves the outputs of wide passes 1.9e-3 off
// (relative 2-norm against 64 bits; 40 rows of 16 / 2 heads, normal values, scores of deviation 3) and two 1.65e-3, what rounding
// the outputs alone makes. us, one / two: 16 rows of 32 heads x 128 over 131072 keys, 100 own 104 / 105; 256 rows over 32768 160 / 211,
// and 640 own 239 / 284; 256 rows of 40 heads x 64 over 32768 141 / 196; 41 rows over 6001, 485 own 19.5 / 21.3.
//
// Bound: memory where few rows share the prefix (16 rows of 32 heads x 128 over 131072 keys, 100 own: 105 to 115 us, 4.7 to 5.2 TB/s), the products
// where many do (256 rows over 32768: 211 us, the fold included; three products for every two of the formula, 975 TFLOP/s of bare
// products' 1384), and both at once where many rows have many own keys (640 each: 284 us, 2.8 TB/s and 495 TFLOP/s).

#include "btb_common.hpp"
#include "btb_tile32.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

constexpr int SH_KEYS = 128;  // keys a stage: a tile a wave loads

struct SharedArgs {
    const uint16_t* q;
    const uint16_t* K;
    const uint16_t* V;
    const int32_t* lay;  // off, len, then (off, len) a row
    float* part_m;       // [T, Hq, S]
    float* part_l;
    float* part_acc;     // [T, Hq, S, D]
    long long hs, rs;
    float scale_log2;
    int T, Hq, Hk, G, cap, prefix_cap, own_cap;
    int pair_tiles, prefix_spans, own_spans;  // workgroups: Hk x pair_tiles x prefix_spans, then Hk x T x own_spans
    int states;                               // states a (row, head)
};

struct Keys {
    int first, count;  // slots
};
// a stretch of slots as the layout gives it, kept within the cache and the capacity the launch was sized for
__device__ __forceinline__ Keys stretch(int off, int len, int most, int cap) {
    Keys k;
    k.first = min(max(off, 0), cap);
    k.count = off < 0 ? 0 : min(max(len, 0), min(most, cap - k.first));
    k.first = __builtin_amdgcn_readfirstlane(k.first);
    k.count = __builtin_amdgcn_readfirstlane(k.count);
    return k;
}
// part `i` of `parts` of a stretch, in whole stages
__device__ __forceinline__ Keys part_of(const Keys& k, int i, int parts) {
    const int per = ((k.count + parts - 1) / parts + SH_KEYS - 1) / SH_KEYS * SH_KEYS;
    Keys r;
    const long long begin = (long long)i * per;
    r.first = k.first + (int)min(begin, (long long)k.count);
    r.count = (int)max(min((long long)k.count - begin, (long long)per), 0LL);
    return r;
}

// A workgroup's pairs against a stretch of keys. QW waves take 32 pairs each, KW = 4 / QW of them share the same pairs and
// divide a stage's four tiles. Every wave brings one tile of K and one of V into LDS a stage. K's is asked for again as soon as
// the scores are made and V's as soon as the outputs are, so each travels while the other product and the softmax run, and one
// buffer of each does: 64 KB, two workgroups a CU, whose products and exponentials run beside one another's. Where waves read
// one another's tiles (QW > 1) a stage costs four barriers, else none. `row(r)`: the q row of the workgroup's pair r;
// `state(r)`: where its state goes, negative: nowhere.
template <int D, int QW, class Row, class State>
__device__ __forceinline__ void walk(const SharedArgs& p, const uint16_t* Kg, const uint16_t* Vg, const Keys& keys, uint8_t* lds,
                                     float* meet, Row row, State state) {
    constexpr int STEPS = D / 16, DT = D / 32, TILE = TK * 2 * D, KW = 4 / QW, TPW = QW, PAIRS = 32 * QW;
    constexpr int N = TileLoads<D>::N;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, h = lane >> 5, qw = wv / KW, kw = wv % KW;
    const float ninf = bits_f32(0xff800000u);
    TileLoads<D> loads;
    loads.make(p.rs, lane);
    const uint16_t* Kb = Kg + (size_t)keys.first * p.rs;
    const uint16_t* Vb = Vg + (size_t)keys.first * p.rs;
    // the wave's tile of the stage that starts at key kb (a tile wholly past the end: the last key)
    auto issue_k = [&](int kb) {
        const int k0 = min(kb + TK * wv, keys.count - 1);
        loads.template issue<true>(Kb + (size_t)k0 * p.rs, p.rs, keys.count - k0, lds + wv * TILE, lane);
    };
    auto issue_v = [&](int kb) {
        const int k0 = min(kb + TK * wv, keys.count - 1);
        loads.template issue<false>(Vb + (size_t)k0 * p.rs, p.rs, keys.count - k0, lds + (4 + wv) * TILE, lane);
    };
    auto barrier = [&] {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (QW > 1) asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    f32x16 o[DT];
    float m = ninf, l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = zero16();
    bf16x8 qf[STEPS];
    {
        const uint16_t* qr = row(32 * qw + c) + 8 * h;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) qf[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(qr + 16 * s));
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): q is here, and no register of the loop waits for a load
    __builtin_amdgcn_sched_barrier(0);
    if (keys.count > 0) {
        issue_k(0);
        issue_v(0);
    }
    // The wave's tiles of a stage in groups of at most two. The order within a stage is written down: left alone the compiler
    // reads a fragment, waits for it and multiplies, an LDS round trip a product. Fragments are asked for AHEAD products early,
    // and what vector arithmetic there is to do meanwhile - a group's weights under the next one's scores, that one's maximum
    // under the first one's outputs - is dealt out between the products.
    constexpr int GT = TPW < 2 ? TPW : 2, GROUPS = TPW / GT, AHEAD = 4;
    f32x16 st[GROUPS][GT];  // scores, then weights
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
    // products GT STEPS; work(i) after each of the STEPS
    auto scores = [&](uint32_t at, int group, f32x16(&to)[GT], auto work) {
        bf16x8 kf[STEPS * GT];
        auto read = [&](int e) { return k_fragment(lds + kw * TILE, at, KW * (GT * group + e % GT) * TILE, e / GT); };
#pragma unroll
        for (int j = 0; j < GT; ++j) to[j] = zero16();
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) kf[e] = read(e);
        fence();
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
#pragma unroll
            for (int j = 0; j < GT; ++j) {
                const int e = i * GT + j;
                if (e + AHEAD < STEPS * GT) kf[e + AHEAD] = read(e + AHEAD);
                to[j] = mfma32(kf[e], qf[i], to[j]);
            }
            work(i);
            fence();
        }
    };
    // keys past the end
    auto mask = [&](int kb, int group) {
#pragma unroll
        for (int j = 0; j < GT; ++j) {
            const int left = keys.count - kb - TK * (kw + KW * (GT * group + j));
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i / 4) + 4 * h + i % 4 >= left) st[group][j][i] = ninf;
        }
    };
    // The state moves to a new maximum only where that is 2^8 past its own: weights of up to 2^8 are as exact, and most groups
    // then leave the outputs alone. A pair's decision is its own, whatever its neighbours'.
    auto settle = [&](float top) {
        top = fmaxf(top, xor32(top)) * p.scale_log2;
        const bool moves = top > m + 8.f || m == ninf;
        if (__any(moves)) {
            const float mn = moves ? top : m;
            const float corr = m == ninf ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= corr;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= corr;
        }
    };
    // scores [from, to) of a group as weights, in their place
    auto weigh = [&](int group, float ref, int from, int to) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < GT * 16; ++e)
            if (e >= from && e < to) {
                const float w = __builtin_amdgcn_exp2f(fmaf(st[group][e / 16][e % 16], p.scale_log2, -ref));
                st[group][e / 16][e % 16] = w;
                sum += w;
            }
        l += sum;
    };
    // products GT 4 DT; work(r), GT DT of them
    auto outputs = [&](uint32_t at, int group, auto work) {
        weighted_sums<DT, 2 * GT>(
            o, [&](int u, int d) { return v_fragment<D>(lds + (4 + kw) * TILE, at, KW * (GT * group + u / 2) * TILE, d, u % 2); },
            [&](int u, int i) { return st[group][u / 2][8 * (u % 2) + i]; }, work);
    };
    auto nothing = [](int) {};
    const uint32_t k_at = k_place<D>(lane), v_at = v_place<D>(lane);
    for (int kb = 0; kb < keys.count; kb += SH_KEYS) {
        const bool more = kb + SH_KEYS < keys.count;
        uint32_t ak = k_at, av = v_at;
        wait_loads<N>(ak);
        barrier();
        scores(ak, 0, st[0], nothing);
        if (!more) mask(kb, 0);
        float top = st[0][0][0];
#pragma unroll
        for (int j = 0; j < GT; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, st[0][j][i]);
        settle(top);
        fence();
        {
            const float ref = m == ninf ? 0.f : m;
            constexpr int EACH = GT * 16 / STEPS;
            if constexpr (GROUPS > 1) {
                scores(ak, 1, st[GROUPS - 1], [&](int i) { weigh(0, ref, i * EACH, i * EACH + EACH); });
                if (!more) mask(kb, GROUPS - 1);
            } else {
                weigh(0, ref, 0, GT * 16);
            }
        }
        barrier();
        if (more) {
            issue_k(kb + SH_KEYS);
            wait_loads<N>(av);
        } else {
            wait_loads<0>(av);
            const int mine = keys.count - kb - TK * wv;
            if (mine < TK) TileLoads<D>::clear_past(lds + (4 + wv) * TILE, mine, lane);
            if constexpr (QW > 1) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        barrier();
        if constexpr (GROUPS > 1) {
            constexpr int EACH = GT * 16 / (GT * DT);
            top = st[1][0][0];
            outputs(av, 0, [&](int r) {
#pragma unroll
                for (int e = 0; e < GT * 16; ++e)
                    if (e >= r * EACH && e < r * EACH + EACH) top = fmaxf(top, st[1][e / 16][e % 16]);
            });
            settle(top);
            weigh(1, m == ninf ? 0.f : m, 0, GT * 16);
            fence();
        }
        outputs(av, GROUPS - 1, nothing);
        barrier();
        if (more) issue_v(kb + SH_KEYS);
    }
    // the waves of the same pairs meet: their maxima and sums, then their outputs, through the stage's LDS
    float* mm = meet;  // [4][32] maxima, then sums
    float* ml = meet + 4 * 32;
    l += xor32(l);
    if (h == 0) {
        mm[wv * 32 + c] = m;
        ml[wv * 32 + c] = l;
    }
    __syncthreads();
    float* all = reinterpret_cast<float*>(lds);  // [4 waves][32 pairs][D], a pair's 16-byte chunks permuted
    {
        float top = ninf;
#pragma unroll
        for (int i = 0; i < KW; ++i) top = fmaxf(top, mm[(qw * KW + i) * 32 + c]);
        const float f = m == ninf ? 0.f : __builtin_amdgcn_exp2f(m - top);
        float* dst = all + (size_t)(wv * 32 + c) * D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float4 v = make_float4(o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]);
                if (KW > 1 && m == ninf) v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (KW > 1) v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
                *reinterpret_cast<float4*>(dst + 4 * ((8 * d + 2 * b + h) ^ (c & (D / 4 - 1)))) = v;
            }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < PAIRS * (D / 4); e += 256) {
        const int r = e / (D / 4), chunk = e % (D / 4), group = r / 32, in = r % 32;
        const long long to = state(r);
        if (to < 0) continue;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < KW; ++i) {
            const float4 x =
                *reinterpret_cast<const float4*>(all + (size_t)((group * KW + i) * 32 + in) * D + 4 * (chunk ^ (in & (D / 4 - 1))));
            v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
        }
        *reinterpret_cast<float4*>(p.part_acc + (size_t)to * D + 4 * chunk) = v;
        if (chunk == 0) {
            float top = ninf, sum = 0.f;
#pragma unroll
            for (int i = 0; i < KW; ++i) top = fmaxf(top, mm[(group * KW + i) * 32 + in]);
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const float mw = mm[(group * KW + i) * 32 + in];
                sum = fmaf(mw == ninf ? 0.f : __builtin_amdgcn_exp2f(mw - top), ml[(group * KW + i) * 32 + in], sum);
            }
            p.part_m[to] = top;
            p.part_l[to] = sum;
        }
    }
}

// 128 pairs against a stretch of keys, every wave 32 of them and all the keys: the prefix of many rows, whose products are what
// it costs. Stages of 64 keys, three of K and two of V in LDS, every wave bringing half a tile of each. A stage's weights are made
// between the products of the next one's scores, and that one's maxima between the products of its outputs: no stretch of a stage
// is vector arithmetic alone. Two barriers a stage where walk has four.
// For head_dim 64, where the vector arithmetic costs as much as the products and so is worth hiding; at 128 one tile's chain of eight
// dependent products sets the pace and walk is faster. us, walk / this: head_dim 64, 41 rows of 40 / 8 heads over 6001 and 485 own 23.2 /
// 21.3, 200 rows of 16 / 2 over 20000 54 / 48, 256 of 40 / 8 over 32768 212 / 209; 256 rows of 32 / 8 heads x 128 over 32768 keys 217 /
// 223, and 640 own 285 / 317.
template <int D, int QW>
constexpr bool overlaps() {
    return D == 64 && QW == 4;
}
template <int D, class Row, class State>
__device__ __forceinline__ void walk_many(const SharedArgs& p, const uint16_t* Kg, const uint16_t* Vg, const Keys& keys, uint8_t* lds,
                                          Row row, State state) {
    constexpr int STEPS = D / 16, DT = D / 32, TILE = TK * 2 * D, STAGE = 2 * TILE, AHEAD = 4, H = TileLoads<D>::N / 2;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, h = lane >> 5;
    const float ninf = bits_f32(0xff800000u);
    const int stages = (keys.count + 63) / 64;
    TileLoads<D> loads;
    loads.make(p.rs, lane);
    const uint16_t* Kb = Kg + (size_t)keys.first * p.rs;
    const uint16_t* Vb = Vg + (size_t)keys.first * p.rs;
    uint8_t* v_lds = lds + 3 * STAGE;
    // (`ln` is the lane again, made unknown to the compiler stage by stage: what is rare comes from it and is not kept in registers)
    int ln = lane;
    auto issue_k = [&](int s, int slot) {
        const int k0 = min(64 * s + 16 * wv, keys.count - 1);
        loads.template issue<true, H>(Kb + (size_t)k0 * p.rs, p.rs, keys.count - k0, lds + slot * STAGE + wv * (TILE / 2), ln);
    };
    auto issue_v = [&](int s) {
        const int k0 = min(64 * s + 16 * wv, keys.count - 1);
        loads.template issue<false, H>(Vb + (size_t)k0 * p.rs, p.rs, keys.count - k0, v_lds + (s & 1) * STAGE + wv * (TILE / 2), ln);
    };
    // all but the youngest n stages' loads have landed
    auto wait = [&](int n, uint32_t& at) {
        if (n == 3)
            wait_loads<3 * H>(at);
        else if (n == 2)
            wait_loads<2 * H>(at);
        else if (n == 1)
            wait_loads<H>(at);
        else
            wait_loads<0>(at);
    };
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
    auto barrier = [&] {
        fence();
        asm volatile("s_barrier" ::: "memory");
        fence();
    };
    f32x16 o[DT];
    float m = ninf, l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = zero16();
    bf16x8 qf[STEPS];
    {
        const uint16_t* qr = row(32 * wv + c) + 8 * h;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) qf[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(qr + 16 * s));
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): q is here, and no register of the loop waits for a load
    fence();
    const uint32_t k_at = k_place<D>(lane), v_at = v_place<D>(lane);
    f32x16 st[2], next[2];  // a stage's scores, then weights; the next one's scores
    // the scores of tile `tile` of a stage; work(i) after each of the STEPS
    next[0] = next[1] = zero16();
    auto scores = [&](uint32_t at, int slot, int tile, f32x16& to, auto work) {
        bf16x8 kf[STEPS];
        const uint8_t* tiles = lds + slot * STAGE;
        to = zero16();
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) kf[i] = k_fragment(tiles, at, tile * TILE, i);
        fence();
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (i + AHEAD < STEPS) kf[i + AHEAD] = k_fragment(tiles, at, tile * TILE, i + AHEAD);
            to = mfma32(kf[i], qf[i], to);
            work(i);
            fence();
        }
    };
    // its outputs; work(r), 2 DT of them
    auto outputs = [&](uint32_t at, int s, auto work) {
        const uint8_t* tiles = v_lds + (s & 1) * STAGE;
        weighted_sums<DT, 4>(
            o, [&](int u, int d) { return v_fragment<D>(tiles, at, u / 2 * TILE, d, u % 2); },
            [&](int u, int i) { return st[u / 2][8 * (u % 2) + i]; }, work);
    };
    auto mask = [&](int s, f32x16(&of)[2]) {  // keys past the end
        if (64 * s + 64 <= keys.count) return;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i / 4) + i % 4 >= keys.count - 64 * s - TK * j - 4 * (ln >> 5)) of[j][i] = ninf;
    };
    auto settle = [&](float top) {  // as in walk
        top = fmaxf(top, xor32(top)) * p.scale_log2;
        const bool moves = top > m + 8.f || m == ninf;
        if (__any(moves)) {
            const float mn = moves ? top : m;
            const float corr = m == ninf ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= corr;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= corr;
        }
    };
    if (stages > 0) {
        issue_k(0, 0);
        if (stages > 1) issue_k(1, 1);
        issue_v(0);
        if (stages > 2) issue_k(2, 2);
        uint32_t ak = k_at;
        wait(stages > 2 ? 3 : stages > 1 ? 2 : 1, ak);
        barrier();
        scores(ak, 0, 0, st[0], [](int) {});
        scores(ak, 0, 1, st[1], [](int) {});
        mask(0, st);
        float top = st[0][0];
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaxf(st[0][i], st[1][i]));
        settle(top);
    }
    int slot = 0;  // of stage s's K
    for (int s = 0; s < stages; ++s) {
        const int left = stages - 1 - s;  // stages behind this one
        uint32_t ak = k_at, av = v_at;
        asm volatile("" : "+v"(ln));
        if (left > 0) wait(left > 1 ? 2 : 1, ak);  // the next one's K; behind it this one's V and the K after
        barrier();
        if (left > 0) issue_v(s + 1);
        if (left > 2) issue_k(s + 3, slot);
        slot = slot == 2 ? 0 : slot + 1;
        const float ref = m == ninf ? 0.f : m;
        float sum = 0.f;
        constexpr int EACH = 16 / STEPS;
        auto weigh = [&](int j, int step) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (e / EACH == step) {
                    st[j][e] = __builtin_amdgcn_exp2f(fmaf(st[j][e], p.scale_log2, -ref));
                    sum += st[j][e];
                }
        };
        if (left > 0) {
            scores(ak, slot, 0, next[0], [&](int i) { weigh(0, i); });
            scores(ak, slot, 1, next[1], [&](int i) { weigh(1, i); });
            mask(s + 1, next);
        } else {
#pragma unroll
            for (int i = 0; i < 2 * STEPS; ++i) weigh(i / STEPS, i % STEPS);
        }
        l += sum;
        wait(left > 2 ? 3 : left > 1 ? 2 : left > 0 ? 1 : 0, av);  // this one's V; behind it K, V and K
        if (64 * s + 64 > keys.count) {
            const int mine = keys.count - 64 * s - 16 * wv;
            if (mine < 16) TileLoads<D>::template clear_past<H>(v_lds + (s & 1) * STAGE + wv * (TILE / 2), mine, ln);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        barrier();
        // (after the last stage `next` holds the last one's scores or none: their maximum goes nowhere)
        float top = next[0][0], other = next[1][0];
        constexpr int EACH_MAX = 16 / (2 * DT);
        outputs(av, s, [&](int r) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i / EACH_MAX == r) {
                    top = fmaxf(top, next[0][i]);
                    other = fmaxf(other, next[1][i]);
                }
        });
        if (left > 0) settle(fmaxf(top, other));
        st[0] = next[0];
        st[1] = next[1];
    }
    l += xor32(l);
    // the outputs through LDS, a pair's 16-byte chunks permuted, so that they are written in whole rows
    __syncthreads();
    float* all = reinterpret_cast<float*>(lds) + (size_t)(wv * 32) * D;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b)
            *reinterpret_cast<float4*>(all + c * D + 4 * ((8 * d + 2 * b + h) ^ (c & (D / 4 - 1)))) =
                make_float4(o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]);
    const long long mine = state(32 * wv + c);
    if (h == 0 && mine >= 0) {
        p.part_m[mine] = m;
        p.part_l[mine] = l;
    }
#pragma unroll 4
    for (int e = lane; e < 32 * (D / 4); e += 64) {
        const int r = e / (D / 4), chunk = e % (D / 4);
        const long long to = state(32 * wv + r);
        if (to >= 0)
            *reinterpret_cast<float4*>(p.part_acc + (size_t)to * D + 4 * chunk) =
                *reinterpret_cast<const float4*>(all + r * D + 4 * (chunk ^ (r & (D / 4 - 1))));
    }
}

// The prefix's workgroups come first, the long ones; the rows' own take what room is left beside them and after them.
template <int D, int QW>
__global__ void __launch_bounds__(256, 2) attn_shared_kernel(SharedArgs p) {
    extern __shared__ __align__(16) uint8_t lds[];  // a stage and where the waves meet, or walk_many's five
    float* meet = reinterpret_cast<float*>(lds + 8 * TK * 2 * D);
    const int pairs = p.T * p.G;
    const int prefix = p.Hk * p.pair_tiles * p.prefix_spans;
    int id = blockIdx.x;
    if (id < prefix) {
        const int g = id % p.Hk, tile = id / p.Hk % p.pair_tiles, sp = id / (p.Hk * p.pair_tiles);
        const Keys keys = part_of(stretch(p.lay[0], p.lay[1], p.prefix_cap, p.cap), sp, p.prefix_spans);
        const int r0 = 32 * QW * tile;
        auto row = [&](int i) {
            const int r = min(r0 + i, pairs - 1), t = r / p.G;
            return p.q + ((size_t)t * p.Hq + g * p.G + (r - t * p.G)) * D;
        };
        auto state = [&](int i) -> long long {
            const int r = r0 + i, t = r / p.G;
            return r < pairs ? ((long long)t * p.Hq + g * p.G + (r - t * p.G)) * p.states + sp : -1;
        };
        if constexpr (overlaps<D, QW>())
            walk_many<D>(p, p.K + (size_t)g * p.hs, p.V + (size_t)g * p.hs, keys, lds, row, state);
        else
            walk<D, QW>(p, p.K + (size_t)g * p.hs, p.V + (size_t)g * p.hs, keys, lds, meet, row, state);
        return;
    }
    id -= prefix;
    const int g = id % p.Hk, t = id / p.Hk % p.T, sp = id / (p.Hk * p.T);
    const Keys keys = part_of(stretch(p.lay[2 + 2 * t], p.lay[3 + 2 * t], p.own_cap, p.cap), sp, p.own_spans);
    auto row = [&](int i) { return p.q + ((size_t)t * p.Hq + g * p.G + min(i, p.G - 1)) * D; };
    auto state = [&](int i) -> long long {
        return i < p.G ? ((long long)t * p.Hq + g * p.G + i) * p.states + p.prefix_spans + sp : -1;
    };
    walk<D, 1>(p, p.K + (size_t)g * p.hs, p.V + (size_t)g * p.hs, keys, lds, meet, row, state);
}

// WAVES waves a (row, head): the states' common maximum, their factors, their outputs in a fixed order - a lane two dims, at
// head_dim 64 the halves of a wave in turn. One wave where there are heads enough to fill the chip, else four: the whole call, us, one
// / four: 16 rows of 32 heads 14.9 / 13.0 (over 700 keys), 64 rows 24.0 / 24.3 (over 4096), 128 rows 33.3 / 35.4, 256 rows 50.5 / 55.3.
template <int D, int WAVES>
__global__ void __launch_bounds__(256) attn_shared_fold_kernel(SharedArgs p, uint16_t* att, float* lse) {
    constexpr int HEADS = 4 / WAVES, PART = 128 / D * WAVES;  // heads a workgroup, parts that the states are taken in
    __shared__ float2 acc[WAVES > 1 ? 4 : 1][64];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x * HEADS + wv / WAVES, w = wv % WAVES;
    const bool live = head < p.T * p.Hq && p.lay[3 + 2 * (min(head, p.T * p.Hq - 1) / p.Hq)] >= 0;  // uniform in the wave
    if (WAVES == 1 && !live) return;
    const size_t base = (size_t)(live ? head : 0) * p.states;
    const float ninf = bits_f32(0xff800000u);
    float m = ninf, l = 0.f;
    for (int s = lane; s < p.states; s += 64) m = fmaxf(m, p.part_m[base + s]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, WAVE));
    auto factor = [&](float ms) { return ms == ninf ? 0.f : __builtin_amdgcn_exp2f(ms - m); };
    for (int s = lane; s < p.states; s += 64) l = fmaf(factor(p.part_m[base + s]), p.part_l[base + s], l);
    l = wave_sum(l);
    const int dl = 2 * lane % D;
    float2 a = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int s = w + WAVES * (2 * lane / D); s < p.states; s += PART) {
        const float ms = p.part_m[base + s];
        const float2 v = *reinterpret_cast<const float2*>(p.part_acc + (base + s) * D + dl);
        const float f = factor(ms);
        a.x = fmaf(f, ms == ninf ? 0.f : v.x, a.x);
        a.y = fmaf(f, ms == ninf ? 0.f : v.y, a.y);
    }
    if (WAVES > 1) {
        acc[wv][lane] = a;
        __syncthreads();
        if (w != 0 || !live) return;
#pragma unroll
        for (int i = 1; i < WAVES; ++i) {
            a.x += acc[wv + i][lane].x;
            a.y += acc[wv + i][lane].y;
        }
    }
    if (D == 64) {
        a.x += xor32(a.x);
        a.y += xor32(a.y);
    }
    if (lane < D / 2) reinterpret_cast<uint32_t*>(att + (size_t)head * D)[lane] = l == 0.f ? 0u : f32x2_bf16(a.x / l, a.y / l);
    if (lane == 0 && lse != nullptr) lse[head] = l == 0.f ? ninf : fmaf(m, 0.693147180559945309f, logf(l));
}

struct SharedPlan {
    int qw;  // waves with 32 pairs of their own
    int pair_tiles, prefix_spans, own_spans, states;
};
// A prefix workgroup a CU, the rows' own beside them; two a CU where the products are what the prefix costs - 128 pairs of a head and
// more, spans of eight stages and more (three at head_dim 64) - and the rows' own keys, read at 5.1 TB/s, cost less than half of that (at
// 640 TFLOP/s). us, one a CU / two: 16 rows x 131072 keys, 100 own 105 / 114; 4 rows 98 / 102; 256 x 32768, 640 own 286 / 306, 400 own
// 273 / 266, 64 own 253 / 218, 64 x 131072, 640 own 269 / 240; 48 heads, 60 rows x 12000 (spans of five) 51 / 53, x 24000 (of nine) 82 / 78;
// 128 x 10000 (of five) 51 / 59, x 17000 (of nine) 76 / 79.5; 24 heads, 200 x 20000 (of thirteen) 117 / 107. Head_dim 64, 2 kv heads of 8, 200
// rows x 8000 (of four) 34 / 32, x 20000 (of eight) 63 / 49, of 4, 36 x 98126 (of six) 46 / 39.5.
static SharedPlan shared_plan(size_t T, size_t Hq, size_t Hk, size_t D, size_t prefix_cap, size_t own_cap) {
    const size_t G = Hq / Hk, pairs = T * G, cus = (size_t)device_info().cus;
    auto spans = [&](size_t groups, size_t cap, size_t wgs) {
        const size_t most = (cap + SH_KEYS - 1) / SH_KEYS, want = (wgs + groups - 1) / groups;
        return (int)(want < most ? want : most);
    };
    SharedPlan r;
    r.qw = pairs <= 32 ? 1 : pairs <= 64 ? 2 : 4;
    const size_t wide = 32 * (size_t)r.qw;
    r.pair_tiles = (int)((pairs + wide - 1) / wide);
    const size_t groups = Hk * r.pair_tiles;
    const bool twice = pairs >= 128 && prefix_cap * groups >= 2 * cus * (D == 64 ? 3 : 8) * SH_KEYS && own_cap * 250 < G * prefix_cap;
    r.prefix_spans = spans(groups, prefix_cap, (twice ? 2 : 1) * cus);
    r.own_spans = spans(Hk * T, own_cap, cus);
    if (r.prefix_spans + r.own_spans == 0) r.own_spans = 1;  // no key anywhere: states that say so
    r.states = r.prefix_spans + r.own_spans;
    return r;
}
template <int D, int QW>
static int32_t launch_one(const dim3& grid, const SharedArgs& p, hipStream_t st) {
    constexpr int lds = overlaps<D, QW>() ? 10 * TK * 2 * D : 8 * TK * 2 * D + 1024;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_shared_kernel<D, QW>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return hip_status(e, "hipFuncSetAttribute");
    }
    hipLaunchKernelGGL((attn_shared_kernel<D, QW>), grid, dim3(256), lds, st, p);
    return hip_status(hipGetLastError(), "attn_shared launch");
}
template <int D>
static int32_t launch_walk(const SharedPlan& s, const dim3& grid, const SharedArgs& p, hipStream_t st) {
    if (s.qw == 1) return launch_one<D, 1>(grid, p, st);
    if (s.qw == 2) return launch_one<D, 2>(grid, p, st);
    return launch_one<D, 4>(grid, p, st);
}
static bool shared_sizes_fit(size_t T, size_t Hq, size_t Hk, size_t D, size_t prefix_cap, size_t own_cap) {
    return T > 0 && T <= 65536 && Hk > 0 && Hk <= 1024 && Hq > 0 && Hq % Hk == 0 && Hq / Hk <= 32 && T * Hq <= (1u << 24) && (D == 64 || D == 128) &&
           prefix_cap <= 0x7FFFFF00u && own_cap <= 0x7FFFFF00u;
}

}  // namespace btb

using namespace btb;

extern "C" {

size_t btb_hip_attn_shared_floats(size_t T, size_t Hq, size_t Hk, size_t D, size_t prefix_cap, size_t own_cap) {
    if (!shared_sizes_fit(T, Hq, Hk, D, prefix_cap, own_cap)) return 0;
    const SharedPlan s = shared_plan(T, Hq, Hk, D, prefix_cap, own_cap);
    const size_t n = T * Hq * (size_t)s.states;
    return (2 * n + 3) / 4 * 4 + n * D;
}

int32_t btb_hip_attn_shared(const void* q, const void* K, const void* V, void* att, float* lse, const int32_t* layout,
                            size_t T, size_t Hq, size_t Hk, size_t D, size_t cap, int64_t hs, int64_t rs, float scale,
                            size_t prefix_cap, size_t own_cap, float* workspace, void* stream) {
    if (!q || !K || !V || !att || !layout || !workspace) return ERR_NULL;
    auto loose = [](const void* a) { return ((uintptr_t)a & 15u) != 0; };
    if (!shared_sizes_fit(T, Hq, Hk, D, prefix_cap, own_cap) || cap == 0 || cap > 0x7FFFFFFFu || hs < 0 || rs < 0 || rs > (1 << 25) || hs % 8 || rs % 8 || !(scale > 0.f) || !(scale < __builtin_inff()) || loose(q) ||
        loose(K) || loose(V) || loose(att) || loose(workspace)) {
        set_error("attn_shared: head_dim 64 or 128, up to 32 query heads a kv head, a positive scale, q, K, V, att "
                  "and the workspace 16-byte aligned with strides in multiples of 8, a row's up to 2^25");
        return ERR_DOMAIN;
    }
    const SharedPlan s = shared_plan(T, Hq, Hk, D, prefix_cap, own_cap);
    const size_t n = T * Hq * (size_t)s.states;
    SharedArgs p;
    p.q = static_cast<const uint16_t*>(q);
    p.K = static_cast<const uint16_t*>(K);
    p.V = static_cast<const uint16_t*>(V);
    p.lay = layout;
    p.part_m = workspace;
    p.part_l = workspace + n;
    p.part_acc = workspace + (2 * n + 3) / 4 * 4;
    p.hs = hs;
    p.rs = rs;
    p.scale_log2 = scale * 1.44269504088896341f;
    p.T = (int)T;
    p.Hq = (int)Hq;
    p.Hk = (int)Hk;
    p.G = (int)(Hq / Hk);
    p.cap = (int)cap;
    p.prefix_cap = (int)prefix_cap;
    p.own_cap = (int)own_cap;
    p.pair_tiles = s.pair_tiles;
    p.prefix_spans = s.prefix_spans;
    p.own_spans = s.own_spans;
    p.states = s.states;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const size_t prefix = Hk * (size_t)s.pair_tiles * s.prefix_spans, own = Hk * T * (size_t)s.own_spans;
    const dim3 grid((unsigned)(prefix + own));
    const int32_t rc = D == 64 ? launch_walk<64>(s, grid, p, st) : launch_walk<128>(s, grid, p, st);
    if (rc != OK) return rc;
    const size_t heads = T * Hq;
    uint16_t* out = static_cast<uint16_t*>(att);
    if (heads >= 2048) {
        const dim3 wgs((unsigned)((heads + 3) / 4));
        if (D == 64)
            hipLaunchKernelGGL((attn_shared_fold_kernel<64, 1>), wgs, dim3(256), 0, st, p, out, lse);
        else
            hipLaunchKernelGGL((attn_shared_fold_kernel<128, 1>), wgs, dim3(256), 0, st, p, out, lse);
    } else {
        const dim3 wgs((unsigned)heads);
        if (D == 64)
            hipLaunchKernelGGL((attn_shared_fold_kernel<64, 4>), wgs, dim3(256), 0, st, p, out, lse);
        else
            hipLaunchKernelGGL((attn_shared_fold_kernel<128, 4>), wgs, dim3(256), 0, st, p, out, lse);
    }
    return hip_status(hipGetLastError(), "attn_shared launch");
}

}  // extern "C"
