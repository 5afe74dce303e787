// Attention of rows that share one long prefix: the prefix's keys are read once for all the rows, each row's own keys
// once for itself.
//
//   s_j = scale q . k_j over the prefix's and the row's own keys;  lse = log sum_j exp s_j;  att = sum_j exp(s_j - lse) v_j
//
// in one pass over the keys with a running maximum and sum. A workgroup is four waves and one of two kinds of work:
//   prefix: one kv head, one span of the prefix, a tile of (row, query head) pairs - a wave takes 32 pairs and every key,
//           or, where the head has no more than 32 pairs, all the pairs and a quarter of the keys
//   own:    one row, one kv head, one span of the row's own keys; a wave a quarter of them
// and leaves states (maximum, sum, output) in the scratch, which a second launch folds in a fixed order. The spans are
// cut from the keys there are (the layout lies on the device), so a recorded launch holds while the rows grow.
//
// Sums and outputs are f32; a weight is rounded to bf16 for the product with V, as the matrix cores take it (relative
// 2-norm against 64 bits 2.1e-3 where rounding the output alone makes 1.7e-3), and the sum takes the unrounded weight.

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
    int prefix_states, states;                // states a (row, head): of the prefix, in all
};

struct Keys {
    int first, count;  // slots
};
// a stretch of slots as the layout gives it, kept within the cache and the capacity the launch was sized for
__device__ __forceinline__ Keys stretch(int off, int len, int most, int cap) {
    Keys k;
    k.first = min(max(off, 0), cap);
    k.count = off < 0 ? 0 : min(max(len, 0), min(most, cap - k.first));
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

// one wave's 32 pairs against its keys of a stretch. ALL: every key of the stretch, else the wave's tile of each stage.
// `row(c)`: the q row of pair c; `state(c)`: where pair c's state goes, negative: nowhere.
template <int D, bool ALL, class Row, class State>
__device__ __forceinline__ void walk(const SharedArgs& p, const uint16_t* Kg, const uint16_t* Vg, const Keys& keys, uint8_t* lds,
                                     Row row, State state) {
    constexpr int STEPS = D / 16, DT = D / 32, TILE = TK * 2 * D, REGS = TILE / 1024;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, h = lane >> 5;
    const float ninf = bits_f32(0xff800000u);
    bf16x8 qf[STEPS];
    {
        const uint16_t* qr = row(c) + 8 * h;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) qf[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(qr + 16 * s));
    }
    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = zero16();
    float m = ninf, l = 0.f;
    uint8_t* k_lds = lds;
    uint8_t* v_lds = lds + 4 * TILE;
    for (int kb = 0; kb < keys.count; kb += SH_KEYS) {
        // the wave's tile of the stage, keys past the end as zeros
        __syncthreads();
#pragma unroll
        for (int i = 0; i < REGS; ++i) {
            const int at = i * 64 + lane, key = at / (D / 8), chunk = at % (D / 8), j = kb + TK * wv + key;
            uint4 kw = make_uint4(0u, 0u, 0u, 0u), vw = kw;
            if (j < keys.count) {
                const size_t from = (size_t)(keys.first + j) * p.rs + 8 * chunk;
                kw = *reinterpret_cast<const uint4*>(Kg + from);
                vw = *reinterpret_cast<const uint4*>(Vg + from);
            }
            *reinterpret_cast<uint4*>(k_lds + wv * TILE + key * 2 * D + 16 * k_chunk<D>(key, chunk)) = kw;
            *reinterpret_cast<uint4*>(v_lds + wv * TILE + key * 2 * D + 16 * v_chunk(key, chunk)) = vw;
        }
        __syncthreads();
#pragma unroll 1
        for (int s = ALL ? 0 : wv; s < (ALL ? 4 : wv + 1); ++s) {
            const int left = keys.count - kb - TK * s;  // keys of this tile
            if (left <= 0) break;
            f32x16 st = zero16();
#pragma unroll
            for (int i = 0; i < STEPS; ++i) st = mfma32(k_fragment<D>(k_lds + s * TILE, i, lane), qf[i], st);
            float w[16];
            float top = ninf;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                w[i] = 8 * (i / 4) + 4 * h + i % 4 < left ? st[i] * p.scale_log2 : ninf;
                top = fmaxf(top, w[i]);
            }
            top = fmaxf(top, xor32(top));
            const float mn = fmaxf(m, top);
            const float corr = m == ninf ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                w[i] = w[i] == ninf ? 0.f : __builtin_amdgcn_exp2f(w[i] - mn);
                sum += w[i];
            }
            l = fmaf(l, corr, sum);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= corr;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const bf16x8 pf = weight_fragment(w + 8 * u);
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] = mfma32(v_fragment<D>(v_lds + s * TILE, d, u, lane), pf, o[d]);
            }
        }
    }
    l += xor32(l);
    const long long at = state(c);
    if (at < 0) return;
    if (h == 0) {
        p.part_m[at] = m;
        p.part_l[at] = l;
    }
    if (m == ninf) return;  // nothing seen (or nothing that is a number, which the sum says): the fold does not read the output
    float* dst = p.part_acc + (size_t)at * D + 4 * h;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b)
            *reinterpret_cast<float4*>(dst + 32 * d + 8 * b) = make_float4(o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]);
}

// MANY: a prefix workgroup takes 128 pairs, 32 a wave; else 32, every wave the same and a quarter of the keys
template <int D, bool MANY>
__global__ void __launch_bounds__(256, 2) attn_shared_kernel(SharedArgs p) {
    __shared__ __align__(16) uint8_t lds[8 * TK * 2 * D];
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pairs = p.T * p.G, prefix_wgs = p.Hk * p.pair_tiles * p.prefix_spans;
    int id = blockIdx.x;
    if (id < prefix_wgs) {
        const int g = id % p.Hk, sp = id / p.Hk % p.prefix_spans, tile = id / (p.Hk * p.prefix_spans);
        const Keys keys = part_of(stretch(p.lay[0], p.lay[1], p.prefix_cap, p.cap), sp, p.prefix_spans);
        const int r0 = MANY ? 128 * tile + 32 * wv : 0;
        auto row = [&](int c) {
            const int r = min(r0 + c, pairs - 1), t = r / p.G;
            return p.q + ((size_t)t * p.Hq + g * p.G + (r - t * p.G)) * D;
        };
        auto state = [&](int c) -> long long {
            const int r = r0 + c, t = r / p.G;
            if (r >= pairs) return -1;
            return ((long long)t * p.Hq + g * p.G + (r - t * p.G)) * p.states + (MANY ? sp : 4 * sp + wv);
        };
        walk<D, MANY>(p, p.K + (size_t)g * p.hs, p.V + (size_t)g * p.hs, keys, lds, row, state);
        return;
    }
    id -= prefix_wgs;
    const int g = id % p.Hk, t = id / p.Hk % p.T, sp = id / (p.Hk * p.T);
    const Keys keys = part_of(stretch(p.lay[2 + 2 * t], p.lay[3 + 2 * t], p.own_cap, p.cap), sp, p.own_spans);
    auto row = [&](int c) { return p.q + ((size_t)t * p.Hq + g * p.G + min(c, p.G - 1)) * D; };
    auto state = [&](int c) -> long long {
        return c < p.G ? ((long long)t * p.Hq + g * p.G + c) * p.states + p.prefix_states + 4 * sp + wv : -1;
    };
    walk<D, false>(p, p.K + (size_t)g * p.hs, p.V + (size_t)g * p.hs, keys, lds, row, state);
}

// a workgroup a (row, head): the states' common maximum, their factors, their outputs in a fixed order
template <int D>
__global__ void __launch_bounds__(256) attn_shared_fold_kernel(SharedArgs p, uint16_t* att, float* lse) {
    constexpr int LANES = D / 2, GROUPS = 256 / LANES;
    __shared__ float red[4], sums[4], acc[GROUPS][D];
    const int t = blockIdx.x / p.Hq, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    if (p.lay[3 + 2 * t] < 0) return;  // padding
    const size_t base = (size_t)blockIdx.x * p.states;
    const float ninf = bits_f32(0xff800000u);
    float m = ninf;
    for (int s = tid; s < p.states; s += 256) m = fmaxf(m, p.part_m[base + s]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, WAVE));
    if (lane == 0) red[wv] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    auto factor = [&](float ms) { return ms == ninf ? 0.f : __builtin_amdgcn_exp2f(ms - m); };
    float l = 0.f;
    for (int s = tid; s < p.states; s += 256) l = fmaf(factor(p.part_m[base + s]), p.part_l[base + s], l);
    l = wave_sum(l);
    if (lane == 0) sums[wv] = l;
    const int group = tid / LANES, dl = 2 * (tid % LANES);
    float a0 = 0.f, a1 = 0.f;
    for (int s = group; s < p.states; s += GROUPS) {
        const float ms = p.part_m[base + s];
        if (ms == ninf) continue;
        const float f = factor(ms);
        const float2 v = *reinterpret_cast<const float2*>(p.part_acc + (base + s) * D + dl);
        a0 = fmaf(f, v.x, a0);
        a1 = fmaf(f, v.y, a1);
    }
    acc[group][dl] = a0;
    acc[group][dl + 1] = a1;
    __syncthreads();
    l = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    if (tid < LANES) {
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            x += acc[i][2 * tid];
            y += acc[i][2 * tid + 1];
        }
        reinterpret_cast<uint32_t*>(att + (size_t)blockIdx.x * D)[tid] = l == 0.f ? 0u : f32x2_bf16(x / l, y / l);
    }
    if (tid == 0 && lse != nullptr) lse[blockIdx.x] = l == 0.f ? ninf : fmaf(m, 0.693147180559945309f, logf(l));
}

struct SharedPlan {
    bool many;
    int pair_tiles, prefix_spans, own_spans, prefix_states, states;
};
static SharedPlan shared_plan(size_t T, size_t Hq, size_t Hk, size_t prefix_cap, size_t own_cap) {
    const size_t pairs = T * (Hq / Hk), target = 2 * (size_t)device_info().cus;
    auto spans = [&](size_t groups, size_t cap) {
        const size_t most = (cap + SH_KEYS - 1) / SH_KEYS, want = (target + groups - 1) / groups;
        const size_t s = want < most ? want : most;
        return (int)(s > 0 ? s : 1);
    };
    SharedPlan r;
    r.many = pairs > 32;
    r.pair_tiles = r.many ? (int)((pairs + 127) / 128) : 1;
    r.prefix_spans = spans(Hk * r.pair_tiles, prefix_cap);
    r.own_spans = spans(Hk * T, own_cap);
    r.prefix_states = r.many ? r.prefix_spans : 4 * r.prefix_spans;
    r.states = r.prefix_states + 4 * r.own_spans;
    return r;
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
    const SharedPlan s = shared_plan(T, Hq, Hk, prefix_cap, own_cap);
    const size_t n = T * Hq * (size_t)s.states;
    return (2 * n + 3) / 4 * 4 + n * D;
}

int32_t btb_hip_attn_shared(const void* q, const void* K, const void* V, void* att, float* lse, const int32_t* layout,
                            size_t T, size_t Hq, size_t Hk, size_t D, size_t cap, int64_t hs, int64_t rs, float scale,
                            size_t prefix_cap, size_t own_cap, float* workspace, void* stream) {
    if (!q || !K || !V || !att || !layout || !workspace) return ERR_NULL;
    auto loose = [](const void* a) { return ((uintptr_t)a & 15u) != 0; };
    if (!shared_sizes_fit(T, Hq, Hk, D, prefix_cap, own_cap) || cap == 0 || cap > 0x7FFFFFFFu || prefix_cap > cap ||
        own_cap > cap || hs < 0 || rs < 0 || hs % 8 || rs % 8 || !(scale > 0.f) || !(scale < __builtin_inff()) || loose(q) ||
        loose(K) || loose(V) || loose(att) || loose(workspace)) {
        set_error("attn_shared: head_dim 64 or 128, up to 32 query heads a kv head, capacities within the cache's, a positive "
                  "scale, q, K, V, att and the workspace 16-byte aligned with strides in multiples of 8");
        return ERR_DOMAIN;
    }
    const SharedPlan s = shared_plan(T, Hq, Hk, prefix_cap, own_cap);
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
    p.prefix_states = s.prefix_states;
    p.states = s.states;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(Hk * ((size_t)s.pair_tiles * s.prefix_spans + T * s.own_spans)));
#define AS(DD)                                                                                   \
    do {                                                                                         \
        if (s.many)                                                                              \
            hipLaunchKernelGGL((attn_shared_kernel<DD, true>), grid, dim3(256), 0, st, p);       \
        else                                                                                     \
            hipLaunchKernelGGL((attn_shared_kernel<DD, false>), grid, dim3(256), 0, st, p);      \
        hipLaunchKernelGGL((attn_shared_fold_kernel<DD>), dim3((unsigned)(T * Hq)), dim3(256), 0, st, p, \
                           static_cast<uint16_t*>(att), lse);                                    \
    } while (0)
    if (D == 64)
        AS(64);
    else
        AS(128);
#undef AS
    return hip_status(hipGetLastError(), "attn_shared launch");
}

}  // extern "C"
