// The attention weight every cached key received from a pass, added to what it had:
//
//   out[g, j] = mass[g, j] + sum over rows t with j < seen[t], query heads h of g, of exp(scale q_{t,h} . k_j - lse[t, h])
//
// lse is what the pass's attention left (btb_hip_attn_shared). Scores are made as S = Q K^T, 32 pairs against 32 keys: lane (c, h)
// ends with key c's against pairs 8 (i / 4) + 4 h + i % 4, so a key's sum over the pairs is a lane's own and one exchange between
// the halves at the end. The order of the additions is fixed. Everything after the product is f32. Two kernels:
//
//   many pairs: a wave holds 64 keys as stationary operands and takes the pass's (row, head) pairs 32 at a time out of LDS, where the
//     workgroup's four waves bring them a stage ahead. A tile's weights are made between the next tile's products. Where keys are
//     few, the pairs are cut over workgroups too, whose sums a second launch adds in order. Bound: the products and the exponentials, a
//     multiply-add, a quarter-rate exponential and an addition a score beside a thirty-second of a product of 32 clocks a lane. 500 rows of
//     32 heads x 128 over 16384 keys 82 to 92 us by the chip (720 to 815 TFLOP/s), of which 13 bring the keys into registers; 4096 rows 544
//     to 566 us (970 to 1010 TFLOP/s), of 544 507 without the stages' loads and 398 (1384 TFLOP/s, the chip's rate for bare products) with no
//     exponential either.
//   few pairs (64 and less): they lie in LDS and the keys go by, a tile of 32 a wave ahead of the one at work. Bound: K's
//     trip from memory. 4 rows of 32 heads x 128 over 32000 keys 14.0 us (4.8 TB/s).

#include "btb_common.hpp"
#include "btb_tile32.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

constexpr int MA_KEYS = 256;   // many pairs: keys a workgroup, four waves of two tiles
constexpr int mass_stage(int D) { return 16384 / D; }  // pairs a stage: eight loads a wave
constexpr int MA_META = 1024;  // pairs whose log-sums and limits lie in LDS at a time
// few pairs, at most: two tiles, the most whose log-sums and limits fit a wave's registers. 64 pairs of 8 heads, us, few / many: over 32000 keys
// 16.4 / 26.3, over 2000 9.0 / 9.6; 72 pairs (many) over 32000: 26.0
constexpr int MA_FEW = 64;

struct MassArgs {
    const uint16_t* q;
    const uint16_t* K;
    const float* lse;      // [T, Hq], strides lr and lh
    const int32_t* seen;   // [T]
    const float* mass;     // rows of `ms` floats, or none
    float* out;            // rows of `os` floats
    float* work;           // [parts][Hk][n] where parts > 1
    long long hs, rs, ms, os, lr, lh;
    float scale_log2;
    int T, Hq, Hk, G, n, parts;
};

// A pair's log-sum in units of log 2 and how many keys it sees. A pair past the last, or one that saw nothing, sees none.
__device__ __forceinline__ void pair_facts(const MassArgs& p, int g, int r, int pairs, int row, float& z, int& seen) {
    z = 0.f;
    seen = 0;
    if (r < pairs) {
        const float raw = p.lse[row * p.lr + (g * p.G + (r - row * p.G)) * p.lh];
        if (raw != -__builtin_inff()) {
            z = raw * 1.44269504088896341f;
            seen = p.seen[row];
        }
    }
}
// the smallest of 32 lanes' numbers, in each
__device__ __forceinline__ int half_min(int v) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) v = min(v, __shfl_xor(v, d, WAVE));
    return v;
}
// sixteen of a tile's 32 values, those of the lane's pairs, from LDS
__device__ __forceinline__ void of_pairs(const float* from, int h, float (&v)[16]) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const float4 x = *reinterpret_cast<const float4*>(from + 8 * b + 4 * h);
        v[4 * b] = x.x;
        v[4 * b + 1] = x.y;
        v[4 * b + 2] = x.z;
        v[4 * b + 3] = x.w;
    }
}

template <int D>
__global__ void __launch_bounds__(256, 2) attn_mass_kernel(MassArgs p) {
    constexpr int STEPS = D / 16, CH = D / 8, KPI = 64 / CH;
    constexpr int STAGE = mass_stage(D), TILES = STAGE / 32, TILE = TK * 2 * D, AHEAD = 4;
    static_assert(STAGE == 32 * KPI, "a wave's eight loads bring a quarter of the stage");
    __shared__ __align__(16) uint8_t q_lds[2][TILES * TILE];
    __shared__ __align__(16) float logs[MA_META];
    __shared__ __align__(16) int limits[MA_META];
    __shared__ int least[MA_META / 32];  // the smallest limit of a tile
    const int g = blockIdx.y, lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
    const int k0 = blockIdx.x * MA_KEYS + 64 * wv;
    const int pairs = p.T * p.G, stages = (pairs + STAGE - 1) / STAGE;
    const int per = (stages + p.parts - 1) / p.parts, first = blockIdx.z * per, end = min(first + per, stages);
    // the lane's pairs of a stage: STAGE s + mine + KPI i. r / G by multiplication (G <= 32, r < 2^24: exact)
    const int mine = 8 * KPI * wv + lane / CH;
    const uint32_t by_g = 0xFFFFFFFFu / (uint32_t)p.G + 1;
    auto row_of = [&](int r) { return p.G == 1 ? r : (int)__umulhi((uint32_t)r, by_g); };
    const char* qb = reinterpret_cast<const char*>(uniform(p.q));
    auto issue = [&](int s, int b) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t off[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = mine + KPI * (4 * half + i), r = min(s * STAGE + at, pairs - 1), t = row_of(r);
                off[i] = (uint32_t)(t * p.Hq + g * p.G + (r - t * p.G)) * (2 * D) + 16 * k_chunk<D>(at & 31, lane % CH);
            }
            const uint32_t to = lds_address(&q_lds[b][(8 * KPI * wv + 4 * KPI * half) * 2 * D]);
            load4_to_lds(qb, 0, off[0], off[1], off[2], off[3], (uint32_t)__builtin_amdgcn_readfirstlane((int)to));
        }
    };
    bf16x8 kf[2][STEPS];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint16_t* kr = p.K + (size_t)g * p.hs + (size_t)min(k0 + 32 * k + c, p.n - 1) * p.rs + 8 * h;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) kf[k][s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(kr + 16 * s));
    }
    // a tile's scores against the wave's two tiles of keys, its pairs' log-sums, its first pair among those in `logs`, and whether
    // its pairs see all of the wave's keys
    struct Tile {
        f32x16 s[2];
        float z[16];
        int pair, least;
    };
    Tile one, two;
    float sum[2] = {0.f, 0.f};
    auto empty = [&](Tile& t) {  // no tile: weights of zero
#pragma unroll
        for (int k = 0; k < 2; ++k) t.s[k] = zero16();
#pragma unroll
        for (int i = 0; i < 16; ++i) t.z[i] = __builtin_inff();
        t.pair = 0;
        t.least = 0x7FFFFFFF;
    };
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
    constexpr int EACH = 16 / STEPS;
    auto weigh = [&](const Tile& t, int step) {  // keys that every pair of the tile sees
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i / EACH == step)
#pragma unroll
                for (int k = 0; k < 2; ++k) sum[k] += __builtin_amdgcn_exp2f(fmaf(t.s[k][i], p.scale_log2, -t.z[i]));
    };
    auto weigh_seen = [&](const Tile& t) {
        float lim[16];
        of_pairs(reinterpret_cast<const float*>(limits) + t.pair, h, lim);
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                sum[k] += k0 + 32 * k + c < __builtin_bit_cast(int, lim[i])
                              ? __builtin_amdgcn_exp2f(fmaf(t.s[k][i], p.scale_log2, -t.z[i]))
                              : 0.f;
    };
    auto settle = [&](const Tile& t) {
        if (t.least >= k0 + 64) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) weigh(t, i);
        } else {
            weigh_seen(t);
        }
    };
    // Tile q of the stage: its scores into `to` while `from` is weighed. Its first fragments are in `head`; the next tile's come
    // into it on the way.
    bf16x8 head[AHEAD];
    auto step = [&](const Tile& from, Tile& to, const uint8_t* tiles, uint32_t at, int q, int pair) {
        to.pair = pair;
        to.least = least[pair / 32];
        of_pairs(logs + pair, h, to.z);
        auto scores = [&](auto work) {
            bf16x8 qf[STEPS + AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) qf[i] = head[i];
#pragma unroll
            for (int k = 0; k < 2; ++k) to.s[k] = zero16();
            fence();
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                if (i + AHEAD < STEPS || q + 1 < TILES)
                    qf[i + AHEAD] = k_fragment(tiles, at, (q + (i + AHEAD) / STEPS) * TILE, (i + AHEAD) % STEPS);
#pragma unroll
                for (int k = 0; k < 2; ++k) to.s[k] = mfma32(qf[i], kf[k][i], to.s[k]);
                work(i);
                fence();
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) head[i] = qf[q + 1 < TILES ? STEPS + i : i];
        };
        if (from.least >= k0 + 64) {
            scores([&](int i) { weigh(from, i); });
        } else {
            scores([](int) {});
            weigh_seen(from);
        }
    };
    empty(one);
    if (first < end) issue(first, 0);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the keys are here, and no register of the loop waits for a load
    fence();
    const uint32_t place = k_place<D>(lane);
    for (int s = first; s < end; ++s) {
        const int b = (s - first) & 1, at_meta = (s - first) * STAGE % MA_META;
        if (at_meta == 0) {  // uniform
            settle(one);
            empty(one);
            __syncthreads();
            for (int e = threadIdx.x; e < MA_META; e += 256) {
                const int r = s * STAGE + e;
                int seen;
                pair_facts(p, g, r, pairs, row_of(min(r, pairs - 1)), logs[e], seen);
                limits[e] = seen;
                const int low = half_min(seen);
                if (c == 0) least[e / 32] = low;
            }
        }
        uint32_t at = place;
        wait_loads<0>(at);
        __syncthreads();  // the stage is here, and the other buffer free
        if (s + 1 < end) issue(s + 1, b ^ 1);
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) head[i] = k_fragment(q_lds[b], at, 0, i);
#pragma unroll
        for (int q = 0; q < TILES; q += 2) {
            asm volatile("" : "+v"(at));  // eight places a lane are made each time and not kept
            step(one, two, q_lds[b], at, q, at_meta + 32 * q);
            step(two, one, q_lds[b], at, q + 1, at_meta + 32 * q + 32);
        }
    }
    settle(one);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float v = sum[k] + xor32(sum[k]);
        const int key = k0 + 32 * k + c;
        if (h == 0 && key < p.n) {
            if (p.parts > 1)
                p.work[((size_t)blockIdx.z * p.Hk + g) * p.n + key] = v;
            else
                p.out[(size_t)g * p.os + key] = v + (p.mass != nullptr ? p.mass[(size_t)g * p.ms + key] : 0.f);
        }
    }
}

// Few pairs: QT tiles of 32. A wave of eight takes every (8 gridDim.x)-th tile of a head's keys, two LDS buffers of its own. Sums
// meet the mass they are added to eight tiles at a time: the wait for a loaded register waits for the keys on their way too.
template <int D, int QT>
__global__ void __launch_bounds__(512, 2) attn_mass_few_kernel(MassArgs p) {
    constexpr int STEPS = D / 16, TILE = TK * 2 * D, N = TileLoads<D>::N;
    extern __shared__ __align__(16) uint8_t lds[];  // [8 waves][2] tiles of keys
    __shared__ __align__(16) float logs[32 * QT];
    __shared__ __align__(16) int limits[32 * QT];
    __shared__ float kept[8][8][32];
    const int g = blockIdx.y, lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
    const int pairs = p.T * p.G, tiles = (p.n + TK - 1) / TK, step = 8 * gridDim.x;
    const uint16_t* Kg = p.K + (size_t)g * p.hs;
    uint8_t* mine = lds + wv * 2 * TILE;
    TileLoads<D> loads;
    loads.make(p.rs, lane);
    auto issue = [&](int tile, int b) {
        loads.template issue<true>(Kg + (size_t)tile * TK * p.rs, p.rs, p.n - tile * TK, mine + b * TILE, lane);
    };
    const int first = blockIdx.x + gridDim.x * wv;
    if (first < tiles) issue(first, 0);
    if (threadIdx.x < 32 * QT) {
        const int r = threadIdx.x;
        int seen;
        pair_facts(p, g, r, pairs, min(r, pairs - 1) / p.G, logs[r], seen);
        limits[r] = seen;
    }
    bf16x8 qf[QT][STEPS];
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        const int r = min(32 * q + c, pairs - 1), t = r / p.G;
        const uint16_t* qr = p.q + ((size_t)t * p.Hq + g * p.G + (r - t * p.G)) * D + 8 * h;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) qf[q][s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(qr + 16 * s));
    }
    __syncthreads();  // (and every load so far: the counted waits below find only the keys')
    float z[QT][16], lim[QT][16];
    int least = 0x7FFFFFFF;
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        of_pairs(logs + 32 * q, h, z[q]);
        of_pairs(reinterpret_cast<const float*>(limits) + 32 * q, h, lim[q]);
        least = min(least, half_min(limits[32 * q + c]));
    }
    least = __builtin_amdgcn_readfirstlane(least);
    const uint32_t place = k_place<D>(lane);
    int held = 0;
    for (int tile = first, b = 0; tile < tiles; tile += step, b ^= 1) {
        uint32_t at = place;
        if (tile + step < tiles) {
            issue(tile + step, b ^ 1);
            wait_loads<N>(at);
        } else {
            wait_loads<0>(at);
        }
        const int key = tile * TK + c;
        f32x16 st[QT];
#pragma unroll
        for (int q = 0; q < QT; ++q) st[q] = zero16();
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const bf16x8 kf = k_fragment(mine + b * TILE, at, 0, i);
#pragma unroll
            for (int q = 0; q < QT; ++q) st[q] = mfma32(qf[q][i], kf, st[q]);
        }
        float sum = 0.f;
        if (least >= tile * TK + TK) {
#pragma unroll
            for (int q = 0; q < QT; ++q)
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(fmaf(st[q][i], p.scale_log2, -z[q][i]));
        } else {
#pragma unroll
            for (int q = 0; q < QT; ++q)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    sum += key < __builtin_bit_cast(int, lim[q][i]) ? __builtin_amdgcn_exp2f(fmaf(st[q][i], p.scale_log2, -z[q][i])) : 0.f;
        }
        sum += xor32(sum);
        if (h == 0) kept[wv][held][c] = sum;
        ++held;
        if (held == 8 || tile + step >= tiles) {  // uniform
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const int key = (tile - (held - 1 - i - h) * step) * TK + c;
                if (i + h < held && key < p.n)
                    p.out[(size_t)g * p.os + key] = kept[wv][i + h][c] + (p.mass != nullptr ? p.mass[(size_t)g * p.ms + key] : 0.f);
            }
            held = 0;
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

__global__ void __launch_bounds__(256) attn_mass_add_kernel(MassArgs p) {
    const int key = blockIdx.x * 256 + threadIdx.x, g = blockIdx.y;
    if (key >= p.n) return;
    float v = 0.f;
#pragma unroll 8
    for (int i = 0; i < p.parts; ++i) v += p.work[((size_t)i * p.Hk + g) * p.n + key];
    p.out[(size_t)g * p.os + key] = v + (p.mass != nullptr ? p.mass[(size_t)g * p.ms + key] : 0.f);
}

// Workgroups the pairs are cut over, a stage each or more: until there are two a CU, and from more than 256 pairs on, whose second
// launch costs less than their stages one after the other. 8 heads of 128, us, cut / whole: 500 rows over 512 keys 13.5 / 43, over 2000
// 22.3 / 60, over 8000 53 / 54; 96 rows over 4000 15.5 / 15.5, 90 over 700 14.2 / 16; 64 rows (256 pairs) over 4000 14.8 / 12.1. Heads of
// 64: 500 rows over 512 14.1 with a stage each, 15.2 with two; 70 rows over 4000 14.3 / 15.5.
static int mass_parts(size_t T, size_t Hq, size_t Hk, size_t D, size_t n) {
    const size_t pairs = T * (Hq / Hk), stage = (size_t)mass_stage((int)D);
    if (pairs <= 256) return 1;
    const size_t wgs = Hk * ((n + MA_KEYS - 1) / MA_KEYS), stages = (pairs + stage - 1) / stage;
    const size_t want = 2 * (size_t)device_info().cus / wgs, parts = want < stages ? want : stages;
    if (parts < 2) return 1;
    const size_t per = (stages + parts - 1) / parts;
    return (int)((stages + per - 1) / per);  // none without a stage
}
static bool mass_sizes_fit(size_t T, size_t Hq, size_t Hk, size_t D, size_t n) {
    return T > 0 && Hk > 0 && Hk <= 1024 && Hq > 0 && Hq % Hk == 0 && Hq / Hk <= 32 && T <= (1u << 23) / Hq && (D == 64 || D == 128) &&
           n > 0 && n <= 0x7FFFFF00u;
}

template <int D, int QT>
static int32_t launch_few(const MassArgs& p, hipStream_t st) {
    constexpr int lds = 16 * TK * 2 * D;
    const void* kern = reinterpret_cast<const void*>(attn_mass_few_kernel<D, QT>);
    if (lds > 60 * 1024) {
        const hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return hip_status(e, "hipFuncSetAttribute");
    }
    // a workgroup a CU, a tile a wave at least
    const int tiles = (p.n + TK - 1) / TK, cus = device_info().cus, most = (tiles + 7) / 8, want = (cus + p.Hk - 1) / p.Hk;
    const dim3 grid((unsigned)(want < most ? want : most), (unsigned)p.Hk);
    hipLaunchKernelGGL((attn_mass_few_kernel<D, QT>), grid, dim3(512), lds, st, p);
    return hip_status(hipGetLastError(), "attn_mass launch");
}

}  // namespace btb

using namespace btb;

extern "C" {

size_t btb_hip_attn_mass_floats(size_t T, size_t Hq, size_t Hk, size_t D, size_t n) {
    if (!mass_sizes_fit(T, Hq, Hk, D, n)) return 0;
    const size_t parts = (size_t)mass_parts(T, Hq, Hk, D, n);
    return parts > 1 ? parts * Hk * n : 0;
}

int32_t btb_hip_attn_mass(const void* q, const void* K, const float* lse, const int32_t* seen, const float* mass, float* out,
                          size_t T, size_t Hq, size_t Hk, size_t D, size_t n, int64_t hs, int64_t rs, int64_t mass_stride,
                          int64_t out_stride, int64_t lse_row, int64_t lse_head, float scale, float* workspace, void* stream) {
    if (!q || !K || !lse || !seen || !out) return ERR_NULL;
    auto loose = [](const void* a) { return ((uintptr_t)a & 15u) != 0; };
    if (!mass_sizes_fit(T, Hq, Hk, D, n) || hs < 0 || rs < 0 || rs > (1 << 25) || hs % 8 || rs % 8 || mass_stride < 0 || out_stride < 0 || (Hk > 1 && (size_t)out_stride < n) || lse_row < 0 || lse_head < 0 ||
        !(scale > 0.f) || !(scale < __builtin_inff()) || loose(q) || loose(K)) {
        set_error("attn_mass: head_dim 64 or 128, up to 32 query heads a kv head, a positive scale, q and K 16-byte aligned "
                  "with strides in multiples of 8, a row's up to 2^25, out's heads apart");
        return ERR_DOMAIN;
    }
    const int parts = mass_parts(T, Hq, Hk, D, n);
    if (parts > 1 && workspace == nullptr) return ERR_NULL;
    MassArgs p;
    p.q = static_cast<const uint16_t*>(q);
    p.K = static_cast<const uint16_t*>(K);
    p.lse = lse;
    p.seen = seen;
    p.mass = mass;
    p.out = out;
    p.work = workspace;
    p.parts = parts;
    p.Hk = (int)Hk;
    p.hs = hs;
    p.rs = rs;
    p.ms = mass_stride;
    p.os = out_stride;
    p.lr = lse_row;
    p.lh = lse_head;
    p.scale_log2 = scale * 1.44269504088896341f;
    p.T = (int)T;
    p.Hq = (int)Hq;
    p.G = (int)(Hq / Hk);
    p.n = (int)n;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const size_t pairs = T * (Hq / Hk);
    if (pairs <= (size_t)MA_FEW) {
        if (D == 64) return pairs <= 32 ? launch_few<64, 1>(p, st) : launch_few<64, 2>(p, st);
        return pairs <= 32 ? launch_few<128, 1>(p, st) : launch_few<128, 2>(p, st);
    }
    const dim3 grid((unsigned)((n + MA_KEYS - 1) / MA_KEYS), (unsigned)Hk, (unsigned)parts);
    if (D == 64)
        hipLaunchKernelGGL(attn_mass_kernel<64>, grid, dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL(attn_mass_kernel<128>, grid, dim3(256), 0, st, p);
    if (parts > 1) hipLaunchKernelGGL(attn_mass_add_kernel, dim3((unsigned)((n + 255) / 256), (unsigned)Hk), dim3(256), 0, st, p);
    return hip_status(hipGetLastError(), "attn_mass launch");
}

}  // extern "C"
