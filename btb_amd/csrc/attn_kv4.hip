// Attention of each sequence's last rows over its pages of a cache held in 4 bits (btb_kv4.hpp).
//
//   s_j = scale q . k_j for j = 0 .. the row's position,  lse = log sum_j exp s_j,  att = sum_j exp(s_j - lse) v_j
//
// A wave has 32 (row, query head) pairs of a sequence and kv head, and walks tiles of 32 tokens with a running maximum and sum.
// S^T = K Q^T by v_mfma_f32_32x32x16_bf16, a key's codes times their power of two as bf16, which they are exactly, two a conversion. (The
// products that take the codes as they lie, v_mfma_scale_f32_32x32x64_f8f6f4, lose what is 2^-13 of the largest term: with q as two e4m3
// terms that was 5e-6 of lse.) A pair's scores against keys 8 (i / 4) + 4 h + i % 4 are then lane
// (pair, h)'s own, and V lies in the same order: out^T += V^T P by v_mfma_f32_32x32x16_f16, the codes as f16, which they are exactly,
// a value's scale in its weight.
//
// Weights are f16, off by 2^-12 of themselves at most: e^(s - maximum) times 2^11 times the value's scale over the power of two `unit`, the
// largest one so far: at most 2^15 (the maximum may lag by 2^4), in full precision down to 2^-25 of the largest, and 2^-36 of it is lost at most. A
// bf16 weight would be off by 2^-9, two of them cost twice the products.

#include "btb_kv4.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float NONE = -3.0e38f;   // a maximum of nothing: what is subtracted from it underflows to weight 0
constexpr float LAG = 4.f;         // how far, in powers of two, scores may pass the maximum in use
constexpr int PAIRS = 32;          // (row, query head) pairs a wave

struct AttnKv4 {
    Kv4Seqs seqs;
    const uint16_t* q;
    const uint8_t* cache;
    uint16_t* att;
    float* lse;
    float* part;     // a pair's spans: maximum and sum [T Hq, S, 2], then outputs [T Hq, S, D]
    float c;         // scale log2(e)
    int Hq, Hk, G;
    int items;       // tiles of pairs a sequence, where each has as many rows
    int S, span;     // spans a sequence at most, tiles a span at least
};

// spans of a sequence of `tiles` tiles: how many, and how long
__device__ __forceinline__ int kv4_span(const AttnKv4& p, int tiles) { return max(p.span, (tiles + p.S - 1) / p.S); }

// q's fragment, exact: 8 dims a product, lane (pair, h) dims 64 step + 32 h + 8 j .. + 7 of the pair's row for product j of a step, as K's
// codes lie (the order of the dims is free as long as both operands have it)
template <int D>
struct QueryFragment {
    bf16x8 x[D / 16];

    __device__ __forceinline__ void make(const uint16_t* q, bool there, int h) {
#pragma unroll
        for (int s = 0; s < D / 64; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (there) w = *reinterpret_cast<const uint4*>(q + 64 * s + 32 * h + 8 * j);
                x[4 * s + j] = __builtin_bit_cast(bf16x8, w);
            }
    }
};

// a tile as a lane holds it
template <int D>
struct Kv4Fragment {
    uint4 k[D / 64], v[D / 64];
    uint32_t e;     // D / 64 exponents
    uint4 s[2];     // the half's sixteen scales

    __device__ __forceinline__ void load(const uint8_t* tile, int lane) {
        using Tile = Kv4Tile<D>;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            k[i] = load_stream16(reinterpret_cast<const uint4*>(tile) + 64 * i + lane);
            v[i] = load_stream16(reinterpret_cast<const uint4*>(tile + Tile::V) + 64 * i + lane);
        }
        e = D == 128 ? reinterpret_cast<const uint16_t*>(tile + Tile::KS)[lane] : tile[Tile::KS + lane];
#pragma unroll
        for (int i = 0; i < 2; ++i) s[i] = reinterpret_cast<const uint4*>(tile + Tile::VS + 32 * (lane >> 5))[i];
    }
};

__device__ __forceinline__ uint32_t dword(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }

__device__ __forceinline__ f16x8 codes_f16(uint32_t w) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 1);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 3);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ bf16x8 codes_bf16(uint32_t w, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// a wave's pairs over the tiles it has been given
template <int D>
struct Walk {
    static constexpr int DT = D / 32;
    f32x16 o[DT];
    float m, l, unit;

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
        m = NONE, l = 0.f;
        unit = bits_f32(27u << 23);  // 2^-100
    }

    // `left`: tokens of the tile the lane's pair sees; `there`: that any pair does; MASKED: some pair does not see all 32
    template <bool MASKED>
    __device__ __forceinline__ void tile(const Kv4Fragment<D>& f, const QueryFragment<D>& q, float c, int left, int there, int lane) {
        const int h = lane >> 5;
        f32x16 z;
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0.f;
#pragma unroll
        for (int s = 0; s < D / 64; ++s) {
            // (the conversion reads the exponent's field alone: 0 is 2^-127, 255 makes of the zeros that go with it NaN)
            const float scale = bits_f32((s ? f.e >> 8 : f.e & 0xFFu) << 23);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(codes_bf16(dword(f.k[s], j), scale), q.x[4 * s + j], z, 0, 0, 0);
        }
        uint32_t sc[8] = {f.s[0].x, f.s[0].y, f.s[0].z, f.s[0].w, f.s[1].x, f.s[1].y, f.s[1].z, f.s[1].w};
        if (MASKED) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int token = kv4_token(h, i);
                if (token >= left) z[i] = -__builtin_inff();
                if (token >= there) sc[i / 2] &= i % 2 ? 0x0000FFFFu : 0xFFFF0000u;
            }
        }
        float top = z[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, z[i]);
        top = fmaxf(top, xor32(top)) * c;
        if (__any(top > m + LAG)) {
            const float to = fmaxf(m, top), by = __builtin_amdgcn_exp2f(m - to);
            l *= by;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= by;
            m = to;
        }
        // the largest scale: as signed 16-bit numbers, of which NaN is the least
        typedef __attribute__((ext_vector_type(2))) short i16x2;
        i16x2 big = __builtin_bit_cast(i16x2, sc[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) big = __builtin_elementwise_max(big, __builtin_bit_cast(i16x2, sc[i]));
        int most = max((int)big[0], (int)big[1]);
        most = max(most, __builtin_bit_cast(int, xor32(__builtin_bit_cast(float, most))));
        most = __builtin_amdgcn_readfirstlane(most);
        const float power = bits_f32(((uint32_t)(max(most, 0) & 0x7F80) + 0x80u) << 16);  // the power of two above it
        if (power > unit) {
            const float by = unit / power;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= by;
            unit = power;
        }
        const float inv = bits_f32((265u << 23) - f32_bits(unit));  // 2^11 / unit
        f16x8 w[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(z[i], c, -m));
            l += p;
            const float sv = (i % 2 ? bf16hi_f32(sc[i / 2]) : bf16lo_f32(sc[i / 2])) * inv;
            float ps = p * sv;
            if (MASKED && kv4_token(h, i) >= left) ps = 0.f;
            w[i / 8][i % 8] = (_Float16)ps;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int d = 0; d < DT; ++d)
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(codes_f16(dword(f.v[d / 2], 2 * (d % 2) + u)), w[u], o[d], 0, 0, 0);
    }
};

// SHARE: the workgroup's four waves have a tile of pairs each and the same span; else one tile of pairs, its span dealt out among them
template <int D, bool SHARE>
__global__ void __launch_bounds__(256, 2) attn_kv4_kernel(AttnKv4 p) {
    constexpr int DT = D / 32, PITCH = D + 4;
    __shared__ float meet[SHARE ? 1 : 2][SHARE ? 1 : PAIRS][SHARE ? 1 : PITCH];
    __shared__ float meet_m[2][PAIRS], meet_l[2][PAIRS];
    const int lane = threadIdx.x & 63, pair = lane & 31, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hk = blockIdx.x % p.Hk, rest = blockIdx.x / p.Hk, span = rest % p.S;
    const int per_group = SHARE ? 4 * PAIRS : PAIRS;
    auto groups = [&](int b) {
        int row0, n;
        p.seqs.of(b, row0, n);
        return (int)(((long long)n * p.G + per_group - 1) / per_group);
    };
    int b, item;
    if (p.seqs.first == nullptr)
        b = rest / p.S / p.items, item = rest / p.S % p.items;
    else
        kv4_find(rest / p.S, p.seqs.B, b, item, groups);
    if (b < 0) return;
    b = __builtin_amdgcn_readfirstlane(b), item = __builtin_amdgcn_readfirstlane(item);
    int row0, n;
    p.seqs.of(b, row0, n);
    const int len = p.seqs.len(b), tiles = (len + KV4_TOKENS - 1) / KV4_TOKENS, length = kv4_span(p, tiles);
    const int spans = max(1, (tiles + length - 1) / length);
    if (span >= spans) return;
    const int pairs = n * p.G, pair0 = item * per_group + (SHARE ? wave * PAIRS : 0);
    if (SHARE && pair0 >= pairs) return;  // (no barrier follows in this form)
    const int mine = pair0 + pair;
    const bool there = mine < pairs;
    const int row = there ? mine / p.G : 0, head = hk * p.G + (there ? mine % p.G : 0);
    const size_t place = (size_t)(row0 + row) * p.Hq + head;  // the pair's row and head in q, att and lse
    QueryFragment<D> q;
    q.make(p.q + place * D, there, h);
    // tokens the pair sees, and what every pair of the wave sees
    const int sees = there ? len - n + row + 1 : 0;
    const int last = min(pair0 + PAIRS, pairs) - 1;
    const int all = len - n + pair0 / p.G + 1, any = len - n + last / p.G + 1;
    const int from = span * length + (SHARE ? 0 : wave), to = min(min((span + 1) * length, tiles), (any + KV4_TOKENS - 1) / KV4_TOKENS);
    constexpr int STEP = SHARE ? 1 : 4;

    Walk<D> w;
    w.begin();
    const uint8_t* cache = p.cache;
    // places of the next 64 tiles, one a lane
    long long at = -1, ahead = -1;
    auto places = [&](int j) { return j + STEP * lane < to ? p.seqs.at(b, j + STEP * lane, hk) : -1; };
    auto take = [&](int i) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)at, i);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)at >> 32), i);
        return (long long)((uint64_t)hi << 32 | lo);
    };
    auto step = [&](const Kv4Fragment<D>& f, long long where, int j) {
        if (where < 0) return;  // no page of the pool: its tokens are not there
        const int first = j * KV4_TOKENS;
        if (first + KV4_TOKENS <= all)
            w.template tile<false>(f, q, p.c, 32, 32, lane);
        else
            w.template tile<true>(f, q, p.c, sees - first, len - first, lane);
    };
    for (int base = from; base < to; base += 64 * STEP) {
        at = base == from ? places(base) : ahead;
        ahead = places(base + 64 * STEP);
        const int count = min((to - base + STEP - 1) / STEP, 64);
        Kv4Fragment<D> f[2];
        long long where[2];
        where[0] = take(0);
        f[0].load(cache + max(where[0], 0ll), lane);
        for (int i = 0; i < count; i += 2) {
            where[1] = -1;
            if (i + 1 < count) {
                where[1] = take(i + 1);
                f[1].load(cache + max(where[1], 0ll), lane);
            }
            step(f[0], where[0], base + STEP * i);
            if (i + 2 < count) {
                where[0] = take(i + 2);
                f[0].load(cache + max(where[0], 0ll), lane);
            }
            if (i + 1 < count) step(f[1], where[1], base + STEP * (i + 1));
        }
    }
    float l = w.l + xor32(w.l), m = w.m;
    const float real = w.unit * bits_f32(116u << 23);  // unit / 2^11
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) w.o[d][i] *= real;
    if constexpr (!SHARE) {
        // the four waves' states, two and two
        for (int half = 2; half >= 1; half /= 2) {
            if (half == 1) __syncthreads();
            if (wave >= half && wave < 2 * half) {
                if (h == 0) meet_m[wave - half][pair] = m, meet_l[wave - half][pair] = l;
                if (there)
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int i = 0; i < 16; i += 4)
                            *reinterpret_cast<float4*>(&meet[wave - half][pair][32 * d + 2 * i + 4 * h]) =
                                make_float4(w.o[d][i], w.o[d][i + 1], w.o[d][i + 2], w.o[d][i + 3]);
            }
            __syncthreads();
            if (wave < half) {
                const float m2 = meet_m[wave][pair], l2 = meet_l[wave][pair], to_m = fmaxf(m, m2);
                const float a = __builtin_amdgcn_exp2f(m - to_m), a2 = __builtin_amdgcn_exp2f(m2 - to_m);
                l = l * a + l2 * a2;
                m = to_m;
                if (there)
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const float4 x = *reinterpret_cast<const float4*>(&meet[wave][pair][32 * d + 2 * i + 4 * h]);
                            w.o[d][i] = fmaf(w.o[d][i], a, x.x * a2);
                            w.o[d][i + 1] = fmaf(w.o[d][i + 1], a, x.y * a2);
                            w.o[d][i + 2] = fmaf(w.o[d][i + 2], a, x.z * a2);
                            w.o[d][i + 3] = fmaf(w.o[d][i + 3], a, x.w * a2);
                        }
            }
        }
        if (wave != 0) return;
    }
    if (!there) return;
    if (spans == 1) {
        const float by = l == 0.f ? 0.f : 1.f / l;
        uint16_t* out = p.att + place * D;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<uint2*>(out + 32 * d + 2 * i + 4 * h) =
                    make_uint2(f32x2_bf16(w.o[d][i] * by, w.o[d][i + 1] * by), f32x2_bf16(w.o[d][i + 2] * by, w.o[d][i + 3] * by));
        if (p.lse != nullptr && h == 0) p.lse[place] = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * LN2;
        return;
    }
    const size_t slot = place * p.S + span;
    if (h == 0) reinterpret_cast<float2*>(p.part)[slot] = make_float2(m, l);
    float* out = p.part + 2 * (size_t)p.seqs.T * p.Hq * p.S + slot * D;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(out + 32 * d + 2 * i + 4 * h) =
                make_float4(w.o[d][i], w.o[d][i + 1], w.o[d][i + 2], w.o[d][i + 3]);
}

// The spans of a row and head, in their order: a workgroup each, its waves a quarter of them each.
template <int D>
__global__ void __launch_bounds__(256) attn_kv4_join_kernel(AttnKv4 p) {
    constexpr int V = D / 64;
    __shared__ float sum_o[4][D], sum_m[4], sum_l[4];
    const int t = blockIdx.x / p.Hq, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int b = -1;
    if (p.seqs.first == nullptr) {
        b = t / p.seqs.rows;
    } else {
        for (int b0 = 0; b0 < p.seqs.B && b < 0; b0 += 64) {
            bool mine = false;
            if (b0 + lane < p.seqs.B) {
                int row0, n;
                p.seqs.of(b0 + lane, row0, n);
                mine = t >= row0 && t < row0 + n;
            }
            const uint64_t found = __ballot(mine);
            if (found != 0) b = b0 + __ffsll((unsigned long long)found) - 1;
        }
        if (b < 0) return;
    }
    const int tiles = (p.seqs.len(b) + KV4_TOKENS - 1) / KV4_TOKENS, length = kv4_span(p, tiles);
    const int spans = (tiles + length - 1) / length;
    if (spans <= 1) return;
    const size_t place = blockIdx.x;
    const float2* ml = reinterpret_cast<const float2*>(p.part) + place * p.S;
    const float* o = p.part + 2 * (size_t)p.seqs.T * p.Hq * p.S + place * p.S * D + V * lane;
    const int quarter = (spans + 3) / 4, first = wave * quarter, end = min(first + quarter, spans);
    float m = NONE, l = 0.f, sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    for (int j = first; j < end; j += 4) {
        float2 x[4];
        float y[4][V];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int at = min(j + u, end - 1);
            x[u] = ml[at];
#pragma unroll
            for (int i = 0; i < V; ++i) y[u][i] = o[(size_t)at * D + i];
            if (j + u >= end) x[u] = make_float2(NONE, 0.f);
        }
        float to = m;
#pragma unroll
        for (int u = 0; u < 4; ++u) to = fmaxf(to, x[u].x);
        const float by = __builtin_amdgcn_exp2f(m - to);
        l *= by;
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] *= by;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (j + u >= end) continue;
            const float a = __builtin_amdgcn_exp2f(x[u].x - to);
            l = fmaf(x[u].y, a, l);
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = fmaf(y[u][i], a, sum[i]);
        }
        m = to;
    }
    if (lane == 0) sum_m[wave] = m, sum_l[wave] = l;
#pragma unroll
    for (int i = 0; i < V; ++i) sum_o[wave][V * lane + i] = sum[i];
    __syncthreads();
    if (wave != 0) return;
    float to = NONE, total = 0.f, out[V];
#pragma unroll
    for (int u = 0; u < 4; ++u) to = fmaxf(to, sum_m[u]);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const float a = __builtin_amdgcn_exp2f(sum_m[u] - to);
        total = fmaf(sum_l[u], a, total);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = fmaf(sum_o[u][V * lane + i], a, out[i]);
    }
    const float by = total == 0.f ? 0.f : 1.f / total;
    uint16_t* att = p.att + place * D + V * lane;
    if constexpr (V == 2)
        *reinterpret_cast<uint32_t*>(att) = f32x2_bf16(out[0] * by, out[1] * by);
    else
        *att = f32_bf16(out[0] * by);
    if (p.lse != nullptr && lane == 0) p.lse[place] = total == 0.f ? -__builtin_inff() : (to + __builtin_amdgcn_logf(total)) * LN2;
}

// How a call is cut, from what the host knows: tiles of pairs a sequence, one or four a workgroup, and spans.
struct Kv4Plan {
    bool share;
    int items;        // workgroups a sequence, where each has as many rows
    long long groups; // workgroups a kv head and span
    int S, span;
};
static Kv4Plan kv4_plan(size_t T, size_t B, size_t Hk, size_t G, size_t keys_cap, bool ragged) {
    Kv4Plan plan;
    const size_t R = T / B;
    plan.share = (T + B - 1) / B * G > 2 * PAIRS;
    const size_t per = plan.share ? 4 * PAIRS : PAIRS;
    plan.items = (int)((R * G + per - 1) / per);
    plan.groups = (long long)(ragged ? T * G / per + B : B * plan.items);
    const size_t tiles = (keys_cap + KV4_TOKENS - 1) / KV4_TOKENS;
    const size_t least = 8;  // tiles a span at least: two a wave
    const size_t want = ((size_t)4 * device_info().cus + plan.groups * Hk - 1) / (plan.groups * Hk);
    size_t S = want < 1 ? 1 : want;
    const size_t most = tiles < least ? 1 : tiles / least;
    if (S > most) S = most;
    if (S > 256) S = 256;
    plan.S = (int)S;
    plan.span = (int)((tiles + S - 1) / S);
    if (plan.span < (int)least) plan.span = (int)least;
    return plan;
}

}  // namespace btb

using namespace btb;

extern "C" size_t btb_hip_attn_kv4_floats(size_t T, size_t B, size_t Hq, size_t Hk, size_t D, size_t keys_cap) {
    if (T == 0 || T > (1u << 24) || B == 0 || B > 65536 || Hk == 0 || Hq % Hk != 0 || Hq == 0 || Hq / Hk > 64 || (D != 64 && D != 128) ||
        keys_cap == 0 || keys_cap > (1u << 30))
        return 0;
    // a call may come with `first` or without
    const Kv4Plan a = kv4_plan(T, B, Hk, Hq / Hk, keys_cap, true);
    size_t S = (size_t)a.S;
    if (T % B == 0) {
        const Kv4Plan e = kv4_plan(T, B, Hk, Hq / Hk, keys_cap, false);
        if ((size_t)e.S > S) S = (size_t)e.S;
    }
    return S == 1 ? 4 : T * Hq * S * (D + 2);
}

extern "C" int32_t btb_hip_attn_kv4(const void* q, const void* cache, const int32_t* tables, const int32_t* lens, const int32_t* first,
                                    void* att, float* lse, size_t B, size_t W, size_t pages, size_t page, int64_t stride, size_t T,
                                    size_t Hq, size_t Hk, size_t D, float scale, size_t keys_cap, float* workspace, void* stream) {
    if (!q || !cache || !tables || !lens || !att || !workspace) return ERR_NULL;
    auto loose = [](const void* a) { return ((uintptr_t)a & 15u) != 0; };
    AttnKv4 p{};
    if (!kv4_seqs(p.seqs, tables, lens, first, B, W, pages, page, stride, T, Hk, D) ||
        btb_hip_attn_kv4_floats(T, B, Hq, Hk, D, keys_cap) == 0 || T * Hq > (1u << 24) || !(scale > 0.f) || loose(q) || loose(cache) || loose(att) ||
        loose(workspace)) {
        set_error("attn_kv4: " KV4_DOMAIN ", up to 64 query heads a kv head, 2^24 rows times query heads, scale > 0, keys_cap 1 .. 2^30; "
                  "q, cache, att and workspace 16-byte aligned");
        return ERR_DOMAIN;
    }
    const Kv4Plan plan = kv4_plan(T, B, Hk, Hq / Hk, keys_cap, first != nullptr);
    p.q = static_cast<const uint16_t*>(q);
    p.cache = static_cast<const uint8_t*>(cache);
    p.att = static_cast<uint16_t*>(att);
    p.lse = lse;
    p.part = workspace;
    p.c = scale * LOG2E;
    p.Hq = (int)Hq, p.Hk = (int)Hk, p.G = (int)(Hq / Hk);
    p.items = plan.items, p.S = plan.S, p.span = plan.span;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(plan.groups * plan.S * (long long)Hk)), threads(256);
    if (D == 64)
        hipLaunchKernelGGL((plan.share ? attn_kv4_kernel<64, true> : attn_kv4_kernel<64, false>), grid, threads, 0, st, p);
    else
        hipLaunchKernelGGL((plan.share ? attn_kv4_kernel<128, true> : attn_kv4_kernel<128, false>), grid, threads, 0, st, p);
    int32_t rc = hip_status(hipGetLastError(), "attn_kv4 launch");
    if (rc != OK || plan.S == 1) return rc;
    if (D == 64)
        hipLaunchKernelGGL(attn_kv4_join_kernel<64>, dim3((unsigned)(T * Hq)), threads, 0, st, p);
    else
        hipLaunchKernelGGL(attn_kv4_join_kernel<128>, dim3((unsigned)(T * Hq)), threads, 0, st, p);
    return hip_status(hipGetLastError(), "attn_kv4 join launch");
}
