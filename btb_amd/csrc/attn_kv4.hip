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
// Weights are f16, off by 2^-11 of themselves at most: e^(s - maximum) times 2^11 times the value's scale over the power of two `unit`, the
// largest one so far: at most 2^15 (the maximum may lag by 2^4), in full precision down to 2^-25 of the largest, and 2^-36 of it is lost at most. A
// bf16 weight would be off by 2^-8, two of them cost twice the products. The unit in the maximum instead of in the scales would save a product
// a weight (1 % of the time), but not the last bits of lse.
//
// Times beside a choice are those of its two sides on the code as it was then. As it is now, 32 query heads over 8 x 128: one row of 700 tokens
// 8.4 us, of 131072 32; 64 sequences of up to 8192 70 .. 75; prompts beside single tokens 54; 500 rows over 16384 150 .. 157 (at head_dim 64 over 4
// heads 109).

#include <cfloat>

#include "btb_kv4.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

constexpr int WAVES = 4;           // waves a workgroup
constexpr int MOST_SPANS = 256;    // a thread each where they are joined
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float NONE = -3.0e38f;   // a maximum of nothing: what is subtracted from it underflows to weight 0
constexpr int ROOM = 11;           // a weight of 1 times the largest scale, in units of the power of two above that, as f16
constexpr float LAG = 4.f;         // how far, in powers of two, scores may pass the maximum in use: f16 ends at 2^16
constexpr float FAR = 0x1p20f;     // a maximum from which on its own rounding, half of 2^-3, would tell in the weights' range
constexpr int PAIRS = 32;          // (row, query head) pairs a workgroup

struct AttnKv4 {
    Kv4Seqs seqs;
    const uint16_t* q;
    const uint8_t* cache;
    uint16_t* att;
    float* lse;
    float* part;     // a pair's spans: maximum and sum [T Hq, S, 2], then, from the next 16 bytes on, outputs [T Hq, S, D]
    float c;         // scale log2(e)
    int Hq, Hk, G;
    int S;           // spans a sequence at most
};

// floats of `states` spans' maxima and sums: the outputs behind them are written and read 16 bytes at a time
__host__ __device__ __forceinline__ size_t kv4_states(size_t states) { return (2 * states + 3) / 4 * 4; }

// tiles a span of a sequence of `tiles`, each span but the last: what S spans come to, two a wave at least
constexpr int LEAST = 2 * WAVES;
__device__ __forceinline__ int kv4_span_tiles(const AttnKv4& p, int tiles) { return max(LEAST, (tiles + p.S - 1) / p.S); }

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

// A pair's running softmax, in the lanes (column, 0) and (column, 1)
template <int D>
struct Softmax {
    static constexpr int DT = D / 32;
    f32x16 o[DT];
    float m, l;
    float over;      // a score past which the maximum lags too far
    uint32_t below;  // the last bf16 number below the unit, twice

    __device__ __forceinline__ uint32_t unit() const { return (below << 16) + (1u << 16); }  // (as bits)

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
        m = NONE, l = 0.f;
        over = -__builtin_inff(), below = 0x0D7F0D7Fu;  // 2^-100
    }

    // The maximum and the unit moved to where a tile's scores z and its scales need them. Whether they do each lane asks of its own scores and
    // scales (`past`), and without working out by how much: 500 rows of 32 heads over 16384 tokens take 161 us instead of 166, at head_dim 64 111
    // instead of 125. Where a maximum is so large that its own rounding would tell in the weights, scores are rounded as it was before it is taken from
    // them: z is then times c, and c 1. most(): the largest of the pair's scales, as bits; NaN is below all.
    template <class Most>
    __device__ __forceinline__ void move(f32x16& z, bool past, float& c, Most most) {
        float top = z[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, z[i]);
        if (__any(top > over || past)) {
            top = fmaxf(top, xor32(top)) * c;
            // the power of two above the largest scale, or the unit as it is
            const float was = bits_f32(unit()), to = fmaxf(m, top);
            const float above = fmaxf(was, bits_f32(((uint32_t)(max(most(), 0) & 0x7F80) + 0x80u) << 16));
            const float by = __builtin_amdgcn_exp2f(m - to);
            l *= by;
            const float both = by * (was / above);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= both;
            const bool large = fabsf(to) > FAR && to != NONE;
            // (a pair with such a maximum comes here with every tile it sees anything of)
            m = to, over = large ? -__builtin_inff() : (m + LAG) / c;
            if (__any(large)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] *= c;
                c = 1.f;
            }
            below = (f32_bits(above) >> 16) * 0x00010001u - 0x00010001u;
        }
    }
    // 2^ROOM / unit
    __device__ __forceinline__ float inverse() const { return bits_f32((uint32_t)(254 + ROOM) * (1u << 23) - unit()); }

    // scores 2 i and 2 i + 1 to weights, r and t their scales over the unit
    __device__ __forceinline__ void weigh(const f32x16& z, float r, float t, u32x4 (&w)[2], float c, int i) {
        const float a = __builtin_amdgcn_exp2f(fmaf(z[2 * i], c, -m)), b = __builtin_amdgcn_exp2f(fmaf(z[2 * i + 1], c, -m));
        l += a;
        l += b;
        const float x = a * r, y = b * t;
        // (two to an instruction: left to itself the compiler folds each product into a conversion of its own, at half the rate)
        uint32_t both;
        asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(both) : "v"(x), "v"(y));
        w[i / 4][i % 4] = both;
    }
};

// a tile's operands as a lane holds them
template <int D>
struct TileWords {
    static constexpr int STEPS = D / 64;
    using Tile = Kv4Tile<D>;
    uint4 k[STEPS], v[STEPS];
    uint32_t e;

    // ONCE: past the caches (another workgroup may read the tile all the same)
    template <bool ONCE>
    __device__ __forceinline__ static uint4 piece(const uint8_t* at, int i) {
        const uint4* from = reinterpret_cast<const uint4*>(at) + i;
        return ONCE ? load_stream16(from) : *from;
    }
    template <bool ONCE>
    __device__ __forceinline__ void load_k(const uint8_t* tile, int lane) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) k[i] = piece<ONCE>(tile, 64 * i + lane);
        e = D == 128 ? reinterpret_cast<const uint16_t*>(tile + Tile::KS)[lane] : tile[Tile::KS + lane];
    }
    template <bool ONCE>
    __device__ __forceinline__ void load_v(const uint8_t* tile, int lane) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) v[i] = piece<ONCE>(tile + Tile::V, 64 * i + lane);
    }
    // K's operand of product j: 8 dims of the lane's 32. (The conversion reads the exponent's field alone: 0 is 2^-127, 255 makes of
    // the zeros that go with it NaN.)
    __device__ __forceinline__ bf16x8 wide_k(int j) const {
        return codes_bf16(dword(k[j / 4], j % 4), bits_f32((j / 4 ? e >> 8 : e & 0xFFu) << 23));
    }
    // V's operand of 32 dims against the u-th 16 tokens
    __device__ __forceinline__ f16x8 wide_v(int d, int u) const { return codes_f16(dword(v[d / 2], 2 * (d % 2) + u)); }
};

// The scales of a lane's half of a tile, over the unit as f32, and the step that comes before: the maximum and the unit moved, tokens that the
// pair does not see hidden. Those are the ones from `left` on of a tile that is `hidden` in part: no score, and no scale (what lies there may be
// anything).
template <int NG>
struct TileScales {
    typedef __attribute__((ext_vector_type(2))) short i16x2;
    uint4 s[2];
    uint32_t x[8];

    __device__ __forceinline__ void load(const uint8_t* scales, int lane) {
#pragma unroll
        for (int i = 0; i < 2; ++i) s[i] = reinterpret_cast<const uint4*>(scales + 32 * (lane >> 5))[i];
    }
    template <int D>
    __device__ __forceinline__ void move(Softmax<D>& to, f32x16& z, float& c, bool hidden, int left, int lane, float*) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = dword(s[i / 4], i % 4);
        if (hidden)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (kv4_token(lane >> 5, i) >= left) {
                    z[i] = -__builtin_inff();
                    x[i / 2] &= i % 2 ? 0x0000FFFFu : 0xFFFF0000u;
                }
        i16x2 big = __builtin_bit_cast(i16x2, to.below);
#pragma unroll
        for (int i = 0; i < 8; ++i) big = __builtin_elementwise_max(big, __builtin_bit_cast(i16x2, x[i]));
        to.move(z, __builtin_bit_cast(uint32_t, big) != to.below, c, [&] {
            const int most = max((int)big[0], (int)big[1]);
            return max(most, __builtin_bit_cast(int, xor32(__builtin_bit_cast(float, most))));
        });
    }
    template <int D>
    __device__ __forceinline__ void weigh(Softmax<D>& to, const f32x16& z, u32x4 (&w)[2], float c, int i) const {
        const float inv = to.inverse();
        to.weigh(z, bf16lo_f32(x[i]) * inv, bf16hi_f32(x[i]) * inv, w, c, i);
    }
};
// One tile at a time, every pair needs the same 32: each lane makes one of them, and all read them out of LDS, where sixteen of them would be two
// more instructions each: 500 rows of 32 heads over 16384 tokens 162 -> 150 us, at head_dim 64 over 4 heads 125 -> 109.
template <>
struct TileScales<1> {
    int s;
    float x[16];

    __device__ __forceinline__ void load(const uint8_t* scales, int lane) { s = reinterpret_cast<const int16_t*>(scales)[lane & 31]; }
    __device__ __forceinline__ void share(float mine, int lane, float* room) {
        room[lane & 31] = mine;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 y = reinterpret_cast<const float4*>(room)[4 * (lane >> 5) + i];
            x[4 * i] = y.x, x[4 * i + 1] = y.y, x[4 * i + 2] = y.z, x[4 * i + 3] = y.w;
        }
        __builtin_amdgcn_wave_barrier();
    }
    template <int D>
    __device__ __forceinline__ void move(Softmax<D>& to, f32x16& z, float& c, bool hidden, int left, int lane, float* room) {
        const float mine = bits_f32((uint32_t)s << 16);
        int big = s;
        if (hidden) {  // (from here on the pairs' units may differ)
            share(mine, lane, room);
            big = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (kv4_token(lane >> 5, i) >= left) z[i] = -__builtin_inff(), x[i] = 0.f;
                big = max(big, (int)f32_bits(x[i]) >> 16);
            }
        }
        to.move(z, big > (int)(to.below & 0xFFFFu), c, [&] {
            int most = max(big, __builtin_bit_cast(int, xor32(__builtin_bit_cast(float, big))));
            if (!hidden)
#pragma unroll
                for (int d = 1; d < 32; d *= 2) most = max(most, __shfl_xor(most, d, WAVE));
            return most;
        });
        const float inv = to.inverse();
        if (hidden) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] *= inv;
        } else {
            share(mine * inv, lane, room);
        }
    }
    template <int D>
    __device__ __forceinline__ void weigh(Softmax<D>& to, const f32x16& z, u32x4 (&w)[2], float c, int i) const {
        to.weigh(z, x[2 * i], x[2 * i + 1], w, c, i);
    }
};

__device__ __forceinline__ f32x16 zeros() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// Up to 32 pairs over tiles NG at a time: lane (column, h)'s pair is column % (32 / NG), and of each NG tiles it weighs tile
// column / (32 / NG) alone. The products of K with q give every column the scores of every tile, of which it keeps
// its own tile's; V's products get weights of zero in the other columns. So the softmax's work is done once for NG tiles where a sequence has few pairs,
// and a column is a running softmax of its own; the columns of a pair meet at the end. A batch's weights are made between the products of
// the next one's scores.
template <int D, int NG>
struct Walk {
    static constexpr int DT = D / 32, COLUMNS = PAIRS / NG, PRODUCTS = NG * D / 16;
    Softmax<D> to;
    QueryFragment<D> q;
    TileWords<D> t[NG];
    TileScales<NG> s;
    f32x16 z;

    __device__ __forceinline__ static int group(int lane) { return NG == 1 ? 0 : (lane & 31) / COLUMNS; }

    // `between`(n) is done behind product n of PRODUCTS
    template <class Between>
    __device__ __forceinline__ f32x16 scores(int lane, Between between) {
        f32x16 all;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            f32x16 x = zeros();
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(t[g].wide_k(j), q.x[j], x, 0, 0, 0);
                between(g * D / 16 + j);
                fence();
            }
            if (g == 0) {
                all = x;
            } else {
                const bool own = group(lane) == g;
#pragma unroll
                for (int i = 0; i < 16; ++i) all[i] = own ? x[i] : all[i];
            }
        }
        return all;
    }

    // a batch whose K has been multiplied: `hidden` and left as for its scales; next_k() asks for the K behind the next batch's, next_v() for the
    // next batch's V
    template <class NextK, class NextV>
    __device__ __forceinline__ void batch(bool hidden, int left, float c, int lane, float* room, NextK next_k, NextV next_v) {
        s.move(to, z, c, hidden, left, lane, room);
        u32x4 w[2];
        // Behind the CU's other workgroup where the vector unit is the bound, ahead of it with V's products and what is asked of memory: two
        // waves in step would multiply together and then wait for the vector unit together. The other way round 500 rows over 16384 tokens take
        // 155.6 us instead of 150.3 and 64 sequences of up to 8192 73 instead of 71; with no difference 158.5 and 75.
        __builtin_amdgcn_s_setprio(0);
        const f32x16 ahead = scores(lane, [&](int n) {
#pragma unroll
            for (int i = 8 * n / PRODUCTS; i < 8 * (n + 1) / PRODUCTS; ++i) s.weigh(to, z, w, c, i);
        });
        __builtin_amdgcn_s_setprio(1);
        next_k();
        f16x8 wide = t[0].wide_v(0, 0);
#pragma unroll
        for (int n = 0; n < NG * 2 * DT; ++n) {
            const int d = n % DT, u = n / DT % 2, g = n / DT / 2;
            u32x4 x = w[u];
            if (NG > 1) {
                const bool own = group(lane) == g;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = own ? x[i] : 0u;
            }
            to.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wide, __builtin_bit_cast(f16x8, x), to.o[d], 0, 0, 0);
            if (n + 1 < NG * 2 * DT) wide = t[(n + 1) / DT / 2].wide_v((n + 1) % DT, (n + 1) / DT % 2);
            fence();
        }
        next_v();
        z = ahead;
    }
};

// A workgroup's span of tiles for up to 32 pairs of a sequence and kv head
struct KvSpan {
    int b, hk, span, spans, from, to;  // its tiles
    int row0, n, len;                  // the sequence's rows and tokens
    int pair0, pairs;                  // the first pair, and how many the sequence has
};

template <int D>
struct Meet {  // the columns of the four waves
    float o[WAVES * PAIRS][D + 4];
    float m[WAVES * PAIRS], l[WAVES * PAIRS];
    float scales[WAVES][KV4_TOKENS];  // of a wave's tile
};

// a tile of pairs' columns, of which `here` are pairs, added up; behind a barrier
template <int D, int NG>
__device__ __forceinline__ void kv4_meet(const AttnKv4& p, const KvSpan& a, const Meet<D>& meet, int pair0, int here) {
    constexpr int COLUMNS = PAIRS / NG;
    // a thread four dims of a pair, over its 4 NG columns
    for (int task = threadIdx.x; task < here * (D / 4); task += 64 * WAVES) {
        const int pair = task / (D / 4), dim = 4 * (task % (D / 4));
        float to = NONE, sum = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES * NG; ++i) to = fmaxf(to, meet.m[i / NG * PAIRS + i % NG * COLUMNS + pair]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < WAVES * NG; ++i) {
            const int from_column = i / NG * PAIRS + i % NG * COLUMNS + pair;
            const float by = __builtin_amdgcn_exp2f(meet.m[from_column] - to);
            sum = fmaf(meet.l[from_column], by, sum);
            const float4 y = *reinterpret_cast<const float4*>(&meet.o[from_column][dim]);
            x = make_float4(fmaf(y.x, by, x.x), fmaf(y.y, by, x.y), fmaf(y.z, by, x.z), fmaf(y.w, by, x.w));
        }
        const int r = (pair0 + pair) / p.G, hd = a.hk * p.G + (pair0 + pair) % p.G;
        const size_t at_pair = (size_t)(a.row0 + r) * p.Hq + hd;
        if (a.spans == 1) {
            const float by = sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<uint2*>(p.att + at_pair * D + dim) = make_uint2(f32x2_bf16(x.x * by, x.y * by), f32x2_bf16(x.z * by, x.w * by));
            if (p.lse != nullptr && dim == 0) p.lse[at_pair] = sum == 0.f ? -__builtin_inff() : (to + __builtin_amdgcn_logf(sum)) * LN2;
        } else {
            const size_t slot = at_pair * p.S + a.span;
            if (dim == 0) reinterpret_cast<float2*>(p.part)[slot] = make_float2(to, sum);
            *reinterpret_cast<float4*>(p.part + kv4_states((size_t)p.seqs.T * p.Hq * p.S) + slot * D + dim) = x;
        }
    }
}

// its four waves' batches of NG tiles, dealt out in turn; the columns meet in LDS
template <int D, int NG, bool ONCE>
__device__ __forceinline__ void kv4_span(const AttnKv4& p, const KvSpan& a, Meet<D>& meet) {
    constexpr int DT = D / 32, COLUMNS = PAIRS / NG;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int mine = a.pair0 + (lane & (COLUMNS - 1)), here = min(a.pairs - a.pair0, COLUMNS);
    const bool there = mine < a.pairs;
    const int row = there ? mine / p.G : 0, head = a.hk * p.G + (there ? mine % p.G : 0);
    Walk<D, NG> w;
    w.to.begin();
    w.q.make(p.q + ((size_t)(a.row0 + row) * p.Hq + head) * D, there, h);
    const int sees = there ? a.len - a.n + row + 1 : 0;  // tokens the lane's pair sees
    const int all = a.len - a.n + a.pair0 / p.G + 1;     // and every pair
    const int own = Walk<D, NG>::group(lane);
    // places of the wave's next 64 tiles, one a lane; -1: no tile, or no page of the pool
    const int from = a.from + wave * NG;
    constexpr int STRIDE = WAVES * NG, REFILL = 64 / NG * STRIDE;
    auto places = [&](int base) {
        const int j = base + lane / NG * STRIDE + lane % NG;
        return j < a.to ? p.seqs.at(a.b, j, a.hk) : -1;
    };
    auto take = [&](long long x, int i) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, i);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)x >> 32), i);
        return (long long)((uint64_t)hi << 32 | lo);
    };
    auto give = [&](long long x, int i) {  // the place of the lane's own tile
        if (NG == 1) return take(x, i);
        const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)x, i + own, WAVE);
        const uint32_t hi = (uint32_t)__shfl((int)(uint32_t)((uint64_t)x >> 32), i + own, WAVE);
        return (long long)((uint64_t)hi << 32 | lo);
    };
    auto request_k = [&](long long x, int i) {
#pragma unroll
        for (int t = 0; t < NG; ++t) w.t[t].template load_k<ONCE>(p.cache + max(take(x, i + t), 0ll), lane);
    };
    auto request_v = [&](long long x, int i) {
#pragma unroll
        for (int t = 0; t < NG; ++t) w.t[t].template load_v<ONCE>(p.cache + max(take(x, i + t), 0ll), lane);
        w.s.load(p.cache + max(give(x, i), 0ll) + Kv4Tile<D>::VS, lane);
    };
    if (from < a.to) {
        // (behind the last tile what is asked for is the pool's first, for nobody)
        long long at = places(from), ahead = places(from + REFILL);
        int i = 0, base = from;  // of the 64 places `at`, and the first one's tile
        auto on = [&] {
            i += NG;
            if (i == 64) {
                i = 0, base += REFILL;
                at = ahead;
                ahead = places(base + REFILL);
            }
        };
        request_k(at, 0);
        request_v(at, 0);
        long long place = give(at, 0);
        w.z = w.scores(lane, [](int) {});
        on();
        request_k(at, i);
        for (int j = from; j < a.to; j += STRIDE) {
            const int left = place < 0 ? 0 : sees - (j + own) * KV4_TOKENS;
            const bool hidden = (j + NG) * KV4_TOKENS > all || j + NG > a.to || __any(place < 0);
            const long long next = at;
            const int next_i = i;
            place = give(next, next_i);
            w.batch(
                hidden, left, p.c, lane, meet.scales[wave],
                [&] {
                    on();
                    request_k(at, i);
                },
                [&] { request_v(next, next_i); });
        }
    }
    const int column = wave * PAIRS + (lane & 31);
    const float l = w.to.l + xor32(w.to.l), real = bits_f32(w.to.unit()) * bits_f32((127u - ROOM) << 23);
    if (h == 0) meet.m[column] = w.to.m, meet.l[column] = l;
    if (there)
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f32x16& o = w.to.o[d];
                *reinterpret_cast<float4*>(&meet.o[column][32 * d + 2 * i + 4 * h]) =
                    make_float4(o[i] * real, o[i + 1] * real, o[i + 2] * real, o[i + 3] * real);
            }
    __syncthreads();
    kv4_meet<D, NG>(p, a, meet, a.pair0, here);
}

template <int D>
__global__ void __launch_bounds__(64 * WAVES, 2) attn_kv4_kernel(AttnKv4 p) {
    extern __shared__ float4 lds[];
    Meet<D>& meet = *reinterpret_cast<Meet<D>*>(lds);
    KvSpan a;
    a.hk = blockIdx.x % p.Hk;
    const int rest = blockIdx.x / p.Hk;
    a.span = rest % p.S;
    // whole tiles of pairs come before what is left of each sequence's: they take longest, and a CU gets one of them rather than two
    // (prompts beside single tokens 58.3 -> 56.9 us; spans that cut the prompts' sequences in two cost 87: the CUs are full as it is)
    int item, x = rest / p.S;
    auto pairs = [&](int b) {
        int row0, n;
        p.seqs.of(b, row0, n);
        return (long long)n * p.G;
    };
    if (p.seqs.first == nullptr) {
        const int each = p.seqs.rows * p.G / PAIRS, whole = p.seqs.B * each;
        a.b = x < whole ? x / each : x - whole, item = x < whole ? x % each : each;
        if (a.b >= p.seqs.B) a.b = -1;
    } else {
        kv4_find(x, p.seqs.B, a.b, item, [&](int b) { return (int)(pairs(b) / PAIRS); });
        if (a.b < 0) {
            kv4_find(x, p.seqs.B, a.b, item, [&](int b) { return pairs(b) % PAIRS != 0 ? 1 : 0; });
            if (a.b >= 0) item = (int)(pairs(a.b) / PAIRS);
        }
    }
    if (a.b < 0) return;
    a.b = __builtin_amdgcn_readfirstlane(a.b), item = __builtin_amdgcn_readfirstlane(item);
    p.seqs.of(a.b, a.row0, a.n);
    a.len = p.seqs.len(a.b);
    const int tiles = (p.seqs.held(a.len) + KV4_TOKENS - 1) / KV4_TOKENS, length = kv4_span_tiles(p, tiles);
    a.spans = max(1, (tiles + length - 1) / length);
    if (a.span >= a.spans) return;
    a.pairs = a.n * p.G, a.pair0 = item * PAIRS;
    const int last = min(a.pair0 + PAIRS, a.pairs) - 1;  // the pair that sees most
    const int any = a.len - a.n + last / p.G + 1;
    a.from = a.span * length;
    a.to = min(min(a.from + length, tiles), any < 1 ? 0 : (any - 1) / KV4_TOKENS + 1);
    // Few pairs: several tiles at a time. At head_dim 128 four of them do not fit the registers: 131072 tokens of one row 32.2 us by two,
    // 33.4 by one, 61 by four; 64 sequences of up to 8192 71, 85 and 135. The tiles of a sequence that has but these pairs go past the caches: 35 -> 32 and
    // 78 -> 71 (55 -> 56 for prompts beside single tokens, 14 -> 15.4 for seven passes of eight rows, if what is left of longer ones does too: the whole tiles of
    // pairs read the same). Branches read their common pages each for itself that way: 16 sequences of 1500 tokens with three branches each take 20.0 instead
    // of 18.7, 64 of 1500 with nothing in common 24 instead of 26; of 6000 52 for 52, and 69 for 77.
    constexpr int NG = D == 64 ? 4 : 2;
    if (a.pairs <= PAIRS / NG)
        kv4_span<D, NG, true>(p, a, meet);
    else if (a.pairs - a.pair0 <= PAIRS / NG)
        kv4_span<D, NG, false>(p, a, meet);
    else
        kv4_span<D, 1, false>(p, a, meet);
}

// A row's spans, and where they lie: false where it has none, or one, which has made its outputs itself
struct KvParts {
    int spans;
    const float2* ml;
    const float* o;
};
__device__ __forceinline__ bool kv4_parts(const AttnKv4& p, unsigned pair, int D, KvParts& parts) {
    const int t = pair / p.Hq, lane = threadIdx.x & 63;
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
        if (b < 0) return false;
    }
    const int tiles = (p.seqs.held(p.seqs.len(b)) + KV4_TOKENS - 1) / KV4_TOKENS, length = kv4_span_tiles(p, tiles);
    parts.spans = (tiles + length - 1) / length;
    parts.ml = reinterpret_cast<const float2*>(p.part) + (size_t)pair * p.S;
    parts.o = p.part + kv4_states((size_t)p.seqs.T * p.Hq * p.S) + (size_t)pair * p.S * D;
    return parts.spans > 1;
}
__device__ __forceinline__ void kv4_lse(const AttnKv4& p, unsigned pair, float m, float l) {
    if (p.lse != nullptr) p.lse[pair] = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * LN2;
}

// Few spans: a wave a row and head, the spans four at a time.
template <int D>
__global__ void __launch_bounds__(256) attn_kv4_join_few(AttnKv4 p) {
    constexpr int V = D / 64;
    const int lane = threadIdx.x & 63;
    const unsigned pair = 4 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    KvParts parts;
    if (pair >= (unsigned)p.seqs.T * p.Hq || !kv4_parts(p, pair, D, parts)) return;
    float m = NONE, l = 0.f, sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    for (int j = 0; j < parts.spans; j += 4) {
        float2 x[4];
        float y[4][V];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int at = min(j + u, parts.spans - 1);
            x[u] = parts.ml[at];
#pragma unroll
            for (int i = 0; i < V; ++i) y[u][i] = parts.o[(size_t)at * D + V * lane + i];
            if (j + u >= parts.spans) x[u] = make_float2(NONE, 0.f);
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
            if (j + u >= parts.spans) continue;
            const float a = __builtin_amdgcn_exp2f(x[u].x - to);
            l = fmaf(x[u].y, a, l);
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = fmaf(y[u][i], a, sum[i]);
        }
        m = to;
    }
    const float by = l == 0.f ? 0.f : 1.f / l;
    uint16_t* att = p.att + (size_t)pair * D + V * lane;
    if constexpr (V == 2)
        *reinterpret_cast<uint32_t*>(att) = f32x2_bf16(sum[0] * by, sum[1] * by);
    else
        *att = f32_bf16(sum[0] * by);
    if (lane == 0) kv4_lse(p, pair, m, l);
}

// Many spans: a workgroup a row and head. All that it reads is asked for at once; the spans' weights are made meanwhile.
constexpr int JOIN_AT_ONCE = 8;
template <int D>
__global__ void __launch_bounds__(256) attn_kv4_join_many(AttnKv4 p) {
    constexpr int GROUPS = 1024 / D;  // of threads, a span each at a time
    __shared__ float by[MOST_SPANS], tops[4], sums[4];
    __shared__ float4 part[GROUPS][D / 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, group = tid / (D / 4), dim = tid % (D / 4);
    KvParts parts;
    if (!kv4_parts(p, blockIdx.x, D, parts)) return;
    const float4* o = reinterpret_cast<const float4*>(parts.o) + dim;
    float4 y[JOIN_AT_ONCE];
    const float2 ml = tid < parts.spans ? parts.ml[tid] : make_float2(NONE, 0.f);
#pragma unroll
    for (int u = 0; u < JOIN_AT_ONCE; ++u) {
        const int j = group + GROUPS * u;
        y[u] = j < parts.spans ? o[(size_t)j * (D / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = ml.x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d, WAVE));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float a = __builtin_amdgcn_exp2f(ml.x - top);
    by[tid] = a;
    const float mine = wave_sum(ml.y * a);
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    const float total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v, int j) {
        const float f = by[j];
        x = make_float4(fmaf(v.x, f, x.x), fmaf(v.y, f, x.y), fmaf(v.z, f, x.z), fmaf(v.w, f, x.w));
    };
#pragma unroll
    for (int u = 0; u < JOIN_AT_ONCE; ++u)
        if (group + GROUPS * u < parts.spans) add(y[u], group + GROUPS * u);
    for (int j = group + GROUPS * JOIN_AT_ONCE; j < parts.spans; j += GROUPS) add(o[(size_t)j * (D / 4)], j);
    part[group][dim] = x;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) {
        const float4 v = part[g][dim];
        x = make_float4(x.x + v.x, x.y + v.y, x.z + v.z, x.w + v.w);
    }
    const float f = total == 0.f ? 0.f : 1.f / total;
    *reinterpret_cast<uint2*>(p.att + (size_t)blockIdx.x * D + 4 * dim) = make_uint2(f32x2_bf16(x.x * f, x.y * f), f32x2_bf16(x.z * f, x.w * f));
    if (dim == 0) kv4_lse(p, blockIdx.x, top, total);
}

// How a call is cut, from what the host knows: tiles of pairs, and spans.
struct Kv4Plan {
    long long groups; // workgroups a kv head and span
    int S;
};
static Kv4Plan kv4_plan(size_t T, size_t B, size_t Hk, size_t G, size_t keys_cap, bool ragged) {
    Kv4Plan plan;
    plan.groups = (long long)(ragged ? T * G / PAIRS + B : B * ((T / B * G + PAIRS - 1) / PAIRS));
    const size_t tiles = (keys_cap + KV4_TOKENS - 1) / KV4_TOKENS;
    // two workgroups a CU, as many as fit (131072 tokens of one row: 32 us, 42 with three, 46 with six; with a span more, and so a second round,
    // 500 rows over 16384 are 165 instead of 150, 64 sequences 77 instead of 71). One of eight waves a CU instead: 64 sequences 71 -> 77, prompts beside single
    // tokens 54 -> 61. Groups are those that B sequences with T rows between them may have, whichever of them have any: with `first` 32 sequences of 8192
    // have one span (60 us, 51 without), and 131072 tokens of one among 64 take 753.
    const size_t want = (size_t)(8 / WAVES) * device_info().cus / (plan.groups * Hk);
    size_t S = want < 1 ? 1 : want;
    // (a second launch, for the join, pays from 32 tiles on: 700 tokens of one row take 10.5 us in two spans, 8.4 in one; the rule goes
    // by keys_cap: under one of 32768 they take 1.1 more)
    const size_t most = tiles < 32 ? 1 : tiles / LEAST;
    if (S > most) S = most;
    if (S > (size_t)MOST_SPANS) S = MOST_SPANS;
    plan.S = (int)S;
    return plan;
}

template <int D>
static int32_t launch_attn_kv4(const AttnKv4& p, const Kv4Plan& plan, hipStream_t st) {
    constexpr int lds = (int)sizeof(Meet<D>);
    const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_kv4_kernel<D>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (rc != hipSuccess) return hip_status(rc, "hipFuncSetAttribute");
    hipLaunchKernelGGL(attn_kv4_kernel<D>, dim3((unsigned)(plan.groups * plan.S * (long long)p.Hk)), dim3(64 * WAVES), lds, st, p);
    const int32_t done = hip_status(hipGetLastError(), "attn_kv4 launch");
    if (done != OK || plan.S == 1) return done;
    const unsigned pairs = (unsigned)(p.seqs.T * p.Hq);
    if (plan.S >= 16)
        hipLaunchKernelGGL(attn_kv4_join_many<D>, dim3(pairs), dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL(attn_kv4_join_few<D>, dim3((pairs + 3) / 4), dim3(256), 0, st, p);
    return hip_status(hipGetLastError(), "attn_kv4 join launch");
}

}  // namespace btb

using namespace btb;

extern "C" size_t btb_hip_attn_kv4_floats(size_t T, size_t B, size_t Hq, size_t Hk, size_t D, size_t keys_cap) {
    if (T == 0 || T > (1u << 24) || B == 0 || B > 65536 || Hk == 0 || Hk > 1024 || Hq % Hk != 0 || Hq == 0 || Hq / Hk > 64 ||
        T * Hq > (1u << 24) || (D != 64 && D != 128) || keys_cap == 0 || keys_cap > (1u << 30))
        return 0;
    // a call may come with `first` or without
    const Kv4Plan a = kv4_plan(T, B, Hk, Hq / Hk, keys_cap, true);
    size_t S = (size_t)a.S;
    if (T % B == 0) {
        const Kv4Plan e = kv4_plan(T, B, Hk, Hq / Hk, keys_cap, false);
        if ((size_t)e.S > S) S = (size_t)e.S;
    }
    return S == 1 ? 4 : kv4_states(T * Hq * S) + T * Hq * S * D;
}

extern "C" int32_t btb_hip_attn_kv4(const void* q, const void* cache, const int32_t* tables, const int32_t* lens, const int32_t* first,
                                    void* att, float* lse, size_t B, size_t W, size_t pages, size_t page, int64_t stride, size_t T,
                                    size_t Hq, size_t Hk, size_t D, float scale, size_t keys_cap, float* workspace, void* stream) {
    if (!q || !cache || !tables || !lens || !att || !workspace) return ERR_NULL;
    auto loose = [](const void* a) { return ((uintptr_t)a & 15u) != 0; };
    AttnKv4 p{};
    if (!kv4_seqs(p.seqs, tables, lens, first, B, W, pages, page, stride, T, Hk, D) ||
        btb_hip_attn_kv4_floats(T, B, Hq, Hk, D, keys_cap) == 0 || !(scale > 0.f) || scale > FLT_MAX / LOG2E || loose(q) || loose(cache) || loose(att) ||
        loose(workspace)) {
        set_error("attn_kv4: " KV4_DOMAIN ", up to 64 query heads a kv head, 2^24 rows times query heads, scale from above 0 to 2^128 / log2(e), keys_cap 1 .. 2^30; "
                  "q, cache, att and workspace 16-byte aligned");
        return ERR_DOMAIN;
    }
    // (att may be q: a pair's row is read, by the workgroups that write it or before the join, ahead of what is written there)
    const uintptr_t from = (uintptr_t)q, to = (uintptr_t)att, bytes = 2 * T * Hq * D;
    if (from != to && from < to + bytes && to < from + bytes) {
        set_error("attn_kv4: att lies across q");
        return ERR_DOMAIN;
    }
    const Kv4Plan plan = kv4_plan(T, B, Hk, Hq / Hk, keys_cap, first != nullptr);
    // (a join's workgroup a pair comes with many spans only, and those with few pairs)
    if (plan.groups * plan.S * (long long)Hk > MOST_GROUPS) {
        set_error("attn_kv4: sequences, with tiles of 32 rows and heads, times kv heads below 2^24");
        return ERR_DOMAIN;
    }
    p.q = static_cast<const uint16_t*>(q);
    p.cache = static_cast<const uint8_t*>(cache);
    p.att = static_cast<uint16_t*>(att);
    p.lse = lse;
    p.part = workspace;
    p.c = scale * LOG2E;
    p.Hq = (int)Hq, p.Hk = (int)Hk, p.G = (int)(Hq / Hk);
    p.S = plan.S;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return D == 64 ? launch_attn_kv4<64>(p, plan, st) : launch_attn_kv4<128>(p, plan, st);
}
