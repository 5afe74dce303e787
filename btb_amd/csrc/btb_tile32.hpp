// Tiles of 32 keys against 32 (row, query head) pairs on the matrix cores, for head_dim 64 and 128: what the attention
// over a shared prefix and the pass over its weights have in common.
//
// Scores are made as S^T = K Q^T (v_mfma_f32_32x32x16_bf16): lane (c, h) = (lane & 31, lane >> 5) ends with pair c's
// scores against keys 8 (i / 4) + 4 h + i % 4, i = 0 .. 15. A pair's maximum and sum are then sixteen values of a lane
// and one exchange between the halves. The order of keys within a product's 16 is free as long as both operands have
// it: element e of half h stands for key 8 (e / 4) + 4 h + e % 4 of the 16, so that a lane's own scores, rounded, are the
// weights' operand as they lie and nothing passes through LDS between the two products.
#pragma once

#include "btb_common.hpp"

namespace btb {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

constexpr int TK = 32;  // keys a tile

// a [32 keys, D] tile in LDS: rows of 2 D bytes in 16-byte chunks, a key's chunks permuted so that what a fragment's
// lanes read together lies in different banks: for K the chunks of one number of 8 neighbouring keys, for V two
// neighbouring chunks of 4
template <int D>
__device__ __forceinline__ int k_chunk(int key, int chunk) {
    return chunk ^ (key & (D / 8 - 1));
}
__device__ __forceinline__ int v_chunk(int key, int chunk) { return chunk ^ ((key & 3) << 1); }

// K's fragment of 16 dims: lane (c, h) key c, dims 16 step + 8 h .. + 7. A lane's place in a tile is one number for all steps:
// the step's chunk is an exclusive or with it.
template <int D>
__device__ __forceinline__ uint32_t k_place(int lane) {
    return (uint32_t)((lane & 31) * 2 * D + 16 * k_chunk<D>(lane & 31, lane >> 5));
}
__device__ __forceinline__ bf16x8 k_fragment(const uint8_t* tiles, uint32_t place, int tile_at, int step) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(tiles + (place ^ (uint32_t)(32 * step)) + tile_at));
}

// V^T's fragment of 32 dims (dt) against 16 keys (u): lane (c, h) dim 32 dt + c, keys 16 u + 8 (e / 4) + 4 h + e % 4.
// Two transposing reads: in each group of 16 lanes, lane l asks for 4 dims of key l / 4 and gets dim l of the four keys.
template <int D>
__device__ __forceinline__ uint32_t v_place(int lane) {
    const int l = lane & 15, group = lane >> 4, key = 4 * (group >> 1) + (l >> 2);
    return (uint32_t)(key * 2 * D + 16 * v_chunk(key, 2 * (group & 1) + ((l & 3) >> 1)) + 8 * (l & 1));
}
template <int D>
__device__ __forceinline__ bf16x8 v_fragment(const uint8_t* tiles, uint32_t place, int tile_at, int dt, int u) {
    const uint8_t* at = tiles + (place ^ (uint32_t)(64 * dt)) + tile_at + u * 16 * 2 * D;
    const i16x4 first = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at));
    const i16x4 second = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + 8 * 2 * D));
    typedef __attribute__((ext_vector_type(8))) short i16x8;
    const i16x8 both = __builtin_shufflevector(first, second, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, both);
}

// ---- a wave's own tiles straight from memory into LDS -----------------------------------------------------------------
// global_load_lds_dwordx4 writes lane l's 16 bytes at a wave's LDS base plus 16 l: the place in the tile is fixed, so the
// permutation of a key's chunks is made on the way out of memory, within the key's own row.

// Four such loads, 16 bytes a lane each: from base, base + step, + 2 step and + 3 step (uniform) + the lane's offsets to LDS bytes
// `to` (uniform) + 16 lane and 1, 2 and 3 KB on. Written out, because behind the builtin the compiler makes every transposing
// read of LDS wait for all such loads there are, the next stage's among them. They write no
// register; what they write is waited for by count (wait_loads), and a wait of the compiler's own for another load can only come out
// longer. M0 is left as it was.
__device__ __forceinline__ void load4_to_lds(const char* base, size_t step, uint32_t o0, uint32_t o1, uint32_t o2, uint32_t o3,
                                             uint32_t to) {
    uint32_t kept;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %6\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %7\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %4, %8\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %5, %9\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(kept)
        : "s"(to), "v"(o0), "v"(o1), "v"(o2), "v"(o3), "s"(base), "s"(base + step), "s"(base + 2 * step), "s"(base + 3 * step)
        : "memory", "scc");
}
// two of them
__device__ __forceinline__ void load2_to_lds(const char* base, size_t step, uint32_t o0, uint32_t o1, uint32_t to) {
    uint32_t kept;
    asm volatile(
        "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %4\n\t"
        "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %3, %5\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(kept)
        : "s"(to), "v"(o0), "v"(o1), "s"(base), "s"(base + step)
        : "memory", "scc");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
template <class T>
__device__ __forceinline__ T* uniform(T* p) {
    const uint64_t v = (uint64_t)p;
    // (the builtin returns a signed number: its top bit must not spread over the other half)
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
    return (T*)((uint64_t)lo | (uint64_t)hi << 32);
}

template <int D>
struct TileLoads {
    static constexpr int N = TK * 2 * D / 1024;      // instructions a tile of K, and of V
    static constexpr int CH = D / 8, KPI = 64 / CH;  // chunks a row, keys an instruction
    static constexpr int KP = D / 8 / KPI;           // instructions after which K's permutation is the same again (V's: each)
    uint32_t k[KP], v;                               // the lane's bytes from the first key of an instruction

    __device__ __forceinline__ void make(long long rs, int lane) {
        const uint32_t row = (uint32_t)(lane / CH * rs * 2);
#pragma unroll
        for (int i = 0; i < KP; ++i) k[i] = row + 16 * k_chunk<D>(KPI * i + lane / CH, lane % CH);
        v = row + 16 * v_chunk(lane / CH, lane % CH);
    }
    // COUNT instructions' keys at `from` (uniform), a whole tile or half of one, into LDS: K's, or V's. `left` >= 1 keys are there;
    // those past the last are the last again.
    template <bool IS_K, int COUNT = N>
    __device__ __forceinline__ void issue(const uint16_t* from, long long rs, int left, uint8_t* tile, int lane) const {
        static_assert(COUNT == N || (2 * COUNT == N && COUNT % KP == 0), "a tile or half of one, whose permutation starts over");
        const char* base = reinterpret_cast<const char*>(uniform(from));
        const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_address(tile));
        const bool whole = left >= COUNT * KPI;
        const size_t step = whole ? (size_t)KPI * rs * 2 : 0;
        auto at = [&](int i) {
            if (whole) return IS_K ? k[i % KP] : v;
            const int key = KPI * i + lane / CH;
            return (uint32_t)(min(key, left - 1) * rs * 2) + 16 * (IS_K ? k_chunk<D>(key, lane % CH) : v_chunk(key, lane % CH));
        };
        if (whole) {
#pragma unroll
            for (int i = 0; i + 3 < COUNT; i += 4)
                load4_to_lds(base + i * step, step, IS_K ? k[i % KP] : v, IS_K ? k[(i + 1) % KP] : v, IS_K ? k[(i + 2) % KP] : v,
                             IS_K ? k[(i + 3) % KP] : v, to + 1024 * i);
            if constexpr (COUNT == 2) load2_to_lds(base, step, IS_K ? k[0] : v, IS_K ? k[1 % KP] : v, to);
        } else {
#pragma unroll
            for (int i = 0; i + 3 < COUNT; i += 4) load4_to_lds(base, 0, at(i), at(i + 1), at(i + 2), at(i + 3), to + 1024 * i);
            if constexpr (COUNT == 2) load2_to_lds(base, 0, at(0), at(1), to);
        }
    }
    // V's rows past the last key as zeros, once the tile has landed: weight 0 times what lies there must not make a NaN
    template <int COUNT = N>
    __device__ __forceinline__ static void clear_past(uint8_t* v_lds, int left, int lane) {
#pragma unroll
        for (int i = 0; i < COUNT; ++i)
            if (KPI * i + lane / CH >= left) *reinterpret_cast<uint4*>(v_lds + 1024 * i + 16 * lane) = make_uint4(0u, 0u, 0u, 0u);
    }
};

// All but the youngest N loads have landed. A direct-to-LDS load is, to the compiler, a store made where it was issued; the
// reads behind the wait take their place from `at`, which this statement "writes", so they stay behind it.
template <int N>
__device__ __forceinline__ void wait_loads(uint32_t& at) {
    asm volatile("s_waitcnt vmcnt(%1)" : "+v"(at) : "n"(N) : "memory");
}

// A weight (0 or more) as two bf16 terms: its upper half, and what that leaves, rounded; 2^-16 of it at most stays out, up as often as
// down. Neither term has another sign than the weight, nor is the second zero where the weight is 2^-100 and more (its lowest bit is
// set, 2^-23 of it), so that an infinite value stays infinite in both products. Two weights at a time.
__device__ __forceinline__ uint32_t first_terms(float a, float b) {
    return __builtin_amdgcn_perm(f32_bits(b), f32_bits(a), 0x07060302u);
}
__device__ __forceinline__ uint32_t second_terms(float a, float b) {
    return f32x2_bf16(bits_f32(f32_bits(a) | 1u) - bits_f32(f32_bits(a) & 0xFFFF0000u),
                      bits_f32(f32_bits(b) | 1u) - bits_f32(f32_bits(b) & 0xFFFF0000u));
}

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// the value is made here, not where it is first used
__device__ __forceinline__ void made(uint32_t& v) { asm volatile("" : "+v"(v)); }

// DT outputs of 32 dims += V^T times a tile's weights, as two terms, against V's fragments as they are asked for: 16 keys and DT
// fragments a unit, UNITS of them. The next unit's fragments come in and a unit's second terms are made between the products of
// its first; what else there is to do - `work`, numbered - goes between those of its second. read(unit, dt): a fragment;
// weight(unit, i): the i-th of a unit's eight weights a lane.
template <int DT, int UNITS, class Read, class Weight, class Work>
__device__ __forceinline__ void weighted_sums(f32x16 (&o)[DT], Read read, Weight weight, Work work) {
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
    bf16x8 vf[UNITS + 1][DT];
    u32x4 first[UNITS + 1], second;
#pragma unroll
    for (int d = 0; d < DT; ++d) vf[0][d] = read(0, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) first[0][i] = first_terms(weight(0, 2 * i), weight(0, 2 * i + 1));
    fence();
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if (u + 1 < UNITS) vf[u + 1][d] = read(u + 1, d);
            o[d] = mfma32(vf[u][d], __builtin_bit_cast(bf16x8, first[u]), o[d]);
#pragma unroll
            for (int i = 4 * d / DT; i < 4 * (d + 1) / DT; ++i) {
                uint32_t w = second_terms(weight(u, 2 * i), weight(u, 2 * i + 1));
                made(w);
                second[i] = w;
            }
            fence();
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            o[d] = mfma32(vf[u][d], __builtin_bit_cast(bf16x8, second), o[d]);
            if (u + 1 < UNITS) {
#pragma unroll
                for (int i = 4 * d / DT; i < 4 * (d + 1) / DT; ++i) {
                    uint32_t w = first_terms(weight(u + 1, 2 * i), weight(u + 1, 2 * i + 1));
                    made(w);
                    first[u + 1][i] = w;
                }
            }
            if (d % 2 == 1) work((u * DT + d) / 2);
            fence();
        }
    }
}

}  // namespace btb
