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

// K's fragment of 16 dims: lane (c, h) key c, dims 16 step + 8 h .. + 7
template <int D>
__device__ __forceinline__ bf16x8 k_fragment(const uint8_t* tile, int step, int lane) {
    const int key = lane & 31;
    return __builtin_bit_cast(
        bf16x8, *reinterpret_cast<const uint4*>(tile + key * 2 * D + 16 * k_chunk<D>(key, 2 * step + (lane >> 5))));
}

// V^T's fragment of 32 dims (dt) against 16 keys (u): lane (c, h) dim 32 dt + c, keys 16 u + 8 (e / 4) + 4 h + e % 4.
// Two transposing reads: in each group of 16 lanes, lane l asks for 4 dims of key l / 4 and gets dim l of the four keys.
template <int D>
__device__ __forceinline__ bf16x8 v_fragment(const uint8_t* tile, int dt, int u, int lane) {
    const int l = lane & 15, group = lane >> 4;
    const int key = 16 * u + 4 * (group >> 1) + (l >> 2);
    const int chunk = 4 * dt + 2 * (group & 1) + ((l & 3) >> 1);
    const uint8_t* at = tile + key * 2 * D + 16 * v_chunk(key, chunk) + 8 * (l & 1);
    const i16x4 first = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at));
    const i16x4 second = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + 8 * 2 * D));
    typedef __attribute__((ext_vector_type(8))) short i16x8;
    const i16x8 both = __builtin_shufflevector(first, second, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(bf16x8, both);
}

// eight weights as an operand
__device__ __forceinline__ bf16x8 weight_fragment(const float* p) {
    return __builtin_bit_cast(bf16x8, make_uint4(f32x2_bf16(p[0], p[1]), f32x2_bf16(p[2], p[3]), f32x2_bf16(p[4], p[5]),
                                                 f32x2_bf16(p[6], p[7])));
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

}  // namespace btb
