// A paged cache held in 4 bits: how its tiles lie in memory and how a kernel finds its sequences.
//
// A tile is 32 tokens of one kv head, laid out as the matrix cores' operands, so that attention reads it in whole 16-byte pieces a
// lane, straight into registers, and nothing passes through LDS:
//   K codes   D / 64 steps x 64 lanes x 16 bytes: lane (c, h) = (lane & 31, lane >> 5) has token c's dims 64 step + 32 h .. + 31,
//             the lower dim of a pair in a byte's low half: one block of 32 dims, with one exponent
//   V codes   D / 64 parts x 64 lanes x 16 bytes: dword 2 d + u of lane (c, h) has dim 64 part + 32 d + c of the 8 tokens
//             16 u + 8 (e / 4) + 4 h + e % 4, e = 0 .. 7: where scores made as K Q^T lie, which are thus the second product's operand
//   K scales  D / 64 bytes a lane in the same order: the exponent of the lane's 32 dims, biased by 127 (255: NaN)
//   V scales  bf16, a token each: token 8 (i / 4) + 4 h + i % 4 at 16 h + i. NaN: 0xFFC0, below every other as a signed number
// A page is page / 32 tiles a head, its heads one after another. Tokens 2 i and 2 i + 1 share V's bytes.
#pragma once

#include "btb_common.hpp"

namespace btb {

constexpr int KV4_TOKENS = 32;

template <int D>
struct Kv4Tile {
    static constexpr int STEPS = D / 64;
    static constexpr int V = 1024 * STEPS, KS = 2 * V, VS = KS + 64 * STEPS, BYTES = VS + 64;
};

__host__ __device__ __forceinline__ size_t kv4_tile_bytes(size_t D) { return D == 64 ? Kv4Tile<64>::BYTES : Kv4Tile<128>::BYTES; }

// where a token's V lies: the half of the wave, and its place among the half's sixteen
__device__ __forceinline__ int kv4_half(int token) { return (token >> 2) & 1; }
__device__ __forceinline__ int kv4_index(int token) { return (token >> 3) * 4 + (token & 3); }
__device__ __forceinline__ int kv4_token(int half, int index) { return 8 * (index >> 2) + 4 * half + (index & 3); }

// The sequences of a pass: their pages, their lengths with the pass's rows, and which rows are theirs: their last ones.
struct Kv4Seqs {
    const int32_t* tables;  // [B, W]
    const int32_t* lens;    // [B]
    const int32_t* first;   // [B + 1], or null: `rows` each
    int B, W, T, rows, pages;
    int per;                // tiles a page
    long long stride;       // bytes from a page to the next
    int tile;               // bytes of a tile

    // what the device arrays say is cut to what there is: a sequence's length, by which its rows stand at their places, and how many of
    // those places its table has
    __device__ __forceinline__ int len(int b) const { return max(lens[b], 0); }
    __device__ __forceinline__ int held(int len) const { return (int)min((long long)len, (long long)W * per * KV4_TOKENS); }
    __device__ __forceinline__ void of(int b, int& row0, int& n) const {
        if (first == nullptr) {
            row0 = b * rows, n = rows;
            return;
        }
        row0 = min(max(first[b], 0), T);
        n = max(min(first[b + 1], T) - row0, 0);
    }
    // the bytes of tile j of a sequence's head, -1 where the table names no page of the pool
    __device__ __forceinline__ long long at(int b, int j, int hk) const {
        const int page = tables[(size_t)b * W + j / per];
        return page < 0 || page >= pages ? -1 : page * stride + ((long long)hk * per + j % per) * tile;
    }
};

// Item `x` of a pass whose sequence b has count(b) of them, one sequence after another: its sequence and which of them it is; b = -1
// behind the last, and x is then how far. Each wave looks for itself, 64 sequences at a time.
template <class Count>
__device__ __forceinline__ void kv4_find(int& x, int B, int& b, int& i, Count count) {
    const int lane = threadIdx.x & 63;
    b = -1, i = 0;
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int mine = b0 + lane < B ? count(b0 + lane) : 0;
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int below = __shfl_up(upto, d, WAVE);
            if (lane >= d) upto += below;
        }
        const uint64_t past = __ballot(x < upto);
        if (past != 0) {
            const int at = __ffsll((unsigned long long)past) - 1;
            b = b0 + at;
            i = x - __builtin_amdgcn_readlane(upto - mine, at);
            return;
        }
        x -= __builtin_amdgcn_readlane(upto, 63);
    }
}

// workgroups of 256 threads that a launch can have: its threads are counted in 32 bits
constexpr long long MOST_GROUPS = ((1ll << 32) - 1) / 256;

// What every entry point over such a cache asks of its sizes; false: refused. The words for it:
#define KV4_DOMAIN "head_dim 64 or 128, pages of a multiple of 32 tokens, 1 .. 65536 sequences of up to 2^30 tokens, up to 2^24 rows (without first: as many a sequence), up to 1024 kv heads"
inline bool kv4_seqs(Kv4Seqs& s, const int32_t* tables, const int32_t* lens, const int32_t* first, size_t B, size_t W, size_t pages,
                     size_t page, int64_t stride, size_t T, size_t Hk, size_t D) {
    if (B == 0 || B > 65536 || W == 0 || W > (1u << 30) || pages == 0 || pages > 0x7FFFFFFFu || page == 0 || page % KV4_TOKENS != 0 ||
        page > (1u << 20) || W * page > (1u << 30) || T == 0 || T > (1u << 24) || Hk == 0 || Hk > 1024 || (D != 64 && D != 128) ||
        (first == nullptr && T % B != 0))
        return false;
    s.per = (int)(page / KV4_TOKENS);
    s.tile = (int)kv4_tile_bytes(D);
    s.stride = stride;
    if (stride < (long long)Hk * s.per * s.tile || stride % 16 != 0 || stride > ((int64_t)1 << 46) / (int64_t)pages) return false;
    s.tables = tables, s.lens = lens, s.first = first;
    s.B = (int)B, s.W = (int)W, s.T = (int)T, s.rows = (int)(T / B), s.pages = (int)pages;
    return true;
}

}  // namespace btb
