// New rows of keys and values into a paged cache held in 4 bits (btb_kv4.hpp), and cached rows back as the values they stand for.
//
//   K, 32 dims of a token and head:  e = the smallest with max |k| <= 7 2^e (-127 .. 125), code = e2m1(k / 2^e)    (an infinity or NaN: all 32 NaN)
//   V, a token and head:             s = bf16(max |v| / 6), code = e2m1(v / s), s = 0: 0             (an infinity or NaN: all of it NaN)
//
// e2m1: 0, 1/2, 1, 3/2, 2, 3, 4, 6, the nearest, a tie to the even code, 7 to 6. Keys keep a power of two a block, which the
// matrix cores apply; a value's scale is a whole token's and goes into its weight, and with bf16's eight bits nothing of the codes' range is
// lost to a power of two.
//
// A workgroup a tile of 32 tokens and a head: whoever writes one of two tokens that share V's bytes writes both. Bound: memory for many rows,
// the launch for few.

#include "btb_kv4.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

struct Kv4Rows {
    Kv4Seqs seqs;
    uint8_t* cache;
    const uint16_t* k;  // written: bf16 rows
    const uint16_t* v;
    void* k_out;        // read: bf16 or f32 rows
    void* v_out;
    long long kt, kh, vt, vh;  // values from a row, and from a head, to the next
    int Hk, items;             // items a sequence, where each has as many rows
    long long groups;
};

// the tiles a sequence's last rows lie in
__device__ __forceinline__ int kv4_tiles(const Kv4Seqs& s, int b) {
    int row0, n;
    s.of(b, row0, n);
    const int len = s.len(b), from = len - min(n, len), to = s.held(len);
    return from >= to ? 0 : (to - 1) / KV4_TOKENS - from / KV4_TOKENS + 1;
}

// the workgroup's tile: its sequence and number, the pass's row of its first token (below 0: that token is no row of the pass) and which
// of its tokens are rows of the pass
struct Kv4Place {
    int b, tile, row;
    uint32_t tokens;
};
__device__ __forceinline__ bool kv4_place(const Kv4Rows& p, int item, Kv4Place& at) {
    int i;
    if (p.seqs.first == nullptr) {
        at.b = item / p.items, i = item % p.items;
        if (i >= kv4_tiles(p.seqs, at.b)) return false;
    } else {
        kv4_find(item, p.seqs.B, at.b, i, [&](int b) { return kv4_tiles(p.seqs, b); });
        if (at.b < 0) return false;
    }
    int row0, n;
    p.seqs.of(at.b, row0, n);
    const int len = p.seqs.len(at.b), from = len - min(n, len);  // the first position that is a row's
    at.tile = from / KV4_TOKENS + i;
    const int first = at.tile * KV4_TOKENS, low = max(from - first, 0), high = min(p.seqs.held(len) - first, KV4_TOKENS);
    at.row = row0 + n - len + first;
    at.tokens = (high == 32 ? 0xFFFFFFFFu : (1u << high) - 1u) & (0xFFFFFFFFu << low);
    return true;
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
// the largest |value| of a lane's eight bf16 numbers, as bits
__device__ __forceinline__ uint32_t largest8(const uint4& w) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = umax(m, umax(x[i] & 0x7FFFu, x[i] >> 16 & 0x7FFFu));
    return m;
}
// eight values as e2m1, the first in the lowest four bits
__device__ __forceinline__ uint32_t codes8(const float (&y)[8]) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.f, 3);
}
__device__ __forceinline__ void widen8(const uint4& w, float (&v)[8]) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16lo_f32(x[i]);
        v[2 * i + 1] = bf16hi_f32(x[i]);
    }
}

constexpr uint16_t KV4_NAN = 0xFFC0;

template <int D>
__global__ void __launch_bounds__(256) kv4_write_kernel(Kv4Rows p) {
    using Tile = Kv4Tile<D>;
    constexpr int STEPS = Tile::STEPS, CH = D / 8, PIECES = 64 * STEPS;
    __shared__ uint4 k_piece[PIECES];
    __shared__ uint32_t v_code[KV4_TOKENS][CH + 1];
    __shared__ uint8_t k_scale[PIECES];
    __shared__ uint16_t v_scale[KV4_TOKENS];
    const int hk = blockIdx.x % p.Hk, tid = threadIdx.x;
    Kv4Place at;
    if (!kv4_place(p, blockIdx.x / p.Hk, at)) return;
    const long long place = p.seqs.at(at.b, at.tile, hk);
    if (place < 0) return;
#pragma unroll
    for (int i = 0; i < 32 * CH / 256; ++i) {
        const int token = (tid + 256 * i) / CH, c = (tid + 256 * i) % CH;
        uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
        if (at.tokens >> token & 1u) {
            const long long row = at.row + token;
            k = load_stream16(reinterpret_cast<const uint4*>(p.k + row * p.kt + hk * p.kh + 8 * c));
            v = load_stream16(reinterpret_cast<const uint4*>(p.v + row * p.vt + hk * p.vh + 8 * c));
        }
        float y[8];
        uint32_t top = largest8(k);  // over four lanes, a block of 32 dims
        top = umax(top, dpp_u32<0xB1>(top));
        top = umax(top, dpp_u32<0x4E>(top));
        const bool lost = top >= 0x7F80u;
        // the exponent of bf16's own field; 1 3/4 is the largest mantissa that the power two below it still holds (up to 2^125: six of
        // it are a number yet)
        const int e = min(max((int)(top >> 7) - 2 + ((top & 0x7Fu) > 0x60u ? 1 : 0), 0), 252);
        widen8(k, y);
        const float down = bits_f32((uint32_t)(254 - e) << 23);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] *= down;
        const int piece = c / 8 * 64 + c / 4 % 2 * 32 + token;
        reinterpret_cast<uint32_t*>(k_piece)[4 * piece + c % 4] = lost ? 0u : codes8(y);
        if (c % 4 == 0) k_scale[(c / 4 % 2 * 32 + token) * STEPS + c / 8] = (uint8_t)(lost ? 255 : e);
        top = largest8(v);  // over the token's lanes
        top = umax(top, dpp_u32<0xB1>(top));
        top = umax(top, dpp_u32<0x4E>(top));
        top = umax(top, dpp_u32<0x141>(top));
        if (CH == 16) top = umax(top, dpp_u32<0x140>(top));
        const uint16_t s = top >= 0x7F80u ? KV4_NAN : f32_bf16(bf16_f32((uint16_t)top) / 6.f);
        widen8(v, y);
        // the quotient by the reciprocal, and what that leaves by it once more: a tie comes out as one, and no other quotient of two bf16 numbers is
        // nearer to one than 2^-12 of it (small scales times 2^64, for their reciprocals' sake)
        const float up = (s & 0x7FFFu) < 0x2000u ? bits_f32(191u << 23) : 1.f, scale = bf16_f32(s) * up, by = __builtin_amdgcn_rcpf(scale);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = y[j] * up, z = x * by;
            y[j] = fmaf(fmaf(-z, scale, x), by, z);
        }
        v_code[token][c] = s == 0 || s == KV4_NAN ? 0u : codes8(y);
        if (c == 0) v_scale[kv4_half(token) * 16 + kv4_index(token)] = s;
    }
    __syncthreads();
    uint8_t* tile = p.cache + place;
    if (tid < PIECES) {
        if (at.tokens >> (tid & 31) & 1u) {
            reinterpret_cast<uint4*>(tile)[tid] = k_piece[tid];
            if (tid < 64) {
                if constexpr (STEPS == 2)
                    reinterpret_cast<uint16_t*>(tile + Tile::KS)[tid] = reinterpret_cast<const uint16_t*>(k_scale)[tid];
                else
                    tile[Tile::KS + tid] = k_scale[tid];
            }
        }
        if (tid < 32 && (at.tokens >> kv4_token(tid >> 4, tid & 15) & 1u)) reinterpret_cast<uint16_t*>(tile + Tile::VS)[tid] = v_scale[tid];
    } else if (tid < 2 * PIECES) {
        const int t = tid - PIECES, c = t & 31, h = t >> 5 & 1, part = t >> 6;
        uint32_t w[4], mine[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (at.tokens >> kv4_token(h, j) & 1u) mine[j >> 3] |= 0xFu << (4 * (j & 7));
        if ((mine[0] | mine[1]) != 0u) {
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const int dim = 64 * part + 32 * d + c;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t x = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) x |= (v_code[kv4_token(h, 8 * u + j)][dim >> 3] >> (4 * (dim & 7)) & 0xFu) << (4 * j);
                    w[2 * d + u] = x;
                }
            }
            uint4* to = reinterpret_cast<uint4*>(tile + Tile::V) + t;
            if ((mine[0] & mine[1]) != 0xFFFFFFFFu) {  // the other tokens' bits stay
                const uint4 was = *to;
                w[0] = (w[0] & mine[0]) | (was.x & ~mine[0]);
                w[1] = (w[1] & mine[1]) | (was.y & ~mine[1]);
                w[2] = (w[2] & mine[0]) | (was.z & ~mine[0]);
                w[3] = (w[3] & mine[1]) | (was.w & ~mine[1]);
            }
            *to = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

__device__ __forceinline__ void kv4_put(uint16_t* to, const float (&y)[8]) {
    const u32x4 x = {f32x2_bf16(y[0], y[1]), f32x2_bf16(y[2], y[3]), f32x2_bf16(y[4], y[5]), f32x2_bf16(y[6], y[7])};
    __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(to));
}
__device__ __forceinline__ void kv4_put(float* to, const float (&y)[4]) {
    const f32x4 x = {y[0], y[1], y[2], y[3]};
    __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(to));
}
// N codes' values times a scale
template <int N>
__device__ __forceinline__ void kv4_values(uint32_t codes, float scale, float (&y)[N]) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 1);
    y[0] = a.x * scale, y[1] = a.y * scale, y[2] = b.x * scale, y[3] = b.y * scale;
    if constexpr (N == 8) {
        const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.f, 3);
        y[4] = c.x * scale, y[5] = c.y * scale, y[6] = d.x * scale, y[7] = d.y * scale;
    }
}

// 16 bytes of output a lane at a time, so that a wave writes whole lines, past the caches: 12001 rows of 8 heads x 128 as f32 19.5 us (25.1
// through them; 28.6 through them and 40.5 past them with 32 bytes a lane), as bf16 11.7
template <int D, class OUT>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4Rows p) {
    using Tile = Kv4Tile<D>;
    constexpr int STEPS = Tile::STEPS, N = 16 / sizeof(OUT), CH = D / N, PIECES = Tile::BYTES / 16;
    __shared__ uint4 held[PIECES];
    const int hk = blockIdx.x % p.Hk, tid = threadIdx.x;
    Kv4Place at;
    if (!kv4_place(p, blockIdx.x / p.Hk, at)) return;
    const long long place = p.seqs.at(at.b, at.tile, hk);
    for (int i = tid; i < PIECES; i += 256)
        held[i] = place < 0 ? make_uint4(0u, 0u, 0u, 0u) : reinterpret_cast<const uint4*>(p.cache + place)[i];
    __syncthreads();
    const uint8_t* tile = reinterpret_cast<const uint8_t*>(held);
#pragma unroll
    for (int i = 0; i < 32 * CH / 256; ++i) {
        const int token = (tid + 256 * i) / CH, dim = (tid + 256 * i) % CH * N;
        if (!(at.tokens >> token & 1u)) continue;
        const long long row = at.row + token;
        const int half = dim / 32 % 2, step = dim / 64, lane = half * 32 + token;
        const uint32_t e = tile[Tile::KS + lane * STEPS + step];
        const uint32_t k = reinterpret_cast<const uint32_t*>(tile)[4 * (step * 64 + lane) + dim / 8 % 4] >> (4 * (dim & 7));
        float y[N];
        kv4_values(k, bits_f32(e == 255u ? 0x7FC00000u : (e == 0u ? 0x00400000u : e << 23)), y);
        kv4_put(static_cast<OUT*>(p.k_out) + row * p.kt + hk * p.kh + dim, y);
        const int h = kv4_half(token), j = kv4_index(token);
        // neighbouring dims of a token lie 16 bytes apart
        const uint8_t* from = tile + Tile::V + 16 * (dim / 64 * 64 + h * 32 + dim % 32) + 8 * (dim / 32 % 2) + 4 * (j >> 3) + ((j & 7) >> 1);
        uint32_t v = 0;
#pragma unroll
        for (int d = 0; d < N; ++d) v |= (uint32_t)(from[16 * d] >> (4 * (j & 1)) & 0xF) << (4 * d);
        kv4_values(v, bf16_f32(reinterpret_cast<const uint16_t*>(tile + Tile::VS)[16 * h + j]), y);
        kv4_put(static_cast<OUT*>(p.v_out) + row * p.vt + hk * p.vh + dim, y);
    }
}

static int32_t kv4_rows(Kv4Rows& p, const void* cache, const int32_t* tables, const int32_t* lens, const int32_t* first, size_t B,
                        size_t W, size_t pages, size_t page, int64_t stride, size_t T, size_t Hk, size_t D, int64_t kt, int64_t kh,
                        int64_t vt, int64_t vh, const void* k, const void* v, const char* what) {
    auto loose = [](const void* a) { return ((uintptr_t)a & 15u) != 0; };
    auto odd = [](size_t n, int64_t s) { return n > 1 && (s < 0 || s % 8 != 0 || s > ((int64_t)1 << 46) / (int64_t)n); };  // (one alone has no next)
    if (!kv4_seqs(p.seqs, tables, lens, first, B, W, pages, page, stride, T, Hk, D) || odd(T, kt) || odd(Hk, kh) || odd(T, vt) || odd(Hk, vh) ||
        loose(cache) || loose(k) || loose(v)) {
        set_error(what);
        return ERR_DOMAIN;
    }
    p.cache = static_cast<uint8_t*>(const_cast<void*>(cache));
    p.kt = kt, p.kh = kh, p.vt = vt, p.vh = vh;
    p.Hk = (int)Hk;
    // workgroups: the tiles that the rows can lie in, each at least one of them, a head each
    const long long rows = p.seqs.T, seqs = p.seqs.B, R = p.seqs.rows;
    p.items = (int)(R < (R + 30) / 32 + 1 ? R : (R + 30) / 32 + 1);
    const long long ragged = rows < rows / 32 + 2 * seqs ? rows : rows / 32 + 2 * seqs;
    p.groups = (first ? ragged : seqs * p.items) * p.Hk;
    if (p.groups > MOST_GROUPS) {
        set_error(what);
        return ERR_DOMAIN;
    }
    return OK;
}

// Whether two outputs of such rows, the second `apart` values behind the first, have a value in common. The differences between their places are
// apart + i head + j row, |i| < heads and |j| < rows, and each of them holds D values; at other strides the outputs are apart where their ranges are. Rows
// of one output are D values apart or more.
static bool kv4_outputs_meet(const Kv4Rows& p, int64_t apart, int64_t D) {
    const int64_t T = p.seqs.T, Hk = p.Hk;
    const int64_t kt = T > 1 ? p.kt : 0, vt = T > 1 ? p.vt : 0, kh = Hk > 1 ? p.kh : 0, vh = Hk > 1 ? p.vh : 0;
    if (apart >= (T - 1) * kt + (Hk - 1) * kh + D || -apart >= (T - 1) * vt + (Hk - 1) * vh + D) return false;
    if (kt != vt || kh != vh) return true;
    for (int64_t i = 1 - Hk; i < Hk; ++i) {
        const int64_t x = apart + i * kh;
        if (T == 1) {
            if (x > -D && x < D) return true;
            continue;
        }
        const int64_t rest = (x % kt + kt) % kt, rows = (x - rest) / kt;  // x = rows kt + rest: the rows next to it
        if ((rest < D && rows > -T && rows < T) || (kt - rest < D && rows + 1 > -T && rows + 1 < T)) return true;
    }
    return false;
}

}  // namespace btb

using namespace btb;

extern "C" size_t btb_hip_kv4_tile_bytes(size_t D) { return D == 64 || D == 128 ? kv4_tile_bytes(D) : 0; }

extern "C" int32_t btb_hip_kv4_write(const void* k, const void* v, void* cache, const int32_t* tables, const int32_t* lens,
                                     const int32_t* first, size_t B, size_t W, size_t pages, size_t page, int64_t stride, size_t T,
                                     size_t Hk, size_t D, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head, void* stream) {
    if (!k || !v || !cache || !tables || !lens) return ERR_NULL;
    Kv4Rows p{};
    const int32_t rc = kv4_rows(p, cache, tables, lens, first, B, W, pages, page, stride, T, Hk, D, k_row, k_head, v_row, v_head, k, v,
                                "kv4_write: " KV4_DOMAIN "; k, v and cache 16-byte aligned, strides in multiples of 8; tiles and heads of the rows below 2^24");
    if (rc != OK) return rc;
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)p.groups);
    if (D == 64)
        hipLaunchKernelGGL(kv4_write_kernel<64>, grid, dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL(kv4_write_kernel<128>, grid, dim3(256), 0, st, p);
    return hip_status(hipGetLastError(), "kv4_write launch");
}

extern "C" int32_t btb_hip_kv4_read(const void* cache, const int32_t* tables, const int32_t* lens, const int32_t* first, size_t B,
                                    size_t W, size_t pages, size_t page, int64_t stride, size_t T, size_t Hk, size_t D, void* k,
                                    void* v, int32_t out_f32, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head,
                                    void* stream) {
    if (!k || !v || !cache || !tables || !lens) return ERR_NULL;
    Kv4Rows p{};
    const int32_t rc = kv4_rows(p, cache, tables, lens, first, B, W, pages, page, stride, T, Hk, D, k_row, k_head, v_row, v_head, k, v,
                                "kv4_read: " KV4_DOMAIN "; k, v and cache 16-byte aligned, strides in multiples of 8; tiles and heads of the rows below 2^24");
    if (rc != OK) return rc;
    // rows or heads in one place
    auto shared = [&](int64_t row, int64_t head) {
        return (T > 1 && row < (int64_t)D) || (Hk > 1 && head < (int64_t)D) ||
               (T > 1 && Hk > 1 && row < (int64_t)Hk * head && head < (int64_t)T * row);
    };
    const int64_t apart = ((int64_t)(uintptr_t)v - (int64_t)(uintptr_t)k) / (out_f32 ? 4 : 2);
    if (shared(k_row, k_head) || shared(v_row, v_head) || kv4_outputs_meet(p, apart, (int64_t)D)) {
        set_error("kv4_read: rows or heads of an output, or both outputs, share memory");
        return ERR_DOMAIN;
    }
    p.k_out = k;
    p.v_out = v;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)p.groups);
    if (D == 64)
        hipLaunchKernelGGL((out_f32 ? kv4_read_kernel<64, float> : kv4_read_kernel<64, uint16_t>), grid, dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((out_f32 ? kv4_read_kernel<128, float> : kv4_read_kernel<128, uint16_t>), grid, dim3(256), 0, st, p);
    return hip_status(hipGetLastError(), "kv4_read launch");
}
