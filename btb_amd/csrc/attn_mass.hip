// The attention weight every cached key received from a pass, added to what it had:
//
//   out[g, j] = mass[g, j] + sum over rows t with j < seen[t], query heads h of g, of exp(scale q_{t,h} . k_j - lse[t, h])
//
// lse is what the pass's attention left (btb_hip_attn_shared). A wave holds 32 keys as a stationary operand and takes the
// pass's (row, head) pairs 32 at a time; a lane's sixteen sums (btb_tile32.hpp) stay in its registers until the end, so the
// order of the additions is fixed. Everything after the product is f32.

#include "btb_common.hpp"
#include "btb_tile32.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

struct MassArgs {
    const uint16_t* q;
    const uint16_t* K;
    const float* lse;      // [T, Hq]
    const int32_t* seen;   // [T]
    const float* mass;     // rows of `ms` floats, or none
    float* out;            // rows of `os` floats
    long long hs, rs, ms, os;
    float scale_log2;
    int T, Hq, G, n;
};

template <int D>
__global__ void __launch_bounds__(256) attn_mass_kernel(MassArgs p) {
    constexpr int STEPS = D / 16;
    const int g = blockIdx.y, lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
    const int k0 = (blockIdx.x * 4 + wv) * TK;
    if (k0 >= p.n) return;
    const uint16_t* kr = p.K + (size_t)g * p.hs + (size_t)min(k0 + c, p.n - 1) * p.rs + 8 * h;
    bf16x8 kf[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) kf[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(kr + 16 * s));
    const int pairs = p.T * p.G;
    float sum[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = 0.f;
    for (int r0 = 0; r0 < pairs; r0 += 32) {
        const int r = min(r0 + c, pairs - 1), t = r / p.G;
        const size_t at = (size_t)t * p.Hq + g * p.G + (r - t * p.G);
        const float z = p.lse[at];
        // a pair past the last, or one that saw nothing, adds nothing
        const int lim = r0 + c < pairs && z != -__builtin_inff() ? p.seen[t] : 0;
        const float zl = z * 1.44269504088896341f;
        f32x16 st = zero16();
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
            st = mfma32(kf[s], __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(p.q + at * D + 16 * s + 8 * h)), st);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sum[i] += k0 + 8 * (i / 4) + 4 * h + i % 4 < lim ? __builtin_amdgcn_exp2f(fmaf(st[i], p.scale_log2, -zl)) : 0.f;
    }
    // over the 32 pairs of a tile: the same key in the 32 lanes of a half
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float v = sum[i];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) v += __shfl_xor(v, d, WAVE);
        const int key = k0 + 8 * (i / 4) + 4 * h + i % 4;
        if (c == i && key < p.n)
            p.out[(size_t)g * p.os + key] = v + (p.mass != nullptr ? p.mass[(size_t)g * p.ms + key] : 0.f);
    }
}

}  // namespace btb

using namespace btb;

extern "C" {

int32_t btb_hip_attn_mass(const void* q, const void* K, const float* lse, const int32_t* seen, const float* mass, float* out,
                          size_t T, size_t Hq, size_t Hk, size_t D, size_t n, int64_t hs, int64_t rs, int64_t mass_stride,
                          int64_t out_stride, float scale, void* stream) {
    if (!q || !K || !lse || !seen || !out) return ERR_NULL;
    auto loose = [](const void* a) { return ((uintptr_t)a & 15u) != 0; };
    if (T == 0 || T > 65536 || Hk == 0 || Hk > 1024 || Hq == 0 || Hq % Hk != 0 || Hq / Hk > 32 || (D != 64 && D != 128) ||
        n == 0 || n > 0x7FFFFF00u || hs < 0 || rs < 0 || hs % 8 || rs % 8 || mass_stride < 0 || out_stride < 0 ||
        !(scale > 0.f) || !(scale < __builtin_inff()) || loose(q) || loose(K)) {
        set_error("attn_mass: head_dim 64 or 128, up to 32 query heads a kv head, a positive scale, q and K 16-byte aligned "
                  "with strides in multiples of 8");
        return ERR_DOMAIN;
    }
    MassArgs p;
    p.q = static_cast<const uint16_t*>(q);
    p.K = static_cast<const uint16_t*>(K);
    p.lse = lse;
    p.seen = seen;
    p.mass = mass;
    p.out = out;
    p.hs = hs;
    p.rs = rs;
    p.ms = mass_stride;
    p.os = out_stride;
    p.scale_log2 = scale * 1.44269504088896341f;
    p.T = (int)T;
    p.Hq = (int)Hq;
    p.G = (int)(Hq / Hk);
    p.n = (int)n;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)((n + 4 * TK - 1) / (4 * TK)), (unsigned)Hk);
    if (D == 64)
        hipLaunchKernelGGL(attn_mass_kernel<64>, grid, dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL(attn_mass_kernel<128>, grid, dim3(256), 0, st, p);
    return hip_status(hipGetLastError(), "attn_mass launch");
}

}  // extern "C"
