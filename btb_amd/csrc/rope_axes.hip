// The q / k norm and a rotation by several position axes, the new keys and values written at slots of their own: what
// a pass needs where a row's place in the cache is not its position - a cache that has been cut down, rows of many
// sequences, pictures among the text.
//
//   r = 1 / sqrt(mean(x^2) + eps), y = x r w           (w: 1 + w where centred; y = x without a weight)
//   out[i]         = y[i] c_i - y[i + D/2] s_i          i < D / 2, c_i and s_i read at the place pos[axes[i]] of the row
//   out[i + D/2]   = y[i + D/2] c_i + y[i] s_i
//
// in f32 throughout, rounded to bf16 once. Bound: memory, the qkv rows read once and q, K and V written once.

#include "btb_common.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

struct RopeAxes {
    const uint16_t* qkv;
    const uint16_t* wq;
    const uint16_t* wk;
    const void* cos_t;
    const void* sin_t;
    const int32_t* pos;    // [A, T]
    const uint8_t* axes;   // [D / 2]
    const int32_t* slots;  // [T]
    uint16_t* K;
    uint16_t* V;
    uint16_t* q;
    long long cs;          // values between two positions of a table
    long long hs, rs;
    float eps;
    int T, A, positions, cap, Hq, Hk, centered;
};

template <class TT>
__device__ __forceinline__ float table_value(const TT* t, size_t at);
template <>
__device__ __forceinline__ float table_value<uint16_t>(const uint16_t* t, size_t at) {
    return bf16_f32(t[at]);
}
template <>
__device__ __forceinline__ float table_value<float>(const float* t, size_t at) {
    return t[at];
}

__device__ __forceinline__ void widen8(const uint4& w, float (&v)[8]) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16lo_f32(x[i]);
        v[2 * i + 1] = bf16hi_f32(x[i]);
    }
}
__device__ __forceinline__ uint4 narrow8(const float (&v)[8]) {
    return make_uint4(f32x2_bf16(v[0], v[1]), f32x2_bf16(v[2], v[3]), f32x2_bf16(v[4], v[5]), f32x2_bf16(v[6], v[7]));
}

// A head by D / 16 lanes: lane l holds dims 8 l .. + 7 and their partners D / 2 further on, so the rotation stays within
// a lane and loads and stores are 16 bytes. A wave takes 1024 / D heads of one row.
template <int D, class TT>
__global__ void __launch_bounds__(64) rope_axes_kernel(RopeAxes p) {
    constexpr int LPH = D / 16, HPW = 64 / LPH, HALF = D / 2;
    const int t = blockIdx.y, lane = threadIdx.x, l = lane % LPH;
    const int head = blockIdx.x * HPW + lane / LPH, heads = p.Hq + 2 * p.Hk;
    if (head >= heads) return;
    const uint16_t* src = p.qkv + ((size_t)t * heads + head) * D + 8 * l;
    const uint4 lo = *reinterpret_cast<const uint4*>(src), hi = *reinterpret_cast<const uint4*>(src + HALF);
    const int slot = p.slots[t];
    const bool kept = slot >= 0 && slot < p.cap;
    if (head >= p.Hq + p.Hk) {
        if (!kept) return;
        uint16_t* dst = p.V + (size_t)(head - p.Hq - p.Hk) * p.hs + (size_t)slot * p.rs + 8 * l;
        *reinterpret_cast<uint4*>(dst) = lo;
        *reinterpret_cast<uint4*>(dst + HALF) = hi;
        return;
    }
    const bool is_q = head < p.Hq;
    float a[8], b[8];
    widen8(lo, a);
    widen8(hi, b);
    const uint16_t* wn = is_q ? p.wq : p.wk;
    if (wn != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
        ss += dpp_f32<0xB1>(ss);
        ss += dpp_f32<0x4E>(ss);
        if (LPH >= 8) ss += dpp_f32<0x141>(ss);
        if (LPH >= 16) ss += dpp_f32<0x140>(ss);
        const float r = 1.f / sqrtf(ss / (float)D + p.eps);
        const float one = p.centered ? 1.f : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a[e] *= r * (bf16_f32(wn[8 * l + e]) + one);
            b[e] *= r * (bf16_f32(wn[HALF + 8 * l + e]) + one);
        }
    }
    const TT* cos_t = static_cast<const TT*>(p.cos_t);
    const TT* sin_t = static_cast<const TT*>(p.sin_t);
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int i = 8 * l + e, axis = min((int)p.axes[i], p.A - 1);
        const int at = min(max(p.pos[(size_t)axis * p.T + t], 0), p.positions - 1);
        const float c = table_value(cos_t, (size_t)at * p.cs + i), s = table_value(sin_t, (size_t)at * p.cs + i);
        x[e] = fmaf(a[e], c, -(b[e] * s));
        y[e] = fmaf(b[e], c, a[e] * s);
    }
    uint16_t* dst;
    if (is_q) {
        dst = p.q + ((size_t)t * p.Hq + head) * D + 8 * l;
    } else {
        if (!kept) return;
        dst = p.K + (size_t)(head - p.Hq) * p.hs + (size_t)slot * p.rs + 8 * l;
    }
    *reinterpret_cast<uint4*>(dst) = narrow8(x);
    *reinterpret_cast<uint4*>(dst + HALF) = narrow8(y);
}

template <int D>
static void launch_rope_axes(const RopeAxes& p, bool wide_table, hipStream_t st) {
    constexpr int HPW = 1024 / D;
    const dim3 grid((unsigned)((p.Hq + 2 * p.Hk + HPW - 1) / HPW), (unsigned)p.T);
    if (wide_table)
        hipLaunchKernelGGL((rope_axes_kernel<D, float>), grid, dim3(64), 0, st, p);
    else
        hipLaunchKernelGGL((rope_axes_kernel<D, uint16_t>), grid, dim3(64), 0, st, p);
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace btb

using namespace btb;

extern "C" int32_t btb_hip_norm_rope_axes(const void* qkv, const void* wq, const void* wk, float eps, const void* cos_t,
                                          const void* sin_t, int32_t table_f32, size_t positions, size_t table_stride,
                                          const int32_t* pos, size_t A, const uint8_t* axes, const int32_t* slots, void* K,
                                          void* V, void* q, size_t T, size_t Hq, size_t Hk, size_t D, size_t cap,
                                          int64_t hs, int64_t rs, int32_t centered, void* stream) {
    if (!qkv || !cos_t || !sin_t || !pos || !axes || !slots || !K || !V || !q) return ERR_NULL;
    if (T == 0 || T > 65535 || Hq == 0 || Hk == 0 || Hq + 2 * Hk > 65535 || (D != 64 && D != 128 && D != 256) || A == 0 ||
        A > 255 || positions == 0 || positions > 0x7FFFFFFFu || cap == 0 || cap > 0x7FFFFFFFu || table_stride < D / 2 ||
        table_stride > 0x7FFFFFFFu || hs < 0 || rs < 0 || hs % 8 || rs % 8 || !aligned16(qkv) || !aligned16(q) ||
        !aligned16(K) || !aligned16(V)) {
        set_error("norm_rope_axes: 1 .. 65535 rows, head_dim 64, 128 or 256, 1 .. 255 axes, tables at least D / 2 wide, qkv, q, "
                  "K and V 16-byte aligned with strides in multiples of 8");
        return ERR_DOMAIN;
    }
    RopeAxes p;
    p.qkv = static_cast<const uint16_t*>(qkv);
    p.wq = static_cast<const uint16_t*>(wq);
    p.wk = static_cast<const uint16_t*>(wk);
    p.cos_t = cos_t;
    p.sin_t = sin_t;
    p.pos = pos;
    p.axes = axes;
    p.slots = slots;
    p.K = static_cast<uint16_t*>(K);
    p.V = static_cast<uint16_t*>(V);
    p.q = static_cast<uint16_t*>(q);
    p.cs = (long long)table_stride;
    p.hs = hs;
    p.rs = rs;
    p.eps = eps;
    p.T = (int)T;
    p.A = (int)A;
    p.positions = (int)positions;
    p.cap = (int)cap;
    p.Hq = (int)Hq;
    p.Hk = (int)Hk;
    p.centered = centered;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (D == 64)
        launch_rope_axes<64>(p, table_f32 != 0, st);
    else if (D == 128)
        launch_rope_axes<128>(p, table_f32 != 0, st);
    else
        launch_rope_axes<256>(p, table_f32 != 0, st);
    return hip_status(hipGetLastError(), "norm_rope_axes launch");
}
