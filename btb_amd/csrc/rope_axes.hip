// The q / k norm and a rotation by several position axes, the new keys and values written at slots of their own: what
// a pass needs where a row's place in the cache is not its position - a cache that has been cut down, rows of many
// sequences, pictures among the text.
//
//   r = 1 / sqrt(mean(x^2) + eps), y = x r w           (w: 1 + w where centred; y = x without a weight)
//   out[i]         = y[i] c_i - y[i + D/2] s_i          i < D / 2, c_i and s_i read at the place pos[axes[i]] of the row
//   out[i + D/2]   = y[i + D/2] c_i + y[i] s_i
//
// in f32 throughout, rounded to bf16 once. Bound: memory, the qkv rows read once and q, K and V written once: 16384 rows of 48 heads x 128 take
// 89 us (4.6 TB/s); one row takes 9.1, the launch.
//
// A head by D / 16 lanes: lane l holds dims 8 l .. + 7 and their partners D / 2 further on, so the rotation stays within a lane and
// loads and stores are 16 bytes. A wave takes 1024 / D heads of one row at a time and keeps the row's sixteen cosines and sines;
// many rows: a row a wave, few: a row's heads over several. AT_ONCE groups of heads are on their way at a time: three, or one where
// a wave has no more (16122 rows of 7 + 1 heads x 64: three 42 us, one 35: fewer registers, more waves).

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
    int split;   // waves a row
    int whole;   // the tables' rows, the axes and the norm weights can be read eight values at a time
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

// the lane's eight values of a table's row
__device__ __forceinline__ void table_run(const uint16_t* t, float (&v)[8]) { widen8(*reinterpret_cast<const uint4*>(t), v); }
__device__ __forceinline__ void table_run(const float* t, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(t)[0], b = reinterpret_cast<const float4*>(t)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

template <int D, class TT, int AT_ONCE>
__global__ void __launch_bounds__(256) rope_axes_kernel(RopeAxes p) {
    constexpr int LPH = D / 16, HPW = 64 / LPH, HALF = D / 2;
    const int lane = threadIdx.x & 63, l = lane % LPH, heads = p.Hq + 2 * p.Hk;
    const long long wave = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = (int)(wave / p.split), part = (int)(wave % p.split);
    if (t >= p.T) return;
    const uint16_t* src = p.qkv + (size_t)t * heads * D + 8 * l;
    uint4 lo[AT_ONCE], hi[AT_ONCE];
    auto request = [&](int h0) {
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const uint16_t* from = src + (size_t)min(h0 + u * p.split * HPW, heads - 1) * D;
            lo[u] = load_stream16(reinterpret_cast<const uint4*>(from));
            hi[u] = load_stream16(reinterpret_cast<const uint4*>(from + HALF));
        }
    };
    int head = part * HPW + lane / LPH;
    request(head);
    const int slot = p.slots[t];
    const bool kept = slot >= 0 && slot < p.cap;
    // the row's angles: a lane's eight frequencies, by the row's place on each one's axis
    float c[8], s[8];
    {
        const TT* cos_t = static_cast<const TT*>(p.cos_t) + 8 * l;
        const TT* sin_t = static_cast<const TT*>(p.sin_t) + 8 * l;
        auto place = [&](int axis) {
            return (size_t)min(max(p.pos[(size_t)min(axis, p.A - 1) * p.T + t], 0), p.positions - 1) * p.cs;
        };
        const uint8_t* ax = p.axes + 8 * l;
        bool run = false;
        uint2 a8 = make_uint2(0u, 0u);
        if (p.whole) {  // uniform
            a8 = *reinterpret_cast<const uint2*>(ax);
            run = a8.x == a8.y && a8.x == (a8.x & 0xFFu) * 0x01010101u;
        }
        if (run) {
            const size_t at = place((int)(a8.x & 0xFFu));
            table_run(cos_t + at, c);
            table_run(sin_t + at, s);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const size_t at = place(ax[e]) + e;
                c[e] = table_value(cos_t, at);
                s[e] = table_value(sin_t, at);
            }
        }
    }
    const float one = p.centered ? 1.f : 0.f;
    uint4 wn[2][2];  // the lane's norm weights, q's and k's
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint16_t* w = i ? p.wk : p.wq;
        wn[i][0] = wn[i][1] = make_uint4(0u, 0u, 0u, 0u);
        if (w != nullptr) {  // uniform
            for (int e = 0; e < 2; ++e) {
                if (p.whole) {
                    wn[i][e] = *reinterpret_cast<const uint4*>(w + e * HALF + 8 * l);
                    continue;
                }
                uint32_t x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = (uint32_t)w[e * HALF + 8 * l + 2 * j] | (uint32_t)w[e * HALF + 8 * l + 2 * j + 1] << 16;
                wn[i][e] = make_uint4(x[0], x[1], x[2], x[3]);
            }
        }
    }
    for (; __any(head < heads); head += AT_ONCE * p.split * HPW) {
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int hd = head + u * p.split * HPW;
            if (hd >= heads) continue;
            if (hd >= p.Hq + p.Hk) {
                if (!kept) continue;
                uint16_t* dst = p.V + (size_t)(hd - p.Hq - p.Hk) * p.hs + (size_t)slot * p.rs + 8 * l;
                *reinterpret_cast<uint4*>(dst) = lo[u];
                *reinterpret_cast<uint4*>(dst + HALF) = hi[u];
                continue;
            }
            const bool is_q = hd < p.Hq;
            float a[8], b[8];
            widen8(lo[u], a);
            widen8(hi[u], b);
            if ((is_q ? p.wq : p.wk) != nullptr) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
                ss += dpp_f32<0xB1>(ss);
                ss += dpp_f32<0x4E>(ss);
                if (LPH >= 8) ss += dpp_f32<0x141>(ss);
                if (LPH >= 16) ss += dpp_f32<0x140>(ss);
                const float r = 1.f / sqrtf(ss / (float)D + p.eps);
                float wa[8], wb[8];
                widen8(is_q ? wn[0][0] : wn[1][0], wa);
                widen8(is_q ? wn[0][1] : wn[1][1], wb);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    a[e] *= r * (wa[e] + one);
                    b[e] *= r * (wb[e] + one);
                }
            }
            float x[8], y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = fmaf(a[e], c[e], -(b[e] * s[e]));
                y[e] = fmaf(b[e], c[e], a[e] * s[e]);
            }
            uint16_t* dst;
            if (is_q) {
                dst = p.q + ((size_t)t * p.Hq + hd) * D + 8 * l;
            } else {
                if (!kept) continue;
                dst = p.K + (size_t)(hd - p.Hq) * p.hs + (size_t)slot * p.rs + 8 * l;
            }
            *reinterpret_cast<uint4*>(dst) = narrow8(x);
            *reinterpret_cast<uint4*>(dst + HALF) = narrow8(y);
        }
        if (__any(head + AT_ONCE * p.split * HPW < heads)) request(head + AT_ONCE * p.split * HPW);
    }
}

template <int D>
static void launch_rope_axes(RopeAxes& p, bool wide_table, hipStream_t st) {
    // waves a row: until eight a CU are there
    const int groups = (p.Hq + 2 * p.Hk + 1024 / D - 1) / (1024 / D), want = (8 * device_info().cus + p.T - 1) / p.T;
    p.split = want < groups ? want : groups;
    const dim3 grid((unsigned)(((long long)p.T * p.split + 3) / 4));
    const bool once = p.split == groups;  // a wave has one group of heads
    if (wide_table)
        hipLaunchKernelGGL((once ? rope_axes_kernel<D, float, 1> : rope_axes_kernel<D, float, 3>), grid, dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((once ? rope_axes_kernel<D, uint16_t, 1> : rope_axes_kernel<D, uint16_t, 3>), grid, dim3(256), 0, st, p);
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
    if (T == 0 || T > (1u << 24) || Hq == 0 || Hk == 0 || Hq + 2 * Hk > 65535 || (D != 64 && D != 128 && D != 256) || A == 0 ||
        A > 255 || positions == 0 || positions > 0x7FFFFFFFu || cap == 0 || cap > 0x7FFFFFFFu || table_stride < D / 2 ||
        table_stride > 0x7FFFFFFFu || hs < 0 || rs < 0 || (hs == 0 && Hk > 1) || (rs == 0 && cap > 1) || hs % 8 || rs % 8 || !aligned16(qkv) || !aligned16(q) ||
        !aligned16(K) || !aligned16(V)) {
        set_error("norm_rope_axes: 1 .. 2^24 rows, head_dim 64, 128 or 256, 1 .. 255 axes, tables at least D / 2 wide, qkv, q, "
                  "K and V 16-byte aligned with strides in multiples of 8, no two rows of K in one place");
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
    p.whole = aligned16(cos_t) && aligned16(sin_t) && aligned16(wq) && aligned16(wk) && table_stride % 8 == 0 && ((uintptr_t)axes & 7u) == 0 ? 1 : 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (D == 64)
        launch_rope_axes<64>(p, table_f32 != 0, st);
    else if (D == 128)
        launch_rope_axes<128>(p, table_f32 != 0, st);
    else
        launch_rope_axes<256>(p, table_f32 != 0, st);
    return hip_status(hipGetLastError(), "norm_rope_axes launch");
}
