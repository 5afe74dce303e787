// A cache cut to its heaviest keys. Of a head's n keys the first `kept` in the order (mass descending, slot ascending)
// stay, where a key among the first positions (pos < sinks) or the newest (pos >= recent_from) counts as +inf and a NaN as
// -inf. Kept keys below slot `kept` stay where they are; those above it, ascending, fill the holes below, ascending:
// idx[j] is the slot that slot j's key comes from. Sources of moved keys lie past every destination, so the same cache may
// be given as input and output. Attention does not depend on the keys' order; `pos` tells what stood where.
//
// Two launches: the choice, a workgroup a head - the mass of the last key that stays by its bits, eight at a time, then
// the ranks by running counts - and the rows' move, 16 bytes a lane.
// Bound: memory: mass and pos read, the moved rows read and written.

#include "btb_common.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

constexpr int EV_THREADS = 1024;

struct EvictArgs {
    const float* mass;
    const int32_t* pos;
    int32_t* idx;        // [heads, kept]
    long long ms, ps;    // values between two heads of mass and of pos
    int n, kept, sinks, recent_from;
};

// a key's rank as an unsigned number, larger stays first
__device__ __forceinline__ uint32_t rank_bits(float m, int pos, int sinks, int recent_from) {
    if (pos < sinks || pos >= recent_from) return 0xFF800000u;  // +inf's
    if (m != m) return 0x007FFFFFu;                              // -inf's
    const uint32_t b = f32_bits(m + 0.f);                        // (-0 as 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// the sum of v over the threads before this one, and over all, in thread order
__device__ __forceinline__ int before(int v, int* waves, int& total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    int run = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(run, d, WAVE);
        if (lane >= d) run += o;
    }
    if (lane == 63) waves[wv] = run;
    __syncthreads();
    int ahead = 0;
    total = 0;
    for (int i = 0; i < EV_THREADS / 64; ++i) {
        if (i < wv) ahead += waves[i];
        total += waves[i];
    }
    __syncthreads();
    return ahead + run - v;
}

__global__ void __launch_bounds__(EV_THREADS) evict_choose_kernel(EvictArgs p) {
    __shared__ int hist[256], waves[EV_THREADS / 64], pick[2];
    const int tid = threadIdx.x;
    const float* mass = p.mass + (size_t)blockIdx.x * p.ms;
    const int32_t* pos = p.pos + (size_t)blockIdx.x * p.ps;
    int32_t* idx = p.idx + (size_t)blockIdx.x * p.kept;
    auto rank = [&](int j) { return rank_bits(mass[j], pos[j], p.sinks, p.recent_from); };
    // the rank of the last key that stays, and how many of that rank do
    uint32_t prefix = 0;
    int left = p.kept;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j = tid; j < p.n; j += EV_THREADS) {
            const uint32_t r = rank(j);
            if (shift == 24 || (r >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(r >> shift) & 255u], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int b = 255, more = 0;
            while (b > 0 && more + hist[b] < left) more += hist[b--];
            pick[0] = b;
            pick[1] = left - more;
        }
        __syncthreads();
        prefix |= (uint32_t)pick[0] << shift;
        left = pick[1];
        __syncthreads();
    }
    const uint32_t last = prefix;
    // of the keys of that rank the first `left` stay
    auto stays = [&](int j, int end, int& equal) {
        const uint32_t r = j < end ? rank(j) : 0u;
        const bool same = j < end && r == last;
        int all;
        const int mine = equal + before(same ? 1 : 0, waves, all);
        equal += all;
        return j < end && (r > last || (same && mine < left));
    };
    int equal = 0;
    for (int j0 = 0; j0 < p.kept; j0 += EV_THREADS) {
        int all;
        const int j = j0 + tid;
        before(j < p.kept && rank(j) == last ? 1 : 0, waves, all);
        equal += all;
    }
    // the kept keys past the end, in order, into the first places of idx
    int over = 0;
    for (int j0 = p.kept; j0 < p.n; j0 += EV_THREADS) {
        const int j = j0 + tid;
        const bool s = stays(j, p.n, equal);
        int all;
        const int at = over + before(s ? 1 : 0, waves, all);
        if (s) idx[at] = j;
        over += all;
    }
    __syncthreads();
    // from the end on, so that a hole's key is read before its place is written: the i-th hole lies at slot i or later
    int end = over, tie = 0;
    for (int j0 = 0; j0 < p.kept; j0 += EV_THREADS) {
        int all;
        const int j = j0 + tid;
        before(j < p.kept && rank(j) == last ? 1 : 0, waves, all);
        tie += all;
    }
    for (int j0 = (p.kept - 1) / EV_THREADS * EV_THREADS; j0 >= 0; j0 -= EV_THREADS) {
        const int j = j0 + tid;
        const uint32_t r = j < p.kept ? rank(j) : 0u;
        const bool same = j < p.kept && r == last;
        int all;
        const int ahead = before(same ? 1 : 0, waves, all);
        tie -= all;
        const bool s = j < p.kept && (r > last || (same && tie + ahead < left));
        const int holes_ahead = before(j < p.kept && !s ? 1 : 0, waves, all);
        end -= all;
        int from = j;
        if (j < p.kept && !s) from = idx[end + holes_ahead];
        __syncthreads();
        if (j < p.kept) idx[j] = from;
        __syncthreads();
    }
}

struct MoveArgs {
    const uint16_t* K;
    const uint16_t* V;
    uint16_t* K_out;
    uint16_t* V_out;
    const float* mass;
    const int32_t* pos;
    float* mass_out;
    int32_t* pos_out;
    const int32_t* idx;
    long long ls, hs, rs, lo, ho, ro;  // strides of the layers, heads and rows, in and out
    long long ms, ps, mo, po;
    int Hk, kept, chunks;  // 16-byte chunks a row
    int in_place;
};

__global__ void __launch_bounds__(256) evict_move_kernel(MoveArgs p) {
    const int head = blockIdx.y, layer = head / p.Hk, g = head % p.Hk;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const int j = (int)(at / p.chunks), c = (int)(at % p.chunks);
    if (j >= p.kept) return;
    const int from = p.idx[(size_t)head * p.kept + j];
    if (p.in_place && from == j) return;
    const size_t src = (size_t)layer * p.ls + (size_t)g * p.hs + (size_t)from * p.rs + 8 * c;
    const size_t dst = (size_t)layer * p.lo + (size_t)g * p.ho + (size_t)j * p.ro + 8 * c;
    *reinterpret_cast<uint4*>(p.K_out + dst) = *reinterpret_cast<const uint4*>(p.K + src);
    *reinterpret_cast<uint4*>(p.V_out + dst) = *reinterpret_cast<const uint4*>(p.V + src);
    if (c == 0) {
        p.mass_out[(size_t)head * p.mo + j] = p.mass[(size_t)head * p.ms + from];
        p.pos_out[(size_t)head * p.po + j] = p.pos[(size_t)head * p.ps + from];
    }
}

}  // namespace btb

using namespace btb;

extern "C" int32_t btb_hip_kv_evict(const float* mass, int64_t ms, const int32_t* pos, int64_t ps, const void* K, const void* V,
                                    int64_t ls, int64_t hs, int64_t rs, size_t L, size_t Hk, size_t D, size_t n, size_t budget,
                                    int32_t sinks, int32_t recent_from, void* K_out, void* V_out, int64_t lo, int64_t ho,
                                    int64_t ro, float* mass_out, int64_t mo, int32_t* pos_out, int64_t po, int32_t* idx,
                                    void* stream) {
    if (!mass || !pos || !K || !V || !K_out || !V_out || !mass_out || !pos_out || !idx) return ERR_NULL;
    auto loose = [](const void* a) { return ((uintptr_t)a & 15u) != 0; };
    auto odd = [](int64_t s) { return s < 0 || s % 8 != 0; };
    const bool in_place = K == K_out;
    if (L == 0 || Hk == 0 || L > 65535 || Hk > 65535 || L * Hk > 65535 || D == 0 || D % 8 || D > 1024 || n == 0 ||
        n > 0x7FFFF000u || budget == 0 || ms < 0 || ps < 0 || mo < 0 || po < 0 || odd(ls) || odd(hs) || odd(rs) || odd(lo) ||
        odd(ho) || odd(ro) || loose(K) || loose(V) || loose(K_out) || loose(V_out) || in_place != (V == V_out) ||
        in_place != (mass == mass_out) || in_place != (pos == pos_out) ||
        (in_place && (ls != lo || hs != ho || rs != ro || ms != mo || ps != po))) {
        set_error("kv_evict: at most 65535 heads in all, head_dim a multiple of 8, K and V 16-byte aligned with strides in "
                  "multiples of 8; in place: all four outputs the inputs with their strides, or none");
        return ERR_DOMAIN;
    }
    EvictArgs e;
    e.mass = mass;
    e.pos = pos;
    e.idx = idx;
    e.ms = ms;
    e.ps = ps;
    e.n = (int)n;
    e.kept = (int)(budget < n ? budget : n);
    e.sinks = sinks;
    e.recent_from = recent_from;
    hipStream_t st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(evict_choose_kernel, dim3((unsigned)(L * Hk)), dim3(EV_THREADS), 0, st, e);
    MoveArgs m;
    m.K = static_cast<const uint16_t*>(K);
    m.V = static_cast<const uint16_t*>(V);
    m.K_out = static_cast<uint16_t*>(K_out);
    m.V_out = static_cast<uint16_t*>(V_out);
    m.mass = mass;
    m.pos = pos;
    m.mass_out = mass_out;
    m.pos_out = pos_out;
    m.idx = idx;
    m.ls = ls;
    m.hs = hs;
    m.rs = rs;
    m.lo = lo;
    m.ho = ho;
    m.ro = ro;
    m.ms = ms;
    m.ps = ps;
    m.mo = mo;
    m.po = po;
    m.Hk = (int)Hk;
    m.kept = e.kept;
    m.chunks = (int)(D / 8);
    m.in_place = in_place ? 1 : 0;
    const unsigned blocks = (unsigned)(((size_t)e.kept * m.chunks + 255) / 256);
    hipLaunchKernelGGL(evict_move_kernel, dim3(blocks, (unsigned)(L * Hk)), dim3(256), 0, st, m);
    return hip_status(hipGetLastError(), "kv_evict launch");
}
