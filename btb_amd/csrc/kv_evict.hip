// A cache cut to its heaviest keys. Of a head's n keys the first `kept` in the order (mass descending, slot ascending)
// stay, where a key among the first positions (pos < sinks) or the newest (pos >= recent_from) counts as +inf and a NaN as
// -inf. Kept keys below slot `kept` stay where they are; those above it, ascending, fill the holes below, ascending:
// idx[j] is the slot that slot j's key comes from. Sources of moved keys lie past every destination, so the same cache may
// be given as input and output. Attention does not depend on the keys' order; `pos` tells what stood where.
//
// The choice, then the rows' move, 16 bytes a lane. The choice finds the rank of the last key that stays, eleven, eleven and
// ten bits at a time from the top (histograms in LDS), counts what stays and then writes the order. A wave takes a stretch of
// the slots below `kept` and one of those above, so its own running count is all that its keys' order needs, and the waves
// meet in one scan. A workgroup takes a head of up to 8192 keys alone, ranks in LDS, one launch; a longer one is cut over
// workgroups of 8192 keys and the rounds are launches (six), since what a key costs is arithmetic. The second round reads every
// workgroup's histogram in every workgroup, 4 KB times the square of their number a head: 1 MB at 131072 keys, 4 GB at 2^23.
//
// us, a workgroup a head / the rounds: 8192 keys to 4096 x 8 heads 18.9 / 30.7, x 32 39.4 / 51.6, x 288 260 / 274; the choice alone of
// 131072 keys x 32 358 / 49. Bound: memory, mass and pos read, the moved rows read and written: 4608 keys to 4096 x 288 heads 245 us
// (5.0 TB/s); 131072 to 16384 x 32 heads 153 us, of which the move 104 and the first round, additions in LDS, 19; 700 to 512 x 8 heads
// 13.5 us, two launches of 6 and 4.

#include "btb_common.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64, EV_BINS = 2048;
constexpr int EV_KEYS = 8192, EV_PER = EV_KEYS / EV_THREADS;  // keys a workgroup, and a thread
constexpr int EV_COPIES = 8;  // words a bin of a long head's histograms (131072 keys x 32 heads: 4 words 158 us a call, 8 153)
constexpr int EV_BLOCKS = 1024;                               // workgroups a head: their counts meet in one scan

// what a long head keeps between the launches, in the call's workspace
struct EvictWork {
    uint32_t* rank;   // [n]
    uint32_t* first;  // [blocks][EV_BINS / 2] two counts a word: the first round's histograms
    int* later;       // [2][EV_BINS]: the later rounds'
    int* state;       // [4][2]: after a round, the bits found so far and how many keys of them stay
    int* counts;      // [blocks][4]: above and with the last rank, below slot `kept` and past it
    int* list;        // [n / 2]: the slots of the kept keys at or past `kept`
};
__host__ __device__ inline size_t evict_words(size_t n) {
    const size_t blocks = (n + EV_KEYS - 1) / EV_KEYS;
    return ((n + 3) / 4 * 4 + blocks * (EV_BINS / 2) + 2 * EV_BINS + 8 + 4 * blocks + n / 2 + 3) / 4 * 4;
}

struct EvictArgs {
    const float* mass;
    const int32_t* pos;
    int32_t* idx;      // [heads, kept]
    uint32_t* work;    // [heads][evict_words(n)]
    long long ms, ps;  // values between two heads of mass and of pos
    int n, kept, sinks, recent_from;
};
__device__ __forceinline__ EvictWork work_of(const EvictArgs& p, int head) {
    const size_t blocks = (p.n + EV_KEYS - 1) / EV_KEYS;
    EvictWork w;
    w.rank = p.work + (size_t)head * evict_words(p.n);
    w.first = w.rank + (p.n + 3) / 4 * 4;
    w.later = reinterpret_cast<int*>(w.first + blocks * (EV_BINS / 2));
    w.state = w.later + 2 * EV_BINS;
    w.counts = w.state + 8;
    w.list = w.counts + 4 * blocks;
    return w;
}

// a key's rank as an unsigned number, larger stays first
__device__ __forceinline__ uint32_t rank_bits(float m, int pos, int sinks, int recent_from) {
    if (pos < sinks || pos >= recent_from) return 0xFF800000u;  // +inf's
    if (m != m) return 0x007FFFFFu;                              // -inf's
    const uint32_t b = f32_bits(m + 0.f);                        // (-0 as 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One more in the bin of every lane that counts. Many keys share one rank - those that received nothing, those that stay
// whatever they weigh - and most others a few exponents, and additions to one word wait for one another: a bin is COPIES words that
// neighbouring lanes take in turn.
template <int COPIES>
__device__ __forceinline__ void count(int* hist, int bin, bool counts, int lane) {
    if (counts) atomicAdd(&hist[COPIES * bin + lane % COPIES], 1);
}
template <int COPIES>
__device__ __forceinline__ int counted(const int* hist, int bin) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < COPIES; ++i) n += hist[COPIES * bin + i];
    return n;
}
__device__ __forceinline__ int digit(uint32_t r, int round) {
    return (int)(round == 0 ? r >> 21 : round == 1 ? (r >> 10) & 2047u : r & 1023u);
}
// whether a rank has the bits that the rounds before this one found
__device__ __forceinline__ bool with(uint32_t r, uint32_t last, int round) {
    return round == 0 || (round == 1 ? (r ^ last) >> 21 == 0 : (r ^ last) >> 10 == 0);
}

// the sum over the lanes up to this one
__device__ __forceinline__ int wave_running(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // lane 15 of a row into the next, lane 31 into the upper half
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
// the sum over the threads before this one; `waves` is free again after the caller's next barrier
__device__ __forceinline__ int before(int v, int* waves, int lane, int wv) {
    const int run = wave_running(v);
    if (lane == 63) waves[wv] = run;
    __syncthreads();
    const int all = wave_running(lane < EV_WAVES ? waves[lane] : 0);
    return run - v + (wv > 0 ? __builtin_amdgcn_readlane(all, wv - 1) : 0);
}

// The bin, from the largest down, in which the count of keys reaches `left`, and how many of that bin that takes: a thread has
// the counts of bins EV_BINS - 1 - 2 tid and the one below.
__device__ __forceinline__ void find(int h0, int h1, int& left, uint32_t& bin, int* waves, int* pick, int tid, int lane, int wv) {
    const int more = before(h0 + h1, waves, lane, wv);
    if (more < left && more + h0 + h1 >= left) {
        const bool upper = more + h0 >= left;
        pick[0] = EV_BINS - 1 - 2 * tid - (upper ? 0 : 1);
        pick[1] = left - more - (upper ? 0 : h0);
    }
    __syncthreads();
    bin = (uint32_t)pick[0];
    left = pick[1];
    __syncthreads();
}

// keys above the last rank and with it, of a wave's stretch
__device__ __forceinline__ void tally(uint32_t r, bool in, uint32_t last, int& above, int& same) {
    above += __popcll(__ballot(in && r > last));
    same += __popcll(__ballot(in && r == last));
}
// whether the lane's key stays: above the last rank, or among the first `left` with it; `ties` counts those so far
__device__ __forceinline__ bool stays(uint32_t r, bool in, uint32_t last, int left, int& ties, int lane) {
    const unsigned long long same = __ballot(in && r == last), mine = 1ull << lane;
    const bool s = in && (r > last || ((same & mine) && ties + __popcll(same & (mine - 1)) < left));
    ties += __popcll(same);
    return s;
}
__device__ __forceinline__ int lanes_before(unsigned long long set, int lane) { return __popcll(set & ((1ull << lane) - 1)); }

// a wave's share of slots [begin, end), whole groups of 64
__device__ __forceinline__ void share(int begin, int end, int wv, int& from, int& to) {
    const int per = ((end - begin + EV_WAVES - 1) / EV_WAVES + 63) / 64 * 64;
    from = min(begin + wv * per, end);
    to = min(from + per, end);
}

// a head of up to EV_KEYS keys
__global__ void __launch_bounds__(EV_THREADS) evict_choose_kernel(EvictArgs p) {
    extern __shared__ __align__(16) uint32_t rank[];  // [n], then the list [n / 2]
    __shared__ __align__(16) int hist[4 * EV_BINS];
    __shared__ int waves[EV_WAVES], pick[2], counts[2][2][EV_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* mass = p.mass + (size_t)blockIdx.x * p.ms;
    const int32_t* pos = p.pos + (size_t)blockIdx.x * p.ps;
    int32_t* idx = p.idx + (size_t)blockIdx.x * p.kept;
    uint32_t* list = rank + p.n;
    uint32_t r[EV_PER];
#pragma unroll
    for (int i = 0; i < EV_PER; ++i) {
        const int j = EV_THREADS * i + tid;
        r[i] = j < p.n ? rank_bits(mass[j], pos[j], p.sinks, p.recent_from) : 0u;
        if (j < p.n) rank[j] = r[i];
    }
    uint32_t last = 0;
    int left = p.kept;
    for (int round = 0; round < 3; ++round) {
        reinterpret_cast<int4*>(hist)[tid] = reinterpret_cast<int4*>(hist)[tid + EV_THREADS] = make_int4(0, 0, 0, 0);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EV_PER; ++i) {
            if (EV_THREADS * i >= p.n) break;  // uniform
            count<4>(hist, digit(r[i], round), EV_THREADS * i + tid < p.n && with(r[i], last, round), lane);
        }
        __syncthreads();
        uint32_t bin;
        find(counted<4>(hist, EV_BINS - 1 - 2 * tid), counted<4>(hist, EV_BINS - 2 - 2 * tid), left, bin, waves, pick, tid, lane, wv);
        last |= bin << (round == 0 ? 21 : round == 1 ? 10 : 0);
    }
    int from[2], to[2];
    share(0, p.kept, wv, from[0], to[0]);
    share(p.kept, p.n, wv, from[1], to[1]);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        int above = 0, same = 0;
        for (int j0 = from[side]; j0 < to[side]; j0 += 64) {
            const bool in = j0 + lane < to[side];
            tally(in ? rank[j0 + lane] : 0u, in, last, above, same);
        }
        if (lane == 0) {
            counts[side][0][wv] = above;
            counts[side][1][wv] = same;
        }
    }
    __syncthreads();
    // ties ahead of the wave's stretches, holes (below) and movers (past) ahead: a lane a stretch
    int tie[2], at[2];
    {
        const int side = (lane / EV_WAVES) & 1, w = lane % EV_WAVES;
        int f, t;
        share(side ? p.kept : 0, side ? p.n : p.kept, w, f, t);
        const bool live = lane < 2 * EV_WAVES;
        const int same = live ? counts[side][1][w] : 0;
        const int ties = wave_running(same) - same;
        const int stay = live ? counts[side][0][w] + min(max(left - ties, 0), same) : 0;
        const int holes = live && !side ? t - f - stay : 0, movers = live && side ? stay : 0;
        const int hole_run = wave_running(holes) - holes, mover_run = wave_running(movers) - movers;
        tie[0] = __builtin_amdgcn_readlane(ties, wv);
        tie[1] = __builtin_amdgcn_readlane(ties, EV_WAVES + wv);
        at[0] = __builtin_amdgcn_readlane(hole_run, wv);
        at[1] = __builtin_amdgcn_readlane(mover_run, EV_WAVES + wv);
    }
    for (int j0 = from[1]; j0 < to[1]; j0 += 64) {
        const bool in = j0 + lane < to[1], s = stays(in ? rank[j0 + lane] : 0u, in, last, left, tie[1], lane);
        const unsigned long long all = __ballot(s);
        if (s) list[at[1] + lanes_before(all, lane)] = j0 + lane;
        at[1] += __popcll(all);
    }
    __syncthreads();
    for (int j0 = from[0]; j0 < to[0]; j0 += 64) {
        const int j = j0 + lane;
        const bool in = j < to[0], hole = !stays(in ? rank[j] : 0u, in, last, left, tie[0], lane) && in;
        const unsigned long long all = __ballot(hole);
        if (in) idx[j] = hole ? (int)list[at[0] + lanes_before(all, lane)] : j;
        at[0] += __popcll(all);
    }
}

// the four tallies of a wave's keys from slot f on; all of them lie on one side of `kept` but for one wave a head
__device__ __forceinline__ void tallies_of(const uint32_t (&r)[EV_PER], int f, const EvictArgs& p, uint32_t last, int lane, int (&c)[4]) {
    if (f < p.kept) {
#pragma unroll
        for (int i = 0; i < EV_PER; ++i) tally(r[i], f + 64 * i + lane < p.kept, last, c[0], c[1]);
    }
    if (f + 64 * EV_PER > p.kept) {
#pragma unroll
        for (int i = 0; i < EV_PER; ++i) tally(r[i], f + 64 * i + lane >= p.kept && f + 64 * i + lane < p.n, last, c[2], c[3]);
    }
}

// A longer head, a workgroup EV_KEYS of its keys; wave w takes 512 of them in a row. Rounds 0, 1 and 2: this round's histogram,
// and before it what the last one's says. Round 3: how many keys stay.
template <int ROUND>
__global__ void __launch_bounds__(EV_THREADS) evict_round_kernel(EvictArgs p) {
    extern __shared__ __align__(16) int hist[];  // [EV_BINS][EV_COPIES]
    __shared__ int waves[EV_WAVES], pick[2];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), block = blockIdx.x;
    const EvictWork w = work_of(p, blockIdx.y);
    const int j0 = block * EV_KEYS + wv * (EV_KEYS / EV_WAVES) + lane;
    uint32_t r[EV_PER];
#pragma unroll
    for (int i = 0; i < EV_PER; ++i) {
        const int j = j0 + 64 * i;
        if (ROUND == 0)
            r[i] = j < p.n ? rank_bits(p.mass[(size_t)blockIdx.y * p.ms + j], p.pos[(size_t)blockIdx.y * p.ps + j], p.sinks,
                                       p.recent_from)
                           : 0u;
        else
            r[i] = j < p.n ? w.rank[j] : 0u;
    }
    for (int i = tid; i < EV_COPIES * EV_BINS / 4; i += EV_THREADS) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
    uint32_t last = 0;
    if constexpr (ROUND > 0) {
        int left = ROUND == 1 ? p.kept : w.state[2 * (ROUND - 1) + 1];
        int h0 = 0, h1 = 0;
        if constexpr (ROUND == 1) {
#pragma unroll 16
            for (int b = 0; b < (int)gridDim.x; ++b) {
                const uint32_t two = w.first[(size_t)b * (EV_BINS / 2) + EV_BINS / 2 - 1 - tid];
                h0 += two >> 16;
                h1 += two & 0xFFFFu;
            }
        } else {
            const int* from = w.later + (ROUND - 2) * EV_BINS;
            h0 = from[EV_BINS - 1 - 2 * tid];
            h1 = from[EV_BINS - 2 - 2 * tid];
        }
        uint32_t bin;
        find(h0, h1, left, bin, waves, pick, tid, lane, wv);
        last = (ROUND == 1 ? 0u : (uint32_t)w.state[2 * (ROUND - 1)]) | bin << (ROUND == 1 ? 21 : ROUND == 2 ? 10 : 0);
        if (block == 0 && tid == 0) {
            w.state[2 * ROUND] = (int)last;
            w.state[2 * ROUND + 1] = left;
        }
    }
    if constexpr (ROUND < 3) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EV_PER; ++i) {
            const bool in = j0 + 64 * i < p.n;
            if (ROUND == 0 && in) w.rank[j0 + 64 * i] = r[i];
            count<EV_COPIES>(hist, digit(r[i], ROUND), in && with(r[i], last, ROUND), lane);
        }
        __syncthreads();
        if constexpr (ROUND == 0) {
            w.first[(size_t)block * (EV_BINS / 2) + tid] = (uint32_t)counted<EV_COPIES>(hist, 2 * tid) | (uint32_t)counted<EV_COPIES>(hist, 2 * tid + 1) << 16;
            if (block == 0)
                for (int i = tid; i < 2 * EV_BINS; i += EV_THREADS) w.later[i] = 0;
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int b = tid + EV_THREADS * i;
                const int n = counted<EV_COPIES>(hist, b);
                if (n != 0) atomicAdd(&w.later[(ROUND - 1) * EV_BINS + b], n);
            }
        }
    } else {
        int c[4] = {0, 0, 0, 0};
        tallies_of(r, j0 - lane, p, last, lane, c);
        if (lane < 4) hist[4 * wv + lane] = lane == 0 ? c[0] : lane == 1 ? c[1] : lane == 2 ? c[2] : c[3];
        __syncthreads();
        if (tid < 4) {
            int sum = 0;
            for (int i = 0; i < EV_WAVES; ++i) sum += hist[4 * i + tid];
            w.counts[4 * block + tid] = sum;
        }
    }
}

// The order: the kept keys past slot `kept` into the list, and for the slots below, idx: themselves, or -1 - i the i-th hole, which
// takes the list's i-th key (the move looks it up). Every wave adds up the counts of the workgroups ahead for itself.
__global__ void __launch_bounds__(EV_THREADS) evict_order_kernel(EvictArgs p) {
    __shared__ int tallies[4][EV_WAVES];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block = blockIdx.x, blocks = gridDim.x;
    const EvictWork w = work_of(p, blockIdx.y);
    const int j0 = block * EV_KEYS + wv * (EV_KEYS / EV_WAVES) + lane;
    uint32_t r[EV_PER];
#pragma unroll
    for (int i = 0; i < EV_PER; ++i) r[i] = j0 + 64 * i < p.n ? w.rank[j0 + 64 * i] : 0u;
    const uint32_t last = (uint32_t)w.state[6];
    const int left = w.state[7];
    int c[4] = {0, 0, 0, 0};
    tallies_of(r, j0 - lane, p, last, lane, c);
    if (lane < 4) tallies[lane][wv] = lane == 0 ? c[0] : lane == 1 ? c[1] : lane == 2 ? c[2] : c[3];
    // all ties below `kept` come before those past it
    int low = 0;
    for (int b = lane; b < blocks; b += 64) low += w.counts[4 * b + 1];
    int tie[2] = {0, __builtin_amdgcn_readlane(wave_running(low), 63)}, at[2] = {0, 0};  // ties, then holes and movers, ahead
    // moves the four on by stretches, a lane each - `n` keys below `kept`, what `v` says of them and of those past it -, up to `upto`
    auto advance = [&](int4 v, int n, int upto) {
        const int run[2] = {wave_running(v.y), wave_running(v.w)};
        const int t[2] = {tie[0] + run[0] - v.y, tie[1] + run[1] - v.w};
        const int holes = n - v.x - min(max(left - t[0], 0), v.y), movers = v.z + min(max(left - t[1], 0), v.w);
        const int ran[2] = {wave_running(holes), wave_running(movers)};
        if (upto == 0) return;
        tie[0] += __builtin_amdgcn_readlane(run[0], upto - 1);
        tie[1] += __builtin_amdgcn_readlane(run[1], upto - 1);
        at[0] += __builtin_amdgcn_readlane(ran[0], upto - 1);
        at[1] += __builtin_amdgcn_readlane(ran[1], upto - 1);
    };
    auto below = [&](int from, int keys) { return max(min(from + keys, p.kept) - from, 0); };
    for (int b = 0; b < block; b += 64) {
        const bool live = b + lane < blocks;
        const int4 v = live ? *reinterpret_cast<const int4*>(w.counts + 4 * (b + lane)) : make_int4(0, 0, 0, 0);
        advance(v, live ? below((b + lane) * EV_KEYS, EV_KEYS) : 0, min(block - b, 64));
    }
    __syncthreads();
    {
        const bool live = lane < EV_WAVES;
        const int4 v = live ? make_int4(tallies[0][lane], tallies[1][lane], tallies[2][lane], tallies[3][lane]) : make_int4(0, 0, 0, 0);
        advance(v, live ? below(block * EV_KEYS + lane * (EV_KEYS / EV_WAVES), EV_KEYS / EV_WAVES) : 0, wv);
    }
    if (j0 - lane < p.kept) {  // uniform
#pragma unroll
        for (int i = 0; i < EV_PER; ++i) {
            const int j = j0 + 64 * i;
            const bool in = j < p.kept, s = stays(r[i], in, last, left, tie[0], lane);
            const unsigned long long holes = __ballot(in && !s);
            if (in) p.idx[(size_t)blockIdx.y * p.kept + j] = s ? j : -1 - (at[0] + lanes_before(holes, lane));
            at[0] += __popcll(holes);
        }
    }
    if (j0 - lane + 64 * EV_PER > p.kept) {
#pragma unroll
        for (int i = 0; i < EV_PER; ++i) {
            const int j = j0 + 64 * i;
            const bool s = stays(r[i], j >= p.kept && j < p.n, last, left, tie[1], lane);
            const unsigned long long movers = __ballot(s);
            if (s) w.list[at[1] + lanes_before(movers, lane)] = j;
            at[1] += __popcll(movers);
        }
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
    int32_t* idx;
    const int* list;  // of head 0, `per` words a head: what idx's negative numbers name
    long long per;
    long long ls, hs, rs, lo, ho, ro;  // strides of the layers, heads and rows, in and out
    long long ms, ps, mo, po;
    int Hk, kept, in_place;
};

// a workgroup takes EV_MOVE rows, a thread 16 bytes of some of them: all of its loads before its first store
constexpr int EV_MOVE = 64;

template <int CHUNKS>
__global__ void __launch_bounds__(256) evict_move_kernel(MoveArgs p) {
    constexpr int STEP = 256 / CHUNKS, ROWS = EV_MOVE / STEP;  // rows at a time, and a thread's
    const int head = blockIdx.y, layer = head / p.Hk, g = head % p.Hk, c = threadIdx.x % CHUNKS;
    const int j0 = blockIdx.x * EV_MOVE + threadIdx.x / CHUNKS;
    const size_t src = (size_t)layer * p.ls + (size_t)g * p.hs + 8 * c, dst = (size_t)layer * p.lo + (size_t)g * p.ho + 8 * c;
    int32_t* idx = p.idx + (size_t)head * p.kept;
    int from[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) from[i] = j0 + STEP * i < p.kept ? idx[j0 + STEP * i] : 0;
    if (p.list != nullptr) {  // uniform
        int named[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) named[i] = from[i] < 0 ? p.list[(size_t)head * p.per - 1 - from[i]] : from[i];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            if (from[i] < 0 && c == 0) idx[j0 + STEP * i] = named[i];  // (this row's lanes, all of this wave, have read it)
            from[i] = named[i];
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        if (j0 + STEP * i >= p.kept || (p.in_place && from[i] == j0 + STEP * i)) from[i] = -1;
    uint4 k[ROWS], v[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        if (from[i] >= 0) {
            k[i] = load_stream16(reinterpret_cast<const uint4*>(p.K + src + (size_t)from[i] * p.rs));
            v[i] = load_stream16(reinterpret_cast<const uint4*>(p.V + src + (size_t)from[i] * p.rs));
        }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        if (from[i] >= 0) {
            const int j = j0 + STEP * i;
            *reinterpret_cast<uint4*>(p.K_out + dst + (size_t)j * p.ro) = k[i];
            *reinterpret_cast<uint4*>(p.V_out + dst + (size_t)j * p.ro) = v[i];
            if (c == 0) {
                p.mass_out[(size_t)head * p.mo + j] = p.mass[(size_t)head * p.ms + from[i]];
                p.pos_out[(size_t)head * p.po + j] = p.pos[(size_t)head * p.ps + from[i]];
            }
        }
}

template <int ROUND>
static int32_t launch_round(const dim3& grid, const EvictArgs& e, hipStream_t st) {
    constexpr int lds = 4 * EV_COPIES * EV_BINS;
    const hipError_t rc = hipFuncSetAttribute(reinterpret_cast<const void*>(evict_round_kernel<ROUND>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (rc != hipSuccess) return hip_status(rc, "hipFuncSetAttribute");
    hipLaunchKernelGGL(evict_round_kernel<ROUND>, grid, dim3(EV_THREADS), lds, st, e);
    return hip_status(hipGetLastError(), "kv_evict launch");
}

}  // namespace btb

using namespace btb;

extern "C" size_t btb_hip_kv_evict_words(size_t L, size_t Hk, size_t n) {
    return n <= (size_t)EV_KEYS ? 0 : L * Hk * evict_words(n);
}

extern "C" int32_t btb_hip_kv_evict(const float* mass, int64_t ms, const int32_t* pos, int64_t ps, const void* K, const void* V,
                                    int64_t ls, int64_t hs, int64_t rs, size_t L, size_t Hk, size_t D, size_t n, size_t budget,
                                    int32_t sinks, int32_t recent_from, void* K_out, void* V_out, int64_t lo, int64_t ho,
                                    int64_t ro, float* mass_out, int64_t mo, int32_t* pos_out, int64_t po, int32_t* idx,
                                    uint32_t* workspace, void* stream) {
    if (!mass || !pos || !K || !V || !K_out || !V_out || !mass_out || !pos_out || !idx) return ERR_NULL;
    if (workspace == nullptr && btb_hip_kv_evict_words(1, 1, n) != 0) return ERR_NULL;
    auto loose = [](const void* a) { return ((uintptr_t)a & 15u) != 0; };
    auto odd = [](int64_t s) { return s < 0 || s % 8 != 0; };
    const bool in_place = K == K_out;
    const size_t kept = budget < n ? budget : n;
    // rows, or a head's numbers, that several workgroups would write
    const bool shared = (lo == 0 && L > 1) || (ho == 0 && Hk > 1) || (ro == 0 && kept > 1) ||
                        (L * Hk > 1 && ((size_t)mo < kept || (size_t)po < kept));
    if (L == 0 || Hk == 0 || L > 65535 || Hk > 65535 || L * Hk > 65535 || (D != 64 && D != 128 && D != 256) || n == 0 ||
        n > (size_t)EV_KEYS * EV_BLOCKS || budget == 0 || shared || ms < 0 || ps < 0 || mo < 0 || po < 0 || odd(ls) || odd(hs) || odd(rs) || odd(lo) ||
        odd(ho) || odd(ro) || loose(K) || loose(V) || loose(K_out) || loose(V_out) || loose(workspace) || in_place != (V == V_out) ||
        in_place != (mass == mass_out) || in_place != (pos == pos_out) ||
        (in_place && (ls != lo || hs != ho || rs != ro || ms != mo || ps != po))) {
        set_error("kv_evict: at most 65535 heads in all of at most 2^23 keys, head_dim 64, 128 or 256, K and V 16-byte aligned with strides in "
                  "multiples of 8, no two outputs in one place; in place: all four outputs the inputs with their strides, or none");
        return ERR_DOMAIN;
    }
    EvictArgs e;
    e.mass = mass;
    e.pos = pos;
    e.idx = idx;
    e.ms = ms;
    e.ps = ps;
    e.n = (int)n;
    e.kept = (int)kept;
    e.sinks = sinks;
    e.recent_from = recent_from;
    hipStream_t st = static_cast<hipStream_t>(stream);
    e.work = workspace;
    const unsigned heads = (unsigned)(L * Hk);
    int32_t rc = OK;
    if (n <= (size_t)EV_KEYS) {
        const size_t lds = 4 * (n + n / 2);
        if (lds > 28 * 1024) {
            const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(evict_choose_kernel),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (set != hipSuccess) return hip_status(set, "hipFuncSetAttribute");
        }
        hipLaunchKernelGGL(evict_choose_kernel, dim3(heads), dim3(EV_THREADS), lds, st, e);
        rc = hip_status(hipGetLastError(), "kv_evict launch");
    } else {
        const int blocks = (int)((n + EV_KEYS - 1) / EV_KEYS);
        const dim3 grid((unsigned)blocks, heads), threads(EV_THREADS);
        // one statement each: a round reads what the one before it left
        rc = launch_round<0>(grid, e, st);
        if (rc == OK) rc = launch_round<1>(grid, e, st);
        if (rc == OK) rc = launch_round<2>(grid, e, st);
        if (rc == OK) rc = launch_round<3>(grid, e, st);
        if (rc == OK) {
            hipLaunchKernelGGL(evict_order_kernel, grid, threads, 0, st, e);
            rc = hip_status(hipGetLastError(), "kv_evict launch");
        }
    }
    if (rc != OK) return rc;  // (the move goes by what the choice wrote)
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
    m.list = nullptr;
    if (n > (size_t)EV_KEYS)
        m.list = reinterpret_cast<const int*>(workspace) + (n + 3) / 4 * 4 + (n + EV_KEYS - 1) / EV_KEYS * (EV_BINS / 2 + 4) + 2 * EV_BINS + 8;
    m.per = (long long)evict_words(n);
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
    m.in_place = in_place ? 1 : 0;
    const dim3 grid((unsigned)((e.kept + EV_MOVE - 1) / EV_MOVE), (unsigned)(L * Hk));
    if (D == 64)
        hipLaunchKernelGGL(evict_move_kernel<8>, grid, dim3(256), 0, st, m);
    else if (D == 128)
        hipLaunchKernelGGL(evict_move_kernel<16>, grid, dim3(256), 0, st, m);
    else
        hipLaunchKernelGGL(evict_move_kernel<32>, grid, dim3(256), 0, st, m);
    return hip_status(hipGetLastError(), "kv_evict launch");
}
