// Pages of a cache as whole pieces of memory, whatever they hold: sequences that go on from another's, and a pool closed up.
//
//   fork     the new sequence names the old one's whole pages; its last page, where it is not whole, is a copy, as both will write to it
//   compact  the pages that some sequence names, n of them, end up as pages 0 .. n - 1: those below n stay, the others go, in ascending
//            order, to the pages below n that nobody names, in ascending order
//
// Bound: memory, a page read and written once, past the caches both ways: 237 MB of pages copied by 48 forks in 46 us (5.1 TB/s; 50 with stores
// through the caches), 948 MB by a compaction in 196 (209). A page is copied by workgroups of COPY bytes, every layer's in the same launch.

#include "btb_common.hpp"
#include "btb_tuning.hpp"

#include "../../include/btb_hip.h"

namespace btb {

constexpr int COPY_AT_ONCE = 4;                    // 16-byte pieces a thread has on their way
constexpr int COPY = 256 * 16 * COPY_AT_ONCE;      // bytes a workgroup copies at a time
constexpr size_t COMPACT_PAGES = (size_t)1 << 19;  // pages whose bits, and their counts, fit a workgroup's LDS
constexpr int COMPACT_THREADS = 1024;

struct Pages {
    uint8_t* pool;
    long long layer, stride;  // bytes from a layer, and from a page, to the next
    int L, pages, pieces;     // 16-byte pieces a page
    int chunks;               // workgroups a page
    int32_t* tables;          // [B, W]
    int32_t* lens;
    int B, W, page;
    // fork
    const int32_t* src;
    const int32_t* dst;
    const int32_t* fresh;
    int F;
    // compact
    int32_t* out;             // the tables as they are then
    int32_t* used;
    int32_t* work;            // the number of moves; where each page goes [pages]; from and to, a move each [pages / 2]
};

__device__ __forceinline__ int length(const Pages& p, int b) {
    return (int)min((long long)max(p.lens[b], 0), (long long)p.W * p.page);
}
__device__ __forceinline__ bool inside(int x, int n) { return x >= 0 && x < n; }

// one chunk of a page of one layer
__device__ __forceinline__ void copy_chunk(const Pages& p, int layer, int from, int to, int chunk) {
    const u32x4* a = reinterpret_cast<const u32x4*>(p.pool + layer * p.layer + from * p.stride);
    u32x4* b = reinterpret_cast<u32x4*>(p.pool + layer * p.layer + to * p.stride);
    const int first = chunk * (COPY / 16) + threadIdx.x;
    u32x4 x[COPY_AT_ONCE];
#pragma unroll
    for (int i = 0; i < COPY_AT_ONCE; ++i)
        if (first + 256 * i < p.pieces) x[i] = __builtin_nontemporal_load(a + first + 256 * i);
#pragma unroll
    for (int i = 0; i < COPY_AT_ONCE; ++i)
        if (first + 256 * i < p.pieces) __builtin_nontemporal_store(x[i], b + first + 256 * i);
}

__global__ void __launch_bounds__(256) pages_fork_kernel(Pages p) {
    const int chunk = blockIdx.x % p.chunks, layer = blockIdx.x / p.chunks % p.L, f = blockIdx.x / p.chunks / p.L;
    const int src = p.src[f], dst = p.dst[f], fresh = p.fresh[f];
    if (!inside(src, p.B) || !inside(dst, p.B) || src == dst) return;
    const int n = length(p, src), whole = n / p.page;
    const bool part = n % p.page != 0;
    if (part && !inside(fresh, p.pages)) return;
    const int32_t* of = p.tables + (size_t)src * p.W;
    const int last = part ? of[whole] : -1;
    if (layer == 0 && chunk == 0) {
        int32_t* to = p.tables + (size_t)dst * p.W;
        for (int j = threadIdx.x; j < p.W; j += 256) to[j] = j < whole ? of[j] : (j == whole && inside(last, p.pages) ? fresh : -1);
        if (threadIdx.x == 0) p.lens[dst] = n;
    }
    if (inside(last, p.pages) && last != fresh) copy_chunk(p, layer, last, fresh, chunk);
}

// which pages are named, how many, and where each goes: one workgroup
__global__ void __launch_bounds__(COMPACT_THREADS) pages_choose_kernel(Pages p) {
    extern __shared__ uint32_t lds[];
    const int words = (p.pages + 31) / 32, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    constexpr int WAVES = COMPACT_THREADS / 64;
    uint32_t* bits = lds;
    int* before = reinterpret_cast<int*>(lds + words);  // named pages before each word's
    __shared__ int sums[WAVES];
    for (int i = tid; i < words; i += COMPACT_THREADS) bits[i] = 0;
    __syncthreads();
    for (int b = wave; b < p.B; b += WAVES) {
        const int count = (length(p, b) + p.page - 1) / p.page;
        for (int j = lane; j < count; j += 64) {
            const int page = p.tables[(size_t)b * p.W + j];
            if (inside(page, p.pages)) atomicOr(&bits[page >> 5], 1u << (page & 31));
        }
    }
    __syncthreads();
    // a thread a run of words, the runs' sums one after another
    const int run = (words + COMPACT_THREADS - 1) / COMPACT_THREADS, first = min(tid * run, words), end = min(first + run, words);
    int mine = 0;
    for (int i = first; i < end; ++i) mine += __popc(bits[i]);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int below = __shfl_up(upto, d, WAVE);
        if (lane >= d) upto += below;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int used = 0, at = upto - mine;
    for (int i = 0; i < WAVES; ++i) {
        if (i < wave) at += sums[i];
        used += sums[i];
    }
    for (int i = first; i < end; ++i) {
        before[i] = at;
        at += __popc(bits[i]);
    }
    __syncthreads();
    auto named_before = [&](int page) {
        return page >= p.pages ? used : before[page >> 5] + __popc(bits[page >> 5] & ((1u << (page & 31)) - 1u));
    };
    const int stay = named_before(used), moves = used - stay;
    int32_t* goes = p.work + 4;
    int32_t* from = goes + p.pages;
    int32_t* to = from + p.pages / 2;
    for (int page = tid; page < p.pages; page += COMPACT_THREADS) {
        const bool named = bits[page >> 5] >> (page & 31) & 1u;
        const int rank = named_before(page);
        if (page < used && !named) to[page - rank] = page;
        if (page >= used && named) from[rank - stay] = page;
        if (page < used && named) goes[page] = page;
    }
    __syncthreads();  // (also for what was written to memory: one workgroup reads it)
    for (int i = tid; i < moves; i += COMPACT_THREADS) goes[from[i]] = to[i];
    if (tid == 0) {
        p.work[0] = moves;
        *p.used = used;
    }
}

__global__ void __launch_bounds__(256) pages_move_kernel(Pages p) {
    const int32_t* goes = p.work + 4;
    const int32_t* from = goes + p.pages;
    const int32_t* to = from + p.pages / 2;
    const long long entries = (long long)p.B * p.W;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < entries; e += (long long)gridDim.x * 256) {
        const int b = (int)(e / p.W), j = (int)(e % p.W), page = p.tables[e];
        const bool named = j < (length(p, b) + p.page - 1) / p.page && inside(page, p.pages);
        p.out[e] = named ? goes[page] : -1;
    }
    const int each = p.L * p.chunks;
    const long long items = (long long)p.work[0] * each;
    for (long long i = blockIdx.x; i < items; i += gridDim.x) {
        const int move = (int)(i / each), rest = (int)(i % each);
        copy_chunk(p, rest / p.chunks, from[move], to[move], rest % p.chunks);
    }
}

static bool pages_of(Pages& p, void* pool, size_t L, size_t pages, size_t bytes, int64_t layer, int64_t stride, size_t B, size_t W,
                     size_t page) {
    if (L == 0 || L > 65535 || pages == 0 || pages > 0x7FFFFFFFu || bytes == 0 || bytes % 16 != 0 || bytes > ((size_t)1 << 30) ||
        stride < (int64_t)bytes || stride % 16 != 0 || stride > ((int64_t)1 << 46) / (int64_t)pages || layer < 0 || layer % 16 != 0 ||
        (L > 1 && layer < (int64_t)bytes) || layer > ((int64_t)1 << 46) / (int64_t)L || ((uintptr_t)pool & 15u) != 0 || B == 0 || B > 65536 || W == 0 || W > (1u << 30) || page == 0 || page > (1u << 30) ||
        W * page > (1u << 30))
        return false;
    // layers one after another, or pages one after another with all their layers
    if (L > 1 && layer < (int64_t)pages * stride && stride < (int64_t)L * layer) return false;
    p.pool = static_cast<uint8_t*>(pool);
    p.layer = layer, p.stride = stride;
    p.L = (int)L, p.pages = (int)pages, p.pieces = (int)(bytes / 16), p.chunks = (int)((bytes + COPY - 1) / COPY);
    p.B = (int)B, p.W = (int)W, p.page = (int)page;
    return true;
}

#define PAGES_DOMAIN "pages of a multiple of 16 bytes, the pool 16-byte aligned, its pages and layers in places of their own, " \
                     "1 .. 65536 sequences of up to 2^30 tokens"

}  // namespace btb

using namespace btb;

extern "C" int32_t btb_hip_pages_fork(void* pool, size_t L, size_t pages, size_t bytes, int64_t layer, int64_t stride, int32_t* tables,
                                      int32_t* lens, size_t B, size_t W, size_t page, const int32_t* src, const int32_t* dst,
                                      const int32_t* fresh, size_t F, void* stream) {
    if (!pool || !tables || !lens || !src || !dst || !fresh) return ERR_NULL;
    Pages p{};
    if (!pages_of(p, pool, L, pages, bytes, layer, stride, B, W, page) || F == 0 || F > 65536 ||
        F * L * p.chunks > ((size_t)1 << 24) - 1) {  // (a launch's threads are counted in 32 bits)
        set_error("pages_fork: " PAGES_DOMAIN ", 1 .. 65536 forks, below 2^24 of 16 KB in all layers");
        return ERR_DOMAIN;
    }
    p.tables = tables, p.lens = lens;
    p.src = src, p.dst = dst, p.fresh = fresh, p.F = (int)F;
    hipLaunchKernelGGL(pages_fork_kernel, dim3((unsigned)(F * L * p.chunks)), dim3(256), 0, static_cast<hipStream_t>(stream), p);
    return hip_status(hipGetLastError(), "pages_fork launch");
}

extern "C" size_t btb_hip_pages_compact_words(size_t pages) {
    return pages == 0 || pages > COMPACT_PAGES ? 0 : 4 + pages + 2 * (pages / 2);
}

extern "C" int32_t btb_hip_pages_compact(void* pool, size_t L, size_t pages, size_t bytes, int64_t layer, int64_t stride,
                                         const int32_t* tables, const int32_t* lens, size_t B, size_t W, size_t page,
                                         int32_t* tables_out, int32_t* used, int32_t* workspace, void* stream) {
    if (!pool || !tables || !lens || !tables_out || !used || !workspace) return ERR_NULL;
    Pages p{};
    const bool crossed = tables_out != tables && tables_out < tables + B * W && tables < tables_out + B * W;
    if (!pages_of(p, pool, L, pages, bytes, layer, stride, B, W, page) || pages > COMPACT_PAGES || crossed) {
        set_error("pages_compact: " PAGES_DOMAIN ", up to 2^19 pages, tables_out the tables or apart from them");
        return ERR_DOMAIN;
    }
    p.tables = const_cast<int32_t*>(tables), p.lens = const_cast<int32_t*>(lens);
    p.out = tables_out, p.used = used, p.work = workspace;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int lds = (int)((pages + 31) / 32 * 8);
    if (lds > 32 * 1024) {
        const hipError_t set =
            hipFuncSetAttribute(reinterpret_cast<const void*>(pages_choose_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (set != hipSuccess) return hip_status(set, "hipFuncSetAttribute");
    }
    hipLaunchKernelGGL(pages_choose_kernel, dim3(1), dim3(COMPACT_THREADS), lds, st, p);
    const int32_t rc = hip_status(hipGetLastError(), "pages_compact launch");
    if (rc != OK) return rc;  // (the move goes by what the choice wrote)
    // as many workgroups as half of the pages could need, up to eight a CU, which go on from chunk to chunk
    const size_t most = pages / 2 * L * p.chunks, fit = (size_t)8 * device_info().cus;
    hipLaunchKernelGGL(pages_move_kernel, dim3((unsigned)(most < 1 ? 1 : most < fit ? most : fit)), dim3(256), 0, st, p);
    return hip_status(hipGetLastError(), "pages_compact move launch");
}
