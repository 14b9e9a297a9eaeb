// kv_pages.cu -- fork, free, extend and compact KV cache pages
// (include/kv_cache.h).
//
// Which pages are in use follows from the tables of each call alone: a mark
// pass writes one key per owned page, a plan pass ranks what has to be
// allocated or moved and the free pages with prefix sums (ids in order, so
// equal inputs give equal tables), an apply pass writes the tables and copies
// the pages of all caches.  A page that is written is one that no row of the
// result owned before the call, so no copy reads what another writes.
//
// Bound: the copied pages' bytes, twice, and the latency of mark and plan under
// one block.  Measured (B200, device time): 24 rows of up to 1000 tokens compacted
// over 92 caches of 9216-byte pages, 144 MB moved, 31 us -- 5.8 TB/s once the plan is
// there; 32 rows forked into 64 over 184 caches of 4 KB pages, 26 MB, 13 us; small
// pools 5 to 7 us.
#include <cuda_runtime.h>

#include <cstdint>

#include "attn_common.cuh"
#include "kv_cache.h"
#include "sm100.cuh"

namespace {

using namespace tb;

// Key of an owned page: the tokens its row has in it, whether that row will
// append to it, and the row, lowest first; the largest key keeps the page.
constexpr int kRowBits = 26;
__device__ __forceinline__ uint32_t page_key(int fill, bool writer, int row) {
    return (static_cast<uint32_t>(fill) << (kRowBits + 1)) | (static_cast<uint32_t>(writer) << kRowBits) |
           ((1u << kRowBits) - 1u - static_cast<uint32_t>(row));
}

struct PageParams {
    uint8_t* caches;
    size_t cache_stride, page_bytes;
    int num_caches, num_pages, max_pages, num_seqs, num_rows;   // num_rows: rows of the result
    const int32_t* table_in;
    const int32_t* lens;
    const int32_t* parents;        // null: row i of table_in (compact)
    const int32_t* reserve;
    int32_t* table_out;
    int32_t* lens_out;
    int32_t* num_used;             // compact
    int* error_word;
    uint32_t* keys;                // [num_pages]
    int32_t* free_list;            // [num_pages] free pages in order
    int32_t* move_src;             // fork: [num_rows] page copied for row i's copy k; compact: [num_pages]
    int32_t* move_dst;
    int32_t* first_req;            // fork: [num_rows] index of the row's first fresh page
    int32_t* counts;               // [0] page copies, [1] fresh pages that exist
};

struct Row {
    int parent, len, have, need;   // have: pages owned, need: with the reservation
    bool writes;                   // appends into a page in part filled
};

// Row i of the result; errors are recorded by the caller that passes `report`.
__device__ __forceinline__ Row row_of(const PageParams& p, int i, bool report) {
    Row r;
    r.parent = p.parents ? p.parents[i] : i;
    int err = 0;
    if (r.parent < -1 || r.parent >= p.num_seqs) {
        err = 7;
        r.parent = -1;
    }
    r.len = r.parent >= 0 ? max(p.lens[r.parent], 0) : 0;
    const long long cap = static_cast<long long>(p.max_pages) * kPage;
    if (r.len > cap) {
        err = 5;
        r.len = static_cast<int>(cap);
    }
    const int reserve = p.reserve ? max(p.reserve[i], 0) : 0;
    long long total = static_cast<long long>(r.len) + reserve;
    if (total > cap) {
        err = 4;
        total = cap;
    }
    r.have = (r.len + kPage - 1) / kPage;
    r.need = static_cast<int>((total + kPage - 1) / kPage);
    r.writes = total > r.len && r.len % kPage != 0;
    if (err && report && p.error_word) atomicExch(p.error_word, err);
    return r;
}

__device__ __forceinline__ int owned_page(const PageParams& p, const Row& r, int j) {
    const int id = p.table_in[static_cast<size_t>(r.parent) * p.max_pages + j];
    return id >= 0 && id < p.num_pages ? id : -1;
}

// ---------------------------------------------------------------- mark

constexpr int kMarkWarps = 8;

// Marks the pages of rows first, first + step, ...: one warp a row.
__device__ __forceinline__ void mark_rows(const PageParams& p, int first, int step) {
    const int lane = threadIdx.x & 31;
    for (int i = first; i < p.num_rows; i += step) {
        const Row r = row_of(p, i, lane == 0);
        for (int j = lane; j < r.have; j += 32) {
            const int id = owned_page(p, r, j);
            if (id < 0) {
                if (p.error_word) atomicExch(p.error_word, 6);
                continue;
            }
            const int fill = min(r.len - j * kPage, kPage);
            atomicMax(&p.keys[id], page_key(fill, r.writes && j == r.have - 1, i));
        }
    }
}

__global__ void __launch_bounds__(kMarkWarps * 32)
pages_mark_kernel(const PageParams p) {
    mark_rows(p, blockIdx.x * kMarkWarps + (threadIdx.x >> 5), gridDim.x * kMarkWarps);
}

// ---------------------------------------------------------------- plan

constexpr int kPlanThreads = 1024;

// Exclusive prefix sum of v over the block; *total receives the sum.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* total,
                                                         unsigned long long* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                   // sh is free
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    if (warp == 0) {
        unsigned long long w = sh[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        sh[lane] = w;
    }
    __syncthreads();
    *total = sh[kPlanThreads / 32 - 1];
    return x - v + (warp ? sh[warp - 1] : 0ull);
}

// By one block of kPlanThreads.
__device__ __forceinline__ void fork_plan(const PageParams& p, unsigned long long* sh) {
    unsigned long long base = 0;       // fresh pages wanted | page copies << 32
    for (int i0 = 0; i0 < p.num_rows; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        unsigned long long v = 0;
        int src = -1;
        if (i < p.num_rows) {
            const Row r = row_of(p, i, false);
            if (r.writes) {
                src = owned_page(p, r, r.have - 1);
                if (src >= 0 && p.keys[src] == page_key(r.len - (r.have - 1) * kPage, true, i)) src = -1;
            }
            v = static_cast<unsigned long long>(r.need - r.have + (src >= 0)) | (static_cast<unsigned long long>(src >= 0) << 32);
            p.lens_out[i] = r.len;
        }
        unsigned long long total;
        const unsigned long long at = base + block_scan(v, &total, sh);
        if (i < p.num_rows) p.first_req[i] = static_cast<int32_t>(at & 0xFFFFFFFFull);
        if (src >= 0) {
            p.move_src[at >> 32] = src;
            p.move_dst[at >> 32] = static_cast<int32_t>(at & 0xFFFFFFFFull);   // index into free_list
        }
        base += total;
    }
    const unsigned int wanted = static_cast<unsigned int>(base & 0xFFFFFFFFull);
    unsigned int found = 0;
    for (int q0 = 0; q0 < p.num_pages && found < wanted; q0 += kPlanThreads) {
        const int q = q0 + threadIdx.x;
        const bool is_free = q < p.num_pages && p.keys[q] == 0;
        unsigned long long total;
        const unsigned long long at = found + block_scan(is_free, &total, sh);
        if (is_free && at < wanted) p.free_list[at] = q;
        found += static_cast<unsigned int>(total);
    }
    if (threadIdx.x == 0) {
        p.counts[0] = static_cast<int32_t>(base >> 32);
        p.counts[1] = static_cast<int32_t>(min(found, wanted));
        if (found < wanted && p.error_word) atomicExch(p.error_word, 8);
    }
}

__device__ __forceinline__ void compact_plan(const PageParams& p, unsigned long long* sh) {
    int used = 0;
    for (int q = threadIdx.x; q < p.num_pages; q += kPlanThreads) used += p.keys[q] != 0;
    unsigned long long total;
    block_scan(used, &total, sh);
    const int U = static_cast<int>(total);
    unsigned long long base = 0;       // free pages below U | used pages from U on << 32
    for (int q0 = 0; q0 < p.num_pages; q0 += kPlanThreads) {
        const int q = q0 + threadIdx.x;
        const bool is_used = q < p.num_pages && p.keys[q] != 0;
        const bool hole = q < U && !is_used, high = q >= U && is_used;
        const unsigned long long at =
            base + block_scan(static_cast<unsigned long long>(hole) | (static_cast<unsigned long long>(high) << 32), &total, sh);
        if (hole) p.move_dst[at & 0xFFFFFFFFull] = q;
        if (high) p.move_src[at >> 32] = q;
        base += total;
    }
    __syncthreads();
    const int moves = static_cast<int>(base >> 32);
    for (int k = threadIdx.x; k < moves; k += kPlanThreads) p.keys[p.move_src[k]] = static_cast<uint32_t>(p.move_dst[k]);
    if (threadIdx.x == 0) {
        p.counts[0] = moves;
        p.counts[1] = U;
        p.num_used[0] = U;
    }
}

// ---------------------------------------------------------------- apply

// Entries tid, tid + threads, ... of the result's table.
__device__ __forceinline__ void write_table(const PageParams& p, bool fork, long long tid, long long threads) {
    const int fresh = p.counts[1];
    for (long long e = tid; e < static_cast<long long>(p.num_rows) * p.max_pages; e += threads) {
        const int i = static_cast<int>(e / p.max_pages), j = static_cast<int>(e % p.max_pages);
        const Row r = row_of(p, i, false);
        int id = -1;
        if (j < r.have) id = owned_page(p, r, j);
        if (!fork) {
            if (id >= fresh) id = static_cast<int>(p.keys[id]);   // counts[1] is U
        } else {
            int req = -1;
            const bool copies = r.writes && j >= r.have - 1 && [&] {
                const int last = owned_page(p, r, r.have - 1);
                return last >= 0 && p.keys[last] != page_key(r.len - (r.have - 1) * kPage, true, i);
            }();
            if (j == r.have - 1 && copies) req = p.first_req[i];
            else if (j >= r.have && j < r.need) req = p.first_req[i] + (j - r.have) + copies;
            if (req >= 0) id = req < fresh ? p.free_list[req] : -1;
        }
        p.table_out[e] = id;
    }
}

constexpr int kApplyThreads = 256;
constexpr int kChunkVecs = 256;        // 16-byte pieces one warp copies at a time (4 KB, 8 in flight a lane)

// The copies: one warp per 4 KB piece of a page of one cache.
__device__ __forceinline__ void copy_pages(const PageParams& p, bool fork, long long warp, long long warps) {
    const int fresh = p.counts[1], lane = threadIdx.x & 31;
    const int vecs = static_cast<int>(p.page_bytes / 16);
    const int chunks = (vecs + kChunkVecs - 1) / kChunkVecs;
    const long long units = static_cast<long long>(p.counts[0]) * p.num_caches * chunks;
    for (long long u = warp; u < units; u += warps) {
        const int chunk = static_cast<int>(u % chunks);
        const int cache = static_cast<int>(u / chunks % p.num_caches);
        const int k = static_cast<int>(u / chunks / p.num_caches);
        int dst = p.move_dst[k];
        if (fork) {
            if (dst >= fresh) continue;
            dst = p.free_list[dst];
        }
        uint8_t* base = p.caches + static_cast<size_t>(cache) * p.cache_stride;
        const uint4* s = reinterpret_cast<const uint4*>(base + static_cast<size_t>(p.move_src[k]) * p.page_bytes);
        uint4* d = reinterpret_cast<uint4*>(base + static_cast<size_t>(dst) * p.page_bytes);
        const int v0 = chunk * kChunkVecs + lane;
        uint4 x[kChunkVecs / 32];
#pragma unroll
        for (int c = 0; c < kChunkVecs / 32; ++c)
            if (v0 + 32 * c < vecs) x[c] = s[v0 + 32 * c];
#pragma unroll
        for (int c = 0; c < kChunkVecs / 32; ++c)
            if (v0 + 32 * c < vecs) d[v0 + 32 * c] = x[c];
    }
}

template <bool kFork>
__global__ void __launch_bounds__(kPlanThreads)
pages_plan_kernel(const PageParams p) {
    __shared__ unsigned long long sh[32];
    if constexpr (kFork) fork_plan(p, sh);
    else compact_plan(p, sh);
}

template <bool kFork>
__global__ void __launch_bounds__(kApplyThreads)
pages_apply_kernel(const PageParams p) {
    const long long threads = static_cast<long long>(gridDim.x) * kApplyThreads;
    const long long tid = static_cast<long long>(blockIdx.x) * kApplyThreads + threadIdx.x;
    write_table(p, kFork, tid, threads);
    copy_pages(p, kFork, tid / 32, threads / 32);
}

// Small tables and pools: keys in shared memory, everything but the copies by
// one block, the copies' launch under it.  The limits are 128 KB of keys and 32 entries a thread.
constexpr int kSmallPages = 32768, kSmallEntries = 32768;

template <bool kFork>
__global__ void __launch_bounds__(kPlanThreads)
pages_small_kernel(PageParams p) {
    extern __shared__ __align__(16) uint32_t keys_s[];
    __shared__ unsigned long long sh[32];
    grid_dependents_launch();
    p.keys = keys_s;
    for (int q = threadIdx.x; q < p.num_pages; q += kPlanThreads) keys_s[q] = 0;
    __syncthreads();
    mark_rows(p, threadIdx.x >> 5, kPlanThreads / 32);
    __syncthreads();
    if constexpr (kFork) fork_plan(p, sh);
    else compact_plan(p, sh);
    __syncthreads();
    write_table(p, kFork, threadIdx.x, kPlanThreads);
}

template <bool kFork>
__global__ void __launch_bounds__(kApplyThreads)
pages_copy_kernel(const PageParams p) {
    grid_dependency_wait();
    const long long tid = static_cast<long long>(blockIdx.x) * kApplyThreads + threadIdx.x;
    copy_pages(p, kFork, tid / 32, static_cast<long long>(gridDim.x) * kApplyThreads / 32);
}

// ---------------------------------------------------------------- host

struct Layout {
    size_t keys, free_list, src, dst, first_req, counts, bytes;
};

Layout layout(int num_pages, int num_rows) {
    auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    const size_t pages = up(static_cast<size_t>(num_pages) * 4), rows = up(static_cast<size_t>(num_rows) * 4);
    const size_t moves = pages > rows ? pages : rows;
    Layout l;
    l.keys = 0;
    l.free_list = l.keys + pages;
    l.src = l.free_list + pages;
    l.dst = l.src + moves;
    l.first_req = l.dst + moves;
    l.counts = l.first_req + rows;
    l.bytes = l.counts + 256;
    return l;
}

bool overlaps(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

moe_status_t check_common(const void* caches, size_t cache_stride, int num_caches, int num_pages, size_t page_bytes,
                          int page_size, int max_pages, int num_seqs, int num_rows) {
    if (num_caches < 0 || num_pages <= 0 || page_size != kPage || max_pages <= 0 || num_seqs <= 0 || num_rows < 0)
        return MOE_ERR_INVALID_ARGUMENT;
    if (max_pages > 0x7FFFFFFF / kPage || num_rows >= (1 << kRowBits) ||
        static_cast<long long>(num_rows) * max_pages > 0x7FFFFFFF)
        return MOE_ERR_UNSUPPORTED;
    if (num_caches > 0) {
        if (!caches || !a16(caches) || page_bytes == 0 || page_bytes % 16 || cache_stride % 16) return MOE_ERR_INVALID_ARGUMENT;
        if (num_caches > 1 && cache_stride / page_bytes < static_cast<size_t>(num_pages)) return MOE_ERR_INVALID_ARGUMENT;
        if (page_bytes / 16 > 0x7FFFFF00u) return MOE_ERR_UNSUPPORTED;
    }
    return MOE_OK;
}

template <bool kFork>
moe_status_t run_pages(PageParams& p, void* workspace, cudaStream_t st) {
    const Layout l = layout(p.num_pages, p.num_rows);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.keys = reinterpret_cast<uint32_t*>(ws + l.keys);
    p.free_list = reinterpret_cast<int32_t*>(ws + l.free_list);
    p.move_src = reinterpret_cast<int32_t*>(ws + l.src);
    p.move_dst = reinterpret_cast<int32_t*>(ws + l.dst);
    p.first_req = reinterpret_cast<int32_t*>(ws + l.first_req);
    p.counts = reinterpret_cast<int32_t*>(ws + l.counts);
    const int copy_blocks = 148 * 4;
    if (p.num_pages <= kSmallPages && static_cast<long long>(p.num_rows) * p.max_pages <= kSmallEntries) {
        static bool attr[kMaxDevices] = {};
        if (smem_optin_once(pages_small_kernel<kFork>, kSmallPages * 4, attr) != cudaSuccess) return MOE_ERR_CUDA;
        pages_small_kernel<kFork><<<1, kPlanThreads, static_cast<size_t>(p.num_pages) * 4, st>>>(p);
        const moe_status_t s = launch_status();
        if (s != MOE_OK || p.num_caches == 0) return s;
        return launch_dependent(pages_copy_kernel<kFork>, copy_blocks, kApplyThreads, st, p) == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
    }
    if (cudaMemsetAsync(p.keys, 0, static_cast<size_t>(p.num_pages) * 4, st) != cudaSuccess) return MOE_ERR_CUDA;
    const int mark_blocks = (p.num_rows + kMarkWarps - 1) / kMarkWarps;
    pages_mark_kernel<<<mark_blocks < 1184 ? mark_blocks : 1184, kMarkWarps * 32, 0, st>>>(p);
    moe_status_t s = launch_status();
    if (s != MOE_OK) return s;
    pages_plan_kernel<kFork><<<1, kPlanThreads, 0, st>>>(p);
    if ((s = launch_status()) != MOE_OK) return s;
    pages_apply_kernel<kFork><<<copy_blocks, kApplyThreads, 0, st>>>(p);
    return launch_status();
}

}  // namespace

extern "C" {

size_t kv_pages_workspace_bytes(int num_pages, int num_rows) {
    return num_pages > 0 && num_rows >= 0 ? layout(num_pages, num_rows).bytes : 0;
}

moe_status_t kv_pages_fork(void* caches, size_t cache_stride, int num_caches, int num_pages, size_t page_bytes,
                           int page_size, const int32_t* table_in, int max_pages, const int32_t* lens, int num_seqs,
                           const int32_t* parents, const int32_t* reserve, int num_out, int32_t* table_out,
                           int32_t* lens_out, void* workspace, size_t workspace_bytes, int* error_word,
                           cwStream_t stream) {
    moe_status_t s = check_common(caches, cache_stride, num_caches, num_pages, page_bytes, page_size, max_pages, num_seqs,
                                  num_out);
    if (s != MOE_OK) return s;
    if (num_out == 0) return MOE_OK;
    if (!table_in || !lens || !parents || !table_out || !lens_out || !workspace || !a16(workspace))
        return MOE_ERR_INVALID_ARGUMENT;
    const size_t tin = static_cast<size_t>(num_seqs) * max_pages * 4, tout = static_cast<size_t>(num_out) * max_pages * 4;
    const size_t rows = static_cast<size_t>(num_out) * 4, seqs = static_cast<size_t>(num_seqs) * 4;
    const void* ins[] = {table_in, lens, parents, reserve};
    const size_t in_bytes[] = {tin, seqs, rows, reserve ? rows : 0};
    for (int i = 0; i < 4; ++i)
        if (overlaps(table_out, tout, ins[i], in_bytes[i]) || overlaps(lens_out, rows, ins[i], in_bytes[i]))
            return MOE_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < layout(num_pages, num_out).bytes) return MOE_ERR_WORKSPACE;
    PageParams p = {};
    p.caches = static_cast<uint8_t*>(caches);
    p.cache_stride = cache_stride;
    p.page_bytes = page_bytes;
    p.num_caches = num_caches;
    p.num_pages = num_pages;
    p.max_pages = max_pages;
    p.num_seqs = num_seqs;
    p.num_rows = num_out;
    p.table_in = table_in;
    p.lens = lens;
    p.parents = parents;
    p.reserve = reserve;
    p.table_out = table_out;
    p.lens_out = lens_out;
    p.error_word = error_word;
    return run_pages<true>(p, workspace, static_cast<cudaStream_t>(stream));
}

moe_status_t kv_pages_compact(void* caches, size_t cache_stride, int num_caches, int num_pages, size_t page_bytes,
                              int page_size, const int32_t* table_in, int max_pages, const int32_t* lens, int num_seqs,
                              int32_t* table_out, int32_t* num_used, void* workspace, size_t workspace_bytes,
                              int* error_word, cwStream_t stream) {
    moe_status_t s = check_common(caches, cache_stride, num_caches, num_pages, page_bytes, page_size, max_pages, num_seqs,
                                  num_seqs);
    if (s != MOE_OK) return s;
    if (!table_in || !lens || !table_out || !num_used || !workspace || !a16(workspace)) return MOE_ERR_INVALID_ARGUMENT;
    const size_t tb = static_cast<size_t>(num_seqs) * max_pages * 4;
    if (table_out != table_in && overlaps(table_out, tb, table_in, tb)) return MOE_ERR_INVALID_ARGUMENT;
    if (overlaps(table_out, tb, lens, static_cast<size_t>(num_seqs) * 4)) return MOE_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < layout(num_pages, num_seqs).bytes) return MOE_ERR_WORKSPACE;
    PageParams p = {};
    p.caches = static_cast<uint8_t*>(caches);
    p.cache_stride = cache_stride;
    p.page_bytes = page_bytes;
    p.num_caches = num_caches;
    p.num_pages = num_pages;
    p.max_pages = max_pages;
    p.num_seqs = num_seqs;
    p.num_rows = num_seqs;
    p.table_in = table_in;
    p.lens = lens;
    p.table_out = table_out;
    p.num_used = num_used;
    p.error_word = error_word;
    return run_pages<false>(p, workspace, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
