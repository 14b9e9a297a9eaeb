// attn_prompt.cu -- causal attention over whole prompts in packed rows
// (attn_prompt_packed in include/attn_block.h).
//
// The (position, query head) pairs of one KV head's group are the M rows of a
// tile, position-major, so a tile spans few positions whatever the group size:
// little of a diagonal tile is masked, and a short prompt fills a tile with its
// heads.  Tiles are taken in the order of the keys they attend, most first, by
// a search over the sequence bounds in each CTA: nothing is planned on the host.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <mutex>

#include "attn_block.h"
#include "attn_common.cuh"
#include "sm100.cuh"

namespace {

using namespace tb;

constexpr int kMaxGroup = 16;

struct PromptParams {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    long long q_stride, k_stride, v_stride;
    const int32_t* cu_seqlens;
    __nv_bfloat16* out;            // [T][nq][128]
    uint8_t* out_q;
    float* out_s;
    int* error_word;
    int num_seqs, T, nq, nkv, G, out_ld;
    float scale_log2;
    bool flip_q;                   // a negative scale: its sign is taken by the queries
};

struct Tile {
    int first, len;                // rows [first, first + len) are the sequence's
    int index;                     // tile of the sequence
    bool some;
};

// Tile number c of `rows`-row tiles in the order of (tile index, descending;
// sequence).  From the first bound that is out of order or range on there are
// no sequences, so no two overlap.  One warp; every lane gets the result.
__device__ __forceinline__ Tile find_tile(const PromptParams& p, long long c, int rows) {
    const int lane = threadIdx.x & 31;
    int seqs = p.num_seqs;
    for (int s = lane; s < p.num_seqs; s += 32) {
        const int a = p.cu_seqlens[s], b = p.cu_seqlens[s + 1];
        if (a < 0 || b < a || b > p.T) seqs = min(seqs, s);
    }
    seqs = __reduce_min_sync(0xffffffffu, seqs);
    if (seqs < p.num_seqs && c == 0 && lane == 0 && p.error_word) atomicExch(p.error_word, 5);
    auto tiles = [&](int s) {
        const long long n = s < seqs ? static_cast<long long>(p.cu_seqlens[s + 1] - p.cu_seqlens[s]) * p.G : 0;
        return static_cast<int>((n + rows - 1) / rows);
    };
    // tiles with an index of at least x
    auto at_least = [&](int x) {
        long long sum = 0;
        for (int s0 = 0; s0 < seqs; s0 += 32) sum += max(tiles(s0 + lane) - x, 0);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return sum;
    };
    int most = 0;
    for (int s0 = 0; s0 < seqs; s0 += 32) most = max(most, tiles(s0 + lane));
    most = __reduce_max_sync(0xffffffffu, most);
    Tile t = {0, 0, 0, false};
    if (c >= at_least(0)) return t;
    int lo = 0, hi = most;             // at_least(lo) > c, at_least(hi) <= c
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (at_least(mid) > c) lo = mid;
        else hi = mid;
    }
    long long skip = c - at_least(lo + 1);
    for (int s0 = 0; s0 < seqs; s0 += 32) {
        const bool has = tiles(s0 + lane) > lo;
        const uint32_t m = __ballot_sync(0xffffffffu, has);
        const int n = __popc(m);
        if (skip < n) {
            const int s = s0 + __fns(m, 0, static_cast<int>(skip) + 1);
            t.first = p.cu_seqlens[s];
            t.len = p.cu_seqlens[s + 1] - t.first;
            t.index = lo;
            t.some = true;
            return t;
        }
        skip -= n;
    }
    return t;
}

// Zeroes the NaN and infinite elements of eight bf16 values; true if any.
__device__ __forceinline__ bool zero_nonfinite(uint4& v) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & 0x7F80u) == 0x7F80u) { w[i] &= 0xFFFF0000u; any = true; }
        if ((w[i] & 0x7F800000u) == 0x7F800000u) { w[i] &= 0x0000FFFFu; any = true; }
    }
    return any;
}

// ---------------------------------------------------------------- mma.sync tiles

constexpr int kRows = 64;          // M rows of a CTA, 16 a warp
constexpr int kKeys = 64;          // keys per step
constexpr int kPad = kD + 8;       // bf16 elements per shared row
constexpr size_t kSmem = (static_cast<size_t>(kRows) + 2 * 2 * kKeys) * kPad * 2;

__global__ void __launch_bounds__(kRows * 2, 2)
prompt_kernel(const PromptParams p) {
    extern __shared__ __align__(128) __nv_bfloat16 sm[];
    __shared__ Tile tile_s;
    __shared__ int dirty;              // V values zeroed behind the tile's first position
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tq = lane & 3;
    const int kvh = blockIdx.y;
    if (warp == 0) {
        const Tile t = find_tile(p, blockIdx.x, kRows);
        if (lane == 0) {
            tile_s = t;
            dirty = 0;
        }
    }
    __syncthreads();
    const Tile tile = tile_s;
    if (!tile.some) return;
    const long long r0 = static_cast<long long>(tile.index) * kRows;
    const int rows = static_cast<int>(min(static_cast<long long>(kRows), static_cast<long long>(tile.len) * p.G - r0));
    const int pos0 = static_cast<int>(r0 / p.G);                  // first position of the tile
    const int pos1 = static_cast<int>((r0 + rows - 1) / p.G);     // last
    const int steps = pos1 / kKeys + 1;

    __nv_bfloat16* q_s = sm;
    __nv_bfloat16* kv_s = sm + kRows * kPad;                      // [2][K 64 | V 64][kPad]
    for (int c = threadIdx.x; c < kRows * (kD / 8); c += blockDim.x) {
        const int i = c / (kD / 8), e = c % (kD / 8) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (i < rows) {
            const int row = tile.first + static_cast<int>((r0 + i) / p.G), h = kvh * p.G + static_cast<int>((r0 + i) % p.G);
            v = *reinterpret_cast<const uint4*>(p.q + row * p.q_stride + h * kD + e);
        }
        *reinterpret_cast<uint4*>(q_s + i * kPad + e) = v;
    }
    auto load = [&](int step, int stage) {
        __nv_bfloat16* dst = kv_s + stage * 2 * kKeys * kPad;
        for (int c = threadIdx.x; c < 2 * kKeys * (kD / 8); c += blockDim.x) {
            const int which = c / (kKeys * (kD / 8)), i = c / (kD / 8) % kKeys, e = c % (kD / 8) * 8;
            const int j = step * kKeys + i;
            const bool in = j < tile.len;
            const long long row = tile.first + (in ? j : 0);
            const __nv_bfloat16* src = which ? p.v + row * p.v_stride : p.k + row * p.k_stride;
            cp_async16(dst + (which * kKeys + i) * kPad + e, src + kvh * kD + e, in ? 16u : 0u);
        }
    };
    load(0, 0);
    cp_async_commit();
    __syncthreads();
    uint32_t qa[kD / 16][4];
    {
        const int mi = lane >> 3, rr = (lane & 7) + 8 * (mi & 1);
#pragma unroll
        for (int ks = 0; ks < kD / 16; ++ks)
            ldsm_x4(smem_u32(q_s + (warp * 16 + rr) * kPad + ks * 16 + 8 * (mi >> 1)), qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3]);
    }
    int pos_r[2];                      // position of this thread's two rows (padding: the last)
#pragma unroll
    for (int h = 0; h < 2; ++h) pos_r[h] = static_cast<int>((r0 + min(warp * 16 + g + 8 * h, rows - 1)) / p.G);
    float o[kD / 8][4];
#pragma unroll
    for (int i = 0; i < kD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m_r[2] = {-INFINITY, -INFINITY}, l_r[2] = {0.0f, 0.0f};
    for (int i = 0; i < steps; ++i) {
        __syncthreads();               // the other stage is free
        if (i + 1 < steps) load(i + 1, (i + 1) & 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        __nv_bfloat16* ks_ = kv_s + (i & 1) * 2 * kKeys * kPad;
        __nv_bfloat16* vs_ = ks_ + kKeys * kPad;
        const int j0 = i * kKeys;
        const bool masked = j0 + kKeys - 1 > pos0;
        if (masked) {
            // a weight of 0 must meet a finite value: V of positions that not every row attends
            for (int c = threadIdx.x; c < kKeys * (kD / 8); c += blockDim.x) {
                const int j = j0 + c / (kD / 8);
                if (j <= pos0) continue;
                uint4* at = reinterpret_cast<uint4*>(vs_ + c / (kD / 8) * kPad + c % (kD / 8) * 8);
                uint4 v = *at;
                if (zero_nonfinite(v)) {
                    *at = v;
                    dirty = 1;
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int half = 0; half < kKeys / 16; ++half) {            // 16 keys at a time
            const __nv_bfloat16* kh = ks_ + half * 16 * kPad;
            const __nv_bfloat16* vh = vs_ + half * 16 * kPad;
            float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
            {
                const int mi = lane >> 3, rr = (lane & 7) + 8 * (mi >> 1), cofs = 8 * (mi & 1);
#pragma unroll
                for (int ks = 0; ks < kD / 16; ++ks) {
                    uint32_t b0, b1, b2, b3;
                    ldsm_x4(smem_u32(kh + rr * kPad + ks * 16 + cofs), b0, b1, b2, b3);
                    mma_bf16(s0, qa[ks], b0, b1);
                    mma_bf16(s1, qa[ks], b2, b3);
                }
            }
            const int j = j0 + half * 16 + 2 * tq;
            float sv[2][4] = {{s0[0], s0[1], s1[0], s1[1]}, {s0[2], s0[3], s1[2], s1[3]}};
            float alpha[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int jj = j + (e & 1) + 8 * (e >> 1);
                    sv[h][e] = jj <= pos_r[h] ? sv[h][e] * p.scale_log2 : -INFINITY;
                    mx = fmaxf(mx, sv[h][e]);
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m_r[h], mx);
                const float ms = mn == -INFINITY ? 0.0f : mn;
                alpha[h] = exp2f(m_r[h] - ms);
                m_r[h] = mn;
                float rs = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sv[h][e] = exp2f(sv[h][e] - ms);
                    rs += sv[h][e];
                }
                l_r[h] = l_r[h] * alpha[h] + rs;
            }
            if (alpha[0] != 1.0f || alpha[1] != 1.0f) {
#pragma unroll
                for (int nd = 0; nd < kD / 8; ++nd) {
                    o[nd][0] *= alpha[0]; o[nd][1] *= alpha[0];
                    o[nd][2] *= alpha[1]; o[nd][3] *= alpha[1];
                }
            }
            uint32_t pa[4] = {pack_bf16(sv[0][0], sv[0][1]), pack_bf16(sv[1][0], sv[1][1]), pack_bf16(sv[0][2], sv[0][3]),
                              pack_bf16(sv[1][2], sv[1][3])};
            const int mi = lane >> 3, rr = (lane & 7) + 8 * (mi & 1), cofs = 8 * (mi >> 1);
#pragma unroll
            for (int nd = 0; nd < kD / 8; nd += 2) {
                uint32_t b0, b1, b2, b3;
                ldsm_x4_t(smem_u32(vh + rr * kPad + nd * 8 + cofs), b0, b1, b2, b3);
                mma_bf16(o[nd], pa, b0, b1);
                mma_bf16(o[nd + 1], pa, b2, b3);
            }
        }
    }
    cp_async_wait<0>();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float l = l_r[h];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int i = warp * 16 + g + 8 * h;
        float amax = 0.0f;
#pragma unroll
        for (int nd = 0; nd < kD / 8; ++nd)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = o[nd][2 * h + e] / l;
                if (dirty) {               // the values zeroed above, for the rows that attend them
                    for (int j = pos0 + 1; j <= pos_r[h]; ++j) {
                        const float y = __bfloat162float(p.v[(tile.first + j) * p.v_stride + kvh * kD + nd * 8 + 2 * tq + e]);
                        if (!isfinite(y)) x += y;
                    }
                }
                o[nd][2 * h + e] = x;
                amax = fmaxf(amax, fabsf(x));
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        if (i >= rows) continue;
        const long long row = tile.first + pos_r[h];
        const int head = kvh * p.G + static_cast<int>((r0 + i) % p.G);
        __nv_bfloat16* orow = p.out + (row * p.nq + head) * kD;
        const float inv = amax > 0.0f ? 448.0f / amax : 0.0f;
#pragma unroll
        for (int nd = 0; nd < kD / 8; ++nd) {
            const int col = nd * 8 + 2 * tq;
            *reinterpret_cast<uint32_t*>(orow + col) = pack_bf16(o[nd][2 * h], o[nd][2 * h + 1]);
            if (p.out_q)
                *reinterpret_cast<uint16_t*>(p.out_q + (row * p.nq + head) * kD + col) =
                    amax > 0.0f ? cvt_e4m3x2(o[nd][2 * h] * inv, o[nd][2 * h + 1] * inv) : 0;
        }
        if (p.out_q && tq == 0) p.out_s[static_cast<size_t>(head) * p.out_ld + row] = amax > 0.0f ? amax / 448.0f : 0.0f;
    }
}

// ---------------------------------------------------------------- tcgen05 tiles
//
// One CTA per 256 rows, two M = 128 tiles with a softmax warpgroup each, one
// thread per row.  While one tile's softmax runs on its scores, the tensor core
// works on the other's: S = Q K^T into TMEM, read as fp32, written back over
// itself as the bf16 weights P, which the second MMA takes from TMEM as its A
// operand with V (MN-major) from shared memory.  K and V arrive by TMA in a
// ring of 128-key stages.  The running maximum is left behind by up to 2^8
// before the output is rescaled, so a rescale is rare and the softmax threads
// do it themselves: the scores' arrival means that the product before is done.

constexpr int kTcRows = 256;
constexpr int kTcKeys = 128;
constexpr int kTcStages = 5;                            // K and V tiles in flight, 32 KB each
constexpr int kTcThreads = 384;
constexpr uint32_t kHalf = kTcKeys * 128;               // 64 dims of a 128-row tile: rows of 128 bytes, swizzled
constexpr uint32_t kTileBytes = 2 * kHalf;
constexpr size_t kTcSmem = 2 * kTileBytes + kTcStages * kTileBytes + 1024;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr int kCleanThreads = 64;
// 256 rows are at most 256 positions (one head a group), so at most three steps hold masked ones
constexpr int kMaxMasked = 3;

struct TcBars {
    uint64_t full[kTcStages], empty[kTcStages];
    uint64_t s_full[2], p_full[2], o_full[2], drain;
    uint64_t v_full[kMaxMasked], clean[kMaxMasked];     // V tiles with masked positions, each used once
};

// Waits without regard to the abort flag, for this thread's own copies.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 < kWaitNs) {}
}

__global__ void __launch_bounds__(kTcThreads, 1)
prompt_tc_kernel(const PromptParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    extern __shared__ uint8_t sm_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* q_s = sm;                                  // [2 tiles][2 halves][128][128 B]
    uint8_t* kv_s = sm + 2 * kTileBytes;                // [stages][2 halves][128][128 B]
    __shared__ TcBars bars;
    __shared__ Tile tile_s;
    __shared__ uint32_t tmem_s;
    __shared__ int dirty_s, abort_s;
    volatile int* abort_flag = &abort_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kvh = blockIdx.x % p.nkv;
    if (warp == 0) {
        const Tile t = find_tile(p, blockIdx.x / p.nkv, kTcRows);
        if (lane == 0) tile_s = t;
    } else if (warp == 9 && lane == 0) {
        for (int i = 0; i < kTcStages; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&bars.s_full[t], 1);
            mbar_init(&bars.p_full[t], 128);
            mbar_init(&bars.o_full[t], 1);
        }
        for (int i = 0; i < kMaxMasked; ++i) {
            mbar_init(&bars.v_full[i], 1);
            mbar_init(&bars.clean[i], kCleanThreads);
        }
        mbar_init(&bars.drain, 1);
        dirty_s = 0;
        abort_s = 0;
        fence_mbar_init();
        prefetch_tmap(&kmap);
        prefetch_tmap(&vmap);
    }
    __syncthreads();
    const Tile tile = tile_s;
    if (!tile.some) return;
    const long long r0 = static_cast<long long>(tile.index) * kTcRows;
    const int rows = static_cast<int>(min(static_cast<long long>(kTcRows), static_cast<long long>(tile.len) * p.G - r0));
    const int pos0 = static_cast<int>(r0 / p.G);
    const int pos1 = static_cast<int>((r0 + rows - 1) / p.G);
    const int steps = pos1 / kTcKeys + 1;
    const int mt = rows > 128 ? 2 : 1;                  // M tiles in use
    // steps from here on hold positions that not every row attends
    const int first_masked = (pos0 + 1) / kTcKeys;

    if (warp < 8) {                                     // Q: a row a thread, as the TMA would swizzle it
        const int i = threadIdx.x;
        uint8_t* dst = q_s + (i >> 7) * kTileBytes + (i & 127) * 128;
        const bool in = i < rows;
        const long long row = tile.first + (in ? (r0 + i) / p.G : 0);
        const uint4* src = reinterpret_cast<const uint4*>(p.q + row * p.q_stride + (kvh * p.G + (in ? (r0 + i) % p.G : 0)) * kD);
        if ((i >> 7) < mt) {
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                uint4 v = in ? src[c] : make_uint4(0, 0, 0, 0);
                if (p.flip_q) { v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u; }
                *reinterpret_cast<uint4*>(dst + (c >> 3) * kHalf + (((c & 7) ^ (i & 7)) << 4)) = v;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    } else if (warp == 8) {
        tmem_alloc(&tmem_s, 512);
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 9 && lane == 0) {
            // ---- loads: K and V tiles of step 0, 1, ...
            const int x = kvh * kD;
            int n = 0;
            bool ok = true;
            for (; n < 2 * steps; ++n) {
                const int st = n % kTcStages, use = n / kTcStages;
                if (!(ok = mbar_wait_bounded(&bars.empty[st], (use & 1) ^ 1, abort_flag, kWaitNs))) break;
                uint8_t* dst = kv_s + st * kTileBytes;
                const int y = tile.first + n / 2 * kTcKeys;
                const bool to_clean = (n & 1) && n / 2 >= first_masked;
                uint64_t* bar = to_clean ? &bars.v_full[n / 2 - first_masked] : &bars.full[st];
                if (to_clean) mbar_arrive(&bars.full[st]);          // keeps the ring's phases; nobody waits for this one
                mbar_arrive_expect_tx(bar, kTileBytes);
                const CUtensorMap* map = (n & 1) ? &vmap : &kmap;
                tma_load_2d(map, bar, dst, x, y);
                tma_load_2d(map, bar, dst + kHalf, x + 64, y);
            }
            if (!ok) {   // loads in flight land before the block leaves
                for (int i = max(n - kTcStages, 0); i < n; ++i) {
                    mbar_drain(&bars.full[i % kTcStages], (i / kTcStages) & 1);
                    if ((i & 1) && i / 2 >= first_masked) mbar_drain(&bars.v_full[i / 2 - first_masked], 0);
                }
            }
        } else if (warp == 8 && lane == 0) {
            // ---- MMA issue
            constexpr uint32_t id_s = idesc_bf16_f32(128, kTcKeys, false), id_o = idesc_bf16_f32(128, kD, true);
            auto wait_full = [&](int n) {
                return mbar_wait_bounded(&bars.full[n % kTcStages], (n / kTcStages) & 1, abort_flag, kWaitNs);
            };
            auto scores = [&](int t, int n) {           // S_t = Q_t K^T, K tile number n of the ring
                const uint32_t q = smem_u32(q_s + t * kTileBytes), k = smem_u32(kv_s + n % kTcStages * kTileBytes);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const uint32_t off = (ks >> 2) * kHalf + (ks & 3) * 32;
                    umma_f16(tmem + t * 128, umma_desc_sw128(q + off), umma_desc_sw128(k + off), id_s, ks > 0);
                }
                umma_commit(&bars.s_full[t]);
            };
            bool ok = wait_full(0);
            if (ok) {
                for (int t = 0; t < mt; ++t) scores(t, 0);
                umma_commit(&bars.empty[0]);
            }
            for (int i = 0; i < steps && ok; ++i) {
                const int nv = 2 * i + 1, nk = 2 * i + 2;
                for (int t = 0; t < mt && ok; ++t) {
                    ok = mbar_wait_bounded(&bars.p_full[t], i & 1, abort_flag, kWaitNs);
                    if (ok && t == 0)
                        ok = i < first_masked ? wait_full(nv)
                                              : mbar_wait_bounded(&bars.clean[i - first_masked], 0, abort_flag, kWaitNs);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t v = smem_u32(kv_s + nv % kTcStages * kTileBytes);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)      // 16 keys: 16 rows of 128 bytes
                        umma_f16_ta(tmem + 256 + t * 128, tmem + t * 128 + ks * 8, umma_desc_mn_sw128(v + ks * 2048, kHalf),
                                    id_o, i > 0 || ks > 0);
                    if (i == steps - 1) umma_commit(&bars.o_full[t]);
                    if (t == mt - 1) umma_commit(&bars.empty[nv % kTcStages]);
                    if (i + 1 < steps) {
                        if (t == 0 && !(ok = wait_full(nk))) break;
                        scores(t, nk);
                        if (t == mt - 1) umma_commit(&bars.empty[nk % kTcStages]);
                    }
                }
            }
            if (!ok) {
                umma_commit(&bars.drain);
                mbar_drain(&bars.drain, 0);
            }
        } else if (warp >= 10) {
            // ---- a weight of 0 must meet a finite value: V of positions that not every row attends
            const int c0 = threadIdx.x - 320;
            bool ok = true, dirty = false;
            for (int i = first_masked; i < steps && ok; ++i) {
                const int n = 2 * i + 1;
                ok = mbar_wait_bounded(&bars.v_full[i - first_masked], 0, abort_flag, kWaitNs);
                if (!ok) break;
                uint8_t* v = kv_s + n % kTcStages * kTileBytes;
                const int j0 = max(pos0 + 1 - i * kTcKeys, 0);     // first such row of the tile
#pragma unroll 4
                for (int c = c0; c < (kTcKeys - j0) * 16; c += kCleanThreads) {
                    uint4* at = reinterpret_cast<uint4*>(v + (c & 1) * kHalf + (j0 + (c >> 4)) * 128 + ((c >> 1) & 7) * 16);
                    uint4 x = *at;
                    if (zero_nonfinite(x)) {
                        *at = x;
                        dirty = true;
                    }
                }
                if (dirty) dirty_s = 1;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&bars.clean[i - first_masked]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int t = warp >> 2;
        const int i_row = threadIdx.x;
        const int pos = static_cast<int>((r0 + min(i_row, rows - 1)) / p.G);
        const uint32_t ts = tmem + (static_cast<uint32_t>(warp & 3) << 21) + t * 128;   // this warp's 32 lanes
        const uint32_t to = ts + 256;
        const float sl2 = p.scale_log2;
        float m = -INFINITY, l = 0.0f;
        bool ok = t < mt;
        for (int i = 0; i < steps && ok; ++i) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.s_full[t], i & 1, abort_flag, kWaitNs));
            if (!ok) break;
            tc_fence_after();
            uint32_t s[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, s[c]);
            tmem_wait_ld();
            if (i >= first_masked) {
                const int lim = pos - i * kTcKeys;
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (32 * c + e > lim) s[c][e] = 0xFF800000u;
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][e]));
            const float mt_ = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            if (i == 0) {
                m = mt_;
            } else {
                const bool need = (mt_ - m) * sl2 > 8.0f;
                if (__any_sync(0xffffffffu, need)) {
                    const float f = need ? ex2((m - mt_) * sl2) : 1.0f;
                    l *= f;
                    if (need) m = mt_;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[32];
                        tmem_ld32(to + 32 * c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st32(to + 32 * c, o);
                    }
                }
            }
            const float nm = m == -INFINITY ? 0.0f : -m * sl2;     // nothing but -inf so far: weights 0, not NaN
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float2 x = ffma2(make_float2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])),
                                     make_float2(sl2, sl2), make_float2(nm, nm));
                    x.x = ex2(x.x);
                    x.y = ex2(x.y);
                    sum.x += x.x;
                    sum.y += x.y;
                    w[e] = pack_bf16(x.x, x.y);         // the weights' rounding, 2^-8 at most; the sum has them whole
                }
                tmem_st16(ts + 16 * c, w);
            }
            l += sum.x + sum.y;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars.p_full[t]);
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.o_full[t], 0, abort_flag, kWaitNs));
        if (ok && steps > first_masked)                 // acquires the flag below
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&bars.clean[steps - 1 - first_masked], 0, abort_flag, kWaitNs));
        if (ok) {
            tc_fence_after();
            const bool dirty = *static_cast<volatile int*>(&dirty_s) != 0;
            const float inv = 1.0f / l;
            const long long row = tile.first + pos;
            const int head = kvh * p.G + static_cast<int>((r0 + min(i_row, rows - 1)) % p.G);
            __nv_bfloat16* orow = p.out + (row * p.nq + head) * kD;
            const __nv_bfloat16* vrow = p.v + static_cast<long long>(tile.first) * p.v_stride + kvh * kD;
            const bool store = i_row < rows;
            auto column = [&](uint32_t bits, int d) {
                float x = __uint_as_float(bits) * inv;
                if (dirty)                              // the values zeroed above, for the rows that attend them
                    for (int j = pos0 + 1; j <= pos; ++j) {
                        const float y = __bfloat162float(vrow[j * p.v_stride + d]);
                        if (!isfinite(y)) x += y;
                    }
                return x;
            };
            float amax = 0.0f;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                tmem_ld32(to + 32 * c, o);
                tmem_wait_ld();
                uint32_t w[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float a = column(o[2 * e], 32 * c + 2 * e), b = column(o[2 * e + 1], 32 * c + 2 * e + 1);
                    amax = fmaxf(amax, fmaxf(fabsf(a), fabsf(b)));
                    w[e] = pack_bf16(a, b);
                }
                if (store)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        *reinterpret_cast<uint4*>(orow + 32 * c + 8 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
            }
            if (p.out_q) {
                const float qi = amax > 0.0f ? 448.0f / amax : 0.0f;
                uint8_t* qrow = p.out_q + (row * p.nq + head) * kD;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t o[32];
                    tmem_ld32(to + 32 * c, o);
                    tmem_wait_ld();
                    uint32_t w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int d = 32 * c + 4 * e;
                        w[e] = amax > 0.0f ? cvt_e4m3x2(column(o[4 * e], d) * qi, column(o[4 * e + 1], d + 1) * qi) |
                                                 static_cast<uint32_t>(cvt_e4m3x2(column(o[4 * e + 2], d + 2) * qi,
                                                                                  column(o[4 * e + 3], d + 3) * qi)) << 16
                                           : 0u;
                    }
                    if (store)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            *reinterpret_cast<uint4*>(qrow + 32 * c + 16 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                }
                if (store) p.out_s[static_cast<size_t>(head) * p.out_ld + row] = amax > 0.0f ? amax / 448.0f : 0.0f;
            }
            tc_fence_before();
        }
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && *abort_flag && p.error_word) atomicExch(p.error_word, 1);
}

// ---------------------------------------------------------------- host

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// bf16 rows [T][cols], `stride` elements apart, boxes of 64 columns x 128 rows.
bool encode_rows(CUtensorMap* map, const void* base, int T, int cols, long long stride) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(T)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
    cuuint32_t box[2] = {64, kTcKeys};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

extern "C" {

moe_status_t attn_prompt_packed(const void* q_bf16, long long q_stride, const void* k_bf16, long long k_stride,
                                const void* v_bf16, long long v_stride, const int32_t* cu_seqlens, int num_seqs, int T,
                                int nq, int nkv, int head_dim, float scale, void* out_bf16, void* out_q, float* out_s,
                                int out_ld, int* error_word, cwStream_t stream) {
    if (T < 0 || num_seqs < 0 || nq <= 0 || nkv <= 0 || nq % nkv || nq / nkv > kMaxGroup || head_dim != kD)
        return MOE_ERR_INVALID_ARGUMENT;
    if (nkv > 65535 || nq > (1 << 20)) return MOE_ERR_UNSUPPORTED;
    if (q_stride < nq * kD || k_stride < nkv * kD || v_stride < nkv * kD || q_stride % 8 || k_stride % 8 || v_stride % 8)
        return MOE_ERR_INVALID_ARGUMENT;
    if (T == 0 || num_seqs == 0) return MOE_OK;
    if (!q_bf16 || !k_bf16 || !v_bf16 || !cu_seqlens || !out_bf16) return MOE_ERR_INVALID_ARGUMENT;
    if (!a16(q_bf16) || !a16(k_bf16) || !a16(v_bf16) || !a16(out_bf16)) return MOE_ERR_INVALID_ARGUMENT;
    if (out_q && (!out_s || out_ld < T || !a16(out_q))) return MOE_ERR_INVALID_ARGUMENT;
    PromptParams p;
    p.q = static_cast<const __nv_bfloat16*>(q_bf16);
    p.k = static_cast<const __nv_bfloat16*>(k_bf16);
    p.v = static_cast<const __nv_bfloat16*>(v_bf16);
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.cu_seqlens = cu_seqlens;
    p.out = static_cast<__nv_bfloat16*>(out_bf16);
    p.out_q = static_cast<uint8_t*>(out_q);
    p.out_s = out_s;
    p.error_word = error_word;
    p.num_seqs = num_seqs;
    p.T = T;
    p.nq = nq;
    p.nkv = nkv;
    p.G = nq / nkv;
    p.out_ld = out_ld;
    p.scale_log2 = scale * kLog2e;
    p.flip_q = false;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const char* form = getenv("PROMPT_FORM");
    if (!form || form[0] == 't') {
        p.flip_q = p.scale_log2 < 0.0f;
        p.scale_log2 = fmaxf(fabsf(p.scale_log2), 1.17549435e-38f);   // 0: every finite score alike, masked ones still -inf
        const long long tiles = ((static_cast<long long>(T) * p.G + kTcRows - 1) / kTcRows + num_seqs) * nkv;
        if (tiles > 0x7FFFFFFF) return MOE_ERR_UNSUPPORTED;
        CUtensorMap kmap, vmap;
        if (!encode_rows(&kmap, k_bf16, T, nkv * kD, k_stride) || !encode_rows(&vmap, v_bf16, T, nkv * kD, v_stride))
            return MOE_ERR_CUDA;
        static bool tc_attr[kMaxDevices] = {};
        if (smem_optin_once(prompt_tc_kernel, static_cast<int>(kTcSmem), tc_attr) != cudaSuccess) return MOE_ERR_CUDA;
        prompt_tc_kernel<<<static_cast<int>(tiles), kTcThreads, kTcSmem, st>>>(p, kmap, vmap);
        return launch_status();
    }
    // every sequence has at most one tile in part filled
    const long long tiles = (static_cast<long long>(T) * p.G + kRows - 1) / kRows + num_seqs;
    if (tiles > 0x7FFFFFFF) return MOE_ERR_UNSUPPORTED;
    static bool attr[kMaxDevices] = {};
    if (smem_optin_once(prompt_kernel, static_cast<int>(kSmem), attr) != cudaSuccess) return MOE_ERR_CUDA;
    prompt_kernel<<<dim3(static_cast<int>(tiles), nkv), kRows * 2, kSmem, static_cast<cudaStream_t>(stream)>>>(p);
    return launch_status();
}

}  // extern "C"
