// attn_prompt.cu -- causal attention over whole prompts in packed rows
// (attn_prompt_packed in include/attn_block.h).
//
// The (position, query head) pairs of one KV head's group are the M rows of a
// tile, position-major, so a tile spans few positions whatever the group size:
// little of a diagonal tile is masked, and a short prompt fills a tile with its
// heads.  Tiles are taken in the order of the keys they attend, most first, by
// a search over the sequence bounds in each CTA: nothing is planned on the host.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

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
    // every sequence has at most one tile in part filled
    const long long tiles = (static_cast<long long>(T) * p.G + kRows - 1) / kRows + num_seqs;
    if (tiles > 0x7FFFFFFF) return MOE_ERR_UNSUPPORTED;
    static bool attr[kMaxDevices] = {};
    if (smem_optin_once(prompt_kernel, static_cast<int>(kSmem), attr) != cudaSuccess) return MOE_ERR_CUDA;
    prompt_kernel<<<dim3(static_cast<int>(tiles), nkv), kRows * 2, kSmem, static_cast<cudaStream_t>(stream)>>>(p);
    return launch_status();
}

}  // extern "C"
