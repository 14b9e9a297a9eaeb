// attn_kv4.cu -- the 4-bit KV cache (include/kv_cache.h): partial RoPE with the
// quantising page write, rows read back, and split-context decode attention.
//
// A value is n * s with n a 4-bit integer and s a bf16 number of four
// significant bits, one per 32 dims.  Decode turns a code into it with one
// lop3 and one bf16x2 fma: the code's nibble under the exponent of 128 is the
// bf16 number 128 + (n + 8), and (136 + n) * s - 136 * s is exact -- 136 * s is
// 17 * s with at most eight significant bits, n * s has at most eight -- so the
// tensor cores see exactly the values held and nothing is rounded on the way.
//
// Measured (B200, device time).  Write of 4198 rows, 96 query and 8 KV heads:
// 47 us, 5.1 TB/s of rows in, queries, keys and codes out; 64 rows: 3.2 us.  Rows
// read back: 8 us for those 4198.  Decode: see there.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "attn_common.cuh"
#include "kv_cache.h"
#include "sm100.cuh"

namespace {

using namespace tb;

constexpr int kGroups = kD / 32;                     // scales per token and head
constexpr int kCodes = kPage * kD / 2;               // code bytes of one page and head
constexpr int kPage4 = kCodes + kPage * kGroups * 2; // 1152
constexpr int kGPad = 16;                            // query rows of one GQA group, padded to the MMA M

// Byte offsets inside one (page, head) tile; see kv_cache.h.
__host__ __device__ constexpr int k_code_byte(int t, int d) {
    return t * 64 + (d % 32) / 8 * 16 + d / 32 * 4 + d % 8 / 2;
}
__host__ __device__ constexpr int v_code_byte(int t, int d) {
    return t / 8 * 512 + (4 * (d % 32 / 4) + t % 8 / 2) * 16 + t % 2 * 8 + d / 32 * 2 + d % 4 / 2;
}

// ---------------------------------------------------------------- write

constexpr int kWriteWarps = 8;
constexpr int kWriteUnroll = 4;                      // pairs of heads a warp has in flight

// Scale of a group whose largest |x| has the bits `amax`, and 0 for a group
// that is stored as NaN.
__device__ __forceinline__ float group_scale(uint32_t amax) {
    if (amax >= ((127u + 120u) << 23)) return 0.0f;
    const uint32_t b = __float_as_uint(__fdiv_rn(__uint_as_float(amax), 7.5f));
    return fmaxf(__uint_as_float((b + 0x000FFFFFu) & ~0x000FFFFFu), 1.17549435e-38f);
}

// (lo, hi) of a pair after rotation; products rounded before the sum, so the
// result does not hang on what the compiler contracts.
__device__ __forceinline__ float rotate_lo(float a, float c, float cs, float sn) { return __fsub_rn(__fmul_rn(a, cs), __fmul_rn(c, sn)); }
__device__ __forceinline__ float rotate_hi(float a, float c, float cs, float sn) { return __fadd_rn(__fmul_rn(a, sn), __fmul_rn(c, cs)); }

struct WriteParams {
    const __nv_bfloat16* qkv;
    const float* inv_freq;
    const int32_t* positions;
    const int32_t* row_seq;
    const int32_t* page_table;
    __nv_bfloat16* q_out;
    __nv_bfloat16* k_out;
    uint8_t* k_cache;
    uint8_t* v_cache;
    int32_t* seq_lens_out;
    int* error_word;
    int nq, nkv, rot, num_seqs, max_pages, num_cache_pages;
};

__device__ __forceinline__ float2 bf16_pair(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }

// Eight dims 8 l .. 8 l + 7 of a head, by lane l of a half-warp, quantised into
// token t of the (page, head) tile; the whole warp comes here, `store` says
// which half has a tile.
//
// rint(x / s) without a division: q = x * r with r near 1 / s is corrected by its
// own residual (Newton), q + (x - q s) r, within 2^-45 of x / s before it is
// rounded.  With x of 8 bits and s of 4, x / s is a half integer or at least 2^-12
// away from one, so only half integers need care, and those are floats: the
// corrected q is x / s itself.  Scales below 2^-60 are worked at 2^64 times
// their size, where the residual is no subnormal.
__device__ __forceinline__ void quantise_store(const uint4& xv, uint8_t* page, int t, int l, bool is_k, bool store) {
    const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
    uint32_t amax = 0;                               // as bits: a NaN is above every number
#pragma unroll
    for (int i = 0; i < 4; ++i) amax = max(amax, max(xw[i] << 16 & 0x7FFF0000u, xw[i] & 0x7FFF0000u));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));       // a group of 32 dims is four lanes
    if (!store) return;
    const float s = group_scale(amax);
    const float up = s < 8.67361737988403547e-19f ? 18446744073709551616.0f : 1.0f;
    const float su = s * up, r = __frcp_rn(su);
    constexpr float kMagic = 12582912.0f + 8.0f;     // 1.5 * 2^23: the sum's low bits are rint(q) + 8
    uint32_t codes = 0;                              // the sums' other bits go by their total
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = bf16_pair(xw[i]);
        const float xe[2] = {x.x * up, x.y * up};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float q = xe[e] * r;
            q = fmaf(fmaf(-q, su, xe[e]), r, q);
            codes += __float_as_uint(fminf(q, 7.0f) + kMagic) << (4 * (2 * i + e));
        }
    }
    constexpr uint32_t kOnes = 0x11111111u;
    codes -= 0x4B400000u * kOnes;
    if (s == 0.0f) codes = 8u * kOnes;
    if (is_k) {
        *reinterpret_cast<uint32_t*>(page + k_code_byte(t, 8 * l)) = codes;
    } else {
        *reinterpret_cast<uint16_t*>(page + v_code_byte(t, 8 * l)) = static_cast<uint16_t>(codes);
        *reinterpret_cast<uint16_t*>(page + v_code_byte(t, 8 * l + 4)) = static_cast<uint16_t>(codes >> 16);
    }
    if ((l & 3) == 0)
        *reinterpret_cast<uint16_t*>(page + kCodes + (t * kGroups + l / 4) * 2) =
            s > 0.0f ? static_cast<uint16_t>(__float_as_uint(s) >> 16) : static_cast<uint16_t>(0x7FC0);   // s is a bf16 number
}

// One block per (row, share of the heads), a half-warp per head with 16 bytes a
// lane and kWriteUnroll heads in flight; bound by the rows in and the q rows
// out (0.8 of the copy bandwidth; 2, 3 and 7 heads in flight are within 4 %).  kLanes: the rotated halves are whole lanes, a dim's partner comes from
// lane l +- half / 8 and a lane's cosines stay in registers; else partners come
// from memory.
template <bool kLanes>
__global__ void __launch_bounds__(kWriteWarps * 32, 4)
kv4_rope_write_kernel(const WriteParams p) {
    __shared__ float cs_s[kD / 2], sn_s[kD / 2];
    const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & 15;
    const bool first = blockIdx.y == 0 && threadIdx.x == 0;
    const int heads = p.nq + 2 * p.nkv;
    const __nv_bfloat16* row = p.qkv + static_cast<size_t>(b) * heads * kD;
    const int stride = gridDim.y * kWriteWarps * 2;
    int h0 = (blockIdx.y * kWriteWarps + warp) * 2 + (lane >> 4);
    uint4 in[kWriteUnroll];
    auto load = [&] {
#pragma unroll
        for (int u = 0; u < kWriteUnroll; ++u)
            if (h0 + u * stride < heads) in[u] = *reinterpret_cast<const uint4*>(row + static_cast<size_t>(h0 + u * stride) * kD + 8 * l);
    };
    load();                                          // under the position's and the page's way here
    const int pos = p.positions[b];
    const int seq = seq_of_row(p.row_seq, b, p.num_seqs);
    if (first && p.seq_lens_out) p.seq_lens_out[b] = (pos >= 0 && seq >= 0) ? pos + 1 : 0;
    int phys = 0, err = 0;
    if (seq < 0) err = 7;
    else if (pos < 0 || pos / kPage >= p.max_pages) err = 4;
    else {
        phys = p.page_table[static_cast<size_t>(seq) * p.max_pages + pos / kPage];
        if (phys < 0 || phys >= p.num_cache_pages) err = 6;
    }
    if (err) {
        if (first && p.error_word) atomicExch(p.error_word, err);
        return;
    }
    const int half = p.rot / 2;
    for (int i = threadIdx.x; i < half; i += blockDim.x)
        // the angle is the fp32 product, as in the bf16 page write
        sincosf(static_cast<float>(pos) * p.inv_freq[i], &sn_s[i], &cs_s[i]);
    __syncthreads();
    const int t = pos % kPage;
    // this lane's dims: below half, above it, or not rotated
    const bool rotated = 8 * l < p.rot, lo = 8 * l < half;
    float2 cs[4], sn[4];                             // sn with the sign that it has in this lane's sum
    if constexpr (kLanes) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = rotated ? 8 * l + 2 * i - (lo ? 0 : half) : 0;
            cs[i] = rotated ? make_float2(cs_s[d], cs_s[d + 1]) : make_float2(1.0f, 1.0f);
            sn[i] = rotated ? make_float2(sn_s[d], sn_s[d + 1]) : make_float2(0.0f, 0.0f);
            if (lo) sn[i] = make_float2(-sn[i].x, -sn[i].y);
        }
    }
    const int partner = lo ? lane + half / 8 : lane - half / 8;
    while (h0 - (lane >> 4) < heads) {
#pragma unroll
        for (int u = 0; u < kWriteUnroll; ++u) {
            const int h = h0 + u * stride;
            if (h - (lane >> 4) >= heads) break;     // for the whole warp: what follows shuffles
            const bool some = h < heads;
            uint4 xv = in[u];
            if constexpr (kLanes) {
                uint4 other;
                other.x = __shfl_sync(0xffffffffu, in[u].x, partner & 31);
                other.y = __shfl_sync(0xffffffffu, in[u].y, partner & 31);
                other.z = __shfl_sync(0xffffffffu, in[u].z, partner & 31);
                other.w = __shfl_sync(0xffffffffu, in[u].w, partner & 31);
                if (rotated && h < p.nq + p.nkv) {
                    auto rotate = [&](uint32_t mine, uint32_t theirs, int i) {
                        // one by one: packed products and their packed sum come out contracted
                        const float2 a = bf16_pair(mine), b = bf16_pair(theirs);
                        return pack_bf16(__fadd_rn(__fmul_rn(a.x, cs[i].x), __fmul_rn(b.x, sn[i].x)),
                                         __fadd_rn(__fmul_rn(a.y, cs[i].y), __fmul_rn(b.y, sn[i].y)));
                    };
                    xv = make_uint4(rotate(xv.x, other.x, 0), rotate(xv.y, other.y, 1), rotate(xv.z, other.z, 2),
                                    rotate(xv.w, other.w, 3));
                }
            } else if (some && h < p.nq + p.nkv) {
                const __nv_bfloat16* src = row + static_cast<size_t>(h) * kD;
                const __nv_bfloat16* ib = reinterpret_cast<const __nv_bfloat16*>(&in[u]);
                __nv_bfloat16* x = reinterpret_cast<__nv_bfloat16*>(&xv);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = 8 * l + e;
                    if (d < half) x[e] = __float2bfloat16_rn(rotate_lo(__bfloat162float(ib[e]), __bfloat162float(src[d + half]), cs_s[d], sn_s[d]));
                    else if (d < p.rot) x[e] = __float2bfloat16_rn(rotate_hi(__bfloat162float(src[d - half]), __bfloat162float(ib[e]), cs_s[d - half], sn_s[d - half]));
                }
            }
            if (some && h < p.nq) *reinterpret_cast<uint4*>(p.q_out + (static_cast<size_t>(b) * p.nq + h) * kD + 8 * l) = xv;
            if (h - (lane >> 4) + 1 < p.nq) continue;        // both heads of the warp are queries
            const bool is_k = h < p.nq + p.nkv;
            const int kvh = is_k ? h - p.nq : h - p.nq - p.nkv;
            const bool kv = some && h >= p.nq;
            if (kv && is_k && p.k_out) *reinterpret_cast<uint4*>(p.k_out + (static_cast<size_t>(b) * p.nkv + kvh) * kD + 8 * l) = xv;
            uint8_t* page = (is_k ? p.k_cache : p.v_cache) + (static_cast<size_t>(phys) * p.nkv + (kv ? kvh : 0)) * kPage4;
            quantise_store(xv, page, t, l, is_k, kv);
        }
        h0 += stride * kWriteUnroll;
        load();
    }
}

// ---------------------------------------------------------------- read

constexpr int kReadWarps = 8;
constexpr int kReadUnroll = 4;

// A warp per eight (K or V, head) tiles of a row, a half-warp per tile with 16
// bytes out a lane.
__global__ void __launch_bounds__(kReadWarps * 32)
kv4_read_kernel(const uint8_t* __restrict__ k_cache, const uint8_t* __restrict__ v_cache, int num_cache_pages,
                const int32_t* __restrict__ positions, const int32_t* __restrict__ row_seq, int num_seqs,
                const int32_t* __restrict__ page_table, int max_pages, int B, int nkv,
                __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int* __restrict__ error_word) {
    const int items = 2 * nkv;                       // K of every head, then V
    const int parts = (items + 2 * kReadUnroll - 1) / (2 * kReadUnroll);
    const int w = blockIdx.x * kReadWarps + (threadIdx.x >> 5);
    const int b = w / parts;
    if (b >= B) return;
    const int lane = threadIdx.x & 31, l = lane & 15;
    const int pos = positions[b];
    const int seq = seq_of_row(row_seq, b, num_seqs);
    int phys = -1, err = 0;
    if (seq < 0) err = 7;
    else if (pos < 0 || pos / kPage >= max_pages) err = 4;
    else {
        phys = page_table[static_cast<size_t>(seq) * max_pages + pos / kPage];
        if (phys < 0 || phys >= num_cache_pages) err = 6;
    }
    if (err && lane == 0 && error_word) atomicExch(error_word, err);
    const int t = err ? 0 : pos % kPage;
    const size_t page0 = static_cast<size_t>(err ? 0 : phys) * nkv * kPage4;
    {
        const int i0 = w % parts * 2 * kReadUnroll + (lane >> 4);
        uint32_t codes[kReadUnroll], scale[kReadUnroll];
#pragma unroll
        for (int u = 0; u < kReadUnroll; ++u) {
            const int i = i0 + 2 * u;
            const bool is_k = i < nkv;
            codes[u] = 0x88888888u;
            scale[u] = 0;
            if (i < items && !err && (is_k ? k_out : v_out)) {
                const uint8_t* page = (is_k ? k_cache : v_cache) + page0 + static_cast<size_t>(is_k ? i : i - nkv) * kPage4;
                if (is_k) codes[u] = *reinterpret_cast<const uint32_t*>(page + k_code_byte(t, 8 * l));
                else codes[u] = *reinterpret_cast<const uint16_t*>(page + v_code_byte(t, 8 * l)) |
                                static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(page + v_code_byte(t, 8 * l + 4))) << 16;
                scale[u] = *reinterpret_cast<const uint16_t*>(page + kCodes + (t * kGroups + l / 4) * 2);
            }
        }
#pragma unroll
        for (int u = 0; u < kReadUnroll; ++u) {
            const int i = i0 + 2 * u;
            const bool is_k = i < nkv;
            __nv_bfloat16* out = is_k ? k_out : v_out;
            if (i >= items || !out) continue;
            const float s = __uint_as_float(scale[u] << 16);
            __nv_bfloat16 x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = __float2bfloat16_rn(static_cast<float>(static_cast<int>((codes[u] >> (4 * e)) & 15u) - 8) * s);
            *reinterpret_cast<uint4*>(out + (static_cast<size_t>(b) * nkv + (is_k ? i : i - nkv)) * kD + 8 * l) =
                *reinterpret_cast<const uint4*>(x);
        }
    }
}

// ---------------------------------------------------------------- decode
//
// One CTA per (context split, row x kv head), four warps that take two pages at
// a time from bulk-copied rings of their own: codes to fragments with the fma of
// the file's head, S = Q K^T and O += P V on mma.sync with the group's query
// heads as M, one online softmax whose maximum is left behind by up to 2^8.
// mma.sync, because its B fragments are registers: a code goes from the ring to
// the tensor core without a way back through shared memory.  On tcgen05 the same
// holds with the page's tokens and dims as M and the heads as N, the unpacked page
// being the operand in TMEM; that form has not been built.
//
// Bound by what a page costs to unpack, not by its bytes: 366 instructions a page
// and KV head, a third of them shifts and masks; the ALU pipe is 52 % busy, the
// tensor pipe 38 %, and three CTAs (168 registers) leave a scheduler under three
// warps.  Measured (B200, device time): 64 contexts of up to 16384, 64 heads on 8
// KV heads, 169 us or 3.2 TB/s of pages; 64 of up to 32768, 12 heads, 53 us or
// 2.5 TB/s, the merge and uneven lengths in it; 16 of up to 8191, 96
// heads, 31 us; one of 32768, 10 us; the e4m3 rows add under 1 us.  Slower: four CTAs of 128 registers, shifts as
// multiplications, scores of the next pair under this one's softmax.

constexpr int kWarps = 4;
constexpr int kNst = 3;                                   // page pairs in flight per warp
constexpr int kTile = 2 * kPage4;                         // K and V of one page
constexpr int kStage = 2 * kTile;
constexpr int kMaxSplitPages = 512;                       // split_tokens <= 8192
constexpr int kMergePad = kD + 4;
constexpr size_t kRingBytes = static_cast<size_t>(kWarps) * kNst * kStage;
constexpr size_t kQFragBytes = kD / 16 * 32 * 16;
constexpr size_t kDecodeSmem = kRingBytes + kMaxSplitPages * 4 + kQFragBytes;
constexpr uint64_t kWaitNs = 2000000000ull;
// the warp merge reuses the rings: per warp 16 x 128 fp32, then (m, l) and factors of its rows
static_assert(static_cast<size_t>(kWarps) * kGPad * (kMergePad + 3) * 4 + kGPad * 8 <= kRingBytes, "merge scratch fits the rings");

struct Kv4Params {
    const __nv_bfloat16* q;
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const int32_t* page_table;
    const int32_t* row_seq;
    const int32_t* seq_lens;
    float* part_o;                 // [B * nkv][max_splits][G][128]
    float* part_ml;                // [B * nkv][max_splits][G][2]
    int* error_word;
    __nv_bfloat16* out;            // [B][nq][128]
    uint8_t* out_q;
    float* out_s;
    int out_ld;
    int nq, nkv, G, max_pages, num_cache_pages, split_tokens, max_splits, num_seqs;
    float scale_log2;              // at least FLT_MIN: a sign is taken by the queries
    uint32_t q_flip;               // 0x80008000 for a negative scale
};

__device__ __forceinline__ int clamp_len(int len, int max_pages, int split_tokens, int max_splits) {
    const long long cap = min(static_cast<long long>(max_pages) * kPage, static_cast<long long>(max_splits) * split_tokens);
    return len < 0 ? 0 : (len > cap ? static_cast<int>(cap) : len);
}

__device__ __forceinline__ uint32_t bf2_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// mma_bf16 for the compiler to place: nothing here depends on its order
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
constexpr uint32_t kMinus136 = 0xC308C308u;   // bf16x2

// The codes at nibble i of both halves of w as the bf16 pair 136 + n, one lop3
// after the shift.  `magic` is 0x43004300 in a register: as an immediate beside
// the mask it would take a second lop3.
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int i, uint32_t magic) {
    uint32_t d;
    asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(d) : "r"(w >> (4 * i)), "r"(magic));
    return d;
}

// One output row (128 threads, one dim each): bf16, and e4m3 with its scale.
__device__ __forceinline__ void write_row(const Kv4Params& p, int b, int h, float v, float* red) {
    const int d = threadIdx.x;
    p.out[(static_cast<size_t>(b) * p.nq + h) * kD + d] = __float2bfloat16_rn(v);
    if (p.out_q) {
        float a = fabsf(v);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        named_bar_sync(1, kD);
        if ((d & 31) == 0) red[d >> 5] = a;
        named_bar_sync(1, kD);
        const float amax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const E4m3Row r = e4m3_row(amax);
        p.out_q[(static_cast<size_t>(b) * p.nq + h) * kD + d] = static_cast<uint8_t>(cvt_e4m3x2(v * r.up * r.inv, 0.0f) & 0xFFu);
        if (d == 0) p.out_s[static_cast<size_t>(h) * p.out_ld + b] = r.scale;
    }
}

__global__ void __launch_bounds__(kWarps * 32, 3)
kv4_decode_kernel(const Kv4Params p) {
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ uint64_t full[kWarps][kNst];
    __shared__ int abort_s;
    __shared__ float red[kWarps];
    const int split = blockIdx.x;
    const int bk = blockIdx.y;
    const int b = bk / p.nkv, kvh = bk % p.nkv;
    const int seq = seq_of_row(p.row_seq, b, p.num_seqs);
    if (seq < 0 && split == 0 && threadIdx.x == 0 && kvh == 0 && p.error_word) atomicExch(p.error_word, 7);
    const int t0 = split * p.split_tokens;
    const int page0 = t0 / kPage;
    // the split's first page ids come with the length, not after it
    const int32_t* ptb = p.page_table + static_cast<size_t>(max(seq, 0)) * p.max_pages + page0;
    const int split_pages = min(p.split_tokens / kPage, p.max_pages - page0);
    int first_id = static_cast<int>(threadIdx.x) < split_pages ? ptb[threadIdx.x] : -1;
    const int len_in = seq < 0 ? 0 : p.seq_lens[b];
    const int len = clamp_len(len_in, p.max_pages, p.split_tokens, p.max_splits);
    if (len < len_in && split == 0 && threadIdx.x == 0 && kvh == 0 && p.error_word) atomicExch(p.error_word, 5);
    if (t0 >= len) {
        if (p.max_splits == 1)                     // there is no merge kernel: an empty row's zeros
            for (int r = 0; r < p.G; ++r) write_row(p, b, kvh * p.G + r, 0.0f, red);
        return;
    }
    const int t1 = min(t0 + p.split_tokens, len);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tq = lane & 3;

    uint8_t* ring = sm + static_cast<size_t>(warp) * kNst * kStage;
    int* pid_s = reinterpret_cast<int*>(sm + kRingBytes);
    const int npages = (t1 - 1) / kPage - page0 + 1;
    bool bad = false;                              // an id outside the cache
    for (int i = threadIdx.x; i < npages; i += blockDim.x) {
        const int phys = i == static_cast<int>(threadIdx.x) ? first_id : ptb[i];
        const bool ok = phys >= 0 && phys < p.num_cache_pages;
        if (!ok && p.error_word) atomicExch(p.error_word, 6);
        pid_s[i] = ok ? phys : -1;
        bad |= !ok;
    }
    if (lane < kNst) mbar_init(&full[warp][lane], 1);
    if (threadIdx.x == 0) abort_s = 0;
    fence_mbar_init();
    // Query fragments: MMA k-step 2j + u takes dims 32 j + 8 tq + {2u, 2u + 4, 2u + 1, 2u + 5} at this lane's
    // four contraction indices, the order the K codes unpack in.
    uint4* qf_s = reinterpret_cast<uint4*>(sm + kRingBytes + kMaxSplitPages * 4);   // [k-step][lane]
    if (warp == 0) {
        uint32_t qa[kD / 16][4];
        const __nv_bfloat16* q0 = p.q + (static_cast<size_t>(b) * p.nq + kvh * p.G) * kD;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h;
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r < p.G) v = *reinterpret_cast<const uint4*>(q0 + static_cast<size_t>(r) * kD + 32 * j + 8 * tq);
                v.x ^= p.q_flip; v.y ^= p.q_flip; v.z ^= p.q_flip; v.w ^= p.q_flip;
                // v: dims 0 1 | 2 3 | 4 5 | 6 7
                qa[2 * j][h] = __byte_perm(v.x, v.z, 0x5410);          // 0, 4
                qa[2 * j][2 + h] = __byte_perm(v.x, v.z, 0x7632);      // 1, 5
                qa[2 * j + 1][h] = __byte_perm(v.y, v.w, 0x5410);      // 2, 6
                qa[2 * j + 1][2 + h] = __byte_perm(v.y, v.w, 0x7632);  // 3, 7
            }
        }
#pragma unroll
        for (int ks = 0; ks < kD / 16; ++ks) qf_s[ks * 32 + lane] = make_uint4(qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3]);
    }
    const bool whole = !__syncthreads_or(bad);
    grid_dependents_launch();                      // the merge may take its places; it waits for this grid's end

    // Pairs of pages, dealt to the warps in turn.
    const int npairs = (npages + 1) / 2;
    const uint8_t* cache = ((lane & 1) ? p.v_cache : p.k_cache) + static_cast<size_t>(kvh) * kPage4;
    const size_t page_stride = static_cast<size_t>(p.nkv) * kPage4;
    const int mine = npairs > warp ? (npairs - warp + kWarps - 1) / kWarps : 0;
    // Lanes 0-3 copy K and V of the pair's two pages.  A page that is not there (none behind the last, or an id outside
    // the cache) reads as zeros: scales of 0.
    auto load_pair = [&](int i, int stage) {
        uint8_t* dst = ring + stage * kStage;
        const int at = 2 * (warp + i * kWarps);
        if (whole && at + 1 < npages) {
            if (lane == 0) mbar_arrive_expect_tx(&full[warp][stage], kStage);
            __syncwarp();
            if (lane < 4)
                bulk_load(dst + lane * kPage4, cache + static_cast<size_t>(pid_s[at + (lane >> 1)]) * page_stride, kPage4,
                          &full[warp][stage]);
            return;
        }
        const int id = lane < 4 && at + (lane >> 1) < npages ? pid_s[at + (lane >> 1)] : -1;
        const uint32_t some = __ballot_sync(0xffffffffu, id >= 0);
        if (lane == 0) mbar_arrive_expect_tx(&full[warp][stage], __popc(some) * kPage4);
        for (int c = 0; c < 4; ++c)
            if (!(some >> c & 1))
                for (int o = lane; o < kPage4 / 16; o += 32)
                    *reinterpret_cast<uint4*>(dst + c * kPage4 + o * 16) = make_uint4(0, 0, 0, 0);
        // a later pair's bulk copy into this stage comes after the zeros
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (id >= 0) bulk_load(dst + lane * kPage4, cache + static_cast<size_t>(id) * page_stride, kPage4, &full[warp][stage]);
    };

    uint32_t magic;
    asm volatile("mov.u32 %0, 0x43004300;" : "=r"(magic));
    float o[kD / 8][4];
#pragma unroll
    for (int i = 0; i < kD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m_r[2] = {-INFINITY, -INFINITY}, top_r[2] = {-INFINITY, -INFINITY}, nm_r[2] = {0.0f, 0.0f};
    float2 l_r[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
    const float lag = 8.0f / p.scale_log2;         // of raw scores

    for (int s = 0; s < kNst - 1 && s < mine; ++s) load_pair(s, s);
    // One pair out of stage `st`; `partial` where only `valid` of its tokens are inside the split (the last pair).
    auto attend = [&](const uint8_t* st, const int valid, auto partial) {
        // S = Q K^T, four tiles of eight tokens side by side: an MMA's result is not waited for by the next
        float s[4][4];
        uint4 kc[4];
        uint2 ks[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint8_t* kt = st + (n >> 1) * kTile;
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
            kc[n] = *reinterpret_cast<const uint4*>(kt + (g + 8 * (n & 1)) * 64 + tq * 16);
            ks[n] = *reinterpret_cast<const uint2*>(kt + kCodes + (g + 8 * (n & 1)) * 8);
        }
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                // volatile: a fragment is read where it is used, not held over the whole loop
                uint32_t qa[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(qa[0]), "=r"(qa[1]), "=r"(qa[2]), "=r"(qa[3])
                             : "r"(smem_u32(qf_s + (2 * j + u) * 32 + lane)));
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t w = j == 0 ? kc[n].x : j == 1 ? kc[n].y : j == 2 ? kc[n].z : kc[n].w;
                    const uint32_t s2 = __byte_perm(j < 2 ? ks[n].x : ks[n].y, 0, (j & 1) ? 0x3232 : 0x1010);
                    const uint32_t c2 = bf2_mul(s2, kMinus136);
                    mma(s[n], qa, bf2_fma(code_pair(w, 2 * u, magic), s2, c2),
                        bf2_fma(code_pair(w, 2 * u + 1, magic), s2, c2));
                }
            }
        if constexpr (partial.value) {
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (8 * n + 2 * tq + (e & 1) >= valid) s[n][e] = -INFINITY;
        }
        // the maximum moves when a score passes it by 8 in log2 units; only then do the lanes of a row compare theirs
        float mx[2];
        bool need = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(s[0][2 * h], s[0][2 * h + 1]);
#pragma unroll
            for (int n = 1; n < 4; ++n) mx[h] = fmaxf(mx[h], fmaxf(s[n][2 * h], s[n][2 * h + 1]));
            need |= mx[h] > top_r[h];
        }
        if (__any_sync(0xffffffffu, need)) {
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                const float mn = fmaxf(m_r[h], mx[h]);
                f[h] = mn == m_r[h] ? 1.0f : ex2((m_r[h] - mn) * p.scale_log2);
                m_r[h] = mn;
                top_r[h] = mn + lag;
                nm_r[h] = mn == -INFINITY ? 0.0f : -mn * p.scale_log2;     // nothing but -inf yet: weights 0, not NaN
                l_r[h].x *= f[h];
                l_r[h].y *= f[h];
            }
#pragma unroll
            for (int nd = 0; nd < kD / 8; ++nd) {
                o[nd][0] *= f[0]; o[nd][1] *= f[0];
                o[nd][2] *= f[1]; o[nd][3] *= f[1];
            }
        }
        // P is rounded to bf16, as the bf16 pages' decode rounds it (2^-8 of each weight at most); l sums the fp32 weights
        uint32_t pa[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                float2 x = ffma2(make_float2(s[n][2 * h], s[n][2 * h + 1]), make_float2(p.scale_log2, p.scale_log2),
                                 make_float2(nm_r[h], nm_r[h]));
                x.x = ex2(x.x);
                x.y = ex2(x.y);
                l_r[h] = fadd2(l_r[h], x);
                pa[n >> 1][(n & 1) * 2 + h] = pack_bf16(x.x, x.y);
            }
        // O += P V, page by page: tokens 2 tq, 2 tq + 1 of its halves a = 0 and 1
#pragma unroll
        for (int pg = 0; pg < 2; ++pg) {
            const uint8_t* vt = st + pg * kTile + kPage4;
            uint4 vc[2], vs[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                vc[a] = *reinterpret_cast<const uint4*>(vt + a * 512 + lane * 16);
                vs[a] = *reinterpret_cast<const uint4*>(vt + kCodes + (8 * a + 2 * tq) * 8);
                if constexpr (partial.value) {                     // a slot past the end may hold anything: weight 0 times value 0
                    const int t = 16 * pg + 8 * a + 2 * tq;
                    if (t >= valid) vs[a].x = vs[a].y = 0;
                    if (t + 1 >= valid) vs[a].z = vs[a].w = 0;
                }
            }
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                uint32_t w[2], s2[2], c2[2];
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const uint32_t sel = (j & 1) ? 0x7632 : 0x5410;
                    w[a] = __byte_perm(j < 2 ? vc[a].x : vc[a].y, j < 2 ? vc[a].z : vc[a].w, sel);
                    s2[a] = __byte_perm(j < 2 ? vs[a].x : vs[a].y, j < 2 ? vs[a].z : vs[a].w, sel);
                    c2[a] = bf2_mul(s2[a], kMinus136);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    mma(o[4 * j + u], pa[pg], bf2_fma(code_pair(w[0], u, magic), s2[0], c2[0]),
                             bf2_fma(code_pair(w[1], u, magic), s2[1], c2[1]));
            }
        }
    };

    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < mine; ++i) {
        if (i + kNst - 1 < mine) load_pair(i + kNst - 1, stage == 0 ? kNst - 1 : stage - 1);
        if (!__all_sync(0xffffffffu, mbar_try_wait(&full[warp][stage], phase)) &&
            !__all_sync(0xffffffffu, mbar_wait_bounded(&full[warp][stage], phase, &abort_s, kWaitNs))) {
            if (p.error_word) atomicExch(p.error_word, 1);
            // the copies in flight get the same time once more before the rings are reused
            const uint64_t begin = globaltimer_ns();
            for (int k = i; k < mine && k < i + kNst; ++k) {
                while (!mbar_try_wait(&full[warp][stage], phase) && globaltimer_ns() - begin < kWaitNs) {}
                if (++stage == kNst) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            break;
        }
        const uint8_t* st = ring + stage * kStage;
        const int valid = t1 - (page0 + 2 * (warp + i * kWarps)) * kPage;   // tokens of the pair inside the split, at least 1
        if (valid < 2 * kPage) attend(st, valid, std::true_type());
        else attend(st, valid, std::false_type());
        __syncwarp();                              // the stage is read
        if (++stage == kNst) {
            stage = 0;
            phase ^= 1;
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l_r[h].x += l_r[h].y;
        l_r[h].x += __shfl_xor_sync(0xffffffffu, l_r[h].x, 1);
        l_r[h].x += __shfl_xor_sync(0xffffffffu, l_r[h].x, 2);
        m_r[h] *= p.scale_log2;                    // from here on in log2 units (-inf stays)
    }
    __syncthreads();   // every warp is done with its ring: reuse as merge scratch
    float* mo = reinterpret_cast<float*>(sm);                       // [warp][16][kMergePad]
    float* mml = mo + kWarps * kGPad * kMergePad;                   // [16][warp][2]
    float* fac = mml + kWarps * kGPad * 2;                          // [16][warp] factors, then [16][2] the split's (m, l)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h;
        float* ow = mo + (warp * kGPad + r) * kMergePad;
        // output tile 4 j + u, column c is dim 32 j + 4 c + u
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                *reinterpret_cast<float4*>(ow + 32 * j + 8 * tq + 4 * e) =
                    make_float4(o[4 * j][2 * h + e], o[4 * j + 1][2 * h + e], o[4 * j + 2][2 * h + e], o[4 * j + 3][2 * h + e]);
        if (tq == 0) *reinterpret_cast<float2*>(mml + (r * kWarps + warp) * 2) = make_float2(m_r[h], l_r[h].x);
    }
    __syncthreads();
    if (threadIdx.x < kGPad) {
        const int r = threadIdx.x;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, mml[(r * kWarps + w) * 2]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float mw = mml[(r * kWarps + w) * 2];
            const float f = mw == -INFINITY ? 1.0f : ex2(mw - M);   // no weight yet: l and o are 0 or NaN
            fac[r * kWarps + w] = f;
            L += mml[(r * kWarps + w) * 2 + 1] * f;
        }
        fac[kGPad * kWarps + r * 2] = M;
        fac[kGPad * kWarps + r * 2 + 1] = L;
    }
    __syncthreads();
    const size_t base = (static_cast<size_t>(bk) * p.max_splits + split) * p.G;
    const int d = threadIdx.x;
    for (int r = 0; r < p.G; ++r) {
        const float4 f = *reinterpret_cast<const float4*>(fac + r * kWarps);
        const float* mr = mo + r * kMergePad + d;
        const float acc = mr[0] * f.x + mr[kGPad * kMergePad] * f.y + mr[2 * kGPad * kMergePad] * f.z + mr[3 * kGPad * kMergePad] * f.w;
        if (p.max_splits == 1) {
            write_row(p, b, kvh * p.G + r, (acc + 0.0f) / fac[kGPad * kWarps + r * 2 + 1], red);   // -0 as the merge's sum has it
        } else {
            p.part_o[(base + r) * kD + d] = acc;
            if (d < 2) p.part_ml[(base + r) * 2 + d] = fac[kGPad * kWarps + r * 2 + d];
        }
    }
}

// Merge of a (row, query head)'s splits: sum g of kSums takes splits g, g + kSums,
// ... in turns of kMergeTurn, and the sums are added in order.  Where there are few
// rows, each sum has 128 threads of its own, one per dim, so that many splits are
// a few loads deep; where the rows fill the GPU, the same threads hold all sums.
// The steps are the same in both, so a row's bits do not tell which it was.  An
// octet of lanes works out the factors of a sum's turn, every warp for itself, and
// the partials' loads wait for nothing but the length.
constexpr int kSums = 4;
constexpr int kMergeTurn = 8;
template <int kGroups>
__global__ void __launch_bounds__(kGroups * kD)
kv4_merge_kernel(const Kv4Params p) {
    static_assert(kGroups == 1 || kGroups == kSums, "a thread holds one sum or all");
    constexpr int kOwn = kSums / kGroups;
    __shared__ float red[kWarps], sum[kGroups][kD + 2];
    const int b = blockIdx.x / p.nq, h = blockIdx.x % p.nq;
    const int kvh = h / p.G, r = h % p.G;
    const int d = threadIdx.x % kD, grp = threadIdx.x / kD, lane = threadIdx.x & 31;
    const int len = seq_of_row(p.row_seq, b, p.num_seqs) < 0
                        ? 0 : clamp_len(p.seq_lens[b], p.max_pages, p.split_tokens, p.max_splits);
    const int ns = (len + p.split_tokens - 1) / p.split_tokens;
    const size_t base = (static_cast<size_t>(b) * p.nkv + kvh) * p.max_splits * p.G + r;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + base;
    const float* po = p.part_o + base * kD + d;
    const int lane_sum = kGroups == 1 ? lane / kMergeTurn : grp;
    grid_dependency_wait();                        // the splits
    float M = -INFINITY, L = 0.0f, acc[kOwn];      // M and L of lane_sum, acc of sums grp ..
#pragma unroll
    for (int u = 0; u < kOwn; ++u) acc[u] = 0.0f;
    float2 x;
    float v[kOwn][kMergeTurn];
    auto load = [&](int s0) {
        const int mine = s0 + lane_sum + lane % kMergeTurn * kSums;
        x = mine < ns ? ml[static_cast<size_t>(mine) * p.G] : make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int c = 0; c < kMergeTurn; ++c) {
            if (kOwn > 1 && s0 + c * kSums >= ns) break;
#pragma unroll
            for (int u = 0; u < kOwn; ++u) {
                const int s = s0 + grp + u + c * kSums;
                v[u][c] = s < ns ? po[static_cast<size_t>(s) * p.G * kD] : 0.0f;
            }
        }
    };
    // A lone sum's next turn is on its way under this one (one context of 32768: 10.3 us instead of 10.9); with all sums in a
    // thread that costs registers, and with them blocks (64 contexts of up to 16384, 64 heads: 171.5 us instead of 169.6).
    constexpr bool kAhead = kOwn == 1;
    if (kAhead) load(0);
    for (int s0 = 0; s0 + grp < ns; s0 += kSums * kMergeTurn) {
        if (!kAhead) load(s0);
        const float2 x0 = x;
        float v0[kOwn][kMergeTurn];
#pragma unroll
        for (int u = 0; u < kOwn; ++u)
#pragma unroll
            for (int c = 0; c < kMergeTurn; ++c) v0[u][c] = v[u][c];
        if (kAhead && s0 + kSums * kMergeTurn < ns) load(s0 + kSums * kMergeTurn);
        float m = x0.x;
#pragma unroll
        for (int o = kMergeTurn / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float mn = fmaxf(M, m);
        const float keep = M == -INFINITY ? 1.0f : ex2(M - mn);
        const float f = x0.x == -INFINITY ? 1.0f : ex2(x0.x - mn);   // no weight: l and o are 0 or NaN
        float l = __fmul_rn(x0.y, f);
#pragma unroll
        for (int o = kMergeTurn / 2; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        L = fmaf(L, keep, l);
        M = mn;
#pragma unroll
        for (int u = 0; u < kOwn; ++u) acc[u] *= __shfl_sync(0xffffffffu, keep, u * kMergeTurn);
#pragma unroll
        for (int c = 0; c < kMergeTurn; ++c) {
            if (s0 + grp + c * kSums >= ns) break;
#pragma unroll
            for (int u = 0; u < kOwn; ++u) acc[u] = fmaf(v0[u][c], __shfl_sync(0xffffffffu, f, u * kMergeTurn + c), acc[u]);
        }
    }
    if constexpr (kGroups > 1) {
        sum[grp][d] = acc[0];
        if (d == 0) {
            sum[grp][kD] = M;
            sum[grp][kD + 1] = L;
        }
        __syncthreads();
        if (grp) return;
    }
    float Ms[kSums], top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int g = 0; g < kSums; ++g) {
        if constexpr (kGroups > 1) Ms[g] = sum[g][kD];
        else Ms[g] = __shfl_sync(0xffffffffu, M, g * kMergeTurn);
        top = fmaxf(top, Ms[g]);
    }
    float Lt = 0.0f;
#pragma unroll
    for (int g = 0; g < kSums; ++g) {
        const float f = Ms[g] == -INFINITY ? 1.0f : ex2(Ms[g] - top);
        if constexpr (kGroups > 1) {
            total = fmaf(sum[g][d], f, total);
            Lt = fmaf(sum[g][kD + 1], f, Lt);
        } else {
            total = fmaf(acc[g], f, total);
            Lt = fmaf(__shfl_sync(0xffffffffu, L, g * kMergeTurn), f, Lt);
        }
    }
    write_row(p, b, h, ns > 0 ? total / Lt : 0.0f, red);
}

}  // namespace

extern "C" {

size_t attn_kv4_page_bytes(int nkv) { return nkv > 0 ? static_cast<size_t>(nkv) * kPage4 : 0; }

moe_status_t attn_kv4_rope_write_rows(const void* qkv_bf16, int B, int nq, int nkv, int head_dim, int rot,
                                      const float* inv_freq, const int32_t* positions, const int32_t* row_seq,
                                      int num_seqs, const int32_t* page_table, int max_pages, int page_size,
                                      int num_cache_pages, void* q_out_bf16, void* k_out_bf16, void* k_cache,
                                      void* v_cache, int32_t* seq_lens_out, int* error_word, cwStream_t stream) {
    if (B < 0 || nq <= 0 || nkv <= 0 || nq % nkv || head_dim != kD || page_size != kPage) return MOE_ERR_INVALID_ARGUMENT;
    if (num_cache_pages <= 0 || rot < 0 || rot > kD || rot % 2 || max_pages <= 0) return MOE_ERR_INVALID_ARGUMENT;
    if (B == 0) return MOE_OK;
    if (num_seqs <= 0) return MOE_ERR_INVALID_ARGUMENT;
    if (!qkv_bf16 || (rot > 0 && !inv_freq) || !positions || !page_table || !q_out_bf16 || !k_cache || !v_cache)
        return MOE_ERR_INVALID_ARGUMENT;
    if (!a16(qkv_bf16) || !a16(q_out_bf16) || !a16(k_out_bf16) || !a16(k_cache) || !a16(v_cache))
        return MOE_ERR_INVALID_ARGUMENT;
    WriteParams p;
    p.qkv = static_cast<const __nv_bfloat16*>(qkv_bf16);
    p.inv_freq = inv_freq;
    p.positions = positions;
    p.row_seq = row_seq;
    p.page_table = page_table;
    p.q_out = static_cast<__nv_bfloat16*>(q_out_bf16);
    p.k_out = static_cast<__nv_bfloat16*>(k_out_bf16);
    p.k_cache = static_cast<uint8_t*>(k_cache);
    p.v_cache = static_cast<uint8_t*>(v_cache);
    p.seq_lens_out = seq_lens_out;
    p.error_word = error_word;
    p.nq = nq;
    p.nkv = nkv;
    p.rot = rot;
    p.num_seqs = num_seqs;
    p.max_pages = max_pages;
    p.num_cache_pages = num_cache_pages;
    // a row's heads over as many blocks as it takes to fill the GPU (four blocks an SM), each warp at least one pair
    const int most = (nq + 2 * nkv + 2 * kWriteWarps - 1) / (2 * kWriteWarps);
    const int want = (4 * 148 + B - 1) / B;
    const dim3 grid(B, want < most ? want : most < 65535 ? most : 65535);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rot % 16 == 0) kv4_rope_write_kernel<true><<<grid, kWriteWarps * 32, 0, st>>>(p);
    else kv4_rope_write_kernel<false><<<grid, kWriteWarps * 32, 0, st>>>(p);
    return launch_status();
}

moe_status_t attn_kv4_read_rows(const void* k_cache, const void* v_cache, int num_cache_pages,
                                const int32_t* positions, const int32_t* row_seq, int num_seqs,
                                const int32_t* page_table, int max_pages, int page_size, int B, int nkv, int head_dim,
                                void* k_out_bf16, void* v_out_bf16, int* error_word, cwStream_t stream) {
    if (B < 0 || nkv <= 0 || head_dim != kD || page_size != kPage || num_cache_pages <= 0 || max_pages <= 0)
        return MOE_ERR_INVALID_ARGUMENT;
    if (B == 0 || (!k_out_bf16 && !v_out_bf16)) return MOE_OK;
    if (num_seqs <= 0) return MOE_ERR_INVALID_ARGUMENT;
    if (!positions || !page_table || (k_out_bf16 && !k_cache) || (v_out_bf16 && !v_cache)) return MOE_ERR_INVALID_ARGUMENT;
    if (!a16(k_cache) || !a16(v_cache) || !a16(k_out_bf16) || !a16(v_out_bf16)) return MOE_ERR_INVALID_ARGUMENT;
    const long long warps = static_cast<long long>(B) * ((2ll * nkv + 2 * kReadUnroll - 1) / (2 * kReadUnroll));
    if (warps > 0x7FFFFFFF - kReadWarps) return MOE_ERR_UNSUPPORTED;
    kv4_read_kernel<<<static_cast<int>((warps + kReadWarps - 1) / kReadWarps), kReadWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), num_cache_pages, positions, row_seq,
        num_seqs, page_table, max_pages, B, nkv, static_cast<__nv_bfloat16*>(k_out_bf16),
        static_cast<__nv_bfloat16*>(v_out_bf16), error_word);
    return launch_status();
}

int attn_kv4_split_tokens(int B, int nkv, int max_context) {
    if (B <= 0 || nkv <= 0 || max_context <= 0) return kPage;
    // One CTA's fixed cost is that of about 14 pages (4 us beside 0.27 us a page, 3 CTAs an SM).  One wave of the 444
    // CTAs at half the longest context, as long as that leaves splits of 256 to 1536 tokens; longer contexts go in two
    // waves or more, which even out uneven lengths (64 rows up to 32K: 2048 tokens 65 us, 1184 59 us).  A context that one
    // split of 512 tokens holds needs no merge.  max_context is what a caller has room for: where its contexts are far
    // shorter, few CTAs get the work (one row of 4096 tokens, 8 KV heads: 8.7 us, and 18.3 with max_context 131072).
    if (max_context <= 512) return (max_context + kPage - 1) / kPage * kPage;
    long long split = static_cast<long long>(B) * nkv * max_context / (2 * 444);
    if (split > 1536) split = split / 2 < 2048 ? split / 2 : 2048;
    constexpr int kTurn = 2 * kPage * kWarps;      // a page pair for every warp
    split = (split + kTurn / 2) / kTurn * kTurn;
    return static_cast<int>(split < 2 * kTurn ? 2 * kTurn : split);
}

size_t attn_kv4_decode_workspace_bytes(int B, int nq, int max_splits) {
    if (B <= 0 || nq <= 0 || max_splits <= 0) return 0;
    return static_cast<size_t>(B) * nq * max_splits * (kD + 2) * sizeof(float);
}

moe_status_t attn_kv4_decode_rows(const void* q_bf16, const void* k_cache, const void* v_cache, int num_cache_pages,
                                  const int32_t* page_table, int max_pages, const int32_t* row_seq, int num_seqs,
                                  const int32_t* seq_lens, int B, int nq, int nkv, int head_dim, int page_size,
                                  float scale, int split_tokens, int max_splits, void* workspace,
                                  size_t workspace_bytes, void* out_bf16, void* out_q, float* out_s, int out_ld,
                                  int* error_word, cwStream_t stream) {
    if (B < 0 || nq <= 0 || nkv <= 0 || nq % nkv || nq / nkv > kGPad || head_dim != kD ||
        page_size != kPage)
        return MOE_ERR_INVALID_ARGUMENT;
    if (split_tokens <= 0 || split_tokens % kPage || split_tokens > kMaxSplitPages * kPage || max_splits <= 0 ||
        max_pages <= 0 || num_cache_pages <= 0 || !std::isfinite(scale * kLog2e))
        return MOE_ERR_INVALID_ARGUMENT;
    if (static_cast<long long>(B) * nkv > 65535 || static_cast<long long>(B) * nq > 0x7FFFFFFF) return MOE_ERR_UNSUPPORTED;
    // positions are 32-bit numbers, one split behind the last included
    if (static_cast<long long>(max_splits) * split_tokens > 0x7FFFFFFF - kMaxSplitPages * kPage) return MOE_ERR_UNSUPPORTED;
    if (B == 0) return MOE_OK;
    if (num_seqs <= 0) return MOE_ERR_INVALID_ARGUMENT;
    if (!q_bf16 || !k_cache || !v_cache || !page_table || !seq_lens || !workspace || !out_bf16)
        return MOE_ERR_INVALID_ARGUMENT;
    if (!a16(q_bf16) || !a16(k_cache) || !a16(v_cache) || !a16(workspace)) return MOE_ERR_INVALID_ARGUMENT;
    if (out_q && (!out_s || out_ld < B)) return MOE_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < attn_kv4_decode_workspace_bytes(B, nq, max_splits)) return MOE_ERR_WORKSPACE;
    static bool attr[kMaxDevices] = {};
    if (smem_optin_once(kv4_decode_kernel, static_cast<int>(kDecodeSmem), attr) != cudaSuccess) return MOE_ERR_CUDA;
    Kv4Params p;
    p.q = static_cast<const __nv_bfloat16*>(q_bf16);
    p.k_cache = static_cast<const uint8_t*>(k_cache);
    p.v_cache = static_cast<const uint8_t*>(v_cache);
    p.page_table = page_table;
    p.row_seq = row_seq;
    p.seq_lens = seq_lens;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = p.part_o + static_cast<size_t>(B) * nq * max_splits * kD;
    p.error_word = error_word;
    p.nq = nq;
    p.nkv = nkv;
    p.G = nq / nkv;
    p.max_pages = max_pages;
    p.num_cache_pages = num_cache_pages;
    p.split_tokens = split_tokens;
    p.max_splits = max_splits;
    p.num_seqs = num_seqs;
    p.out = static_cast<__nv_bfloat16*>(out_bf16);
    p.out_q = static_cast<uint8_t*>(out_q);
    p.out_s = out_s;
    p.out_ld = out_ld;
    p.q_flip = scale < 0.0f ? 0x80008000u : 0u;
    p.scale_log2 = fmaxf(fabsf(scale * kLog2e), 1.17549435e-38f);   // 0: every finite score alike, masked ones still -inf
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    kv4_decode_kernel<<<dim3(max_splits, B * nkv), kWarps * 32, kDecodeSmem, st>>>(p);
    const moe_status_t s = launch_status();
    if (s != MOE_OK || max_splits == 1) return s;
    const cudaError_t e = B * nq < 4 * 148 ? launch_dependent(kv4_merge_kernel<kSums>, B * nq, kSums * kD, st, p)
                                           : launch_dependent(kv4_merge_kernel<1>, B * nq, kD, st, p);
    return e == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

}  // extern "C"
