// attn_prompt.cu -- causal attention over whole prompts in packed rows
// (attn_prompt_packed in include/attn_block.h).
//
// The query heads of one KV head's group at 256 / G consecutive positions are
// the rows of a tile, position-major, so a tile spans few positions: little of a
// diagonal tile is masked, a short prompt fills a tile with its heads, and Q
// comes in one TMA box.  Tiles are taken in the order of the keys they attend,
// most first, by a search over the sequence bounds in each CTA: nothing is
// planned on the host.
//
// Bound: the tensor pipe, 4 * 128 * nq * sum of L (L + 1) / 2 operations over
// the lengths L.  Measured (B200, device time): one prompt of 16384 tokens, 12 query
// heads on one KV head, 632 us or 1300 TFLOP/s in a short run and 722 us or 1140 in
// a long one, where the power limit sets the clock; one of 4096 with 96 heads on 8
// KV heads, 399 us or 1030, and four of 1024, 123-143 us, after those; seven of up to
// 1201, 95 us or 800: a CTA has nine tiles there, and first and last steps take
// longer than those between; 24 of up to 201, 12 heads, 9.8 us: under one wave,
// launch, first loads, four steps and output in a row.  With the e4m3 rows 734, 110
// and 10.8 us for the first, the seven and the 24.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
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
    int tile_pos;                  // positions of a tile
    float scale_log2;
    bool flip_q;                   // a negative scale: its sign is taken by the queries
};

struct Tile {
    int first, len;                // rows [first, first + len) are the sequence's
    int index;                     // tile of the sequence
    bool some;
};

// Tiles of `span` positions in the order of (tile index, descending; sequence),
// asked for in ascending numbers by one warp.  From the first bound that is out
// of order or range on there are no sequences, so no two overlap.  Up to 32
// sequences are counted in registers and a tile is found by bisection over the
// indices; more are walked 32 at a time from the last tile found, so that the
// whole run walks each index's sequences once.
struct TileOrder {
    const PromptParams& p;
    int span, lane, seqs;          // positions of a tile; sequences
    int own;                       // tiles of sequence `lane`
    int most;                      // tiles of the longest sequence
    int level, s0;                 // walk: tile index and first of the 32 sequences looked at,
    unsigned int before;           // and the tiles that come before them

    __device__ __forceinline__ int tiles(int s) const {
        return s < seqs ? (p.cu_seqlens[s + 1] - p.cu_seqlens[s] + span - 1) / span : 0;
    }

    __device__ __forceinline__ TileOrder(const PromptParams& params, int positions, bool report)
        : p(params), span(positions), lane(threadIdx.x & 31), seqs(params.num_seqs), most(0), s0(0), before(0) {
        for (int s = lane; s < p.num_seqs; s += 32) {
            const int a = p.cu_seqlens[s], b = p.cu_seqlens[s + 1];
            if (a < 0 || b < a || b > p.T) seqs = min(seqs, s);
        }
        seqs = __reduce_min_sync(0xffffffffu, seqs);
        if (seqs < p.num_seqs && report && lane == 0 && p.error_word) atomicExch(p.error_word, 5);
        own = tiles(lane);
        most = own;
        for (int s = lane + 32; s < seqs; s += 32) most = max(most, tiles(s));
        most = __reduce_max_sync(0xffffffffu, most);
        level = most - 1;
    }

    // Sequence number `skip` of those in `m`, the sequences from s on with a tile `index`.
    __device__ __forceinline__ Tile pick(uint32_t m, int skip, int s, int index) const {
        const uint32_t hit = __ballot_sync(0xffffffffu, (m >> lane & 1) && __popc(m & ((1u << lane) - 1u)) == skip);
        s += __ffs(hit) - 1;
        Tile t;
        t.first = p.cu_seqlens[s];
        t.len = p.cu_seqlens[s + 1] - t.first;
        t.index = index;
        t.some = true;
        return t;
    }

    // Tile number c, the same in every lane.
    __device__ __forceinline__ Tile find(unsigned int c) {
        const Tile none = {0, 0, 0, false};
        if (seqs <= 32) {
            // tiles with an index of at least x; all together are below 2^31
            auto at_least = [&](int x) { return __reduce_add_sync(0xffffffffu, static_cast<unsigned int>(max(own - x, 0))); };
            if (c >= at_least(0)) return none;
            int lo = 0, hi = most;     // at_least(lo) > c, at_least(hi) <= c
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (at_least(mid) > c) lo = mid;
                else hi = mid;
            }
            const uint32_t m = __ballot_sync(0xffffffffu, own > lo);
            return pick(m, static_cast<int>(c - at_least(lo + 1)), 0, lo);
        }
        while (level >= 0) {
            const uint32_t m = __ballot_sync(0xffffffffu, tiles(s0 + lane) > level);
            const unsigned int n = __popc(m);
            if (c - before < n) return pick(m, static_cast<int>(c - before), s0, level);
            before += n;
            s0 += 32;
            if (s0 >= seqs) {
                s0 = 0;
                --level;
            }
        }
        return none;
    }
};

// Zeroes the NaN and infinite elements of eight bf16 values.
__device__ __forceinline__ void zero_nonfinite(uint4& v) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & 0x7F80u) == 0x7F80u) w[i] &= 0xFFFF0000u;
        if ((w[i] & 0x7F800000u) == 0x7F800000u) w[i] &= 0x0000FFFFu;
    }
}

// ---------------------------------------------------------------- kernel
//
// A CTA per SM takes tiles of 256 rows, two M = 128 tiles of 128 rows each:
//
//   warps 0-3, 4-7   softmax of M tile 0 and 1, one thread per row
//   warps 8-11       epilogue: output rows from TMEM to memory
//   warps 12, 13     MMA issue for M tile 0 and 1
//   warp 14          tiles, Q, and the ring of K and V stages, by TMA
//   warp 15          V of masked positions
//
// S = Q K^T of 64 keys goes to one of two TMEM buffers per M tile, is read as
// fp32 and written back over itself as the bf16 weights P, which the second MMA
// takes from TMEM as its A operand with V (MN-major) from shared memory; the
// scores of the next step are computed meanwhile.  TMEM holds 2 x 2 x 64 columns
// of scores and 2 x 128 of output.  (128 keys a step with one buffer would read
// the queries half as often from shared memory, 64 cycles for 64 of products instead
// of 48 for 32, but leaves the softmax alone with nothing to run under: 141 us
// instead of 126 for four prompts of 1024 x 96 heads.)  The running maximum is left behind by up to
// 2^8 before the output is rescaled, so a rescale is rare and the softmax threads
// do it themselves.  An M tile's MMAs have a warp of their own, so that what one
// spends between MMAs (barriers, descriptors) is covered by the other's; a
// whole warp issues them, with uniform operands, for a lane of a divergent branch
// takes longer to issue an MMA than the MMA takes.  Steps run on from tile to
// tile: with Q in two buffers, the next tile's first scores are issued under the
// last weights of a tile, and its output rows leave through the buffer of the
// queries that are done with.  The six ring stages that are left hold three steps
// of K and V (four stages: 109 us instead of 99 for seven prompts).

constexpr int kSms = 148;
constexpr int kRows = 256;
constexpr int kStep = 64;                               // keys of a softmax step and of a ring stage
constexpr int kFmaPairs = 2;                            // pairs of eight whose exponentials go to the FMA pipe; three or four gain nothing
constexpr int kStages = 6;                              // K and V tiles in flight, 16 KB each
constexpr int kThreads = 512;
constexpr uint32_t kHalf = kStep * 128;                 // 64 dims of a 64-key tile: rows of 128 bytes, swizzled
constexpr uint32_t kTileBytes = 2 * kHalf;
constexpr uint32_t kQHalf = kRows * 128;                // 64 dims of the queries
constexpr uint32_t kQBytes = 2 * kQHalf;
constexpr size_t kSmem = 2 * kQBytes + kStages * kTileBytes + 1024;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr int kTileReaders = 8 + 1 + 2 + 1;             // softmax warps, the epilogue, MMA warps and the cleaner

// A tile is at most 256 positions (one head a group): steps with masked ones.
constexpr int kMaskedSteps = 5;

// Ring items of a tile: K0 K1 V0 K2 V1 .. in the order of their MMAs.
__device__ __forceinline__ int k_item(int j) { return j ? 2 * j - 1 : 0; }
__device__ __forceinline__ int v_item(int j, int steps) { return min(2 * j + 2, 2 * steps - 1); }

// A tile as the load warp hands it to the others.
struct TileWork {
    int some, kvh;
    int first;                                          // row of the sequence's first token
    int pos0;                                           // position of the tile's first rows
    int rows, mt;                                       // rows, M tiles in use
    int steps, first_masked;                            // steps of 64 keys; from that one on there are positions that
                                                        // not every row attends
    int last;                                           // keys of the last step, up to a multiple of 16
    int dirty;                                          // V values zeroed behind pos0
};

// x / G for x < 4096, G <= 16
__device__ __forceinline__ int group_div(int x, uint32_t g_inv) { return static_cast<int>(static_cast<uint32_t>(x) * g_inv >> 16); }

struct Bars {
    uint64_t full[kStages], empty[kStages];             // ring of K and V
    uint64_t s_full[2][2], p_full[2][2];                // [M tile][score buffer]
    uint64_t pv_done[2], o_full[2], o_free[2];
    // Output rows in shared memory, by the tile's slot: an epilogue warp may be a tile ahead of the others, and two only
    // when the slot is free again.
    uint64_t staged[2];
    uint64_t tile_full[2], tile_empty[2], q_full[2], drain[2];      // by the tile's slot; an empty slot's Q is empty
    // V with masked positions, by the tile's slot; every one of them completes once a tile, so its phase is the slot's
    uint64_t v_full[2][kMaskedSteps], clean[2][kMaskedSteps];
};

// Bounded wait that reads the clock and the abort flag every 256 tries only: a
// read of the global timer takes longer than most of the waits here.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    uint64_t t0 = 0;
    for (uint32_t tries = 1; !mbar_try_wait(bar, parity); ++tries) {
        if (tries & 255u) continue;
        if (*abort_flag) return false;
        const uint64_t now = globaltimer_ns();
        if (t0 == 0) t0 = now;
        if (now - t0 > kWaitNs) {
            *abort_flag = 1;
            return false;
        }
    }
    return true;
}

// Waits without regard to the abort flag, for this thread's own copies.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 < kWaitNs) {}
}

// 32 bytes to a 32-byte aligned address.
__device__ __forceinline__ void st_global_32(void* dst, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "l"(dst), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// 2^x for x up to 127 on the FMA pipe, which the softmax leaves idle while the
// MUFU is its limit: x = n + f with n the nearest integer, a polynomial for 2^f
// on [-1/2, 1/2] (least largest relative error with P(0) = 1: 2.8e-6), n added
// to the exponent.  x below -127 gives 0.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
    constexpr float kMagic = 12582912.0f;               // 1.5 * 2^23: the sum's low bits are n
    x.x = fmaxf(x.x, -127.0f);
    x.y = fmaxf(x.y, -127.0f);
    const float2 t = fadd2(x, make_float2(kMagic, kMagic));
    const float2 n = fadd2(t, make_float2(-kMagic, -kMagic));
    const float2 f = ffma2(n, make_float2(-1.0f, -1.0f), x);
    float2 r = ffma2(f, make_float2(0.009582852944731712f, 0.009582852944731712f), make_float2(0.055906426161527634f, 0.055906426161527634f));
    r = ffma2(f, r, make_float2(0.24024099111557007f, 0.24024099111557007f));
    r = ffma2(f, r, make_float2(0.6931241750717163f, 0.6931241750717163f));
    r = ffma2(f, r, make_float2(1.0f, 1.0f));
    return make_float2(__int_as_float(__float_as_int(r.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(r.y) + (__float_as_int(t.y) << 23)));
}

// The largest of three, NaN if any is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// The larger of each of two bf16 pairs, NaN if either is.
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// NaN and infinities in V.  A weight is positive however small, so a row that
// attends infinities of one sign is that infinity in their dim, and with both
// signs or a NaN it is NaN.  The MMAs give that but for two cases: a weight, or the
// factor of a rescale, too small for fp32 makes NaN of an infinity, and V behind a
// tile's first position has zeros in place of such values.  So where a row is NaN
// although its sum of weights is a number, the epilogue looks for such values in
// those dims of all of the sequence's V, and where V was cleaned, in all dims behind
// the first position: what a row is depends on no tile.  (One NaN in V at the start
// of a prompt of 16384 tokens: 954 us instead of 632; a whole row of them 1284.)
struct Settled {
    uint32_t over;                                      // chunks of 8 dims whose outcome stands in place of the row's value,
                                                        // not beside it; alike in the warp
    uint16_t dims[16];                                  // 2 bits a dim of this lane's row: 0 nothing, 1 inf, 2 -inf, 3 NaN
};
__device__ __forceinline__ float settle(float x, const Settled& s, int c, int e) {
    const uint32_t k = s.dims[c] >> (2 * e) & 3u;
    if (k == 0) return x;
    const float y = __uint_as_float(k == 1 ? 0x7F800000u : k == 2 ? 0xFF800000u : 0x7FFFFFFFu);
    return s.over >> c & 1 ? y : x + y;
}

// By a warp, its lanes' rows at `pos`; `nan_chunks`: the chunks of this lane's row with a NaN to be settled.  A lane
// looks at a row of V at a time, eight dims of it.
__device__ __noinline__ void find_settled(const PromptParams& p, long long first, int pos0, int pos, int kvh, bool dirty,
                                          uint32_t nan_chunks, Settled& out) {
    constexpr int kNone = 0x7FFFFFFF, kBatch = 8;
    const int lane = threadIdx.x & 31, n = __reduce_max_sync(0xffffffffu, pos) + 1;
    out.over = __reduce_or_sync(0xffffffffu, nan_chunks);
#pragma unroll 1
    for (int c = 0; c < 16; ++c) {
        const __nv_bfloat16* v = p.v + first * p.v_stride + kvh * kD + 8 * c;
        int at[3][8];                                   // first position with inf, -inf, NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) at[0][e] = at[1][e] = at[2][e] = kNone;
        bool any = false;
        for (int j0 = out.over >> c & 1 ? 0 : dirty ? pos0 + 1 : n; j0 < n; j0 += 32 * kBatch) {
            uint4 x[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int j = j0 + 32 * i + lane;
                x[i] = j < n ? *reinterpret_cast<const uint4*>(v + j * p.v_stride) : make_uint4(0, 0, 0, 0);
            }
            uint32_t found = 0;                         // an exponent of all ones carries into the sign's place
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                found |= ((x[i].x & 0x7F807F80u) + 0x00800080u) | ((x[i].y & 0x7F807F80u) + 0x00800080u) |
                         ((x[i].z & 0x7F807F80u) + 0x00800080u) | ((x[i].w & 0x7F807F80u) + 0x00800080u);
            if (!__any_sync(0xffffffffu, found & 0x80008000u)) continue;
            any = true;
            uint32_t nans = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const uint32_t w = e < 2 ? x[i].x : e < 4 ? x[i].y : e < 6 ? x[i].z : x[i].w;
                    const uint32_t y = w >> (16 * (e & 1)) & 0xFFFFu;
                    const int j = j0 + 32 * i + lane;
                    if (y == 0x7F80u) at[0][e] = min(at[0][e], j);
                    else if (y == 0xFF80u) at[1][e] = min(at[1][e], j);
                    else if ((y & 0x7F80u) == 0x7F80u) at[2][e] = min(at[2][e], j);
                }
                nans |= static_cast<uint32_t>(at[2][e] != kNone) << e;
            }
            if (__reduce_or_sync(0xffffffffu, nans) == 0xFFu) break;       // NaN from there on whatever comes
        }
        uint32_t dims = 0;
        if (any) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool plus = __reduce_min_sync(0xffffffffu, at[0][e]) <= pos, minus = __reduce_min_sync(0xffffffffu, at[1][e]) <= pos;
                const bool nan = __reduce_min_sync(0xffffffffu, at[2][e]) <= pos;
                dims |= (nan ? 3u : static_cast<uint32_t>(plus) | static_cast<uint32_t>(minus) << 1) << (2 * e);
            }
        }
        out.dims[c] = static_cast<uint16_t>(dims);
    }
}

// 16-byte chunk c of output row i in shared memory (see the epilogue).
__device__ __forceinline__ uint4* row_chunk(uint8_t* rows_sm, int i, int c) {
    return reinterpret_cast<uint4*>(rows_sm + (c >> 3) * kQHalf + i * 128 + (((c ^ i) & 7) << 4));
}

// The bf16 rows in shared memory, one a lane; `sums`: the row's sum of weights is a number above 0.
__device__ __noinline__ void settle_rows(const PromptParams& p, uint8_t* rows_sm, int i_row, long long first, int pos0, int pos, int kvh,
                                         bool dirty, bool sums) {
    uint32_t nan_chunks = 0;
    for (int c = 0; c < 16; ++c) {
        const uint4 x = *row_chunk(rows_sm, i_row, c);
        const uint32_t m = max2_nan(max2_nan(x.x, x.y), max2_nan(x.z, x.w));
        if (sums && ((m & 0x7FFFu) > 0x7F80u || (m & 0x7FFF0000u) > 0x7F800000u)) nan_chunks |= 1u << c;
    }
    Settled s;
    find_settled(p, first, pos0, pos, kvh, dirty, nan_chunks, s);
    if (!sums) return;
    for (int c = 0; c < 16; ++c) {
        if (!s.dims[c]) continue;
        __nv_bfloat16* x = reinterpret_cast<__nv_bfloat16*>(row_chunk(rows_sm, i_row, c));
        for (int e = 0; e < 8; ++e) x[e] = __float2bfloat16_rn(settle(__bfloat162float(x[e]), s, c, e));
    }
}

// The e4m3 rows and their scales, from the output in TMEM.
__device__ __noinline__ void settle_quantised(const PromptParams& p, uint32_t to, float inv, long long first, int pos0, int pos, int kvh,
                                              int head, bool dirty, bool sums, bool store) {
    auto columns = [&](int b, float (&x)[16]) {
        uint32_t o[16];
        __syncwarp();
        tmem_ld16(to + 16 * b, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(o[e]) * inv;
    };
    float x[16];
    uint32_t nan_chunks = 0;
    for (int b = 0; b < 8; ++b) {
        columns(b, x);
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (sums && store && x[e] != x[e]) nan_chunks |= 1u << (2 * b + e / 8);
    }
    Settled s;
    find_settled(p, first, pos0, pos, kvh, dirty, nan_chunks, s);
    if (!sums)
        for (int c = 0; c < 16; ++c) s.dims[c] = 0;
    const long long out_row = (first + pos) * p.nq + head;
    float amax = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
        const E4m3Row r = e4m3_row(amax);
        for (int b = 0; b < 8; ++b) {
            columns(b, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                x[e] = settle(x[e], s, 2 * b + e / 8, e % 8);
                if (pass == 0) amax = fmaxf(amax, fabsf(x[e]));
                else if (store) p.out_q[out_row * kD + 16 * b + e] = static_cast<uint8_t>(cvt_e4m3x2(x[e] * r.up * r.inv, 0.0f));
            }
        }
    }
    if (store) p.out_s[static_cast<size_t>(head) * p.out_ld + first + pos] = e4m3_row(amax).scale;
}

// The e4m3 rows and their scales.  (Not a call: the whole kernel comes out slower with one more, 97 us instead of 95 for
// seven prompts of up to 1201 with 96 heads, 728 instead of 722 for one of 16384.)
__device__ __forceinline__ void quantise_output(const PromptParams& p, uint32_t to, float inv, long long first, int pos0, int pos, int kvh,
                                             int head, bool dirty, bool sums, bool store) {
    auto columns = [&](int c, float (&x)[32]) {         // 32 dims of the row
        uint32_t o[32];
        __syncwarp();
        tmem_ld32(to + 32 * c, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = __uint_as_float(o[e]) * inv;
    };
    const long long out_row = (first + pos) * p.nq + head;
    float amax = 0.0f, nan = 0.0f;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        float x[32];
        columns(c, x);
#pragma unroll
        for (int e = 0; e < 32; ++e) amax = fmaxf(amax, fabsf(x[e]));
#pragma unroll
        for (int e = 0; e < 32; e += 2) nan = max3_nan(nan, x[e], x[e + 1]);
    }
    if (dirty || __any_sync(0xffffffffu, nan != nan && sums && store)) {
        settle_quantised(p, to, inv, first, pos0, pos, kvh, head, dirty, sums, store);
        return;
    }
    const E4m3Row r = e4m3_row(amax);
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        float x[32];
        columns(c, x);
        uint32_t wt[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            wt[e] = cvt_e4m3x2(x[4 * e] * r.up * r.inv, x[4 * e + 1] * r.up * r.inv) |
                    static_cast<uint32_t>(cvt_e4m3x2(x[4 * e + 2] * r.up * r.inv, x[4 * e + 3] * r.up * r.inv)) << 16;
        if (store) st_global_32(p.out_q + out_row * kD + 32 * c, wt);
    }
    if (store) p.out_s[static_cast<size_t>(head) * p.out_ld + first + pos] = r.scale;
}

__global__ void __launch_bounds__(kThreads, 1)
prompt_kernel(const __grid_constant__ PromptParams p, const __grid_constant__ CUtensorMap qmap,
              const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
              const __grid_constant__ CUtensorMap omap) {
    extern __shared__ uint8_t sm_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* q_s = sm;                                  // [2 slots][2 halves][256 rows][128 B]
    uint8_t* kv_s = sm + 2 * kQBytes;                   // [stages][2 halves][64][128 B]
    __shared__ Bars bars;
    __shared__ TileWork tile_s[2];
    __shared__ float l_s[kRows];                        // row sums
    __shared__ uint32_t tmem_s;
    __shared__ int abort_s;
    volatile int* abort_flag = &abort_s;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform for the compiler
    if (warp == 15 && lane == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.empty[i], 2);
        }
        for (int t = 0; t < 2; ++t) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&bars.s_full[t][b], 1);
                mbar_init(&bars.p_full[t][b], 128);
            }
            mbar_init(&bars.pv_done[t], 1);
            mbar_init(&bars.o_full[t], 2);
            mbar_init(&bars.o_free[t], 128);
            mbar_init(&bars.tile_full[t], 1);
            mbar_init(&bars.tile_empty[t], kTileReaders);
            mbar_init(&bars.drain[t], 1);
            mbar_init(&bars.staged[t], 4);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&bars.q_full[t], 1);
            for (int i = 0; i < kMaskedSteps; ++i) {
                mbar_init(&bars.v_full[t][i], 1);
                mbar_init(&bars.clean[t][i], 1);
            }
        }
        abort_s = 0;
        fence_mbar_init();
        prefetch_tmap(&qmap);
        prefetch_tmap(&kmap);
        prefetch_tmap(&vmap);
        prefetch_tmap(&omap);
    } else if (warp == 12) {
        tmem_alloc(&tmem_s, 512);
        tc_fence_before();
    }
    const uint32_t g_inv = (65536u + p.G - 1) / p.G;
    const int tile_pos = p.tile_pos;
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_phase(bar, parity, abort_flag); };
    auto all = [&](bool x) { return __all_sync(0xffffffffu, x); };

    if (warp < 8) {
        // ---- softmax
        const int t = warp >> 2;
        const int i_row = threadIdx.x;
        const uint32_t ts = tmem + (static_cast<uint32_t>(warp & 3) << 21) + t * 128;   // this warp's 32 lanes
        const uint32_t to = ts + 256;
        const float sl2 = p.scale_log2;
        int g = 0, tiles = 0;                           // steps and tiles of this M tile so far
        bool ok = true;
        for (int n = 0; ok; ++n) {
            if (!(ok = all(wait(&bars.tile_full[n & 1], (n >> 1) & 1)))) break;
            const TileWork& w = tile_s[n & 1];
            if (!w.some) break;
            if (t < w.mt) {
                const int steps = w.steps, first_masked = w.first_masked;
                const int pos = w.pos0 + group_div(min(i_row, w.rows - 1), g_inv);
                const bool used = i_row < w.rows;
                float m = -INFINITY, l = 0.0f;
                for (int j = 0; j < steps; ++j, ++g) {
                    const uint32_t sb = ts + (g & 1) * kStep;
                    if (!(ok = all(wait(&bars.s_full[t][g & 1], (g >> 1) & 1)))) break;
                    tc_fence_after();
                    uint32_t s[2][32];
#pragma unroll
                    for (int c = 0; c < 2; ++c) tmem_ld32(sb + 32 * c, s[c]);
                    tmem_wait_ld();
                    if (j >= first_masked) {
                        const int lim = pos - j * kStep;
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (32 * c + e > lim) s[c][e] = 0xFF800000u;
                    }
                    // a NaN score makes the maximum NaN, and with it the row
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            mx[c] = max3_nan(mx[c], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
                    const float mt = max3_nan(mx[0], mx[1], -INFINITY);
                    if (j == 0) {
                        m = mt;
                    } else {
                        const bool need = !((mt - m) * sl2 <= 8.0f) && mt != m && used;
                        if (__any_sync(0xffffffffu, need)) {
                            const float f = need ? ex2((m - mt) * sl2) : 1.0f;
                            l *= f;
                            if (need) m = mt;
                            // the product of the step before has to be in
                            if (!(ok = all(wait(&bars.pv_done[t], (g - 1) & 1)))) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < 8; ++c) {
                                uint32_t o[16];
                                tmem_ld16(to + 16 * c, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tmem_st16(to + 16 * c, o);
                            }
                        }
                    }
                    const float nm = m == -INFINITY ? 0.0f : -m * sl2;     // nothing but -inf so far: weights 0, not NaN
                    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t wt[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float2 x = ffma2(make_float2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1])),
                                             make_float2(sl2, sl2), make_float2(nm, nm));
                            if (e % 8 < kFmaPairs) {
                                x = ex2_fma(x);
                            } else {
                                x.x = ex2(x.x);
                                x.y = ex2(x.y);
                            }
                            sum[e & 1] = fadd2(sum[e & 1], x);
                            wt[e] = pack_bf16(x.x, x.y);    // the weights' rounding, 2^-8 at most; the sum has them whole
                        }
                        tmem_st16(sb + 16 * c, wt);
                    }
                    sum[0] = fadd2(sum[0], sum[1]);
                    l += sum[0].x + sum[0].y;
                    if (j + 1 == steps) {               // goes to the epilogue with the last weights
                        if (tiles && !(ok = all(wait(&bars.o_free[t], (tiles - 1) & 1)))) break;   // it has the last tile's
                        l_s[i_row] = l;
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    mbar_arrive(&bars.p_full[t][g & 1]);
                }
                ++tiles;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.tile_empty[n & 1]);
        }
    } else if (warp < 12) {
        // ---- epilogue
        uint32_t o_phase = 0;                           // of o_full[t], bit t
        bool ok = true;
        for (int n = 0; ok; ++n) {
            if (!(ok = all(wait(&bars.tile_full[n & 1], (n >> 1) & 1)))) break;
            const TileWork& w = tile_s[n & 1];
            if (!w.some) break;
            const int rows = w.rows, pos0 = w.pos0, kvh = w.kvh, mt = w.mt;
            const long long first = w.first;
            // Rows go through shared memory in place of the queries, in their layout: a full tile leaves as one box, and of
            // one in part filled a store instruction covers two rows and not a sector of each of 32.
            uint8_t* rows_sm = q_s + (n & 1) * kQBytes;
            auto chunk = [&](int i, int c) { return row_chunk(rows_sm, i, c); };
            const bool box = rows == tile_pos * p.G;
#pragma unroll 1
            for (int t = 0; t < mt; ++t) {
                const int i_row = t * 128 + (threadIdx.x & 127);
                const uint32_t to = tmem + (static_cast<uint32_t>(warp & 3) << 21) + 256 + t * 128;
                if (!(ok = all(wait(&bars.o_full[t], (o_phase >> t) & 1)))) break;
                o_phase ^= 1u << t;
                tc_fence_after();
                const float l = l_s[i_row], inv = 1.0f / l;
                const bool dirty = *static_cast<volatile const int*>(&w.dirty) != 0;
                const int at = group_div(min(i_row, rows - 1), g_inv);
                const int pos = pos0 + at;
                const int head = kvh * p.G + min(i_row, rows - 1) - at * p.G;
                const bool store = i_row < rows;
                const bool sums = l > 0.0f;             // else the row is NaN, whatever V holds
                if (p.out_q) {
                    quantise_output(p, to, inv, first, pos0, pos, kvh, head, dirty, sums, store);
                    __syncwarp();
                }
                uint32_t nan = 0;
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    uint32_t o[64];
                    tmem_ld32(to + 64 * c, *reinterpret_cast<uint32_t(*)[32]>(o));
                    tmem_ld32(to + 64 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(o + 32));
                    tmem_wait_ld();
                    if (c == 1) {
                        tc_fence_before();
                        mbar_arrive(&bars.o_free[t]);   // the next tile may write its output
                    }
                    auto pack = [&](int e) {
                        const uint32_t x = pack_bf16(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
                        nan = max2_nan(nan, x);
                        return x;
                    };
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        *chunk(i_row, 8 * c + e) = make_uint4(pack(8 * e), pack(8 * e + 2), pack(8 * e + 4), pack(8 * e + 6));
                }
                const bool is_nan = (nan & 0x7FFFu) > 0x7F80u || (nan & 0x7FFF0000u) > 0x7F800000u;
                if (dirty || __any_sync(0xffffffffu, is_nan && sums && store))
                    settle_rows(p, rows_sm, i_row, first, pos0, pos, kvh, dirty, sums && store);
                if (box) continue;
                __syncwarp();
                const int row0 = t * 128 + (warp & 3) * 32;
#pragma unroll 4
                for (int i = row0 + (lane >> 4); i < min(rows, row0 + 32); i += 2) {
                    const int row_at = group_div(i, g_inv);
                    *reinterpret_cast<uint4*>(p.out + ((first + pos0 + row_at) * p.nq + kvh * p.G + i - row_at * p.G) * kD +
                                              (lane & 15) * 8) = *chunk(i, lane & 15);
                }
            }
            if (!ok) break;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");        // before the box, and the slot's next queries
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.staged[n & 1]);
            if (warp == 8) {
                if (!(ok = all(wait(&bars.staged[n & 1], (n >> 1) & 1)))) break;
                if (lane == 0) {
                    if (box) {
                        tma_store_3d(&omap, rows_sm, 0, kvh * p.G, static_cast<int>(first) + pos0);
                        tma_store_3d(&omap, rows_sm + kQHalf, 64, kvh * p.G, static_cast<int>(first) + pos0);
                        bulk_store_wait_read();
                    }
                    mbar_arrive(&bars.tile_empty[n & 1]);
                }
                __syncwarp();
            }
        }
    } else if (warp < 14) {
        // ---- MMA issue, by a whole warp for M tile t
        const int t = warp - 12;
        const bool el = lane == 0;
        auto uni = [](int x) { return __shfl_sync(0xffffffffu, x, 0); };       // uniform for the compiler as well
        const uint32_t negate = p.flip_q ? 1u << 13 : 0u;      // of A
        constexpr uint32_t id_o = idesc_bf16_f32(128, kD, true);
        const uint32_t tm = uni(tmem) + t * 128;
        const uint32_t q_lo = desc_lo_k(smem_u32(q_s)) + t * (128 * 128 >> 4);
        const uint32_t k_lo = desc_lo_k(smem_u32(kv_s)), v_lo = desc_lo_mn(smem_u32(kv_s), kHalf);
        auto wait_item = [&](int x) { return all(wait(&bars.full[x % kStages], (x / kStages) & 1)); };
        int n = 0, base = 0, tiles = 0, g = 0;          // tile, its first ring item; tiles and products of this M tile so far
        bool ok = true;
        // Scores, up to two steps before the products and at most one tile: as far as tile `next` they are issued where
        // their operands are there, and waited for with `block`.
        int sn = -1, sj = 0, s_steps = 0, s_last = 0, s_base = 0, sg = 0;
        auto scores = [&](int next, int next_base, bool block) {
            auto got = [&](uint64_t* bar, uint32_t phase) {
                if (!block) return all(mbar_test(bar, phase)) != 0;
                return ok = all(wait(bar, phase));
            };
            while (sg - g < 2) {
                if (sj == s_steps) {
                    if (sn >= next) return;
                    if (!got(&bars.tile_full[next & 1], (next >> 1) & 1)) return;
                    const TileWork& w = tile_s[next & 1];
                    if (!uni(w.some) || t >= uni(w.mt)) return;
                    if (!got(&bars.q_full[next & 1], (next >> 1) & 1)) return;
                    sn = next;
                    sj = 0;
                    s_steps = uni(w.steps);
                    s_last = uni(w.last);
                    s_base = next_base;
                }
                const int x = s_base + k_item(sj), st = x % kStages;
                if (!got(&bars.full[st], (x / kStages) & 1)) return;
                tc_fence_after();
                const uint32_t id_s = idesc_bf16_f32(128, sj + 1 == s_steps ? s_last : kStep, false) | negate;
                const uint32_t q = q_lo + (sn & 1) * (kQBytes >> 4), k = k_lo + st * (kTileBytes >> 4);
                const uint32_t d = tm + (sg & 1) * kStep;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    umma_f16_warp(d, q + (ks >> 2) * (kQHalf >> 4) + (ks & 3) * 2, k + (ks >> 2) * (kHalf >> 4) + (ks & 3) * 2,
                                  id_s, ks > 0);
                umma_commit_warp(&bars.s_full[t][sg & 1]);
                umma_commit_warp(&bars.empty[st]);
                ++sj;
                ++sg;
            }
        };
        for (; ok; ++n) {
            if (!(ok = all(wait(&bars.tile_full[n & 1], (n >> 1) & 1)))) break;
            const TileWork& slot = tile_s[n & 1];
            if (!uni(slot.some)) break;
            const int steps = uni(slot.steps), last = uni(slot.last), first_masked = uni(slot.first_masked);
            if (t >= uni(slot.mt)) {
                // the other M tile has it alone: this warp only keeps the counts of the ring
                for (int x = base; x < base + 2 * steps && ok; ++x)
                    if ((ok = wait_item(x)) && el) mbar_arrive(&bars.empty[x % kStages]);
                if (!ok) break;
            } else {
                const uint32_t slot_phase = (n >> 1) & 1;
                for (int j = 0; j < steps; ++j) {
                    // scores and these weights, whichever comes first; the next tile may be handed out only once these are used
                    bool ready = false;
                    for (int i = 0; i < 512 && !ready && sg - g < 2; ++i) {
                        const bool own = sg == g;       // those that the weights are made of
                        scores(own ? n : n + 1, own ? base : base + 2 * steps, own);
                        if (!ok) break;
                        ready = all(mbar_test(&bars.p_full[t][g & 1], (g >> 1) & 1));
                    }
                    if (!ok || !(ready || (ok = all(wait(&bars.p_full[t][g & 1], (g >> 1) & 1))))) break;
                    if (j == 0 && !(ok = all(wait(&bars.o_free[t], (tiles++ & 1) ^ 1)))) break;
                    // V, cleaned where it has to be
                    const int x = base + v_item(j, steps), st = x % kStages;
                    ok = j < first_masked ? wait_item(x) : all(wait(&bars.clean[n & 1][j - first_masked], slot_phase));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t v = v_lo + st * (kTileBytes >> 4);
                    const uint32_t pa = tm + (g & 1) * kStep;
                    const int ksteps = j + 1 == steps ? last / 16 : kStep / 16;
#pragma unroll
                    for (int ks = 0; ks < kStep / 16; ++ks)     // 16 keys: 16 rows of 128 bytes
                        if (ks < ksteps) umma_f16_ta_warp(tm + 256, pa + ks * 8, v + ks * (2048 >> 4), id_o, j > 0 || ks > 0);
                    umma_commit_warp(&bars.pv_done[t]);
                    if (j + 1 == steps) {
                        if (el) mbar_arrive(&bars.o_full[t]);   // the cleaner's word on the tile and the row sums go with it
                        umma_commit_warp(&bars.o_full[t]);
                    }
                    umma_commit_warp(&bars.empty[st]);
                    ++g;
                }
            }
            base += 2 * steps;
            if (el) mbar_arrive(&bars.tile_empty[n & 1]);
        }
        if (!ok) {
            umma_commit_warp(&bars.drain[t]);
            mbar_drain(&bars.drain[t], 0);
        }
    } else if (warp == 14) {
        // ---- tiles, their Q, and K and V of each step
        // A tile is handed out, and its Q on the way, as soon as its slot is free, between the loads of the tile before; it
        // is found under those of that tile's first steps.
        TileOrder order(p, tile_pos, blockIdx.x == 0);
        int item = 0, q_tiles = 0;                      // ring items so far, tiles whose Q is loaded
        int armed[2] = {0, 0};                          // V barriers with a copy, by slot
        bool ok = true;
        auto find = [&](int n) {
            // every other round backwards: a CTA's tiles even out
            const unsigned int c = n * gridDim.x + ((n & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
            const Tile tl = order.find(c / p.nkv);
            TileWork w;
            w.some = tl.some;
            w.kvh = static_cast<int>(c % p.nkv);
            w.first = tl.first;
            w.pos0 = tl.index * tile_pos;
            w.rows = min(tile_pos, tl.len - w.pos0) * p.G;
            w.mt = w.rows > 128 ? 2 : 1;
            const int pos1 = min(w.pos0 + tile_pos, tl.len) - 1;
            w.steps = tl.some ? pos1 / kStep + 1 : 0;
            w.last = (pos1 % kStep + 16) / 16 * 16;
            w.first_masked = (w.pos0 + 1) / kStep;
            w.dirty = 0;
            return w;
        };
        auto hand_out = [&](int n, const TileWork& w) {         // into a free slot
            tile_s[n & 1] = w;
            mbar_arrive(&bars.tile_full[n & 1]);
            armed[n & 1] = 0;
            if (!w.some) return;
            uint8_t* q = q_s + (n & 1) * kQBytes;
            mbar_arrive_expect_tx(&bars.q_full[n & 1], tile_pos * p.G * 256);
            tma_load_3d(&qmap, &bars.q_full[n & 1], q, 0, w.kvh * p.G, w.first + w.pos0);
            tma_load_3d(&qmap, &bars.q_full[n & 1], q + kQHalf, 64, w.kvh * p.G, w.first + w.pos0);
            q_tiles = n + 1;
        };
        // own_bar: V that has to be cleaned lands at a barrier of its own; the ring's only keeps its phase
        auto load = [&](const CUtensorMap* map, int x, int y, int n, uint64_t* own_bar) {
            const int st = item % kStages;
            if (!(ok = wait(&bars.empty[st], ((item / kStages) & 1) ^ 1))) return;
            uint64_t* bar = own_bar ? own_bar : &bars.full[st];
            if (own_bar) mbar_arrive(&bars.full[st]);
            mbar_arrive_expect_tx(bar, kTileBytes);
            uint8_t* dst = kv_s + st * kTileBytes;
            tma_load_2d(map, bar, dst, x, y);
            tma_load_2d(map, bar, dst + kHalf, x + 64, y);
            ++item;
            if (own_bar) ++armed[n & 1];
        };
        auto load_step = [&](int n, const TileWork& w, int j) { // K of the step behind, V of this one; the first K with it
            const int x = w.kvh * kD, y = w.first + j * kStep;
            if (j == 0) load(&kmap, x, y, n, nullptr);
            if (ok && j + 1 < w.steps) load(&kmap, x, y + kStep, n, nullptr);
            if (ok) load(&vmap, x, y, n, j < w.first_masked ? nullptr : &bars.v_full[n & 1][j - w.first_masked]);
        };
        TileWork w = find(0);
        if (lane == 0) hand_out(0, w);
        for (int n = 0; w.some; ++n) {
            const int early = min(w.steps, 2);
            if (lane == 0)
                for (int j = 0; j < early && ok; ++j) load_step(n, w, j);
            __syncwarp();
            const TileWork next = find(n + 1);
            if (lane == 0) {
                uint64_t* slot = &bars.tile_empty[(n + 1) & 1];
                const uint32_t slot_phase = (((n + 1) >> 1) & 1) ^ 1;
                bool out = false;
                for (int j = early; j < w.steps && ok; ++j) {
                    if (!out && (out = mbar_test(slot, slot_phase))) hand_out(n + 1, next);
                    load_step(n, w, j);
                }
                if (ok)
                    for (int i = armed[n & 1]; i < kMaskedSteps; ++i) mbar_arrive(&bars.v_full[n & 1][i]);
                if (ok && !out && (ok = wait(slot, slot_phase))) hand_out(n + 1, next);
                if (!ok) {   // loads in flight land before the block leaves
                    for (int i = max(item - kStages, 0); i < item; ++i) mbar_drain(&bars.full[i % kStages], (i / kStages) & 1);
                    for (int m = max(q_tiles - 2, 0); m < q_tiles; ++m) {
                        mbar_drain(&bars.q_full[m & 1], (m >> 1) & 1);
                        for (int i = 0; i < armed[m & 1]; ++i) mbar_drain(&bars.v_full[m & 1][i], (m >> 1) & 1);
                    }
                }
            }
            if (!__shfl_sync(0xffffffffu, ok, 0)) break;
            w = next;
        }
    } else {
        // ---- a weight of 0 must meet a finite value: V of positions that not every row attends
        int item = 0;
        bool ok = true;
        for (int n = 0; ok; ++n) {
            if (!(ok = all(wait(&bars.tile_full[n & 1], (n >> 1) & 1)))) break;
            TileWork& w = tile_s[n & 1];
            if (!w.some) break;
            const int steps = w.steps, first_masked = w.first_masked;
            for (int i = first_masked; i < steps; ++i) {
                if (!(ok = all(wait(&bars.v_full[n & 1][i - first_masked], (n >> 1) & 1)))) break;
                uint8_t* v = kv_s + (item + v_item(i, steps)) % kStages * kTileBytes;
                const int j0 = max(w.pos0 + 1 - i * kStep, 0);       // first such row of the step
                const int j1 = i + 1 == steps ? w.last : kStep;
                auto at = [&](int c) {
                    return reinterpret_cast<uint4*>(v + (c & 1) * kHalf + (j0 + (c >> 4)) * 128 + ((c >> 1) & 7) * 16);
                };
                // an exponent of all ones carries into the sign's place
                uint32_t found = 0;
#pragma unroll 8
                for (int c = lane; c < (j1 - j0) * 16; c += 32) {
                    const uint4 x = *at(c);
                    found |= ((x.x & 0x7F807F80u) + 0x00800080u) | ((x.y & 0x7F807F80u) + 0x00800080u) |
                             ((x.z & 0x7F807F80u) + 0x00800080u) | ((x.w & 0x7F807F80u) + 0x00800080u);
                }
                if (found & 0x80008000u) {
                    w.dirty = 1;
                    for (int c = lane; c < (j1 - j0) * 16; c += 32) {
                        uint4 x = *at(c);
                        zero_nonfinite(x);
                        *at(c) = x;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.clean[n & 1][i - first_masked]);
            }
            if (!ok) break;
            if (lane == 0)
                for (int i = max(steps - first_masked, 0); i < kMaskedSteps; ++i) mbar_arrive(&bars.clean[n & 1][i]);
            item += 2 * steps;
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.tile_empty[n & 1]);
        }
    }
    __syncthreads();
    if (warp == 12) {
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

// bf16 rows [T][cols], `stride` elements apart, boxes of 64 columns x 64 rows.
bool encode_rows(CUtensorMap* map, const void* base, int T, int cols, long long stride) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(T)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
    cuuint32_t box[2] = {64, kStep};
    cuuint32_t estr[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// q rows [T][nq][128], boxes of 64 dims x G heads x the positions of a tile.
bool encode_q(CUtensorMap* map, const void* base, int T, int nq, int G, int tile_pos, long long stride) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {kD, static_cast<cuuint64_t>(nq), static_cast<cuuint64_t>(T)};
    cuuint64_t strides[2] = {kD * 2, static_cast<cuuint64_t>(stride) * 2};
    cuuint32_t box[3] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(tile_pos)};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
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
    if (!std::isfinite(scale * kLog2e)) return MOE_ERR_INVALID_ARGUMENT;
    if (nkv > 65535 || nq > (1 << 20)) return MOE_ERR_UNSUPPORTED;
    if (q_stride < nq * kD || k_stride < nkv * kD || v_stride < nkv * kD || q_stride % 8 || k_stride % 8 || v_stride % 8)
        return MOE_ERR_INVALID_ARGUMENT;
    if (T == 0 || num_seqs == 0) return MOE_OK;
    if (!q_bf16 || !k_bf16 || !v_bf16 || !cu_seqlens || !out_bf16) return MOE_ERR_INVALID_ARGUMENT;
    if (!a16(q_bf16) || !a16(k_bf16) || !a16(v_bf16) || !a16(out_bf16)) return MOE_ERR_INVALID_ARGUMENT;
    if (out_q && (!out_s || out_ld < T || (reinterpret_cast<uintptr_t>(out_q) & 31))) return MOE_ERR_INVALID_ARGUMENT;
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
    p.flip_q = p.scale_log2 < 0.0f;
    p.scale_log2 = fmaxf(fabsf(p.scale_log2), 1.17549435e-38f);   // 0: every finite score alike, masked ones still -inf
    // every sequence has at most one tile in part filled
    auto tiles_of = [&](int pos) { return ((T + pos - 1ll) / pos + num_seqs) * nkv; };
    // Where tiles of one M tile find an SM each, twice as many SMs run half as many rows (24 prompts of up to 201 tokens, 12
    // heads: 9.8 us instead of 11.9; one of 128: 8.1 instead of 9.7).  A step of one M tile takes two thirds of one of
    // two, so long prompts gain up to two tiles an SM (one of 2000: 29.9 instead of 34.5), while for short ones the second
    // tile costs more (20 of 100: 12.2 instead of 11.0).  A row's bits are the same either way.
    const long long small = tiles_of(128 / p.G);
    p.tile_pos = small <= kSms || (small <= 2 * kSms && T >= 500ll * num_seqs) ? 128 / p.G : kRows / p.G;
    const long long tiles = tiles_of(p.tile_pos);
    if (tiles > 0x7FFFFFFF - 1024) return MOE_ERR_UNSUPPORTED;
    CUtensorMap qmap, kmap, vmap, omap;
    if (!encode_q(&qmap, q_bf16, T, nq, p.G, p.tile_pos, q_stride) || !encode_rows(&kmap, k_bf16, T, nkv * kD, k_stride) ||
        !encode_rows(&vmap, v_bf16, T, nkv * kD, v_stride) || !encode_q(&omap, out_bf16, T, nq, p.G, p.tile_pos, nq * kD))
        return MOE_ERR_CUDA;
    static bool attr[kMaxDevices] = {};
    if (smem_optin_once(prompt_kernel, static_cast<int>(kSmem), attr) != cudaSuccess) return MOE_ERR_CUDA;
    prompt_kernel<<<static_cast<int>(tiles < kSms ? tiles : kSms), kThreads, kSmem, static_cast<cudaStream_t>(stream)>>>(
        p, qmap, kmap, vmap, omap);
    return launch_status();
}

}  // extern "C"
