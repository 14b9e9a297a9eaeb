// attn_common.cuh -- what the attention kernels share: head and page sizes,
// page-table rows, the mma.sync bf16 fragments and launch checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "moe_layer.h"

namespace tb {

constexpr int kD = 128;            // head_dim (the kernels are specialised)
constexpr int kPage = 16;          // tokens per KV page
constexpr float kLog2e = 1.4426950408889634f;

// Page-table row of row b: row_seq[b] when the rows are tokens of several
// sequences (prefill chunks, slot-indexed batches), else b; -1 when outside
// [0, num_seqs).
__device__ __forceinline__ int seq_of_row(const int32_t* row_seq, int b, int num_seqs) {
    const int s = row_seq ? row_seq[b] : b;
    return (s >= 0 && s < num_seqs) ? s : -1;
}

// ---------------------------------------------------------------- mma.sync helpers

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
// D = A (16x16 bf16, row) * B (16x8 bf16, col) + D, fp32 accumulate
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
                 "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// ---------------------------------------------------------------- e4m3 rows

// Codes of a row whose largest number is amax are e4m3(x * up * inv), values code
// * scale.  The scale goes by the numbers: a NaN gets the code NaN, also where there
// is no number or only zeros (inv = 0).  448 / amax is past the fp32 range below
// 1.3e-36, so rows that small are taken 2^64 times their size.
struct E4m3Row {
    float up, inv, scale;
};
__device__ __forceinline__ E4m3Row e4m3_row(float amax) {
    E4m3Row r;
    r.up = amax < 7.8886090522101181e-31f ? 18446744073709551616.0f : 1.0f;      // 2^-100, 2^64
    r.inv = amax > 0.0f ? 448.0f / (amax * r.up) : 0.0f;
    r.scale = amax > 0.0f ? amax / 448.0f : 0.0f;
    return r;
}

// ---------------------------------------------------------------- host

inline moe_status_t launch_status() {
    return cudaGetLastError() == cudaSuccess ? MOE_OK : MOE_ERR_CUDA;
}

inline bool a16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; }

}  // namespace tb
