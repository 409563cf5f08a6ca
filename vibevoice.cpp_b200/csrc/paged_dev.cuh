// paged_dev.cuh -- device helpers of the operators over caller-owned K/V
// pages: bounded reads of the device-side lengths and tables.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace vvq2 {

__device__ __forceinline__ void paged_fault(int* err, int code) {
    if (err) *(volatile int*)err = code;
}

struct SeqRows {
    int row0 = 0, n = 0;   // packed rows of the sequence
    int len = 0;           // its cached keys
};

// Sequence s's rows and keys, cut to the bounds the host gave (so no later
// index leaves the arrays, whatever the device words hold).
__device__ __forceinline__ SeqRows paged_seq(const PagesView& kv, const int* q_start, const int* kv_len, int total_q,
                                             int max_q, int max_kv, int s, int* err) {
    SeqRows r;
    const int a = __ldg(q_start + s), b = __ldg(q_start + s + 1), l = __ldg(kv_len + s);
    r.row0 = min(max(a, 0), total_q);
    const int end = min(max(b, r.row0), total_q);
    r.n = min(end - r.row0, max_q);
    r.len = min(max(l, 0), min(max_kv, kv.max_pages * KV_PAGE));
    if (r.row0 != a || r.row0 + r.n != b || r.len != l) paged_fault(err, PERR_LENGTH);
    return r;
}

// Physical page of a sequence's logical page, or -1 (and the error word) if
// the table names none of the pool's.
__device__ __forceinline__ int paged_page(const int* table, int max_pages, int n_pages, int s, int lp, int* err) {
    const int p = __ldg(table + (size_t)s * max_pages + lp);
    if ((unsigned)p < (unsigned)n_pages) return p;
    paged_fault(err, PERR_PAGE);
    return -1;
}

template <bool BF16>
__device__ __forceinline__ float from16(uint16_t x) {
    if (BF16) return __uint_as_float((uint32_t)x << 16);
    return __half2float(__ushort_as_half(x));
}
template <bool BF16>
__device__ __forceinline__ uint16_t to16(float x) {
    if (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
    return __half_as_ushort(__float2half_rn(x));
}

}  // namespace vvq2
