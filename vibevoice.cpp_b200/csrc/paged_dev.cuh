// paged_dev.cuh -- device helpers of the operators over caller-owned K/V
// pages: bounded reads of the device-side lengths and tables.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "tc.cuh"

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

__device__ __forceinline__ float ex2(float x) {   // 2^x on the special-function unit (~2 ulp, -inf -> +0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two f32 operations in one instruction, each rounded as the plain one
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {   // in one instruction
    float m;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// ---- between the warps of a block.  CT: the block's control block in shared
// memory, with abort_flag, the kernel's arguments a, and a two-slot item queue
// (item, it_full, it_empty).
template <class CT>
__device__ __forceinline__ bool aborted(const CT& ctl) {
    return *(volatile const int*)&ctl.abort_flag != 0;
}
// bounded, and cut short when another warp gave up
template <class CT>
__device__ __forceinline__ bool wait(CT& ctl, uint64_t* bar, uint32_t parity) {
    for (int i = 0; i < (1 << 12); ++i) {
        if (tc::mbar_wait(bar, parity, 1u << 10)) return true;
        if (aborted(ctl)) return false;
    }
    paged_fault(ctl.a.err, PERR_WAIT);
    *(volatile int*)&ctl.abort_flag = 1;
    return false;
}
// A role's n-th item, in shared memory until the role says it is done with it;
// null when there are no more (or a wait gave up).
template <class CT>
__device__ __forceinline__ auto take(CT& ctl, int n) -> decltype(&ctl.item[0]) {
    const bool ok = wait(ctl, &ctl.it_full[n & 1], (n >> 1) & 1);
    return __all_sync(0xffffffffu, ok) && ctl.item[n & 1].valid ? &ctl.item[n & 1] : nullptr;
}
template <class CT>
__device__ __forceinline__ void done_with(CT& ctl, int n) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc::mbar_arrive(&ctl.it_empty[n & 1]);
}

}  // namespace vvq2
