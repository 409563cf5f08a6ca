// attn_paged.cuh -- what the two kernels of the paged attention share: the plan
// of a launch, and the treatment of V rows that not every row may see.
#pragma once

#include "paged_dev.cuh"

namespace vvq2 {

constexpr int BKV = KV_PAGE;                // keys per tile: one page
constexpr int PAGE_BYTES = KV_PAGE * 128;   // one 64-key box of 64 columns, 128-byte swizzle

struct AttnPlan {
    int T = 0, G = 0, direct = 0, few = 0;
    int n_tiles = 0;      // upper bound of (sequence, 2T tokens) tiles
    int nsplit = 1, spt = 0;   // key splits and key tiles per split
    float c = 0.f;        // scale * log2(e)
    // A split's rows: (token, head), tokens numbered as packed, or, with a tile
    // per sequence (direct), max_q to each sequence: total_q may be far larger,
    // where the call has a few sequences of a packed batch.
    int64_t tokens = 0;
    float* part = nullptr;     // [nsplit][tokens * nq][hd]
    float2* part_ml = nullptr; // [nsplit][tokens * nq] (m in log2 units, sum)
    // row of a split: token t of sequence s, which is packed row `tok`
    __device__ __forceinline__ size_t part_row(const PagedAttnArgs& a, int split, int s, int t, int tok, int h) const {
        return ((size_t)split * tokens + (direct ? (size_t)s * a.max_q + t : (size_t)tok)) * a.nq + h;
    }
};

// Calls of at most FEW_ROWS rows a sequence (max_q x G) go to attn_paged_few.cu:
// 128 sequences of 7 rows and up to 2047 keys take 23 us there, 46 in the 128-row
// kernel.  It has forms of one and two row tiles.
constexpr int FEW_ROWS = 32;
cudaError_t attn_paged_few_launch(const PagedAttnArgs& a, const AttnPlan& p, const CUtensorMap& mk,
                                  const CUtensorMap& mv, cudaStream_t st);

// Records that the V element of key lim0 + off in this column is +inf, -inf or
// NaN (kind 0, 1, 2): a byte per kind with the first such off (255: none; off
// <= 254, since an item has at most 256 tokens).
constexpr uint32_t NO_BAD = 0xffffffu;
__device__ __forceinline__ void note_bad(uint32_t* word, int off, int kind) {
    const uint32_t sh = 8 * kind;
    uint32_t old = *(volatile uint32_t*)word;
    while ((int)(old >> sh & 0xff) > off) {
        const uint32_t seen = atomicCAS(word, old, (old & ~(0xffu << sh)) | (uint32_t)off << sh);
        if (seen == old) return;
        old = seen;
    }
}
// What a row that sees `seen` keys from lim0 on gets added in a column.
__device__ __forceinline__ float add_bad(float x, uint32_t word, int seen) {
    if ((int)(word & 0xff) < seen) x += INFINITY;
    if ((int)(word >> 8 & 0xff) < seen) x -= INFINITY;
    if ((int)(word >> 16 & 0xff) < seen) x += NAN;
    return x;
}

// Takes out of a V tile in shared memory what some row must not read, in keys
// [r0, r2): those from r1 on (no row sees them) become zeros, and non-finite
// elements of those before it (some rows see them) are recorded in bad[], with
// has_bad set, and become zeros.  off0: key 0 of the tile less lim0.  By
// `nthreads` threads, of which this is number `th`.  Few tiles need it, and
// inlined it takes registers of the softmax loop (24 packed prompts 181.8
// against 177.9 us).
template <int HD, bool BF16>
__device__ __noinline__ void clean_v(uint8_t* vt, int r0, int r1, int r2, int off0, uint32_t* bad, int* has_bad,
                                        int th, int nthreads) {
    constexpr int CH = HD / 8;   // 16-byte chunks per row
    constexpr uint32_t EXP = BF16 ? 0x7f80u : 0x7c00u;
    for (int i = th; i < (r2 - r0) * CH; i += nthreads) {
        const int r = r0 + i / CH, e = i % CH, b = e >> 3;
        const int ch = (e & 7) ^ (r & 7);   // 128-byte swizzle: the logical chunk
        uint4* q = reinterpret_cast<uint4*>(vt + b * PAGE_BYTES + r * 128 + (e & 7) * 16);
        if (r >= r1) {
            *q = make_uint4(0, 0, 0, 0);
            continue;
        }
        const uint4 v = *q;
        uint32_t u[4] = {v.x, v.y, v.z, v.w};
        bool hit = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) hit |= (u[k] & EXP) == EXP || ((u[k] >> 16) & EXP) == EXP;
        if (!hit) continue;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t sh = (k & 1) * 16, x = (u[k >> 1] >> sh) & 0xffffu;
            if ((x & EXP) != EXP) continue;
            const int kind = (x & 0x7fffu) != EXP ? 2 : x >> 15;   // nan, -inf, +inf
            note_bad(bad + b * 64 + ch * 8 + k, off0 + r, kind);
            u[k >> 1] &= ~(0xffffu << sh);
        }
        *(volatile int*)has_bad = 1;
        *q = make_uint4(u[0], u[1], u[2], u[3]);
    }
    tc::fence_proxy_async_smem();
}

}  // namespace vvq2
