// pages_evict.cu -- shortens paged caches to the keys that received most
// attention weight (vvq2_pages_evict), sm_100a.
//
// Per (layer, sequence, KV head) with L keys and m = min(L, keep): the first
// n_first and the last n_recent keys stay, and the m - n_first - n_recent
// others of largest w (ties: the earlier key; NaN below every number).
//   k_evict_select  one CTA per group: a key stays if fewer others beat it
//                   than places are left; writes the kept positions in order
//   k_evict_move    the kept K and V rows to the destination pages
#include "paged_dev.cuh"

namespace vvq2 {

namespace {

// order-preserving unsigned key of a weight; NaN -> 0, -0 -> +0
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int evict_len(const EvictArgs& a, int s) {
    const int l = __ldg(a.kv_len + s), n = min(max(l, 0), min(a.max_kv, a.kv.max_pages * KV_PAGE));
    if (n != l) paged_fault(a.err, PERR_LENGTH);
    return n;
}

__global__ void __launch_bounds__(1024) k_evict_select(const EvictArgs a) {
    __shared__ int count[32], base;
    const int s = (blockIdx.x / a.kv.nkv) % a.kv.n_seqs;
    const int n = evict_len(a, s), m = min(n, a.keep);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0 && blockIdx.x / a.kv.nkv < a.kv.n_seqs && blockIdx.x % a.kv.nkv == 0) a.new_len[s] = m;
    const float* w = a.w + (size_t)blockIdx.x * a.w_stride;
    int* kept = a.kept + (size_t)blockIdx.x * a.keep;
    const int tail = n - a.n_recent, places = m - a.n_first - a.n_recent;
    if (threadIdx.x == 0) base = 0;
    for (int j0 = 0; j0 < n; j0 += 1024) {
        const int j = j0 + threadIdx.x;
        bool stay = j < n;
        if (stay && n > a.keep && j >= a.n_first && j < tail) {
            const uint32_t u = weight_key(w[j]);
            int better = 0;
            for (int i = a.n_first; i < tail; ++i) {
                const uint32_t x = weight_key(__ldg(w + i));
                better += x > u || (x == u && i < j);
            }
            stay = better < places;
        }
        const unsigned b = __ballot_sync(0xffffffffu, stay);
        if (lane == 0) count[warp] = __popc(b);
        __syncthreads();
        int at = base;
        for (int i = 0; i < warp; ++i) at += count[i];
        if (stay) {
            at += __popc(b & ((1u << lane) - 1));
            kept[at] = j;
            if (a.w_out) a.w_out[(size_t)blockIdx.x * a.keep + at] = w[j];
        }
        __syncthreads();
        if (threadIdx.x == 0)
            for (int i = 0; i < 32; ++i) base += count[i];
        __syncthreads();
    }
    for (int i = m + threadIdx.x; i < a.keep; i += 1024) kept[i] = -1;
}

__global__ void __launch_bounds__(256) k_evict_move(const EvictArgs a) {
    const int grp = blockIdx.x, g = grp % a.kv.nkv, s = (grp / a.kv.nkv) % a.kv.n_seqs;
    const int layer = grp / a.kv.nkv / a.kv.n_seqs;
    const int m = min(evict_len(a, s), a.keep), chunks = a.kv.hd / 8;
    const size_t pool = (size_t)layer * a.kv.n_pages * a.kv.nkv * KV_PAGE * a.kv.hd;
    for (int x = blockIdx.y * 256 + threadIdx.x; x < m * chunks; x += gridDim.y * 256) {
        const int i = x / chunks, c = x % chunks, j = a.kept[(size_t)grp * a.keep + i];
        const int sp = paged_page(a.kv.table, a.kv.max_pages, a.kv.n_pages, s, j / KV_PAGE, a.err);
        const int dp = paged_page(a.dst_table, a.dst_max_pages, a.kv.n_pages, s, i / KV_PAGE, a.err);
        if (dp < 0) continue;
        const size_t from = pool + (((size_t)max(sp, 0) * a.kv.nkv + g) * KV_PAGE + j % KV_PAGE) * a.kv.hd + c * 8;
        const size_t to = pool + (((size_t)dp * a.kv.nkv + g) * KV_PAGE + i % KV_PAGE) * a.kv.hd + c * 8;
        const uint4 z = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(const_cast<uint16_t*>(a.kv.k) + to) =
            sp < 0 ? z : *reinterpret_cast<const uint4*>(a.kv.k + from);
        *reinterpret_cast<uint4*>(const_cast<uint16_t*>(a.kv.v) + to) =
            sp < 0 ? z : *reinterpret_cast<const uint4*>(a.kv.v + from);
    }
}

}  // namespace

cudaError_t pages_evict_launch(const EvictArgs& a, int, cudaStream_t st) {
    const unsigned groups = (unsigned)(a.n_layers * a.kv.n_seqs * a.kv.nkv);
    k_evict_select<<<groups, 1024, 0, st>>>(a);
    const int m = min(a.keep, a.max_kv);
    k_evict_move<<<dim3(groups, (unsigned)min(64, (m * (a.kv.hd / 8) + 255) / 256)), 256, 0, st>>>(a);
    note_launch(2);
    return cudaGetLastError();
}

}  // namespace vvq2
