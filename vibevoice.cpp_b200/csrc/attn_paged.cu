// attn_paged.cu -- causal attention of packed chunks of new tokens over a
// paged K/V cache (vvq2_attention_paged), sm_100a.
//
// Token t of sequence s, with n new tokens and L cached keys, sees the keys
// j < lim = L - n + t + 1:
//   out = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale q.K_j - m),  m = max_j,
//   lse = m + log sum_j p_j,
// in one pass over the keys with a running m, sum and output.
//
// One warp per (token, head): each lane holds hd / 32 of the head's columns.
#include "paged_dev.cuh"

namespace vvq2 {

namespace {

template <int HD, bool BF16>
__global__ void __launch_bounds__(128) k_attn_paged(const PagedAttnArgs a) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s = blockIdx.y, G = a.nq / a.kv.nkv;
    const SeqRows r = paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, s, a.err);
    for (int64_t i = (int64_t)blockIdx.x * 4 + warp; i < (int64_t)r.n * a.nq; i += (int64_t)gridDim.x * 4) {
        const int t = (int)(i / a.nq), h = (int)(i % a.nq), g = h / G, row = r.row0 + t;
        const int lim = min(r.len - r.n + t + 1, r.len);
        float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            q[e] = from16<BF16>(a.q[row * a.q_stride + h * HD + lane * E + e]) * a.scale;
            o[e] = 0.f;
        }
        for (int j = 0; j < lim; ++j) {
            const int page = paged_page(a.kv.table, a.kv.max_pages, a.kv.n_pages, s, j / KV_PAGE, a.err);
            const size_t at = (((size_t)max(page, 0) * a.kv.nkv + g) * KV_PAGE + j % KV_PAGE) * HD + lane * E;
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) x += q[e] * (page < 0 ? 0.f : from16<BF16>(a.kv.k[at + e]));
            x = warp_sum(x);
            const float mn = fmaxf(m, x);
            const float c = m == -INFINITY ? 0.f : expf(m - mn);   // a first key replaces an empty sum
            const float p = x == -INFINITY ? 0.f : expf(x - mn);
            l = l * c + p;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * (page < 0 ? 0.f : from16<BF16>(a.kv.v[at + e]));
            m = mn;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int e = 0; e < E; ++e) a.out[row * a.out_stride + h * HD + lane * E + e] = to16<BF16>(o[e] * inv);
        if (a.lse && lane == 0) a.lse[(size_t)row * a.nq + h] = l == 0.f ? -INFINITY : m + logf(l);
    }
}

}  // namespace

size_t attn_paged_workspace(const PagesView&, int, int, int, int, int) { return 0; }

cudaError_t attn_paged_launch(const PagedAttnArgs& a, int, cudaStream_t st) {
    const long long warps = (long long)min(a.max_q, a.total_q) * a.nq;
    const dim3 grid((unsigned)min((warps + 3) / 4, 1LL << 16), (unsigned)a.kv.n_seqs);
    if (a.kv.n_seqs > 65535) return cudaErrorInvalidValue;
    if (a.kv.hd == 64) {
        if (a.kv.bf16) k_attn_paged<64, true><<<grid, 128, 0, st>>>(a);
        else k_attn_paged<64, false><<<grid, 128, 0, st>>>(a);
    } else {
        if (a.kv.bf16) k_attn_paged<128, true><<<grid, 128, 0, st>>>(a);
        else k_attn_paged<128, false><<<grid, 128, 0, st>>>(a);
    }
    note_launch();
    return cudaGetLastError();
}

}  // namespace vvq2
