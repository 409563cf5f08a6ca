// key_weights.cu -- the attention weight each cached key receives from a
// packed chunk of queries (vvq2_attention_key_weights), sm_100a.
//
//   W[s][g][j] = sum over rows t, h of s in group g with j < lim(t) of
//                exp(scale q[t][h].K[j][g] - lse[t][h])
//
// One warp per (sequence, KV head, key): lanes take the (t, h) pairs in turn,
// a shuffle tree in fixed order adds their sums.
#include "paged_dev.cuh"

namespace vvq2 {

namespace {

template <int HD, bool BF16>
__global__ void __launch_bounds__(128) k_key_weights(const KeyWeightArgs a) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s = blockIdx.y, g = blockIdx.z, G = a.nq / a.kv.nkv;
    const SeqRows r = paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, s, a.err);
    for (int j = blockIdx.x * 4 + warp; j < r.len; j += gridDim.x * 4) {
        const int page = paged_page(a.kv.table, a.kv.max_pages, a.kv.n_pages, s, j / KV_PAGE, a.err);
        const uint16_t* k = a.kv.k + (((size_t)max(page, 0) * a.kv.nkv + g) * KV_PAGE + j % KV_PAGE) * HD;
        const int t0 = max(0, j - (r.len - r.n));   // the first token that sees key j
        float w = 0.f;
        for (int64_t i = (int64_t)t0 * G + lane; i < (int64_t)r.n * G; i += 32) {
            const int row = r.row0 + (int)(i / G), h = g * G + (int)(i % G);
            const uint16_t* q = a.q + row * a.q_stride + h * HD;
            float x = 0.f;
            for (int e = 0; e < HD; ++e) x += from16<BF16>(q[e]) * (page < 0 ? 0.f : from16<BF16>(k[e]));
            w += expf(x * a.scale - a.lse[(size_t)row * a.nq + h]);
        }
        w = warp_sum(w);
        if (lane == 0) {
            const size_t at = ((size_t)s * a.kv.nkv + g) * a.w_stride + j;
            if (a.w_in && j < r.len - r.n) w += a.w_in[at];
            a.w_out[at] = w;
        }
    }
}

}  // namespace

cudaError_t key_weights_launch(const KeyWeightArgs& a, int, cudaStream_t st) {
    if (a.kv.n_seqs > 65535 || a.kv.nkv > 65535) return cudaErrorInvalidValue;
    const dim3 grid((unsigned)((a.max_kv + 3) / 4), (unsigned)a.kv.n_seqs, (unsigned)a.kv.nkv);
    if (a.kv.hd == 64) {
        if (a.kv.bf16) k_key_weights<64, true><<<grid, 128, 0, st>>>(a);
        else k_key_weights<64, false><<<grid, 128, 0, st>>>(a);
    } else {
        if (a.kv.bf16) k_key_weights<128, true><<<grid, 128, 0, st>>>(a);
        else k_key_weights<128, false><<<grid, 128, 0, st>>>(a);
    }
    note_launch();
    return cudaGetLastError();
}

}  // namespace vvq2
