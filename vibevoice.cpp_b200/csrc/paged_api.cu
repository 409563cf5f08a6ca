// paged_api.cu -- C entry points of the operators over caller-owned K/V pages
// (attn_paged.cu, key_weights.cu, pages_evict.cu): argument checks, the device
// the pointers live on, and the launches.  Nothing here allocates, copies or
// synchronizes, so every call may be captured.
#include <math.h>

#include "../../include/vvq2_capi.h"
#include "common.cuh"
#include "kernels.h"

using namespace vvq2;

namespace {

constexpr int MAX_DIM = 1 << 30;   // counts below this keep sums of a few of them in 32 bits

int bad(const char* what) { return set_error(VVQ2_ERR_INVALID_ARG, "%s", what); }

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool overlap(const void* a, size_t an, const void* b, size_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + bn && y < x + an;
}

int check_pages(const vvq2_pages* p, bool need_v) {
    if (!p) return bad("null pages");
    if (!p->k || (need_v && !p->v) || !p->block_table) return bad("null K, V or block table");
    if (p->n_layers <= 0 || p->n_pages <= 0 || p->max_pages <= 0 || p->n_seqs <= 0 || p->n_kv_heads <= 0 ||
        p->n_layers > MAX_DIM || p->n_pages > MAX_DIM || p->max_pages > MAX_DIM / KV_PAGE || p->n_seqs > MAX_DIM / 2)
        return bad("bad page counts");
    if (p->head_dim != 64 && p->head_dim != 128) return bad("head_dim of pages must be 64 or 128");
    if (p->type != VVQ2_TYPE_F16 && p->type != VVQ2_TYPE_BF16) return bad("pages must be f16 or bf16");
    // key rows of a layer are 32-bit coordinates of the tile copies
    if ((int64_t)p->n_pages * p->n_kv_heads > (int64_t)(MAX_DIM / KV_PAGE)) return bad("too many pages x KV heads");
    if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->block_table, 4)) return bad("misaligned pages");
    return 0;
}

PagesView view(const vvq2_pages* p, int layer) {
    PagesView v;
    const int64_t off = (int64_t)layer * p->n_pages * p->n_kv_heads * KV_PAGE * p->head_dim;
    v.k = static_cast<const uint16_t*>(p->k) + off;
    v.v = p->v ? static_cast<const uint16_t*>(p->v) + off : nullptr;
    v.table = p->block_table;
    v.n_pages = p->n_pages;
    v.max_pages = p->max_pages;
    v.n_seqs = p->n_seqs;
    v.nkv = p->n_kv_heads;
    v.hd = p->head_dim;
    v.bf16 = p->type == VVQ2_TYPE_BF16;
    return v;
}

int check_rows(const vvq2_pages* p, int layer, const void* q, int64_t q_stride, const int* q_start, const int* kv_len,
               int total_q, int max_q, int max_kv, int n_heads, float scale) {
    if (layer < 0 || layer >= p->n_layers) return bad("layer outside the pages' layers");
    if (!q_start || !kv_len || (total_q > 0 && !q)) return bad("null q, q_start or kv_len");
    if (total_q < 0 || max_q < 0 || max_kv < 0 || total_q > MAX_DIM || max_q > MAX_DIM || max_kv > MAX_DIM ||
        (total_q > 0 && max_q == 0))
        return bad("bad row or key counts");
    if (n_heads <= 0 || n_heads % p->n_kv_heads || n_heads / p->n_kv_heads > 128)
        return bad("n_heads must be a multiple of n_kv_heads, at most 128 times it");
    if ((int64_t)total_q * n_heads > MAX_DIM) return bad("too many rows x heads");
    if (!(scale > 0.f) || isinf(scale)) return bad("scale must be finite and positive");
    if (q_stride < (int64_t)n_heads * p->head_dim || q_stride % 8 || q_stride > ((int64_t)1 << 38))
        return bad("q_stride must cover a token's heads and be a multiple of 8");
    if (!aligned(q, 16) || !aligned(q_start, 4) || !aligned(kv_len, 4)) return bad("misaligned q, q_start or kv_len");
    return 0;
}

// Runs the call on the GPU that holds its memory, and puts the caller's
// current device back.  All pointers must lie on that one sm_100 GPU.
struct OnDevice {
    int prev = -1, n_sm = 0;
    int enter(const void* const* ptrs, int n, const int* err = nullptr) {
        int dev = -1;
        for (int i = 0; i < n; ++i) {
            if (!ptrs[i]) continue;
            cudaPointerAttributes at{};
            const cudaError_t e = cudaPointerGetAttributes(&at, ptrs[i]);
            if (e != cudaSuccess) {
                cudaGetLastError();
                return e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver
                           ? set_error(VVQ2_ERR_NO_DEVICE, "no sm_100 GPU: %s", cudaGetErrorString(e))
                           : set_error(VVQ2_ERR_CUDA, "cudaPointerGetAttributes: %s", cudaGetErrorString(e));
            }
            if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
                return bad("a pointer is not device memory");
            if (dev < 0) dev = at.device;
            if (at.device != dev && at.type == cudaMemoryTypeDevice) return bad("pointers on different devices");
        }
        if (err) {   // kernels store to it: this GPU's memory, or host memory they can reach
            cudaPointerAttributes at{};
            if (cudaPointerGetAttributes(&at, err) != cudaSuccess || at.type == cudaMemoryTypeUnregistered ||
                (at.type == cudaMemoryTypeDevice && at.device != dev)) {
                cudaGetLastError();
                return bad("err must be device, pinned or managed memory");
            }
        }
        int major = 0;
        cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev);
        int cur = -1;
        if (e == cudaSuccess) e = cudaGetDevice(&cur);
        if (e == cudaSuccess && major != 10)
            return set_error(VVQ2_ERR_NO_DEVICE, "device %d is not an sm_100 GPU", dev);
        if (e == cudaSuccess && cur != dev) {
            e = cudaSetDevice(dev);
            if (e == cudaSuccess) prev = cur;
        }
        if (e != cudaSuccess) return set_error(VVQ2_ERR_CUDA, "%s", cudaGetErrorString(e));
        return 0;
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

int done(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return 0;
    cudaGetLastError();
    return set_error(VVQ2_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

static bool sizes_ok(const vvq2_pages* p, bool need_v, int total_q, int max_q, int max_kv, int n_heads) {
    return !check_pages(p, need_v) && total_q > 0 && max_q > 0 && max_kv > 0 && n_heads > 0 &&
           n_heads % p->n_kv_heads == 0 && n_heads / p->n_kv_heads <= 128 && (int64_t)total_q * n_heads <= MAX_DIM &&
           max_q <= MAX_DIM && max_kv <= MAX_DIM;
}

size_t vvq2_attention_key_weights_workspace(const vvq2_pages* p, int total_q, int max_q, int max_kv, int n_heads) {
    if (!sizes_ok(p, false, total_q, max_q, max_kv, n_heads)) return 0;
    return key_weights_workspace(view(p, 0), total_q, max_q, max_kv, n_heads);
}

size_t vvq2_attention_paged_workspace(const vvq2_pages* p, int total_q, int max_q, int max_kv, int n_heads) {
    if (!sizes_ok(p, true, total_q, max_q, max_kv, n_heads)) return 0;
    OnDevice on;
    const void* ptrs[] = {p->k};
    if (on.enter(ptrs, 1)) return 0;
    return attn_paged_workspace(view(p, 0), total_q, max_q, max_kv, n_heads, on.n_sm);
}

int vvq2_attention_paged(const vvq2_pages* p, int layer, const void* q, int64_t q_stride, const int* q_start,
                         const int* kv_len, int total_q, int max_q, int max_kv, int n_heads, float scale, void* out,
                         int64_t out_stride, float* lse, void* workspace, size_t workspace_bytes, int* err,
                         void* stream) {
    if (int rc = check_pages(p, true)) return rc;
    if (int rc = check_rows(p, layer, q, q_stride, q_start, kv_len, total_q, max_q, max_kv, n_heads, scale)) return rc;
    if (total_q > 0 && !out) return bad("null out");
    if (out_stride < (int64_t)n_heads * p->head_dim || out_stride % 8)
        return bad("out_stride must cover a token's heads and be a multiple of 8");
    if (!aligned(out, 16) || !aligned(lse, 4) || !aligned(workspace, 16) || !aligned(err, 4))
        return bad("misaligned out, lse, workspace or err");
    if (total_q == 0) return 0;
    OnDevice on;
    const void* ptrs[] = {p->k, p->v, p->block_table, q, q_start, kv_len, out, lse, workspace};
    if (int rc = on.enter(ptrs, 9, err)) return rc;
    PagedAttnArgs a;
    a.kv = view(p, layer);
    a.q = static_cast<const uint16_t*>(q);
    a.q_stride = q_stride;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.total_q = total_q;
    a.max_q = max_q;
    a.max_kv = max_kv;
    a.nq = n_heads;
    a.scale = scale;
    a.out = static_cast<uint16_t*>(out);
    a.out_stride = out_stride;
    a.lse = lse;
    a.workspace = workspace;
    a.workspace_bytes = workspace ? workspace_bytes : 0;
    a.err = err;
    return done(attn_paged_launch(a, on.n_sm, static_cast<cudaStream_t>(stream)), "attention_paged");
}

int vvq2_attention_key_weights(const vvq2_pages* p, int layer, const void* q, int64_t q_stride, const float* lse,
                               const int* q_start, const int* kv_len, int total_q, int max_q, int max_kv, int n_heads,
                               float scale, const float* w_in, float* w_out, int64_t w_stride, void* workspace,
                               size_t workspace_bytes, int* err, void* stream) {
    if (int rc = check_pages(p, false)) return rc;
    if (int rc = check_rows(p, layer, q, q_stride, q_start, kv_len, total_q, max_q, max_kv, n_heads, scale)) return rc;
    if (!w_out || (total_q > 0 && !lse)) return bad("null lse or w_out");
    if (w_stride < max_kv || w_stride > MAX_DIM) return bad("w_stride must be at least max_kv");
    if (!aligned(lse, 4) || !aligned(w_in, 4) || !aligned(w_out, 4) || !aligned(workspace, 16) || !aligned(err, 4))
        return bad("misaligned lse, w_in, w_out, workspace or err");
    const size_t wn = (size_t)p->n_seqs * p->n_kv_heads * w_stride * 4;
    if (w_in != w_out && overlap(w_in, wn, w_out, wn)) return bad("w_in and w_out overlap without being the same");
    if (max_kv == 0) return 0;
    OnDevice on;
    const void* ptrs[] = {p->k, p->block_table, q, lse, q_start, kv_len, w_in, w_out, workspace};
    if (int rc = on.enter(ptrs, 9, err)) return rc;
    KeyWeightArgs a;
    a.kv = view(p, layer);
    a.q = static_cast<const uint16_t*>(q);
    a.q_stride = q_stride;
    a.lse = lse;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.total_q = total_q;
    a.max_q = max_q;
    a.max_kv = max_kv;
    a.nq = n_heads;
    a.scale = scale;
    a.w_in = w_in;
    a.w_out = w_out;
    a.w_stride = w_stride;
    a.workspace = workspace;
    a.workspace_bytes = workspace ? workspace_bytes : 0;
    a.err = err;
    return done(key_weights_launch(a, on.n_sm, static_cast<cudaStream_t>(stream)), "attention_key_weights");
}

int vvq2_pages_evict(const vvq2_pages* p, const int* dst_table, int dst_max_pages, const int* kv_len, int max_kv,
                     const float* w, int64_t w_stride, int keep, int n_first, int n_recent, int* kept, float* w_out,
                     int* new_len, int* err, void* stream) {
    if (int rc = check_pages(p, true)) return rc;
    if (!dst_table || !kv_len || !w || !kept || !new_len) return bad("null dst_table, kv_len, w, kept or new_len");
    if (max_kv <= 0 || max_kv > MAX_DIM || w_stride < max_kv || w_stride > MAX_DIM)
        return bad("w_stride must be at least max_kv, max_kv positive");
    if (keep <= 0 || keep > MAX_DIM || n_first < 0 || n_recent < 0 || n_first > keep || n_recent > keep - n_first)
        return bad("n_first + n_recent must be at most keep, keep positive");
    if (dst_max_pages <= 0 || dst_max_pages > MAX_DIM / KV_PAGE ||
        (int64_t)dst_max_pages * KV_PAGE < (keep < max_kv ? keep : max_kv))
        return bad("dst_table has too few pages for keep keys");
    const int64_t groups = (int64_t)p->n_layers * p->n_seqs * p->n_kv_heads;
    if (groups > MAX_DIM / 64) return bad("too many layers x sequences x KV heads");
    if (groups * (((keep < max_kv ? keep : max_kv) + KV_PAGE - 1) / KV_PAGE) > 0x7fffffff)   // (a block each)
        return bad("too many pages to move");
    if (!aligned(dst_table, 4) || !aligned(kv_len, 4) || !aligned(w, 4) || !aligned(kept, 4) || !aligned(w_out, 4) ||
        !aligned(new_len, 4) || !aligned(err, 4))
        return bad("misaligned argument");
    const size_t lens = (size_t)p->n_seqs * 4, wn = (size_t)groups * w_stride * 4, kn = (size_t)groups * keep * 4;
    if (overlap(new_len, lens, kv_len, lens)) return bad("new_len overlaps kv_len");
    if (overlap(dst_table, lens * dst_max_pages, p->block_table, lens * p->max_pages))
        return bad("dst_table overlaps the block table");
    if (overlap(w_out, kn, w, wn) || overlap(kept, kn, w, wn) || overlap(w_out, kn, kept, kn))
        return bad("w, kept and w_out must not overlap");
    OnDevice on;
    const void* ptrs[] = {p->k, p->v, p->block_table, dst_table, kv_len, w, kept, w_out, new_len};
    if (int rc = on.enter(ptrs, 9, err)) return rc;
    EvictArgs a;
    a.kv = view(p, 0);
    a.n_layers = p->n_layers;
    a.dst_table = dst_table;
    a.dst_max_pages = dst_max_pages;
    a.kv_len = kv_len;
    a.max_kv = max_kv;
    a.w = w;
    a.w_stride = w_stride;
    a.keep = keep;
    a.n_first = n_first;
    a.n_recent = n_recent;
    a.kept = kept;
    a.w_out = w_out;
    a.new_len = new_len;
    a.err = err;
    return done(pages_evict_launch(a, on.n_sm, static_cast<cudaStream_t>(stream)), "pages_evict");
}

}  // extern "C"
