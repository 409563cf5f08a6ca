// pages_evict.cu -- shortens paged caches to the keys that received most
// attention weight (vvq2_pages_evict), sm_100a.
//
// Per (layer, sequence, KV head) with L keys and m = min(L, keep): the first
// n_first and the last n_recent keys stay, and the m - n_first - n_recent
// others of largest w (ties: the earlier key; NaN below every number).
//   k_evict_select  a block per group.  Weights become order-preserving 32-bit
//                   keys in shared memory (read from global memory again where
//                   they do not fit); four 8-bit histogram passes from the top
//                   find the key T of the last place and how many of its equals
//                   stay; each warp then lists its range in order, after a scan
//                   of the warps' counts.  One read of w; the passes run at the
//                   rate of shared memory.
//   k_evict_move    a block per destination page: 64 kept rows of K and V, all
//                   loads in flight before the first store.  Bound by HBM:
//                   source and destination pages differ, so blocks need no order.
// Measured: 27,000 keys to 8192, 28 layers, 4 heads of 128, 188 us for 0.96 GB =
// 5.1 TB/s over both; 16 ragged streams, 24 layers, 2 heads of 64, 59 us,
// about 17 of them the selection.
#include "paged_dev.cuh"

namespace vvq2 {

namespace {

constexpr int CACHED_KEYS = 50 * 1024;   // 200 KB of shared memory

// order-preserving unsigned key of a weight; NaN -> 0, -0 -> +0
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int evict_len(const EvictArgs& a, int s, int* err) {
    const int l = __ldg(a.kv_len + s), n = min(max(l, 0), min(a.max_kv, a.kv.max_pages * KV_PAGE));
    if (n != l) paged_fault(err, PERR_LENGTH);
    return n;
}

template <bool CACHED>
__global__ void __launch_bounds__(1024) k_evict_select(const EvictArgs a) {
    extern __shared__ uint32_t keys[];
    __shared__ int hist[8][256], sure_of[32], same_of[32], digit, rest;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int s = (blockIdx.x / a.kv.nkv) % a.kv.n_seqs;
    const int n = evict_len(a, s, threadIdx.x ? nullptr : a.err), m = min(n, a.keep);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
    // 32 warps count into eight histograms: weights crowd in few leading digits
    // (27,000 keys x 112 groups 204 us in one, 188 in eight; smaller blocks lose 3 %)
    const int copies = nwarps == 32 ? 8 : 1;
    if (threadIdx.x == 0 && blockIdx.x / a.kv.nkv < a.kv.n_seqs && blockIdx.x % a.kv.nkv == 0) a.new_len[s] = m;
    const float* w = a.w + (size_t)blockIdx.x * a.w_stride;
    int* kept = a.kept + (size_t)blockIdx.x * a.keep;
    float* w_out = a.w_out ? a.w_out + (size_t)blockIdx.x * a.keep : nullptr;
    for (int i = m + threadIdx.x; i < a.keep; i += blockDim.x) kept[i] = -1;
    if (n <= a.keep) {   // all stay
        for (int j = threadIdx.x; j < n; j += blockDim.x) {
            kept[j] = j;
            if (w_out) w_out[j] = w[j];
        }
        return;
    }
    const int first = a.n_first, tail = n - a.n_recent;   // [first, tail) compete
    if (CACHED)
        for (int j = threadIdx.x; j < n; j += blockDim.x) keys[j] = weight_key(w[j]);
    auto key_of = [&](int j) { return CACHED ? keys[j] : weight_key(__ldg(w + j)); };
    // T: the key of the last place; `places` of T's equals stay
    uint32_t T = 0xffffffffu;   // (no weight has this key)
    int places = m - a.n_first - a.n_recent;
    if (places > 0) {
        uint32_t mask = 0;
        T = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = threadIdx.x; i < copies * 256; i += blockDim.x) hist[0][i] = 0;
            __syncthreads();
            for (int j = first + threadIdx.x; j < tail; j += blockDim.x) {
                const uint32_t k = key_of(j);
                if ((k & mask) == T) atomicAdd(&hist[warp & (copies - 1)][k >> shift & 255], 1);
            }
            __syncthreads();
            if (warp == 0) {   // lane l holds digits 255 - 8l .. 248 - 8l
                int c[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    c[i] = 0;
                    for (int z = 0; z < copies; ++z) c[i] += hist[z][255 - lane * 8 - i];
                    sum += c[i];
                }
                int upto = sum;   // keys with this lane's digits or higher ones
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                if (upto >= places && upto - sum < places) {   // one lane
                    int above = upto - sum, i = 0;
                    while (above + c[i] < places) above += c[i++];
                    digit = 255 - lane * 8 - i;
                    rest = places - above;
                }
            }
            __syncthreads();
            T |= (uint32_t)digit << shift;
            places = rest;
            mask |= 255u << shift;
        }
    } else {
        __syncthreads();
    }
    // warp's range of keys: whole groups of 32
    const int span = ((n + nwarps - 1) / nwarps + 31) / 32 * 32, j0 = warp * span, j1 = min(n, j0 + span);
    auto sure = [&](int j, uint32_t k) { return j < first || j >= tail || k > T; };
    int sures = 0, sames = 0;
    for (int j = j0 + lane; j < j1; j += 32) {
        const uint32_t k = key_of(j);
        const bool y = sure(j, k);
        sures += y;
        sames += !y && k == T;
    }
    sures = __reduce_add_sync(0xffffffffu, sures);
    sames = __reduce_add_sync(0xffffffffu, sames);
    if (lane == 0) {
        sure_of[warp] = sures;
        same_of[warp] = sames;
    }
    __syncthreads();
    int at = 0, equal = 0;   // keys listed, and equals of T passed, before this warp's range
    for (int i = 0; i < warp; ++i) {
        at += sure_of[i] + min(same_of[i], max(0, places - equal));
        equal += same_of[i];
    }
    const unsigned below = (1u << lane) - 1;
    for (int j = j0; j < j1; j += 32) {
        const bool in = j + lane < j1;
        const uint32_t k = in ? key_of(j + lane) : 0;
        const bool y = in && sure(j + lane, k), e = in && !y && k == T;
        const unsigned eb = __ballot_sync(0xffffffffu, e);
        const bool stay = y || (e && equal + __popc(eb & below) < places);
        const unsigned sb = __ballot_sync(0xffffffffu, stay);
        if (stay) {
            const int i = at + __popc(sb & below);
            kept[i] = j + lane;
            if (w_out) w_out[i] = w[j + lane];
        }
        at += __popc(sb);
        equal += __popc(eb);
    }
}

// HC: 16-byte chunks of a row
template <int HC>
__global__ void __launch_bounds__(256) k_evict_move(const EvictArgs a) {
    __shared__ int64_t from[KV_PAGE];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int pages = (min(a.keep, a.max_kv) + KV_PAGE - 1) / KV_PAGE;
    const int grp = blockIdx.x / pages, page = blockIdx.x % pages;
    const int g = grp % a.kv.nkv, s = (grp / a.kv.nkv) % a.kv.n_seqs, layer = grp / a.kv.nkv / a.kv.n_seqs;
    const int rows = min(KV_PAGE, min(evict_len(a, s, nullptr), a.keep) - page * KV_PAGE);
    if (rows <= 0) return;
    const int dp = paged_page(a.dst_table, a.dst_max_pages, a.kv.n_pages, s, page, threadIdx.x ? nullptr : a.err);
    if (dp < 0) return;
    const int64_t head = (int64_t)layer * a.kv.n_pages * a.kv.nkv;   // rows are counted in (page, head) blocks
    if (threadIdx.x < rows) {
        const int j = a.kept[(size_t)grp * a.keep + page * KV_PAGE + threadIdx.x];
        const int sp = paged_page(a.kv.table, a.kv.max_pages, a.kv.n_pages, s, j / KV_PAGE, a.err);
        from[threadIdx.x] = sp < 0 ? -1 : ((head + (int64_t)sp * a.kv.nkv + g) * KV_PAGE + j % KV_PAGE) * HC;
    }
    __syncthreads();
    const uint4 *k = reinterpret_cast<const uint4*>(a.kv.k), *v = reinterpret_cast<const uint4*>(a.kv.v);
    const int64_t to = (head + (int64_t)dp * a.kv.nkv + g) * KV_PAGE * HC;
    constexpr int N = KV_PAGE * HC / 256;
    uint4 x[N], y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = threadIdx.x + i * 256, r = c / HC;
        x[i] = y[i] = make_uint4(0, 0, 0, 0);
        if (r < rows && from[r] >= 0) {
            x[i] = __ldcs(k + from[r] + c % HC);
            y[i] = __ldcs(v + from[r] + c % HC);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = threadIdx.x + i * 256;
        if (c / HC < rows) {
            const_cast<uint4*>(k)[to + c] = x[i];
            const_cast<uint4*>(v)[to + c] = y[i];
        }
    }
}

}  // namespace

cudaError_t pages_evict_launch(const EvictArgs& a, int, cudaStream_t st) {
    const unsigned groups = (unsigned)(a.n_layers * a.kv.n_seqs * a.kv.nkv);
    // (512 threads for 27,000 keys: 22 us more; 256 for 2000: 1 % more)
    const int threads = a.max_kv <= 1024 ? 256 : a.max_kv <= 4096 ? 512 : 1024;
    if (a.max_kv <= CACHED_KEYS) {
        const cudaError_t e = cudaFuncSetAttribute(k_evict_select<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   CACHED_KEYS * 4);
        if (e != cudaSuccess) return e;
        k_evict_select<true><<<groups, threads, a.max_kv * 4, st>>>(a);
    } else {
        k_evict_select<false><<<groups, threads, 0, st>>>(a);
    }
    note_launch();
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const unsigned blocks = groups * ((min(a.keep, a.max_kv) + KV_PAGE - 1) / KV_PAGE);   // (checked by the caller)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    e = a.kv.hd == 64 ? cudaLaunchKernelEx(&cfg, k_evict_move<8>, a) : cudaLaunchKernelEx(&cfg, k_evict_move<16>, a);
    note_launch();
    return e;
}

}  // namespace vvq2
