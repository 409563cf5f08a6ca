// attn_paged_few.cu -- vvq2_attention_paged for sequences with few rows (a
// decode step, some drafted tokens): at most FEW_ROWS = 32 (token, head) rows
// per KV head, sm_100a.
//
// With so few rows the work is reading K and V once.  A 128-row tensor-core
// tile would spend its softmax on rows that do not exist (one thread per row:
// 64 exponentials a page in each, whatever the number of rows; that kernel
// takes some 0.6 us a page, 2-4 TB/s over the GPU), so here warp-level
// 16-row products spread the scores of a page over all lanes.
//
// A block takes one (sequence, KV head, key range).  The G heads of the KV head
// times the new tokens are its rows, in MT tiles of 16.  Pages of K and V come
// by TMA into a ring and go in turn to two teams of four warps; of a page's 64
// keys, warp w of the team takes 16 MT (part w / MT) for row tile w % MT, with
// its own running maximum, sum and output, which all parts add up in shared
// memory at the end.  A page is a short chain of dependent steps (wait, scores,
// maximum, exponentials, output), so the second team nearly halves its time.
//   S = Q K^T   m16n8k16, Q in registers, K rows by ldmatrix
//   O += P V    P from the S accumulators, rounded to V's type (the product
//               takes one), V by ldmatrix.trans
// Masked V rows are treated as in attn_paged.cu.
//
// Measured: 128 rows of 64 to 2047 keys, 14/2 heads of 64, 22.6 us = 3.1 TB/s of
// K and V; one row of 27,001 keys, 28/4 heads of 128, 22 us with the merge.
// Bound by a page's chain of dependent steps in each team, not by HBM.
#include "attn_paged.cuh"

namespace vvq2 {

namespace {

constexpr int TEAM = 4;                       // warps that share a page
constexpr int WARPS = 2 * TEAM;               // of products; one more loads
constexpr int THREADS = (WARPS + 1) * 32;

template <int HD>
struct Cfg {
    static constexpr int NB = HD / 64;
    static constexpr int HALF = NB * PAGE_BYTES;            // K or V of a page
    static constexpr int SLOT = 2 * HALF;
    // An even number: a slot's pages all go to one team, so a team that waits
    // for a slot's phase has seen the phase before it.
    static constexpr int NS = 6;                            // 192 or 96 KB
    static constexpr int PER_SM = HD == 128 ? 1 : 2;        // blocks
    static constexpr int CTL_OFF = NS * SLOT;
};

template <int HD>
struct Ctl {
    uint64_t full[Cfg<HD>::NS], empty[Cfg<HD>::NS];
    PagedAttnArgs a;
    int abort_flag, has_bad;
    uint32_t bad[HD];
    float2 ml[WARPS][16];
};

template <int HD>
constexpr int smem_bytes() {
    return Cfg<HD>::CTL_OFF + (int)sizeof(Ctl<HD>);
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16-byte chunk ch (8 columns) of key row r in a page's swizzled 64-column blocks
__device__ __forceinline__ uint32_t chunk(uint32_t page, int r, int ch) {
    return page + (ch >> 3) * PAGE_BYTES + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
}

template <int HD, bool BF16, int MT>
__global__ void __launch_bounds__(THREADS, Cfg<HD>::PER_SM)
    k_attn_paged_few(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                     const PagedAttnArgs a, const AttnPlan p) {
    using C = Cfg<HD>;
    constexpr int PARTS = TEAM / MT, NT = 2 * MT, KS = HD / 16;   // n-tiles of 8 keys per warp; k steps
    extern __shared__ __align__(1024) uint8_t sm[];
    Ctl<HD>& ctl = *reinterpret_cast<Ctl<HD>*>(sm + C::CTL_OFF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % p.nsplit, g = blockIdx.x / p.nsplit % a.kv.nkv, s = blockIdx.x / p.nsplit / a.kv.nkv;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const SeqRows seq = paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, s,
                                  threadIdx.x || split || g ? nullptr : a.err);
    if (seq.n == 0) return;
    if (tc::smem_u32(sm) & 1023) {   // the swizzle's atoms; the kernel has no static shared memory
        paged_fault(a.err, PERR_WAIT);
        return;
    }
    const int rows = seq.n * p.G, lim0 = seq.len - seq.n + 1, last = seq.len;   // keys of the first, the last token
    const int kt0 = split * p.spt;
    const int J = max(0, min((last + BKV - 1) / BKV, kt0 + p.spt) - kt0);
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NS; ++i) {
            tc::mbar_init(&ctl.full[i], 1);
            tc::mbar_init(&ctl.empty[i], TEAM);
        }
        ctl.abort_flag = 0;
        ctl.has_bad = 0;
        ctl.a = a;
        tc::mbar_fence_init();
    }
    for (int i = threadIdx.x; i < HD; i += THREADS) ctl.bad[i] = NO_BAD;
    __syncthreads();

    // a row's keys: its token's limit
    const int mt = warp % MT, part = warp % TEAM / MT, team = warp / TEAM;
    const int r0 = mt * 16 + (lane >> 2);   // this lane's rows: r0 and r0 + 8
    float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][k] = 0.f;

    if (warp == WARPS) {
        // ---- loads
        bool ok = true;
        int j = 0, page = -1;
        for (; j < J; ++j) {
            if (j % 32 == 0)
                page = j + lane < J ? paged_page(a.kv.table, a.kv.max_pages, a.kv.n_pages, s, kt0 + j + lane, a.err)
                                    : -1;
            const int pg = __shfl_sync(0xffffffffu, page, j & 31);
            // no page: rows past the pool's, which read as zeros
            const int y = (pg >= 0 ? pg * a.kv.nkv + g : a.kv.n_pages * a.kv.nkv) * KV_PAGE;
            const int st = j % C::NS, use = j / C::NS;
            ok = use == 0 || wait(ctl, &ctl.empty[st], (use - 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) break;
            if (lane == 0) {
                uint8_t* dst = sm + st * C::SLOT;
                tc::mbar_arrive_expect_tx(&ctl.full[st], C::SLOT);
#pragma unroll
                for (int b = 0; b < C::NB; ++b) {
                    tc::tma_load_2d(dst + b * PAGE_BYTES, &mk, b * 64, y, &ctl.full[st]);
                    tc::tma_load_2d(dst + C::HALF + b * PAGE_BYTES, &mv, b * 64, y, &ctl.full[st]);
                }
            }
            __syncwarp();
        }
        // copies still in flight land before the block reuses the ring or exits
        for (int i = max(0, j - C::NS); i < j; ++i) tc::mbar_wait(&ctl.full[i % C::NS], (i / C::NS) & 1, 1u << 20);
    } else {
        const bool work = mt * 16 < rows;
        // Q fragments, straight from global memory; rows that do not exist are zeros
        uint32_t q[KS][4];
        int lim[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int r = r0 + x * 8;
            const bool valid = r < rows;
            const int tok = r / p.G;
            lim[x] = valid ? lim0 + tok : 0x7fffffff;
            const uint16_t* src = a.q + (size_t)(seq.row0 + (valid ? tok : 0)) * a.q_stride +
                                  (size_t)(g * p.G + (valid ? r % p.G : 0)) * HD + (lane & 3) * 2;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                q[k][x] = valid ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16)) : 0u;
                q[k][x + 2] = valid ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16 + 8)) : 0u;
            }
        }
        const int kb = part * 16 * MT;   // this warp's keys of a page
        const float c = p.c;
        bool ok = true;
        for (int j = team; j < J; j += 2) {
            const int st = j % C::NS, k0 = (kt0 + j) * BKV;
            ok = wait(ctl, &ctl.full[st], (j / C::NS) & 1);
            if (!__all_sync(0xffffffffu, ok)) break;
            const uint32_t kp = tc::smem_u32(sm + st * C::SLOT), vp = kp + C::HALF;
            if (work) {
                const bool edge = k0 + BKV > lim0;
                if (edge) {
                    // (row tiles that share these keys each do this: what one has
                    // taken out, another finds taken out)
                    const int c0 = min(max(max(lim0 - k0, 0), kb), kb + 16 * MT);
                    clean_v<HD, BF16>(sm + st * C::SLOT + C::HALF, c0, min(last - k0, BKV), kb + 16 * MT, k0 - lim0,
                                      ctl.bad, &ctl.has_bad, lane, 32);
                    __syncwarp();
                }
                float sc[NT][4];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float odd[4] = {0.f, 0.f, 0.f, 0.f};   // two chains instead of one
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[t][x] = 0.f;
#pragma unroll
                    for (int k = 0; k < KS; k += 2) {
                        uint32_t b[4];   // columns 16k .. 16k + 31 of 8 keys
                        ldsm4(chunk(kp, kb + t * 8 + (lane & 7), 2 * k + (lane >> 3)), b);
                        mma16<BF16>(sc[t], q[k], b[0], b[1]);
                        mma16<BF16>(odd, q[k + 1], b[2], b[3]);
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) sc[t][x] += odd[x];
                }
                float alpha[2], mc[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if (edge) {
                            const int left = lim[x] - k0 - kb - t * 8 - (lane & 3) * 2;
                            if (left <= 0) sc[t][2 * x] = -INFINITY;
                            if (left <= 1) sc[t][2 * x + 1] = -INFINITY;
                        }
                        mx = max_nan(mx, sc[t][2 * x], sc[t][2 * x + 1]);
                    }
                    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    alpha[x] = 1.f;
                    // the reference maximum follows when a row's grows by more than 2^8
                    if (mx != -INFINITY && (m[x] == -INFINITY || (mx - m[x]) * c > 8.f)) {
                        if (m[x] != -INFINITY) alpha[x] = ex2((m[x] - mx) * c);
                        m[x] = mx;
                    }
                    mc[x] = m[x] == -INFINITY ? 0.f : m[x] * c;
                    // a score of NaN or +inf makes the row NaN
                    l[x] = mx < INFINITY ? l[x] * alpha[x] : NAN;
                }
                if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i) {
                        o[i][0] *= alpha[0];
                        o[i][1] *= alpha[0];
                        o[i][2] *= alpha[1];
                        o[i][3] *= alpha[1];
                    }
                }
#pragma unroll
                for (int t = 0; t < NT; t += 2) {   // 16 keys
                    uint32_t pa[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float p0 = ex2(fmaf(sc[t + h][2 * x], c, -mc[x]));
                            const float p1 = ex2(fmaf(sc[t + h][2 * x + 1], c, -mc[x]));
                            l[x] += p0 + p1;
                            pa[2 * h + x] = pack2<BF16>(p0, p1);
                        }
#pragma unroll
                    for (int i = 0; i < HD / 8; i += 2) {
                        uint32_t b[4];   // 16 keys x columns 8i .. 8i + 15
                        ldsm4t(chunk(vp, kb + t * 8 + (lane & 15), i + (lane >> 4)), b);
                        mma16<BF16>(o[i], pa, b[0], b[1]);
                        mma16<BF16>(o[i + 1], pa, b[2], b[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&ctl.empty[st]);
        }
        // the four lanes of a row hold its columns' sums
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            if ((lane & 3) == 0) ctl.ml[warp][(lane >> 2) + x * 8] = make_float2(m[x], l[x]);
        }
    }
    __syncthreads();   // every page has been read: the ring holds the parts' outputs now
    if (aborted(ctl)) return;
    float* part_o = reinterpret_cast<float*>(sm);   // [warp][16 rows][HD]
    if (warp < WARPS) {
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x)
                *reinterpret_cast<float2*>(part_o + (warp * 16 + (lane >> 2) + x * 8) * HD + i * 8 + (lane & 3) * 2) =
                    make_float2(o[i][2 * x], o[i][2 * x + 1]);
    }
    __syncthreads();
    constexpr int E = HD / 32;   // a lane's columns
    const bool whole = p.nsplit == 1, has_bad = *(volatile int*)&ctl.has_bad != 0;
    for (int r = warp; r < rows; r += WARPS + 1) {
        const int rt = r / 16, rr = r % 16, tok = seq.row0 + r / p.G, h = g * p.G + r % p.G;
        float mx = -INFINITY, sum = 0.f, v[E] = {};
#pragma unroll
        for (int i = 0; i < 2 * PARTS; ++i) mx = fmaxf(mx, ctl.ml[i * MT + rt][rr].x);
#pragma unroll
        for (int i = 0; i < 2 * PARTS; ++i) {
            const float2 ml = ctl.ml[i * MT + rt][rr];
            // a part without a score adds nothing; a NaN sum stays one
            const float f = ml.x == -INFINITY ? 0.f : ex2((ml.x - mx) * p.c);
            sum += ml.y == ml.y ? ml.y * f : ml.y;
            const float* x = part_o + ((i * MT + rt) * 16 + rr) * HD + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = f != 0.f ? fmaf(x[e], f, v[e]) : v[e];
        }
        const float inv = sum != sum ? sum : !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] *= inv;
            if (has_bad) v[e] = add_bad(v[e], *(volatile uint32_t*)&ctl.bad[lane * E + e], r / p.G);
        }
        const size_t prow = (size_t)tok * a.nq + h, srow = p.part_row(a, split, s, r / p.G, tok, h);
        const float mlog = mx == -INFINITY ? 0.f : mx * p.c;
        if (whole) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + (size_t)tok * a.out_stride + (size_t)h * HD + lane * E);
#pragma unroll
            for (int e = 0; e < E; e += 2) dst[e / 2] = pack2<BF16>(v[e], v[e + 1]);
            if (a.lse && lane == 0) a.lse[prow] = sum == 0.f ? -INFINITY : (mlog + log2f(sum)) * 0.69314718056f;
        } else {
            float* dst = p.part + srow * HD + lane * E;
#pragma unroll
            for (int e = 0; e < E; e += 2) *reinterpret_cast<float2*>(dst + e) = make_float2(v[e], v[e + 1]);
            if (lane == 0) p.part_ml[srow] = make_float2(sum == 0.f ? -INFINITY : mlog, sum);
        }
    }
}

template <int HD, bool BF16, int MT>
cudaError_t launch(const PagedAttnArgs& a, const AttnPlan& p, const CUtensorMap& mk, const CUtensorMap& mv,
                   cudaStream_t st) {
    const long long grid = (long long)a.kv.n_seqs * a.kv.nkv * p.nsplit;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
    const cudaError_t e = cudaFuncSetAttribute(k_attn_paged_few<HD, BF16, MT>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<HD>());
    if (e != cudaSuccess) return e;
    k_attn_paged_few<HD, BF16, MT><<<(unsigned)grid, THREADS, smem_bytes<HD>(), st>>>(mk, mv, a, p);
    note_launch();
    return cudaGetLastError();
}

template <int HD, bool BF16>
cudaError_t launch_tiles(const PagedAttnArgs& a, const AttnPlan& p, const CUtensorMap& mk, const CUtensorMap& mv,
                         cudaStream_t st) {
    const int rows = a.max_q * p.G;
    static_assert(FEW_ROWS == 32, "two row tiles");
    return rows <= 16 ? launch<HD, BF16, 1>(a, p, mk, mv, st) : launch<HD, BF16, 2>(a, p, mk, mv, st);
}

}  // namespace

cudaError_t attn_paged_few_launch(const PagedAttnArgs& a, const AttnPlan& p, const CUtensorMap& mk,
                                  const CUtensorMap& mv, cudaStream_t st) {
    if (a.kv.hd == 64)
        return a.kv.bf16 ? launch_tiles<64, true>(a, p, mk, mv, st) : launch_tiles<64, false>(a, p, mk, mv, st);
    return a.kv.bf16 ? launch_tiles<128, true>(a, p, mk, mv, st) : launch_tiles<128, false>(a, p, mk, mv, st);
}

}  // namespace vvq2
