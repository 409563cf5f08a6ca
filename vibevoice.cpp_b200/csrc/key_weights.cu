// key_weights.cu -- the attention weight each cached key receives from a
// packed chunk of queries (vvq2_attention_key_weights) on the 5th-generation
// tensor cores, sm_100a.
//
//   W[s][g][j] = sum over rows t, h of s in group g with j < lim(t) of
//                exp(scale q[t][h].K[j][g] - lse[t][h]),  lim(t) = L - n + t + 1
//
// The product is taken transposed, S = K Q^T: a key is a TMEM lane, so its sum
// over the queries stays in a thread and is made in one fixed order, without
// atomics.  An item is (sequence, KV head, 256 keys): its two
// tiles of 128 keys stay in shared memory while tiles of
// T tokens x G heads (G = nq / nkv, T = floor(128 / G)) stream past both, every
// other one for each of a key tile's two warpgroups.
// Blocks (one per SM) stride over the items.  The first keys of a long prompt
// see all its rows, so its rows are cut into chunks that are items of their own;
// k_key_weights_join adds a key's chunks up in their order.  Sequences of no more
// rows than a chunk have no chunks and need no join.
// Bound by the special-function unit when there are many rows (one exponential
// per row, head and key), by reading K when there are few.
//
//   warp 0      TMA producer: K tiles (two pages each), query tiles
//   warp 1      MMA issuer: S into the TMEM buffer of a warpgroup
//   warp 2      scheduler: finds the items
//   warp 3      log-sum-exps and visibility limits of each query tile's columns
//   warps 4-19  four warpgroups, one key per thread: sums 2^(c S - lse log2 e)
//               (two warps to a scheduler leave its special-function unit idle
//               more than half of the time)
// Every wait is bounded; a timeout sets error word 1 and the block unwinds.
//
// Measured: 6 prompts of 131 to 4001 tokens over themselves and up to 500 keys
// more, 12/2 heads of 128, 114 us (59 % of the special-function unit); one row of
// each of 64 streams of up to 2048 keys 16 us, mostly the blocks' start and end.
#include <limits.h>

#include "paged_dev.cuh"

namespace vvq2 {

namespace {

constexpr int THREADS = 640;
constexpr int BK = 128;                     // keys per tile
constexpr int BLK = 16384;                  // one [128 rows][128 bytes] swizzled block
constexpr int PAGE_BYTES = KV_PAGE * 128;   // one 64-key box of 64 columns
constexpr uint32_t TMEM_COLS = 512;         // one S buffer of each warpgroup

template <int HD>
struct Cfg {
    static constexpr int NB = HD / 64;
    static constexpr int TILE = NB * BLK;               // 128 rows of K or of queries
    static constexpr int NQ = HD == 128 ? 2 : 3;        // query slots
    static constexpr int NL = 4;                        // slots of query columns
    static constexpr int K_OFF = 0;                     // two items x two tiles
    static constexpr int Q_OFF = 4 * TILE;
    static constexpr int CTL_OFF = Q_OFF + NQ * TILE;   // 192 KB with 128 columns
};

struct KeyItem {
    int valid;          // 0: no more items
    int seq, g, k0;     // first key
    int len, lim0;      // the sequence's keys; keys that its first token sees
    int row0, n;        // its rows
    int t0, t1;         // the tokens of this item, none before the first that sees key k0
    int line;           // line of the chunk's sums in the scratch; -1: the sums are whole
};

struct KeyPlan {
    int T = 0, G = 0;   // tokens per query tile, heads per KV head
    float c = 0.f;      // scale * log2(e)
    int chunks = 1, per = 0;   // most row chunks of a sequence, tokens in each
    int items = 0;             // at most so many, if q_start ascends
    // Sums of chunks, [2 (total_q / per)][nkv][max_kv].  A sequence with more than
    // `per` rows has its lines from 2 (row0 / per) on: those of k per + f rows,
    // k >= 1, f < per, are k or k + 1, and the next sequence's start 2k or more
    // further on.
    float* part = nullptr;
    int* taken = nullptr;      // items given out, if blocks take them as they come free
    __device__ __forceinline__ int chunks_of(int n) const { return n > per ? (n + per - 1) / per : 1; }
    __device__ __forceinline__ size_t part_at(const KeyWeightArgs& a, int line, int g, int key) const {
        return ((size_t)line * a.kv.nkv + g) * a.max_kv + key;
    }
};

template <int HD>
struct Ctl {
    uint64_t k_full[2], k_empty[2], q_full[3], q_empty[3], l_full[4], l_empty[4], s_full[4], s_empty[4], c_full[2],
        c_empty[2], it_full[2], it_empty[2], mma_done;
    KeyWeightArgs a;
    KeyItem item[2];
    uint32_t tmem_base;
    int abort_flag;
    float half[2][BK];   // sums of the second warpgroup of each key tile
};
// the columns of a query tile: lse in log2 units, and the keys the row sees
struct Columns {
    float lse2[BK];   // -lse log2(e)
    int lim[BK];
};

// 2^x of two values with the FMA unit: x = i + f, |f| <= 1/2, 2^f by the degree-5
// polynomial of least relative error there (Remez exchange: 7.5e-8, 2.1e-7 with
// its f32 evaluation) times 2^i.  x <= -126 gives about 2^-126, NaN NaN; x past
// 127 (an lse that is not these rows') gives no useful value.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    const float BIG = 12582912.f;   // 1.5 * 2^23: adding it rounds to a whole number
    x.x = max_nan(x.x, -126.f);
    x.y = max_nan(x.y, -126.f);
    const float2 t = add2(x, make_float2(BIG, BIG));
    const float2 i = add2(t, make_float2(-BIG, -BIG));
    const float2 f = fma2(i, make_float2(-1.f, -1.f), x);
    float2 r = make_float2(0.0013276472454890609f, 0.0013276472454890609f);
    r = fma2(r, f, make_float2(0.009675540961325169f, 0.009675540961325169f));
    r = fma2(r, f, make_float2(0.05550713092088699f, 0.05550713092088699f));
    r = fma2(r, f, make_float2(0.24022120237350464f, 0.24022120237350464f));
    r = fma2(r, f, make_float2(0.6931469440460205f, 0.6931469440460205f));
    r = fma2(r, f, make_float2(1.0000001192092896f, 1.0000001192092896f));
    return mul2(r, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                               __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}

// *s0, *s1 += 2^(c S - lse log2 e) of 32 columns, or 0 where the row does not see the key.
template <bool EDGE>
__device__ __forceinline__ void add_columns(const uint32_t* r, const float* lse2, const int* lim, int key, float2 c2,
                                            float2* s0, float2* s1) {
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
        const float4 l = *reinterpret_cast<const float4*>(lse2 + e);
        float2 x = fma2(make_float2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), c2, make_float2(l.x, l.y));
        float2 y = fma2(make_float2(__uint_as_float(r[e + 2]), __uint_as_float(r[e + 3])), c2, make_float2(l.z, l.w));
        x = make_float2(ex2(x.x), ex2(x.y));
        // 6 of 32 on the FMA unit: the special-function unit is the busiest (7 %)
        y = !EDGE && (e == 4 || e == 12 || e == 20) ? ex2_poly(y) : make_float2(ex2(y.x), ex2(y.y));
        if (EDGE) {
            const int4 m = *reinterpret_cast<const int4*>(lim + e);
            x.x = key < m.x ? x.x : 0.f;
            x.y = key < m.y ? x.y : 0.f;
            y.x = key < m.z ? y.x : 0.f;
            y.y = key < m.w ? y.y : 0.f;
        }
        *s0 = add2(*s0, x);
        *s1 = add2(*s1, y);
    }
}

template <int HD>
constexpr int smem_bytes() {
    constexpr int n = Cfg<HD>::CTL_OFF + (int)sizeof(Ctl<HD>) + Cfg<HD>::NL * (int)sizeof(Columns);
    static_assert(n <= 227 * 1024, "shared memory");
    return n;
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
    k_key_weights(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                  const KeyWeightArgs a, const KeyPlan p) {
    using C = Cfg<HD>;
    extern __shared__ __align__(1024) uint8_t sm[];
    Columns* cols = reinterpret_cast<Columns*>(sm + C::CTL_OFF);
    Ctl<HD>& ctl = *reinterpret_cast<Ctl<HD>*>(sm + C::CTL_OFF + C::NL * sizeof(Columns));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (tc::smem_u32(sm) & 1023) {   // the swizzle's atoms; the kernel has no static shared memory
        paged_fault(a.err, PERR_WAIT);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&ctl.k_full[i], 1);
            tc::mbar_init(&ctl.k_empty[i], 1);
            tc::mbar_init(&ctl.it_full[i], 1);
            tc::mbar_init(&ctl.it_empty[i], 19);   // producer, issuer, columns, 16 warps of sums
            tc::mbar_init(&ctl.c_full[i], 4);
            tc::mbar_init(&ctl.c_empty[i], 4);
        }
        for (int i = 0; i < 4; ++i) {
            tc::mbar_init(&ctl.s_full[i], 1);
            tc::mbar_init(&ctl.s_empty[i], 4);
        }
        for (int i = 0; i < C::NQ; ++i) {
            tc::mbar_init(&ctl.q_full[i], 1);
            tc::mbar_init(&ctl.q_empty[i], 1);
        }
        for (int i = 0; i < C::NL; ++i) {
            tc::mbar_init(&ctl.l_full[i], 1);
            tc::mbar_init(&ctl.l_empty[i], 8);     // the warps of the tile's two warpgroups
        }
        tc::mbar_init(&ctl.mma_done, 1);
        ctl.abort_flag = 0;
        ctl.a = a;
        tc::mbar_fence_init();
    }
    // rows of the query slots that no copy ever writes: zeros, so that their
    // scores are 0 for a finite key, and their log-sum-exp of +inf makes their
    // terms 0 (any other key: see below)
    {
        const int rows = p.T * p.G, per = (128 - rows) * 8;   // 16-byte chunks per 64-column block
        for (int i = threadIdx.x; i < C::NQ * C::NB * per; i += THREADS)
            *reinterpret_cast<uint4*>(sm + C::Q_OFF + (i / per) * BLK + rows * 128 + (i % per) * 16) =
                make_uint4(0, 0, 0, 0);
        tc::fence_proxy_async_smem();
    }
    if (warp == 0) {
        tc::tmem_alloc(&ctl.tmem_base, TMEM_COLS);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = ctl.tmem_base;

    if (warp == 2) {
        // ---- scheduler: items in the order (sequence, key tile, KV head, chunk),
        // every gridDim.x-th one or the next that no block has taken (make_plan)
        int n = 0, s0 = 0, held = -1, of = 1;
        // (key tile, chunk) pairs of the sequences before s0, and up to a lane's; no
        // more than CAP, for a q_start that does not ascend (its items end at p.items
        // all the same)
        constexpr int CAP = (1 << 30) - 1;
        int before = 0, sum = 0;
        SeqRows mine;
        int id = blockIdx.x;
        auto next = [&]() {
            if (!p.taken) {
                id += gridDim.x;
                return;
            }
            if (lane == 0) id = atomicAdd(p.taken, 1);
            id = __shfl_sync(0xffffffffu, id, 0);
        };
        if (p.taken) next();
        bool ok = true, more = true;
        while (more) {
            // (g aside; past the last: on through all sequences, for their error words)
            const int pair = id < p.items ? id / a.kv.nkv : INT_MAX;
            more = false;
            while (s0 < a.kv.n_seqs) {
                if (held != s0) {   // lane l holds sequence s0 + l, and the pairs up to its last
                    mine = SeqRows();
                    if (s0 + lane < a.kv.n_seqs)
                        mine = paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, s0 + lane,
                                         blockIdx.x ? nullptr : a.err);
                    of = p.chunks_of(mine.n);
                    sum = (mine.len + 2 * BK - 1) / (2 * BK) * of;   // (2^22 tiles, 64 chunks at most)
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int v = __shfl_up_sync(0xffffffffu, sum, o);
                        if (lane >= o) sum = min(sum + v, CAP);
                    }
                    held = s0;
                }
                const int all = __shfl_sync(0xffffffffu, sum, 31);
                if (pair >= before + all) {   // past these 32 sequences
                    before = min(before + all, CAP);
                    s0 += 32;
                    continue;
                }
                const int f = __ffs(__ballot_sync(0xffffffffu, before + sum > pair)) - 1;
                const int first = before + (f ? __shfl_sync(0xffffffffu, sum, f - 1) : 0);
                const int chunks = __shfl_sync(0xffffffffu, of, f);
                const int local = id - first * a.kv.nkv, line = local / chunks;
                const int kt = line / a.kv.nkv, g = line % a.kv.nkv;
                // The chunks turn with the tile: early ones see no late key, and a
                // block that met the same chunk each time could have most or least.
                const int chunk = (local + kt) % chunks;
                SeqRows r;
                r.row0 = __shfl_sync(0xffffffffu, mine.row0, f);
                r.n = __shfl_sync(0xffffffffu, mine.n, f);
                r.len = __shfl_sync(0xffffffffu, mine.len, f);
                next();
                more = true;
                const int t0 = max(chunk * p.per, kt * 2 * BK - (r.len - r.n)), t1 = min(r.n, (chunk + 1) * p.per);
                // nothing to add, nor (without chunks) anything to write
                if (chunks > 1 && t0 >= t1) break;
                ok = n < 2 || wait(ctl, &ctl.it_empty[n & 1], ((n >> 1) - 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) {
                    more = false;
                    break;
                }
                if (lane == 0) {
                    KeyItem& it = ctl.item[n & 1];
                    it.valid = 1;
                    it.seq = s0 + f;
                    it.g = g;
                    it.k0 = kt * 2 * BK;
                    it.len = r.len;
                    it.lim0 = r.len - r.n + 1;
                    it.row0 = r.row0;
                    it.n = r.n;
                    it.t0 = t0;
                    it.t1 = t1;
                    it.line = chunks > 1 ? 2 * (r.row0 / p.per) + chunk : -1;
                    tc::mbar_arrive(&ctl.it_full[n & 1]);
                }
                ++n;
                break;
            }
        }
        if (ok && n >= 2) wait(ctl, &ctl.it_empty[n & 1], ((n >> 1) - 1) & 1);
        if (lane == 0) {
            ctl.item[n & 1].valid = 0;
            tc::mbar_arrive(&ctl.it_full[n & 1]);
        }
    } else if (warp == 0) {
        // ---- TMA producer
        unsigned qi = 0;   // query slots filled so far
        int n = 0;
        bool ok = true;
        for (; ok; ++n) {
            const KeyItem* it = take(ctl, n);
            if (!it) break;
            const int seq = it->seq, g = it->g, k0 = it->k0, len = it->len, row0 = it->row0, rows = it->t1, t0 = it->t0;
            done_with(ctl, n);
            // page ids of the item's four pages, in lanes 0-3
            int page = -1;
            if (lane < 4 && k0 + lane * KV_PAGE < len)
                page = paged_page(a.kv.table, a.kv.max_pages, a.kv.n_pages, seq, k0 / KV_PAGE + lane, a.err);
            ok = n < 2 || wait(ctl, &ctl.k_empty[n & 1], ((n >> 1) - 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) break;
            const int pages = k0 + BK < len ? 4 : 2;   // the second tile only if it has keys
            if (lane == 0) tc::mbar_arrive_expect_tx(&ctl.k_full[n & 1], (uint32_t)(pages * C::NB * PAGE_BYTES));
            __syncwarp();
            for (int i = 0; i < pages; ++i) {
                const int pg = __shfl_sync(0xffffffffu, page, i);
                // no page: rows past the pool's, which read as zeros
                const int y = (pg >= 0 ? pg * a.kv.nkv + g : a.kv.n_pages * a.kv.nkv) * KV_PAGE;
                uint8_t* dst = sm + C::K_OFF + ((n & 1) * 2 + (i >> 1)) * C::TILE + (i & 1) * PAGE_BYTES;
                if (lane == 0)
                    for (int b = 0; b < C::NB; ++b)
                        tc::tma_load_2d(dst + b * BLK, &mk, b * 64, y, &ctl.k_full[n & 1]);
            }
            for (int t = t0; ok && t < rows; t += p.T, ++qi) {
                const unsigned st = qi % C::NQ, use = qi / C::NQ;
                ok = use == 0 || wait(ctl, &ctl.q_empty[st], (use - 1) & 1);
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    tc::mbar_arrive_expect_tx(&ctl.q_full[st], (uint32_t)(C::NB * p.T * p.G * 128));
                    for (int b = 0; b < C::NB; ++b)
                        tc::tma_load_3d(sm + C::Q_OFF + st * C::TILE + b * BLK, &mq, b * 64, g * p.G, row0 + t,
                                        &ctl.q_full[st]);
                }
                __syncwarp();
            }
        }
        // copies still in flight land before the block exits
        if (aborted(ctl)) {
            for (int i = max(0, n - 2); i < n; ++i) tc::mbar_wait(&ctl.k_full[i & 1], (i >> 1) & 1, 1u << 20);
            for (unsigned i = qi > C::NQ ? qi - C::NQ : 0; i < qi; ++i)
                tc::mbar_wait(&ctl.q_full[i % C::NQ], (i / C::NQ) & 1, 1u << 20);
        }
    } else if (warp == 1) {
        // ---- MMA issuer
        constexpr uint32_t TY = BF16 ? (1u << 7) | (1u << 10) : 0u;
        constexpr uint32_t idS = tc::idesc_f16(BK, 128) | TY;
        unsigned qi = 0;
        unsigned made[4] = {0, 0, 0, 0};   // S tiles made for each warpgroup
        bool ok = true;
        for (int n = 0; ok; ++n) {
            const KeyItem* it = take(ctl, n);
            if (!it) break;
            const int rows = it->t1, t0 = it->t0, tiles = it->k0 + BK < it->len ? 2 : 1;
            done_with(ctl, n);
            ok = wait(ctl, &ctl.k_full[n & 1], (n >> 1) & 1);
            auto tile = [&](int t, unsigned* mk0, unsigned* mk1, int u) {
                const unsigned st = qi % C::NQ;
                ok = ok && wait(ctl, &ctl.q_full[st], (qi / C::NQ) & 1);
                const uint64_t qd = tc::desc_sw128(sm + C::Q_OFF + st * C::TILE);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    unsigned* m = w ? mk1 : mk0;
                    if (w >= tiles) continue;
                    ok = ok && (*m == 0 || wait(ctl, &ctl.s_empty[2 * u + w], (*m - 1) & 1));
                    if (!__all_sync(0xffffffffu, ok)) continue;
                    tc::tc_fence_after();
                    const uint64_t kd = tc::desc_sw128(sm + C::K_OFF + ((n & 1) * 2 + w) * C::TILE);
                    if (tc::elect_one()) {
#pragma unroll
                        for (int k16 = 0; k16 < HD / 16; ++k16) {
                            const int o = (k16 >> 2) * (BLK / 16) + 2 * (k16 & 3);
                            tc::mma_f16(tmem + (2 * u + w) * 128, kd + o, qd + o, idS, k16 > 0);
                        }
                        tc::mma_commit(&ctl.s_full[2 * u + w]);
                    }
                    __syncwarp();
                    ++*m;
                }
                if (tc::elect_one()) tc::mma_commit(&ctl.q_empty[st]);
                __syncwarp();
                ++qi;
            };
            for (int t = t0; __all_sync(0xffffffffu, ok) && t < rows; t += 2 * p.T) {
                tile(t, &made[0], &made[1], 0);
                if (t + p.T < rows) tile(t + p.T, &made[2], &made[3], 1);
            }
            ok = __all_sync(0xffffffffu, ok);
            if (tc::elect_one()) tc::mma_commit(&ctl.k_empty[n & 1]);
            __syncwarp();
        }
        if (tc::elect_one()) tc::mma_commit(&ctl.mma_done);   // completes after every MMA issued above
        __syncwarp();
    } else if (warp == 3) {
        // ---- columns of the query tiles: lse in log2 units, visibility limits.
        // The words of the next tile are on their way while this one is written.
        int dt[4], dh[4];   // token and head of this lane's columns within a tile
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = k * 32 + lane;
            dt[k] = c < p.T * p.G ? c / p.G : 0x40000000;   // no such column
            dh[k] = c % p.G;
        }
        unsigned qi = 0;
        bool ok = true;
        for (int n = 0; ok; ++n) {
            const KeyItem* it = take(ctl, n);
            if (!it) break;
            const int rows = it->t1, t0 = it->t0, row0 = it->row0, g = it->g, lim0 = it->lim0;
            done_with(ctl, n);
            float v[4];
            auto fetch = [&](int t) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    v[k] = dt[k] < rows - t
                               ? __ldg(a.lse + (size_t)(row0 + t + dt[k]) * a.nq + g * p.G + dh[k])
                               : INFINITY;
            };
            if (t0 < rows) fetch(t0);
            for (int t = t0; t < rows; t += p.T, ++qi) {
                const unsigned st = qi % C::NL, use = qi / C::NL;
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = v[k];
                const int left = rows - t;
                if (t + p.T < rows) fetch(t + p.T);
                ok = use == 0 || wait(ctl, &ctl.l_empty[st], (use - 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    cols[st].lse2[k * 32 + lane] = x[k] * -1.4426950408889634f;
                    cols[st].lim[k * 32 + lane] = dt[k] < left ? lim0 + t + dt[k] : 0;
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&ctl.l_full[st]);
            }
        }
    } else {
        // ---- sums: thread owns key rr of its key tile w (TMEM lane rr) and sums
        // the query tiles of parity u
        const int v = (warp - 4) >> 2, w = v & 1, u = v >> 1, quarter = warp & 3, rr = quarter * 32 + lane;
        const uint32_t ts = tmem + ((uint32_t)(quarter * 32) << 16) + v * 128;
        unsigned qi = 0, steps = 0;
        bool ok = true;
        for (int n = 0; ok; ++n) {
            const KeyItem* it = take(ctl, n);
            if (!it) break;
            const int key = it->k0 + w * BK + rr, len = it->len, rows = it->t1, t0 = it->t0, lim0 = it->lim0;
            const size_t at = ((size_t)it->seq * a.kv.nkv + it->g) * a.w_stride + key;
            const bool whole = it->line < 0;
            const size_t part = p.part_at(a, whole ? 0 : it->line, it->g, key);
            const bool mine = key < len, active = it->k0 + w * BK < len;
            const int top = it->k0 + (w + 1) * BK;   // a token that sees so many keys sees the whole tile
            done_with(ctl, n);
            const float old = u == 0 && whole && a.w_in && mine && key < lim0 - 1 ? a.w_in[at] : 0.f;
            float total = 0.f;
            for (int t = t0 + u * p.T; ok && t < rows; t += 2 * p.T) {
                const unsigned q = qi + (unsigned)((t - t0) / p.T), st = q % C::NL;
                const int ncol = min(p.T, rows - t) * p.G;
                // some column not seen by some key of the tile, or a token past
                // the last in it
                const bool edge = lim0 + t < top || t + p.T > rows;
                ok = wait(ctl, &ctl.l_full[st], (q / C::NL) & 1);
                if (active) ok = ok && wait(ctl, &ctl.s_full[v], steps & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (active) {
                    tc::tc_fence_after();
                    const Columns& col = cols[st];
                    float2 s0 = make_float2(0.f, 0.f), s1 = s0;
                    const float2 c2 = make_float2(p.c, p.c);
#pragma unroll 1
                    for (int c0 = 0; c0 < ncol; c0 += 32) {
                        uint32_t r[32];
                        tc::tmem_ld32_async(ts + c0, r);
                        tc::tmem_wait_ld32(r);
                        if (c0 + 32 >= ncol) {   // S has been read: the next one may come
                            tc::tc_fence_before();
                            __syncwarp();
                            if (lane == 0) tc::mbar_arrive(&ctl.s_empty[v]);
                        }
                        // Columns past the tile's have zeros for queries: their
                        // scores are 0, or NaN with a key that is not finite
                        // (whose scores may be -inf, for a weight of 0).
                        const bool odd = c0 + 32 > ncol &&
                                         __any_sync(0xffffffffu, __uint_as_float(r[31]) != __uint_as_float(r[31]));
                        if (edge || odd) add_columns<true>(r, &col.lse2[c0], &col.lim[c0], key, c2, &s0, &s1);
                        else add_columns<false>(r, &col.lse2[c0], nullptr, key, c2, &s0, &s1);
                    }
                    total += (s0.x + s0.y) + (s1.x + s1.y);   // tile by tile: long sums lose less
                    ++steps;
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&ctl.l_empty[st]);
            }
            if (rows > t0) qi += (unsigned)((rows - t0 + p.T - 1) / p.T);
            if (!ok) break;
            // the second warpgroup's sums join the first's
            if (u == 1) {
                ok = n == 0 || wait(ctl, &ctl.c_empty[w], (n - 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ctl.half[w][rr] = total;
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&ctl.c_full[w]);
            } else {
                ok = wait(ctl, &ctl.c_full[w], n & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                total += ctl.half[w][rr];
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&ctl.c_empty[w]);
                if (mine) {
                    if (whole) a.w_out[at] = old + total;
                    else p.part[part] = total;
                }
            }
        }
    }

    tc::tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        // no MMA may still be writing TMEM when it is released
        tc::mbar_wait(&ctl.mma_done, 0, 1u << 20);
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, TMEM_COLS);
    }
}

// Adds the chunks of every key up, in order, to what the key had.
__global__ void __launch_bounds__(256) k_key_weights_join(const KeyWeightArgs a, const KeyPlan p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int s = blockIdx.y / a.kv.nkv, g = blockIdx.y % a.kv.nkv, key = blockIdx.x * 256 + threadIdx.x;
    const SeqRows r = paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, s, nullptr);
    const int chunks = p.chunks_of(r.n);
    if (key >= r.len || chunks == 1) return;
    // the chunks that were made for the key's tile
    const int t0 = max(0, key / (2 * BK) * (2 * BK) - (r.len - r.n)), line = 2 * (r.row0 / p.per);
    const size_t at = (size_t)blockIdx.y * a.w_stride + key;
    float w = 0.f;
#pragma unroll 8
    for (int c = t0 / p.per; c < chunks; ++c) w += p.part[p.part_at(a, line + c, g, key)];
    if (a.w_in && key < r.len - r.n) w += a.w_in[at];
    a.w_out[at] = w;
}

constexpr size_t HEAD = 16;   // of the workspace: the counter of items
// two lines for every `per` rows (KeyPlan::part)
size_t line_bytes(const KeyWeightArgs& a) { return (size_t)a.kv.nkv * a.max_kv * sizeof(float); }
int64_t max_items(const KeyWeightArgs& a, const KeyPlan& p) {
    const int64_t chunks = a.kv.n_seqs + (p.per < min(a.max_q, a.total_q) ? a.total_q / p.per : 0);
    return chunks * a.kv.nkv * ((a.max_kv + 2 * BK - 1) / (2 * BK));
}
size_t scratch_bytes(const KeyWeightArgs& a, int per) { return 2 * (size_t)(a.total_q / per) * line_bytes(a); }

// Row chunks of at least 8 query tiles, at most 64 in a sequence, and no more
// than fit the workspace or make ITEMS items of all sequences' rows: those are
// some 90 for each block, and more balance nothing.  So the scratch is at most
// 2 KB x ITEMS, whatever the bounds.  From COUNTED items on, blocks take them as
// they come free instead of every gridDim.x-th one, which costs the reset of a
// counter: 48 prompts of 500 to 2239 rows, 20/4 heads of 64 (13,000 items) take
// 427 us that way, 529 dealt out; one of 4000 rows, 14/2 heads (900) 82 and 89;
// 3 of up to 2000 rows, 12/2 of 128 (430) 41 and 45; one of 2000 rows, 14/2 of 64
// (220) 39 and 37.
constexpr int ITEMS = 14000, COUNTED = 300;
constexpr int64_t MAX_ITEMS = 1 << 29;   // (the scheduler's CAP)
KeyPlan make_plan(const KeyWeightArgs& a, size_t workspace) {
    KeyPlan p;
    p.G = a.nq / a.kv.nkv;
    p.T = min(128 / p.G, max(1, min(a.max_q, a.total_q)));
    p.c = (float)((double)a.scale * 1.4426950408889634);
    const int rows = min(a.max_q, a.total_q), tiles = (rows + p.T - 1) / p.T, n = min(64, tiles / 8);
    const int kt = (a.max_kv + 2 * BK - 1) / (2 * BK);
    const long long seq_heads = (long long)a.kv.n_seqs * a.kv.nkv;
    p.per = max(1, rows);
    if (n > 1 && seq_heads <= 65535 && workspace > HEAD) {   // (a join's grid y)
        const double lines = floor((double)(workspace - HEAD) / (2.0 * line_bytes(a)));
        const double per = max(max((double)((tiles + n - 1) / n) * p.T, (double)a.total_q * a.kv.nkv * kt / ITEMS),
                               floor(a.total_q / (lines + 1)) + 1);   // total_q / per <= lines
        if (per < rows) p.per = min(rows, ((int)ceil(per) + p.T - 1) / p.T * p.T);
        if (max_items(a, p) > MAX_ITEMS) p.per = rows;
    }
    p.chunks = max(1, (rows + p.per - 1) / p.per);
    p.items = (int)min(max_items(a, p), MAX_ITEMS);
    if (p.chunks > 1) {
        if (p.items >= COUNTED) p.taken = static_cast<int*>(a.workspace);
        p.part = static_cast<float*>(a.workspace) + HEAD / sizeof(float);
    }
    return p;
}

template <int HD, bool BF16>
cudaError_t launch(const KeyWeightArgs& a, int n_sm, cudaStream_t st) {
    const KeyPlan p = make_plan(a, a.workspace_bytes);
    if (max_items(a, p) > MAX_ITEMS) return cudaErrorInvalidValue;
    CUtensorMap mq, mk;
    const int64_t rows = (int64_t)a.kv.n_pages * a.kv.nkv * KV_PAGE;
    if (!make_kv_map(&mk, reinterpret_cast<const __half*>(a.kv.k), rows, HD)) return cudaErrorInvalidValue;
    // without rows no query tile is ever loaded
    if (a.total_q > 0 && !make_heads_map(&mq, a.q, HD, a.nq, a.total_q, a.q_stride, p.G, p.T))
        return cudaErrorInvalidValue;
    if (a.total_q == 0) mq = mk;
    cudaError_t e = cudaFuncSetAttribute(k_key_weights<HD, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         smem_bytes<HD>());
    if (e != cudaSuccess) return e;
    if (p.taken) {
        e = cudaMemsetAsync(p.taken, 0, sizeof(int), st);
        if (e != cudaSuccess) return e;
    }
    k_key_weights<HD, BF16><<<(unsigned)min(p.items, n_sm), THREADS, smem_bytes<HD>(), st>>>(mq, mk, a, p);
    note_launch();
    e = cudaGetLastError();
    if (e != cudaSuccess || p.chunks == 1) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.max_kv + 255) / 256), (unsigned)(a.kv.n_seqs * a.kv.nkv));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, k_key_weights_join, a, p);
    note_launch();
    return e;
}

}  // namespace

size_t key_weights_workspace(const PagesView& kv, int total_q, int max_q, int max_kv, int nq) {
    KeyWeightArgs a;
    a.kv = kv;
    a.total_q = total_q;
    a.max_q = max_q;
    a.max_kv = max_kv;
    a.nq = nq;
    const KeyPlan p = make_plan(a, ~(size_t)0);
    return p.chunks > 1 ? HEAD + scratch_bytes(a, p.per) : 0;
}

cudaError_t key_weights_launch(const KeyWeightArgs& a, int n_sm, cudaStream_t st) {
    if (a.kv.hd == 64) return a.kv.bf16 ? launch<64, true>(a, n_sm, st) : launch<64, false>(a, n_sm, st);
    return a.kv.bf16 ? launch<128, true>(a, n_sm, st) : launch<128, false>(a, n_sm, st);
}

}  // namespace vvq2
