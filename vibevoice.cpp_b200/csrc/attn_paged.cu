// attn_paged.cu -- causal attention of packed chunks of new tokens over a
// paged K/V cache (vvq2_attention_paged) on the 5th-generation tensor cores,
// sm_100a.
//
// Token t of sequence s, with n new tokens and L cached keys, sees the keys
// j < lim = L - n + t + 1:
//   out = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale q.K_j - m),  m >= all,
//   lse = m + log sum_j p_j,
// in one pass over the keys with a running m, sum and output per row.
//
// Rows.  The G = nq / nkv query heads of a KV head share its keys, so a tile
// packs T = floor(128 / G) tokens x G heads into the 128 rows of one MMA: a
// decode step's heads cost one pass over K and V, and a causal tile spans T
// tokens only, so little of its last key tile is masked.
//
// Work.  An item is (sequence, 2T tokens, KV head, key range).  With more
// than T tokens its two row tiles ("dual") walk the same key tiles, so K and V
// are loaded once for both; with at most T tokens ("solo") the one row tile has
// its even and its odd key tiles treated as those of two, with an accumulator
// each, added up at the end.
// The grid has one block per possible item, a sequence's later tokens (which
// see more keys) before its earlier ones and the last sequence first; a running
// block takes over blocks that have not started (cluster launch control), so
// barriers, TMEM and the load pipeline stay alive from item to item.  When
// there are fewer items than SMs, the key range is cut into splits whose
// (O, m, l) k_attn_paged_merge joins.  Sequences of few rows go to
// attn_paged_few.cu.
//
//   warp 0      TMA producer: queries (3-D boxes of T tokens x G heads), and a
//               ring of key tiles, K and V of one 64-key page each
//   warps 1, 3  MMA issuers, one per row tile w: S = Q K_j^T (both from shared
//               memory) into one of the tile's two 64-column TMEM buffers;
//               O += P_j V_j with P read from TMEM.  Issue keeps pace with the
//               tensor core, so a single issuer's barrier waits leave it idle
//   warp 2      scheduler: asks for the next block, finds its sequence
//   warps 4-    softmax warpgroups, one row per thread: S from TMEM,
//               P = exp2(scale' S - m') over it, while the issuer works on the
//               other buffer; O is rescaled in TMEM only when a row's maximum
//               grows by more than 2^8.  With 128 columns one warpgroup per row
//               tile; with 64 there is room for two, which take turns at the
//               key tiles and have an accumulator each
// Tiles of 64 keys make room for two score buffers next to the accumulators
// (2 x 2 x 64 + 2 x 128 or 4 x 64 = 512 TMEM columns), so the softmax of a tile
// does not wait for the products of the one before.
// Masks: scores past a row's limit become -inf.  V rows past the sequence's
// keys (the rest of its last page) are zeroed in shared memory; a non-finite
// V element that only some rows of a tile may see is taken out there and
// added to those rows at the end, since 0 x inf would reach all of them.
// Every wait is bounded; a timeout sets error word 1 and the block unwinds.  A
// warp gives up as one: lanes that went on alone would meet no one at its next
// shuffle.
//
// Measured: a 16,384-token prompt of 28/4 heads of 128 2.06 ms (0.94 PFLOP/s,
// under the power cap), one of 8000 tokens 0.49 ms, and of 14/2 heads of 64 0.21
// ms (a third more with one warpgroup per row tile).  Bound by the chain from
// scores to probabilities (the special-function unit is 44 % busy with 64
// columns) and, with 128, by the shared-memory reads of N = 64 products.
#include "attn_paged.cuh"

namespace vvq2 {

namespace {

constexpr int BLK = 16384;                  // queries: one [128 rows][128 bytes] swizzled block
constexpr uint32_t TMEM_COLS = 512;         // two S buffers of each row tile | the accumulators

template <int HD>
struct Cfg {
    // Warpgroups per row tile: with 64 columns there is room for two accumulators
    // each, and four warps to a scheduler hide each other's waits
    static constexpr int NU = HD == 64 ? 2 : 1;
    static constexpr int THREADS = 128 + 256 * NU;
    static constexpr int NB = HD / 64;                    // 64-column blocks along hd
    static constexpr int HALF = NB * PAGE_BYTES;          // K or V of a tile
    static constexpr int SLOT = 2 * HALF;
    static constexpr int NS = HD == 128 ? 5 : 10;         // ring slots
    static constexpr int Q_OFF = 0;                       // two query tiles
    static constexpr int RING_OFF = 2 * NB * BLK;
    static constexpr int CTL_OFF = RING_OFF + NS * SLOT;
    static constexpr uint32_t O_COL = 4 * BKV;
};

struct Item {
    int valid;       // 0: no more items
    int seq, g, tok0, ntok;   // tokens tok0 .. tok0 + ntok of the packed rows
    int lim0, last;  // keys the first and the last token see (may be <= 0)
    int kt0, nkt;    // key tiles
    int split;
};

// everything that is not a tile
template <int HD>
struct Ctl {
    uint64_t ring_full[Cfg<HD>::NS], ring_empty[Cfg<HD>::NS];
    uint64_t q_full, q_empty, s_full[2][2], p_full[2][2], pv_done[2][2], o_full[2][2], it_full[2], it_empty[2],
        clc_full, mma_done, halves, pair[2];
    uint4 clc;
    PagedAttnArgs a;           // the kernel's arguments, for the warps compiled apart
    AttnPlan p;
    Item item[2];
    uint32_t tmem_base;
    int abort_flag;
    uint32_t asked;            // ring slot uses whose loads are under way or done
    int has_bad[2];            // an even / odd item has non-finite V elements set aside
    uint32_t bad[2][HD];       // per column: see note_bad
    // (m, l) of a row's other parts, then the parts' factors (see softmax_role)
    float2 ml[Cfg<HD>::NU == 1 ? 1 : 4][128];
};

template <int HD>
constexpr int smem_bytes() {
    static_assert(Cfg<HD>::CTL_OFF + sizeof(Ctl<HD>) <= 227 * 1024, "shared memory");
    return Cfg<HD>::CTL_OFF + (int)sizeof(Ctl<HD>);
}

// N of a row's scores: those from `left` on become -inf.
template <int N>
__device__ __forceinline__ void mask_row(uint32_t* r, int left) {
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e >= left) r[e] = 0xff800000u;
}
template <int N>
__device__ __forceinline__ float row_max(const uint32_t* r) {   // NaN if one is
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const int k = (e >> 1) & 3;
        m[k] = max_nan(m[k], __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
    }
    return max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3]));
}
// P = 2^(c S - mc) of 32 scores, in 16 packed pairs; *s0, *s1 += their sums
// (before the rounding to 16 bits).  P has V's type because both operands of the
// product must: each p is off by half a step at most, so an output by eps / 2 of
// sum p |V|, no more than its own rounding to that type where V has one sign.
template <bool BF16>
__device__ __forceinline__ void row_exp(const uint32_t* r, float c, float mc, uint32_t* pu, float2* s0, float2* s1) {
    const float2 c2 = make_float2(c, c), m2 = make_float2(-mc, -mc);
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
        float2 a = fma2(make_float2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), c2, m2);
        float2 b = fma2(make_float2(__uint_as_float(r[e + 2]), __uint_as_float(r[e + 3])), c2, m2);
        a = make_float2(ex2(a.x), ex2(a.y));
        b = make_float2(ex2(b.x), ex2(b.y));
        *s0 = add2(*s0, a);
        *s1 = add2(*s1, b);
        pu[e / 2] = pack2<BF16>(a.x, a.y);
        pu[e / 2 + 1] = pack2<BF16>(b.x, b.y);
    }
}

// The rows' outputs so far times alpha, in TMEM (rare: see the caller).
template <int HD>
__device__ __forceinline__ void rescale(uint32_t to, float alpha) {
#pragma unroll 1
    for (int cc = 0; cc < HD; cc += 32) {
        float v[32];
        tc::tmem_ld32(to + cc, v);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] *= alpha;
        tc::tmem_st32(to + cc, v);
    }
}

// Ring slot use i is loaded.  A parity names a phase only to one who knows
// that the phase before it is over: the producer's count says that use i has
// been asked for, so the slot's earlier uses have come and gone (the reader may
// not have waited for those, if they were the other warpgroup's tiles).
template <class CT>
__device__ __forceinline__ bool slot_full(CT& ctl, unsigned i, unsigned ns) {
    uint32_t asked = 0;
    for (int k = 0; k < (1 << 24); ++k) {
        asm volatile("ld.acquire.cta.shared.u32 %0, [%1];" : "=r"(asked) : "r"(tc::smem_u32(&ctl.asked)) : "memory");
        if (asked > i) return wait(ctl, &ctl.ring_full[i % ns], (i / ns) & 1);
        if (aborted(ctl)) return false;
    }
    paged_fault(ctl.a.err, PERR_WAIT);
    *(volatile int*)&ctl.abort_flag = 1;
    return false;
}
// Sequence and first token of a block's tile; false if there is no such tile.
// Whole warp.
__device__ __forceinline__ bool find_item(const PagedAttnArgs& a, const AttnPlan& p, int x, int* seq, int* t0_out) {
    const int lane = threadIdx.x & 31, step = 2 * p.T;
    const int tile = p.n_tiles - 1 - x / p.nsplit / a.kv.nkv;   // later tokens see more keys: first
    int s = tile, t0 = 0;
    if (!p.direct) {
        int before = 0;
        s = -1;
        for (int s0 = 0; s0 < a.kv.n_seqs && s < 0; s0 += 32) {
            int n = 0;
            if (s0 + lane < a.kv.n_seqs)
                n = paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, s0 + lane, nullptr).n;
            const int tiles = (n + step - 1) / step;
            int sum = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += v;
            }
            const unsigned here = __ballot_sync(0xffffffffu, before + sum > tile);
            if (here) {
                const int w = __ffs(here) - 1;
                s = s0 + w;
                t0 = (tile - before - __shfl_sync(0xffffffffu, sum - tiles, w)) * step;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (s < 0) return false;
    }
    *seq = s;
    *t0_out = t0;
    return true;
}

// Writes an item's rows: the sum of f_i O_i over the row tile's accumulators,
// O_i of warpgroup (w, u) being number w NU + u: a dual row tile has its own NU,
// a solo one all of them.  Results, or, when the keys are split, sums next to
// (m, l) for the merge.  The warpgroups share the columns.  Which of a tile's two
// warpgroups had its first keys hangs on the block's earlier items; they are
// added up in the order of their keys all the same (bit i of flip: parts 2i and
// 2i + 1 are each other's accumulators), so that a call's sums are repeatable.
template <int HD, bool BF16>
__device__ __noinline__ void results(Ctl<HD>& ctl, int n, uint32_t tmem, float m_ref, float l, float4 f,
                                     unsigned flip) {
    using C = Cfg<HD>;
    const PagedAttnArgs& a = ctl.a;
    const AttnPlan& p = ctl.p;
    const Item& it = ctl.item[n & 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int v = (warp - 4) >> 2, w = v & 1, u = v >> 1, quarter = warp & 3, rr = quarter * 32 + lane;
    const bool dual = it.ntok > p.T, last = p.nsplit == 1;
    const int t0 = dual ? w * p.T : 0, rows = min(p.T, it.ntok - t0) * p.G;
    const int share = C::NU == 2 ? u : dual ? 0 : w;   // which part of the columns
    if (quarter * 32 >= rows || (C::NU == 2 && !dual && w == 1)) return;
    const uint32_t to = tmem + ((uint32_t)(quarter * 32) << 16) + C::O_COL + (dual ? w * C::NU : 0) * HD;
    const bool valid = rr < rows;
    const int row = it.tok0 + t0 + rr / p.G, h = it.g * p.G + rr % p.G;
    const int seen = t0 + rr / p.G;   // keys from lim0 on that the row sees
    const size_t prow = (size_t)row * a.nq + h;
    const size_t split_row = p.part_row(a, it.split, it.seq, row - it.tok0, row, h);   // (one tile: it has all tokens)
    const float mlog = m_ref == -INFINITY ? 0.f : m_ref * p.c;
    if (valid && share == 0) {
        if (!last) p.part_ml[split_row] = make_float2(l == 0.f ? -INFINITY : mlog, l);
        else if (a.lse) a.lse[prow] = l == 0.f ? -INFINITY : (mlog + log2f(l)) * 0.69314718056f;
    }
    const bool has_bad = *(volatile int*)&ctl.has_bad[n & 1] != 0;
    constexpr int MAXP = 2 * C::NU;
    const int parts = dual ? C::NU : MAXP;
    const float fs[4] = {f.x, f.y, f.z, f.w};
    const int width = C::NU == 2 || !dual ? HD / 2 : HD, c0 = share * width;
#pragma unroll 1
    for (int cc = c0; cc < c0 + width; cc += 32) {
        float o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0.f;
#pragma unroll
        for (int i = 0; i < MAXP; ++i) {
            // an accumulator that no key of the row reached may hold anything
            if (i >= parts || !__any_sync(0xffffffffu, fs[i] != 0.f)) continue;
            float x[32];
            tc::tmem_ld32(to + (i ^ (int)(flip >> (i >> 1) & 1)) * HD + cc, x);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = fs[i] != 0.f ? fmaf(x[e], fs[i], o[e]) : o[e];
        }
        if (has_bad) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = add_bad(o[e], ctl.bad[n & 1][cc + e], seen);
        }
        if (!valid) continue;
        if (last) {
            uint16_t* dst = a.out + (size_t)row * a.out_stride + (size_t)h * HD + cc;
#pragma unroll
            for (int d = 0; d < 32; d += 8)
                *reinterpret_cast<uint4*>(dst + d) =
                    make_uint4(pack2<BF16>(o[d], o[d + 1]), pack2<BF16>(o[d + 2], o[d + 3]),
                               pack2<BF16>(o[d + 4], o[d + 5]), pack2<BF16>(o[d + 6], o[d + 7]));
        } else {
            float* dst = p.part + split_row * HD + cc;
#pragma unroll
            for (int d = 0; d < 32; d += 4)
                *reinterpret_cast<float4*>(dst + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
        }
    }
}

// Softmax warpgroups meet for the k-th time at a barrier of theirs (bounded,
// unlike a named barrier).
template <class CT>
__device__ __forceinline__ bool meet(CT& ctl, uint64_t* bar, unsigned k) {
    tc::tc_fence_before();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc::mbar_arrive(bar);
    const bool all = __all_sync(0xffffffffu, wait(ctl, bar, k & 1));
    tc::tc_fence_after();
    return all;
}

struct Walk {
    float m, l;              // the row's reference maximum and sum
    unsigned steps, meets;   // the caller's counts, carried on
    bool ok, any;            // no wait gave up; there was a tile
};

// One item's key tiles.  The two loops of the softmax warps are functions of
// their own: compiled together with what comes before and after it, this one
// has spills inside (and next to 227 KB of shared memory there is hardly any
// L1 to catch them; they cost more than the arithmetic).
template <int HD, bool BF16>
__device__ __noinline__ Walk walk_tiles(Ctl<HD>& ctl, uint8_t* sm, const uint32_t tmem, const int n,
                                        const unsigned base, unsigned steps, unsigned meets) {
    using C = Cfg<HD>;
    const Item& it = ctl.item[n & 1];
    const AttnPlan& p = ctl.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int v = (warp - 4) >> 2, w = v & 1, u = v >> 1, quarter = warp & 3, rr = quarter * 32 + lane;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const float c = p.c;
    const int J = it.nkt, lim0 = it.lim0;
    const bool dual = it.ntok > p.T;
    bool ok = true;
    int lim = 0x7fffffff;   // keys the row sees (no row: no limit)
    bool wvalid;
    {
        const int rows = min(p.T, it.ntok - (dual ? w * p.T : 0)) * p.G;
        wvalid = quarter * 32 < rows;
        if (rr < rows) lim = lim0 + (dual ? w * p.T : 0) + rr / p.G;
    }
    float m_ref = -INFINITY, l = 0.f;
    bool any_step = false;
    const int j0 = dual ? 0 : w, dj = dual ? 1 : 2;   // the row tile's key tiles
    const unsigned after = steps + (unsigned)max(0, (J - j0 + dj - 1) / dj);
    const int skip = C::NU == 2 && (steps & 1) != (unsigned)u;   // of two, this warpgroup has buffer u
    steps += skip;
    for (int j = j0 + skip * dj; j < J; j += C::NU * dj) {
        const unsigned b = steps & 1;
        const uint32_t ts = lane_base + (2 * w + b) * BKV;
        ok = wait(ctl, &ctl.s_full[w][b], (steps >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::tc_fence_after();
        const int k0 = (it.kt0 + j) * BKV;
        // V rows some row must not read: by the warpgroups that use the tile
        if (k0 + BKV > lim0) {
            ok = slot_full(ctl, base + j, C::NS);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            uint8_t* vt = sm + C::RING_OFF + (base + j) % C::NS * C::SLOT + C::HALF;
            // rows from lim0 on are seen by some rows only, those from `last` on by none
            clean_v<HD, BF16>(vt, max(lim0 - k0, 0), min(it.last - k0, BKV), BKV, k0 - lim0, ctl.bad[n & 1],
                              &ctl.has_bad[n & 1], dual && C::NU == 1 ? threadIdx.x - 128 : threadIdx.x & 127,
                              dual && C::NU == 1 ? 256 : 128);
            // the other row tile's warpgroup cleans half of it, too, before this
            // one's P V (with four warpgroups all of it: what one has taken out,
            // another finds taken out)
            if (dual && C::NU == 1) {
                ok = meet(ctl, &ctl.halves, meets++);
                if (!ok) break;
            }
        }
        if (wvalid) {
            // a limit inside (or before) the tile
            const bool edge = __any_sync(0xffffffffu, k0 + BKV > lim);
            // All 64 scores in registers, or, for the four warpgroups' fewer
            // registers, 32 at a time, read twice.
            uint32_t r[C::NU == 1 ? BKV : 32];
            auto load = [&](int e) {
                tc::tmem_ld32_async(ts + e * 32, r);
                tc::tmem_wait_ld32(r);
                if (edge) mask_row<32>(r, lim - k0 - e * 32);
            };
            float m;
            if constexpr (C::NU == 1) {
                tc::tmem_ld32_async(ts, r);
                tc::tmem_ld32_async(ts + 32, r + 32);
                tc::tmem_wait_ld32(r);
                tc::tmem_wait_ld32(r + 32);
                if (edge) mask_row<BKV>(r, lim - k0);
                m = row_max<BKV>(r);
            } else {
                load(1);
                m = row_max<32>(r);
                load(0);
                m = max_nan(m, row_max<32>(r));
            }
            float alpha = 1.f;
            if (lim != 0x7fffffff && m != -INFINITY && (m_ref == -INFINITY || (m - m_ref) * c > 8.f)) {
                if (m_ref != -INFINITY) alpha = ex2((m_ref - m) * c);
                m_ref = m;
            }
            const float mc = m_ref == -INFINITY ? 0.f : m_ref * c;
            float2 s0 = make_float2(0.f, 0.f), s1 = s0;
            // (each half stored as soon as it is made: together they spill; P of
            // the first goes over scores that have been read for the last time)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t pu[16];
                if (C::NU == 2 && e == 1) load(1);
                row_exp<BF16>(C::NU == 1 ? r + e * 32 : r, c, mc, pu, &s0, &s1);
                tc::tmem_st16_async(ts + e * 16, pu);
            }
            // a score of NaN or +inf makes the row NaN
            l = m < INFINITY ? l * alpha + ((s0.x + s0.y) + (s1.x + s1.y)) : NAN;
            tc::tmem_wait_st();
            if (__any_sync(0xffffffffu, alpha != 1.f) && any_step) {
                // P V of the step before may still be running (its buffer's
                // earlier one is not: S of that step came after it, and with two
                // warpgroups that one is this accumulator's last)
                if (C::NU == 1) {
                    ok = wait(ctl, &ctl.pv_done[w][b ^ 1], ((steps - 1) >> 1) & 1);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc::tc_fence_after();
                }
                rescale<HD>(lane_base + C::O_COL + (w * C::NU + u) * HD, alpha);
            }
        }
        any_step = true;
        steps += C::NU;
        tc::tc_fence_before();   // S reads, P stores and the O rescale are done
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&ctl.p_full[w][b]);
    }
    return Walk{m_ref, l, after, meets, (bool)__all_sync(0xffffffffu, ok), any_step};
}

// The softmax warps' items.
template <int HD, bool BF16>
__device__ __noinline__ void softmax_role(uint8_t* sm, const uint32_t tmem) {
    Ctl<HD>& ctl = *reinterpret_cast<Ctl<HD>*>(sm + Cfg<HD>::CTL_OFF);
    const AttnPlan& p = ctl.p;
    using C = Cfg<HD>;
    const int v = ((int)threadIdx.x - 128) >> 7, w = v & 1, u = v >> 1, rr = threadIdx.x & 127;
    unsigned finals = 0, base = 0;
    Walk k{0.f, 0.f, 0, 0, true, false};   // step i uses buffer i & 1
    unsigned theirs = 0;                   // steps of the other row tile
    for (int n = 0;; ++n) {
        const Item* mine = take(ctl, n);
        if (!mine) break;
        const Item& it = *mine;
        k = walk_tiles<HD, BF16>(ctl, sm, tmem, n, base, k.steps, k.meets);
        if (!k.ok) break;
        if (k.any) {
            const bool ok = wait(ctl, &ctl.o_full[w][u], finals++ & 1);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc::tc_fence_after();
        }
        base += it.nkt;
        const bool dual = it.ntok > p.T;
        // with two warpgroups to a row tile, the one of odd steps has an item's first key tile at times
        // (a solo item's even tiles are the first row tile's)
        const unsigned own_flip = C::NU == 2 ? (k.steps - (dual ? it.nkt : (it.nkt + 1 - w) / 2)) & 1 : 0;
        const unsigned their_flip = C::NU == 2 ? theirs & 1 : 0;
        theirs += dual ? it.nkt : (it.nkt + w) / 2;
        // a row's parts: accumulators first .. first + parts - 1
        const int parts = dual ? C::NU : 2 * C::NU, first = dual ? w * C::NU : 0;
        const int me = w * C::NU + (u ^ (int)own_flip) - first;   // in the order of their first keys
        const unsigned flip = dual ? own_flip : own_flip << w | their_flip << (w ^ 1);
        float4 f = make_float4(k.m == -INFINITY ? k.l : 1.f, 0.f, 0.f, 0.f);   // (without a score: 0, or NaN)
        if (parts > 1) {
            // The parts show one another (m, l).  Where there is room for it all,
            // each adds up for itself; else the first does, and answers the second.
            uint64_t* bar = dual ? &ctl.pair[w] : &ctl.halves;
            if constexpr (C::NU == 2) ctl.ml[first + me][rr] = make_float2(k.m, k.l);
            else if (me == 1) ctl.ml[0][rr] = make_float2(k.m, k.l);
            // (two warpgroups to a row tile meet twice an item, so always an even time here)
            if (!meet(ctl, bar, C::NU == 2 ? 0 : k.meets++)) break;
            if (C::NU == 2 || me == 0) {
                const float2 none = make_float2(-INFINITY, 0.f);
                float2 o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (C::NU == 2) o[i] = i < parts ? ctl.ml[first + (i < parts ? i : 0)][rr] : none;
                    else o[i] = i == 0 ? make_float2(k.m, k.l) : i == 1 ? ctl.ml[0][rr] : none;
                }
                k.m = fmaxf(fmaxf(o[0].x, o[1].x), fmaxf(o[2].x, o[3].x));
                k.l = 0.f;
                float g[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // a part without a score adds nothing; NaN scores may leave m
                    // at -inf, with a NaN sum
                    g[i] = o[i].x == -INFINITY ? 0.f : ex2((o[i].x - k.m) * p.c);
                    k.l += o[i].y == o[i].y ? o[i].y * g[i] : o[i].y;
                }
                f = make_float4(g[0], g[1], g[2], g[3]);
            }
        }
        if (C::NU == 2 || me == 0 || dual) {
            const float scale = k.l != k.l ? k.l : p.nsplit > 1 ? 1.f : k.l == 0.f ? 0.f : 1.f / k.l;
            f = make_float4(f.x * scale, f.y * scale, f.z * scale, f.w * scale);
            if (k.l != k.l) f.x = k.l;   // a NaN row is NaN in every column
        }
        if (C::NU == 1 && !dual) {
            if (me == 0) ctl.ml[0][rr] = make_float2(f.x, f.y);
            if (!meet(ctl, &ctl.halves, k.meets++)) break;
            if (me == 1) {
                const float2 o = ctl.ml[0][rr];
                f.x = o.x;
                f.y = o.y;
            }
        }
        results<HD, BF16>(ctl, n, tmem, k.m, k.l, f, flip);
        // all parts have been read before one is written again
        if (parts > 1) {
            if (!meet(ctl, dual ? &ctl.pair[w] : &ctl.halves, C::NU == 2 ? 1 : k.meets++)) break;
        }
        done_with(ctl, n);
        tc::tc_fence_before();
    }
}

// Error words of all sequences, by one warp.  (Inlined, it changes the code of
// the issuers: 8000 rows of 28/4 heads of 128 510 against 491 us.)
__device__ __noinline__ void look_at_all(const PagedAttnArgs& a) {
    for (int s = threadIdx.x & 31; s < a.kv.n_seqs; s += 32)
        paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, s, a.err);
}

template <int HD, bool BF16>
__global__ void __launch_bounds__(Cfg<HD>::THREADS, 1)
    k_attn_paged(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                 const __grid_constant__ CUtensorMap mv, const PagedAttnArgs a, const AttnPlan p) {
    using C = Cfg<HD>;
    extern __shared__ __align__(1024) uint8_t sm[];
    Ctl<HD>& ctl = *reinterpret_cast<Ctl<HD>*>(sm + C::CTL_OFF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (tc::smem_u32(sm) & 1023) {   // the swizzle's atoms; the kernel has no static shared memory
        paged_fault(a.err, PERR_WAIT);
        return;
    }

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NS; ++i) {
            tc::mbar_init(&ctl.ring_full[i], 1);
            tc::mbar_init(&ctl.ring_empty[i], 2);
        }
        tc::mbar_init(&ctl.q_full, 1);
        tc::mbar_init(&ctl.q_empty, 2);
        for (int i = 0; i < 2; ++i) {
            for (int b = 0; b < 2; ++b) {
                tc::mbar_init(&ctl.s_full[i][b], 1);
                tc::mbar_init(&ctl.p_full[i][b], 4);
                tc::mbar_init(&ctl.pv_done[i][b], 1);
            }
            for (int b = 0; b < 2; ++b) tc::mbar_init(&ctl.o_full[i][b], 1);
            tc::mbar_init(&ctl.pair[i], 4 * C::NU);
            tc::mbar_init(&ctl.it_full[i], 1);
            tc::mbar_init(&ctl.it_empty[i], 3 + 8 * C::NU);   // producer, issuers, softmax warps
            ctl.has_bad[i] = 0;
        }
        tc::mbar_init(&ctl.clc_full, 1);
        tc::mbar_init(&ctl.mma_done, 2);
        tc::mbar_init(&ctl.halves, 8 * C::NU);
        ctl.abort_flag = 0;
        ctl.asked = 0;
        ctl.a = a;
        ctl.p = p;
        tc::mbar_fence_init();
    }
    for (int i = threadIdx.x; i < 2 * HD; i += C::THREADS) ctl.bad[i / HD][i % HD] = NO_BAD;
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
        // ---- scheduler
        int x = blockIdx.x, n = 0;
        for (int asked = 0; x >= 0; ++asked) {
            if (lane == 0) {
                tc::fence_proxy_async_smem();   // the last answer was read before this one lands
                tc::mbar_arrive_expect_tx(&ctl.clc_full, 16);
                tc::clc_try_cancel(&ctl.clc, &ctl.clc_full);
            }
            int seq, t0;
            if (find_item(a, p, x, &seq, &t0)) {
                const SeqRows r = paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, seq,
                                            lane ? nullptr : a.err);
                if (t0 < r.n) {
                    const bool free = n < 2 || wait(ctl, &ctl.it_empty[n & 1], ((n >> 1) - 1) & 1);
                    if (!__all_sync(0xffffffffu, free)) {
                        wait(ctl, &ctl.clc_full, asked & 1);
                        break;
                    }
                    // the records of the last item but one: every role is done with it
                    if (*(volatile int*)&ctl.has_bad[n & 1]) {
                        for (int i = lane; i < HD; i += 32) ctl.bad[n & 1][i] = NO_BAD;
                        __syncwarp();
                        if (lane == 0) ctl.has_bad[n & 1] = 0;
                    }
                    __syncwarp();
                    if (lane == 0) {
                        Item& it = ctl.item[n & 1];
                        const int ntok = min(2 * p.T, r.n - t0), lim0 = r.len - r.n + t0 + 1, last = lim0 + ntok - 1;
                        const int kt0 = x % p.nsplit * p.spt, nkt = last > 0 ? (last + BKV - 1) / BKV : 0;
                        it.valid = 1;
                        it.seq = seq;
                        it.g = x / p.nsplit % a.kv.nkv;
                        it.split = x % p.nsplit;
                        it.tok0 = r.row0 + t0;
                        it.ntok = ntok;
                        it.lim0 = lim0;
                        it.last = last;
                        it.kt0 = kt0;
                        it.nkt = max(0, min(nkt, kt0 + p.spt) - kt0);
                        tc::mbar_arrive(&ctl.it_full[n & 1]);
                    }
                    ++n;
                }
            }
            // item 0's block looks at all sequences: one that is cut to no rows at
            // all has no tile that would say so (direct: each has a tile)
            if (x == 0 && !p.direct) look_at_all(ctl.a);
            const bool answered = wait(ctl, &ctl.clc_full, asked & 1);
            if (!__all_sync(0xffffffffu, answered)) break;
            x = tc::clc_answer(&ctl.clc);
            __syncwarp();
        }
        if (n >= 2) wait(ctl, &ctl.it_empty[n & 1], ((n >> 1) - 1) & 1);
        if (lane == 0) {
            ctl.item[n & 1].valid = 0;
            tc::mbar_arrive(&ctl.it_full[n & 1]);
        }
    } else if (warp == 0) {
        // ---- TMA producer
        int qn = 0;              // items with keys so far
        unsigned idx = 0;        // ring slots filled so far
        bool ok = true;
        for (int n = 0; ok; ++n) {
            const Item* it = take(ctl, n);
            if (!it) break;
            const int ntok = it->ntok, nkt = it->nkt, g = it->g, tok0 = it->tok0, kt0 = it->kt0, seq = it->seq;
            done_with(ctl, n);
            if (nkt == 0) continue;
            const bool dual = ntok > p.T;
            ok = qn == 0 || wait(ctl, &ctl.q_empty, (qn - 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (lane == 0) {
                const int tiles = dual ? 2 : 1;
                tc::mbar_arrive_expect_tx(&ctl.q_full, (uint32_t)(tiles * C::NB * p.T * p.G * 128));
                for (int w = 0; w < tiles; ++w)
                    for (int b = 0; b < C::NB; ++b)
                        tc::tma_load_3d(sm + C::Q_OFF + (w * C::NB + b) * BLK, &mq, b * 64, g * p.G,
                                        tok0 + w * p.T, &ctl.q_full);
            }
            ++qn;
            int pages = -1;      // lane l: page id of the tile that is l after the last multiple of 32
            for (int j = 0; ok && j < nkt; ++j, ++idx) {
                if (j % 32 == 0) {
                    const int lp = kt0 + j + lane;
                    pages = j + lane < nkt
                                ? paged_page(a.kv.table, a.kv.max_pages, a.kv.n_pages, seq, lp, a.err)
                                : -1;
                }
                const int pg = __shfl_sync(0xffffffffu, pages, j & 31);
                // no page: rows past the pool's, which read as zeros
                const int y = (pg >= 0 ? pg * a.kv.nkv + g : a.kv.n_pages * a.kv.nkv) * KV_PAGE;
                const unsigned st = idx % C::NS, use = idx / C::NS;
                ok = use == 0 || wait(ctl, &ctl.ring_empty[st], (use - 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) {
                    uint8_t* dst = sm + C::RING_OFF + st * C::SLOT;
                    tc::mbar_arrive_expect_tx(&ctl.ring_full[st], C::SLOT);
#pragma unroll
                    for (int b = 0; b < C::NB; ++b) {
                        tc::tma_load_2d(dst + b * PAGE_BYTES, &mk, b * 64, y, &ctl.ring_full[st]);
                        tc::tma_load_2d(dst + C::HALF + b * PAGE_BYTES, &mv, b * 64, y, &ctl.ring_full[st]);
                    }
                    asm volatile("st.release.cta.shared.u32 [%0], %1;" ::"r"(tc::smem_u32(&ctl.asked)), "r"(idx + 1)
                                 : "memory");
                }
                __syncwarp();
            }
        }
        // copies still in flight land before the block exits
        if (aborted(ctl)) {
            if (qn > 0) tc::mbar_wait(&ctl.q_full, (qn - 1) & 1, 1u << 20);
            for (unsigned i = idx > C::NS ? idx - C::NS : 0; i < idx; ++i)
                tc::mbar_wait(&ctl.ring_full[i % C::NS], (i / C::NS) & 1, 1u << 20);
        }
    } else if (warp < 4) {
        // ---- MMA issuers: warp 1 for warpgroup 0's tiles, warp 3 for warpgroup 1's
        constexpr uint32_t TY = BF16 ? (1u << 7) | (1u << 10) : 0u;
        constexpr uint32_t idS = tc::idesc_f16(128, BKV) | TY;
        constexpr uint32_t idO = tc::idesc_f16_bmn(128, HD) | TY;
        const int w = warp >> 1;
        int qn = 0;              // items with keys
        unsigned steps = 0;      // this warpgroup's softmax steps; step i uses buffer i & 1
        unsigned base = 0;       // ring slots used by earlier items
        bool ok = true;
        for (int n = 0; ok; ++n) {
            const Item* it = take(ctl, n);
            if (!it) break;
            const int J = it->nkt;
            const bool dual = it->ntok > p.T;
            done_with(ctl, n);
            if (J == 0) continue;
            // Key tiles j0, j0 + dj, ...: tile j is ring slot base + j.  A dual
            // item's slots are freed by both issuers, a solo item's by two
            // arrivals of the one that uses them.
            const int j0 = dual ? 0 : w, dj = dual ? 1 : 2;
            const uint64_t qd = tc::desc_sw128(sm + C::Q_OFF + (dual ? w : 0) * C::NB * BLK);
            auto slot = [&](int j) { return sm + C::RING_OFF + (base + j) % C::NS * C::SLOT; };
            auto s_mma = [&](int j, unsigned step) {   // S = Q K_j^T
                const uint64_t kd = tc::desc_sw128(slot(j));
                const uint32_t tS = tmem + (2 * w + (step & 1)) * BKV;
#pragma unroll
                for (int k16 = 0; k16 < HD / 16; ++k16)
                    tc::mma_f16(tS, qd + (k16 >> 2) * (BLK / 16) + 2 * (k16 & 3),
                                kd + (k16 >> 2) * (PAGE_BYTES / 16) + 2 * (k16 & 3), idS, k16 > 0);
                tc::mma_commit(&ctl.s_full[w][step & 1]);
                if (j + dj >= J) tc::mma_commit(&ctl.q_empty);
            };
            ok = wait(ctl, &ctl.q_full, qn & 1);
            if (j0 >= J && lane == 0) tc::mbar_arrive(&ctl.q_empty);
            for (int i = 0; i < 2; ++i) {   // the first S of both buffers
                const int j = j0 + i * dj;
                if (j >= J) break;
                ok = ok && slot_full(ctl, base + j, C::NS);
                if (!__all_sync(0xffffffffu, ok)) break;
                tc::tc_fence_after();
                if (tc::elect_one()) s_mma(j, steps + i);
                __syncwarp();
            }
            for (int j = j0; __all_sync(0xffffffffu, ok) && j < J; j += dj, ++steps) {
                const bool more = j + 2 * dj < J;
                const unsigned b = steps & 1;
                // the tiles are usually there long before P, whose wait is last:
                // then P V and the next S go out in one run
                ok = (!more || slot_full(ctl, base + j + 2 * dj, C::NS)) &&
                     wait(ctl, &ctl.p_full[w][b], (steps >> 1) & 1);
                if (!__all_sync(0xffffffffu, ok)) break;
                tc::tc_fence_after();
                if (tc::elect_one()) {
                    // A = P (TMEM, over S's columns), B = V (MN-major: hd contiguous per key)
                    const uint64_t vd = tc::desc_sw128_mn(slot(j) + C::HALF, PAGE_BYTES);
                    const uint32_t tP = tmem + (2 * w + b) * BKV;
                    // (of two warpgroups the one with buffer b accumulates this tile)
                    const int u = C::NU == 2 ? b : 0;
                    const uint32_t tO = tmem + C::O_COL + (w * C::NU + u) * HD;
#pragma unroll
                    for (int k16 = 0; k16 < BKV / 16; ++k16)
                        tc::mma_f16_ts(tO, tP + k16 * 8, vd + k16 * (16 * 128 / 16), idO,
                                       j >= j0 + C::NU * dj || k16 > 0);
                    if (C::NU == 1) tc::mma_commit(&ctl.pv_done[w][b]);
                    tc::mma_commit(&ctl.ring_empty[(base + j) % C::NS]);
                    if (!dual) tc::mma_commit(&ctl.ring_empty[(base + j) % C::NS]);
                    if (j + C::NU * dj >= J) tc::mma_commit(&ctl.o_full[w][u]);
                    if (more) s_mma(j + 2 * dj, steps + 2);
                }
                __syncwarp();
            }
            ok = __all_sync(0xffffffffu, ok);
            ++qn;
            base += J;
        }
        if (tc::elect_one()) tc::mma_commit(&ctl.mma_done);   // completes after every MMA issued above
        __syncwarp();
    } else {
        softmax_role<HD, BF16>(sm, tmem);
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

// The packed row of the splits' token i, or -1 if no sequence has it: then
// nothing was written for it, and its outputs are not this call's.  Whole warp.
__device__ __forceinline__ int merge_row(const PagedAttnArgs& a, const AttnPlan& p, int i) {
    if (p.direct) {
        const SeqRows r = paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, i / a.max_q, nullptr);
        return i % a.max_q < r.n ? r.row0 + i % a.max_q : -1;
    }
    // the last sequence that begins at or before row i, 32 probes at a time
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = a.kv.n_seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, s = lo + lane * step;
        const int n = __popc(__ballot_sync(0xffffffffu, s < hi && __ldg(a.q_start + s) <= i));
        if (n == 0) return -1;
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    const SeqRows r = paged_seq(a.kv, a.q_start, a.kv_len, a.total_q, a.max_q, a.max_kv, lo, nullptr);
    return i >= r.row0 && i < r.row0 + r.n ? i : -1;
}

// Joins the key splits of a row, W warps (token, head), a lane holds hd / 32
// columns; the splits' factors are 2^(m_i - m) / l.  One warp walks up to
// MERGE_WARP splits; more are dealt out to four and added in their order.
constexpr int MERGE_WARP = 8;
template <int HD, bool BF16, int W>
__global__ void __launch_bounds__(128) k_attn_paged_merge(const PagedAttnArgs a, const AttnPlan p) {
    constexpr int E = HD / 32;
    __shared__ float so[W][HD], sl[W];
    const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) % W;
    const int64_t all = p.tokens * a.nq;
    const unsigned row = W == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x, i = row / a.nq;
    // (the lengths were there before the splits' kernel began)
    const int tok = i < p.tokens ? merge_row(a, p, (int)i) : -1, h = (int)(row % a.nq);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (tok < 0) return;   // (whole blocks where they share a row)
    const int64_t r = row;
    float m = -INFINITY;
    for (int i = lane; i < p.nsplit; i += 32) m = fmaxf(m, p.part_ml[i * all + r].x);
    m = warp_max(m);
    float l = 0.f, o[E] = {};
#pragma unroll 4
    for (int i = w; i < p.nsplit; i += W) {
        const float2 ml = p.part_ml[i * all + r];
        const float* x = p.part + (i * all + r) * HD + lane * E;
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = x[e];
        const float f = ex2(ml.x - m);
        // the row sees no key of a split whose sum is 0 (and nothing was written)
        l = ml.y == 0.f ? l : fmaf(ml.y, f, l);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = ml.y == 0.f ? o[e] : fmaf(v[e], f, o[e]);
    }
    if (W > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) so[w][lane * E + e] = o[e];
        if (lane == 0) sl[w] = l;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int k = 1; k < W; ++k) {
            l += sl[k];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += so[k][lane * E + e];
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + (size_t)tok * a.out_stride + (size_t)h * HD + lane * E);
#pragma unroll
    for (int e = 0; e < E; e += 2) dst[e / 2] = pack2<BF16>(o[e] * inv, o[e + 1] * inv);
    if (a.lse && lane == 0) a.lse[(size_t)tok * a.nq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718056f;
}

size_t split_bytes(const PagedAttnArgs& a, const AttnPlan& p) { return (size_t)p.tokens * a.nq * (a.kv.hd * 4 + 8); }

// Tiles, and as many key splits as fill the SMs and fit the workspace.
AttnPlan make_plan(const PagedAttnArgs& a, int n_sm, size_t workspace) {
    AttnPlan p;
    p.G = a.nq / a.kv.nkv;
    p.T = min(128 / p.G, max(1, a.max_q));   // (a box of queries no larger than a sequence's)
    p.c = (float)((double)a.scale * 1.4426950408889634);
    const int step = 2 * p.T, kt = (a.max_kv + BKV - 1) / BKV;
    p.few = (long long)a.max_q * p.G <= FEW_ROWS;
    p.direct = a.max_q <= step;
    const long long busy = p.direct ? a.kv.n_seqs : (a.total_q + step - 1) / step;
    // whole tiles of every sequence, and one more each for what is left over
    const long long most = p.direct ? a.kv.n_seqs : (long long)a.total_q / step + a.kv.n_seqs;
    p.n_tiles = (int)most;
    // (of `few` two blocks fit an SM with 64 columns)
    const long long items = busy * a.kv.nkv, slots = p.few && a.kv.hd == 64 ? 2 * n_sm : n_sm;
    long long ns = items > 0 && items < slots ? slots / items : 1;
    // Enough key tiles each to be worth the merge's launch (some 3 us).
    const int least = p.few ? 4 : 8;
    ns = min(ns, kt > 16 ? (long long)(kt + least - 1) / least : 1LL);
    p.tokens = p.direct ? (int64_t)a.kv.n_seqs * a.max_q : a.total_q;
    if (ns > 1) ns = max(1LL, min(ns, (long long)(workspace / split_bytes(a, p))));   // (few sequences: no overflow)
    p.spt = max(1, (int)((kt + ns - 1) / ns));
    p.nsplit = max(1, (kt + p.spt - 1) / p.spt);
    p.part = static_cast<float*>(a.workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part + (size_t)p.nsplit * p.tokens * a.nq * a.kv.hd);
    return p;
}

template <int HD, bool BF16>
cudaError_t launch_merge(const PagedAttnArgs& a, const AttnPlan& p, cudaStream_t st) {
    const int64_t rows = p.tokens * a.nq;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.nsplit > MERGE_WARP ? rows : (rows + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = p.nsplit > MERGE_WARP ? cudaLaunchKernelEx(&cfg, k_attn_paged_merge<HD, BF16, 4>, a, p)
                                                : cudaLaunchKernelEx(&cfg, k_attn_paged_merge<HD, BF16, 1>, a, p);
    note_launch();
    return e;
}

template <int HD, bool BF16>
cudaError_t launch(const PagedAttnArgs& a, const AttnPlan& p, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    const int64_t rows = (int64_t)a.kv.n_pages * a.kv.nkv * KV_PAGE;
    if (!make_kv_map(&mk, reinterpret_cast<const __half*>(a.kv.k), rows, HD) ||
        !make_kv_map(&mv, reinterpret_cast<const __half*>(a.kv.v), rows, HD))
        return cudaErrorInvalidValue;
    if (p.few) {
        const cudaError_t e = attn_paged_few_launch(a, p, mk, mv, st);
        return e != cudaSuccess || p.nsplit == 1 ? e : launch_merge<HD, BF16>(a, p, st);
    }
    if (!make_heads_map(&mq, a.q, HD, a.nq, a.total_q, a.q_stride, p.G, p.T))
        return cudaErrorInvalidValue;
    const long long grid = (long long)p.n_tiles * a.kv.nkv * p.nsplit;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
    cudaError_t e = cudaFuncSetAttribute(k_attn_paged<HD, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         smem_bytes<HD>());
    if (e != cudaSuccess) return e;
    k_attn_paged<HD, BF16><<<(unsigned)grid, Cfg<HD>::THREADS, smem_bytes<HD>(), st>>>(mq, mk, mv, a, p);
    note_launch();
    e = cudaGetLastError();
    return e != cudaSuccess || p.nsplit == 1 ? e : launch_merge<HD, BF16>(a, p, st);
}

}  // namespace

size_t attn_paged_workspace(const PagesView& kv, int total_q, int max_q, int max_kv, int nq, int n_sm) {
    PagedAttnArgs a;
    a.kv = kv;
    a.total_q = total_q;
    a.max_q = max_q;
    a.max_kv = max_kv;
    a.nq = nq;
    const AttnPlan p = make_plan(a, n_sm, ~(size_t)0);
    return p.nsplit > 1 ? p.nsplit * split_bytes(a, p) : 0;
}

cudaError_t attn_paged_launch(const PagedAttnArgs& a, int n_sm, cudaStream_t st) {
    const AttnPlan p = make_plan(a, n_sm, a.workspace_bytes);
    if (a.kv.hd == 64) return a.kv.bf16 ? launch<64, true>(a, p, st) : launch<64, false>(a, p, st);
    return a.kv.bf16 ? launch<128, true>(a, p, st) : launch<128, false>(a, p, st);
}

}  // namespace vvq2
