/*
 * Attention of a step's new tokens over a pool of pages: token j that request r brings attends positions [0, rows[r] + j] of
 * that request, with the query heads of a kv head sharing every row that is read.
 *
 *     o = sum_p w_p v_p / sum_p w_p,  w_p = 2^(scale log2(e) q.k_p - m),  m the running maximum;  out = o sigmoid(gate)
 *
 * q4_pg_few_k, tokens of requests that bring few.  Bound by memory: every row is read once, for 8 to 32 (token, head) pairs.
 * Both contractions run on warp-level MMA with the positions as M, so that 8 pairs are a whole tile of the product:
 * S^T = K Q^T and O^T += V^T P^T, 16 positions per step of a warp.
 *
 * Requests differ in length by orders of magnitude, so blocks are not given requests but equal shares of the step's whole work:
 * the steps (128 positions) of all units (request, kv head, group of tokens) lie one behind the other, and block c takes steps
 * [T c / C, T (c + 1) / C).  Where a share ends inside a unit the block leaves (acc, m, l) records, at most two, and the unit's
 * blocks meet and join them.  The division is computed by every block itself from the lengths on the device (one scan), which
 * the host need not know.
 */
#include <cuda_bf16.h>
#include <math_constants.h>
#include <string.h>
#include <type_traits>

#include "q4_paged.h"

namespace {

constexpr uint32_t PG_SPIN_LIMIT = 1u << 20;
__device__ uint32_t g_few_meet[PG_MAX_BLOCKS];

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done != 0u;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/* the same with an initial accumulator of its own, one value per column */
__device__ __forceinline__ void mma16816_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
/* fp16 1024 + 128 + code has (code ^ 0x80) in its low byte: two bytes picked out of word x (its codes ^ 0x80), and the exact codes */
template <uint32_t SEL>
__device__ __forceinline__ uint32_t raised2(uint32_t x) { return __byte_perm(x, 0x64646464u, SEL); }
template <uint32_t SEL>
__device__ __forceinline__ uint32_t codes2(uint32_t x) { return h2u(__hsub2(u2h(raised2<SEL>(x)), u2h(0x64806480u))); }

/* the rows of the tile at sb (by a whole warp) whose V holds a number that is not finite; rows behind the last position may be among them */
template <int KIND, int HD>
__device__ __forceinline__ uint32_t not_finite(uint32_t sb, uint32_t lane) {
    constexpr uint32_t TILE = PgTile<KIND, HD>::BYTES;
    uint32_t rows = 0;
    if constexpr (KIND == Q4K_Q8) {   /* fp16(127 x scale) is not from 516 on */
        const uint32_t a = sb + (lane & 15u) * (TILE / 16u) + 2u * HD + HD / 16u;
#pragma unroll
        for (uint32_t b = 0; b < HD / 64u; b++) {
            const uint32_t x = lds32(a + 4u * b);
            if ((x & 0x7fffu) > 0x6007u || (x >> 16 & 0x7fffu) > 0x6007u) rows = 1u << (lane & 15u);
        }
    } else {   /* exponents of ones only */
#pragma unroll 4
        for (uint32_t i = 0; i < HD / 8u; i++) {   /* 8 bytes at a time: two rows of a block of 64 dims */
            const uint2 w = lds64(sb + TILE / 2u + i * 256u + lane * 8u);
            const bool x = (w.x & 0x7c00u) == 0x7c00u || (w.x & 0x7c000000u) == 0x7c000000u || (w.y & 0x7c00u) == 0x7c00u || (w.y & 0x7c000000u) == 0x7c000000u;
            if (x) rows |= 1u << ((2u * i + (lane >> 4)) & 15u);
        }
    }
    return __reduce_or_sync(0xffffffffu, rows);
}

/* warps per block, blocks per SM, tiles of a warp's ring: as many bytes in flight as an SM's shared memory holds */
template <int KIND, int HD, int NT>
struct FewCfg {
    static constexpr uint32_t TILE = PgTile<KIND, HD>::BYTES;
    static constexpr uint32_t ROWS = 8u * NT;
    static constexpr uint32_t CTAS = (TILE <= 4352u && NT * HD <= 128) ? 2u : 1u;   /* 128 registers: more columns do not fit */
    static constexpr uint32_t WARPS = TILE > 8704u ? 4u : 8u;
    static constexpr uint32_t FIT = 209000u / (CTAS * WARPS * TILE), DEPTH = FIT < 6u ? FIT : 6u;
    static constexpr uint32_t THREADS = WARPS * 32u;
    static constexpr uint32_t STEP = WARPS * 16u;            /* positions per step */
    static constexpr uint32_t EXTRA = 3u;                    /* steps that a piece costs besides its own, where blocks have several */
    static constexpr uint32_t Q_STRIDE = HD * 2u + 32u;      /* the four rows of a half-warp's 8-byte reads on different banks */
    static constexpr uint32_t RING = WARPS * DEPTH * TILE;
    static constexpr uint32_t REC = HD + 4u;
    /* the warps' records reuse the ring: of all warps at once, or of half of them, which have taken over the others' fragments */
    static constexpr uint32_t FRAG = (HD / 16u * 4u + 4u) * NT * 32u * 4u, PARTS = WARPS * ROWS * REC * 4u <= RING ? WARPS : WARPS / 2u;
    static_assert(ROWS <= (WARPS - 1u) * 16u + 1u, "masks in a warp's last tile only");
    static_assert(WARPS / 2u * FRAG <= RING && PARTS * ROWS * REC * 4u <= RING, "merge does not fit");
    static constexpr uint32_t DIRECT = 16u;                  /* records that the unit's last block joins alone */
    static constexpr uint32_t SMEM = RING + ROWS * Q_STRIDE + WARPS * DEPTH * 8u + 1024u;
};

template <int KIND, int HD, int NT>
__global__ void __launch_bounds__(FewCfg<KIND, HD, NT>::THREADS, FewCfg<KIND, HD, NT>::CTAS) q4_pg_few_k(const PagedParams P) {
    using C = FewCfg<KIND, HD, NT>;
    constexpr uint32_t TILE = C::TILE, WARPS = C::WARPS, DEPTH = C::DEPTH, STEP = C::STEP, MT = HD / 16u;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint64_t s_sum[2u * WARPS];
    __shared__ uint64_t s_off, s_end2[2];
    __shared__ PgShares s_shares;   /* what only the ends of pieces need is kept here: registers are short in the loop between */
    __shared__ PgSplit s_split[2];  /* units that began before this block; that go on behind it */
    __shared__ uint32_t s_req, s_last;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t s_base = (smem_u32(smem) + 1023u) & ~1023u;   /* swizzled tiles are anchored to multiples of 1024 */
    uint8_t *base = smem + (s_base - smem_u32(smem));
    const uint32_t ring = s_base + warp * DEPTH * TILE, s_q = s_base + C::RING, bars = s_q + C::ROWS * C::Q_STRIDE + warp * DEPTH * 8u;
    if (lane == 0)
        for (uint32_t i = 0; i < DEPTH; i++) bar_init(bars + 8u * i, 1u);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    /* Beside the chunks of its own call it takes the SMs that they leave: that launch began behind everything before it, and nothing
     * here reads what it writes (a mixed step 279 -> 256 us in a burst, 291 -> 273 over a second of them; in q8_0 297 -> 277 and 296 -> 281).  What it reads may be two launches old: by loads that do not look into L1.  The
     * end of that launch is waited for at the end, for those behind this one. */
    if (!P.beside) q4d_pdl_wait();

    /* ---- this block's share of all steps */
    auto mine_of = [&](uint32_t r, bool &bad) -> PgReq {
        PgReq q = pg_request(P, r, bad);
        if (q.add > P.add_split) q.add = 0u;
        return q;
    };
    const uint32_t per = (P.n_req + C::THREADS - 1u) / C::THREADS, r0 = min(tid * per, P.n_req), r1 = min(r0 + per, P.n_req);
    uint64_t mine = 0, units = 0, total, all_units, before, units_before;
    bool bad, any_bad = false;
    PgReq mine_is = {0u, 0u, 0u};
    auto units_of = [&](const PgReq &q) -> uint64_t { return (uint64_t)((q.add + P.tpg - 1u) / P.tpg) * P.n_kvh; };   /* no tokens: none */
    auto steps_in = [&](const PgReq &q) -> uint32_t { return (q.held + q.add + STEP - 1u) / STEP; };
    for (uint32_t r = r0; r < r1; r++) {
        mine_is = mine_of(r, bad);
        units += units_of(mine_is);
        mine += units_of(mine_is) * steps_in(mine_is);
        any_bad |= bad;
    }
    {
        uint64_t x = mine, y = units;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
            if (lane >= (uint32_t)d) { x += u; y += v; }
        }
        if (lane == 31u) { s_sum[warp] = x; s_sum[WARPS + warp] = y; }
        __syncthreads();
        total = all_units = before = units_before = 0;
#pragma unroll
        for (uint32_t w = 0; w < WARPS; w++) {
            if (w < warp) { before += s_sum[w]; units_before += s_sum[WARPS + w]; }
            total += s_sum[w];
            all_units += s_sum[WARPS + w];
        }
        before += x - mine;
        units_before += y - units;
    }
    /* Where the blocks have many steps each, a unit counts as EXTRA more, that a piece costs, and short ones stay whole (a token of 64
     * sessions 116 -> 113 us).  Where they have few, the way through the launch counts: units are cut as finely as there are
     * blocks, down to one step (a token of four short chats 13.4 us whole, 11.4 so), but where a unit has three at most (one such chat 9.7 us cut, 8.5 whole). */
    const uint32_t extra = total >= 4u * gridDim.x ? C::EXTRA : 0u;   /* also shares.near */
    total += all_units * extra; before += units_before * extra; mine += units * extra;
    if (blockIdx.x == 0 && any_bad) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    PgShares shares;
    shares.set(total, extra, extra ? 8u : 3u, extra ? 4u : 1u);
    if (blockIdx.x >= shares.blocks) {
        if (P.beside) q4d_pdl_wait();
        return;
    }
    if (tid == 0) {
        s_end2[0] = s_end2[1] = total;
        s_shares = shares;
        s_split[0] = s_split[1] = {1u, 0u, 0u, 0u, 0u};
    }
    __syncthreads();
    for (uint32_t i = 0; i < 2u && mine && blockIdx.x + i < shares.blocks; i++) {   /* the two cuts */
        const uint64_t x = shares.cut(blockIdx.x + i);
        if (x < before || x >= before + mine) continue;
        uint64_t at = before;
        for (uint32_t r = r0; r < r1; r++) {
            if (per > 1u) mine_is = mine_of(r, bad);
            const uint32_t steps = steps_in(mine_is) + extra;
            const uint64_t n = units_of(mine_is) * steps;
            if (x < at + n) {
                const uint64_t in = x - at, u0 = in >> 32 ? in / steps * steps : (uint32_t)in / steps * steps, to = u0 + shares.snap(in - u0, steps);
                if (i == 0u) {
                    s_req = r;
                    s_off = to;
                }
                s_end2[i] = at + to;
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    uint32_t req = s_req, issued = 0, taken = 0;   /* of the warp's ring, over all pieces */
    uint64_t off = s_off, s = s_end2[0];
    bool ok = true;

    /* ---- pieces of units */
    while (s < s_end2[1]) {
        const PgReq R = mine_of(req, bad);
        const uint32_t groups = (R.add + P.tpg - 1u) / P.tpg, n_steps = steps_in(R), extra = s_shares.near, steps = n_steps + extra;
        if (off >= (uint64_t)groups * P.n_kvh * steps) {   /* on to the next request; requests without tokens are passed over */
            off -= (uint64_t)groups * P.n_kvh * steps;
            req++;
            continue;
        }
        const uint32_t unit = off >> 32 ? (uint32_t)(off / steps) : (uint32_t)off / steps, at = (uint32_t)(off - (uint64_t)unit * steps);
        const uint32_t take = (uint32_t)min((uint64_t)(steps - at), s_end2[1] - s);
        const uint32_t st = max(at, extra) - extra, here = max(at + take, extra) - extra - st;   /* the first `extra` steps are none */
        const uint32_t kh = unit / groups, j0 = (unit - kh * groups) * P.tpg, n_here = min(P.tpg, R.add - j0);
        const uint32_t n_kv = R.held + j0 + n_here, live_rows = n_here * P.gqa, tok0 = R.tok0 + j0;

        __syncthreads();   /* the piece before has been read */
        /* positions that column 2 t + e of row tile i may see */
        uint32_t lim[NT][2], lim_min = n_kv;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (uint32_t e = 0; e < 2; e++) {
                const uint32_t row = 8u * i + 2u * t + e;
                lim[i][e] = row < live_rows ? R.held + j0 + row / P.gqa + 1u : n_kv;
                lim_min = min(lim_min, lim[i][e]);
            }
        lim_min = __reduce_min_sync(0xffffffffu, lim_min);

        /* ---- this warp's tiles of the piece, numbered i = 0 .. : tile (st + i) * WARPS + warp of the unit */
        const uint32_t tiles = (n_kv + 15u) / 16u;
        uint32_t n_my = 0;
        if (ok && st * WARPS + warp < tiles) n_my = min(here, (tiles - 1u - st * WARPS - warp) / WARPS + 1u);
        auto entry = [&](uint32_t i) -> int32_t { return i < n_my ? __ldcg(P.table + (size_t)req * P.table_stride + ((((st + i) * WARPS + warp) * 16u) >> P.page_shift)) : 0; };
        int32_t cur = -1, nxt = entry(lane);
        uint32_t dead = 0, dead_nxt = 0;   /* tiles of the present / the next 32 whose page is not the pool's */
        const uint8_t *src = P.mem;
        uint32_t ahead = 0;
        auto issue = [&]() {   /* tile `ahead`, by the lane that holds its page */
            if ((ahead & 31u) == 0u) {
                cur = nxt;
                nxt = entry(ahead + 32u + lane);
                const uint32_t p = ((st + ahead + lane) * WARPS + warp) * 16u;
                const bool there = cur >= 0 && (uint32_t)cur < P.n_pages;
                src = P.mem + (uint64_t)(there ? (uint32_t)cur : 0u) * P.page_bytes + (uint64_t)kh * P.part_bytes + ((p & ((1u << P.page_shift) - 1u)) >> 4) * TILE;
                cur = there ? 0 : -1;
                dead_nxt = __ballot_sync(0xffffffffu, !there);
                if (ahead == 0u) dead = dead_nxt;
            }
            const uint32_t slot = issued % DEPTH;
            if (lane == (ahead & 31u)) {
                if (cur >= 0) {
                    bar_expect(bars + 8u * slot, TILE);
                    bulk_load(ring + slot * TILE, src, TILE, bars + 8u * slot);
                } else {
                    bar_arrive(bars + 8u * slot);
                    atomicOr(P.err, (uint32_t)Q4E_RANGE);
                }
            }
            ahead++;
            issued++;
        };
        while (ahead < n_my && ahead < DEPTH) issue();

        /* ---- the unit's queries as fp16, while the first tiles come in */
        for (uint32_t i = tid; i < C::ROWS * (HD / 4u); i += C::THREADS) {
            const uint32_t row = i / (HD / 4u), d = i % (HD / 4u) * 4u;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row < live_rows) {
                const size_t at = ((size_t)(tok0 + row / P.gqa) * P.n_head + kh * P.gqa + row % P.gqa) * HD + d;
                if (P.q_bf16) {
                    const uint2 w = __ldcg(reinterpret_cast<const uint2 *>(reinterpret_cast<const __nv_bfloat16 *>(P.q) + at));
                    x = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
                } else {
                    x = __ldcg(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(P.q) + at));
                }
            }
            const uint32_t lo = h2u(__floats2half2_rn(x.x, x.y)), hi = h2u(__floats2half2_rn(x.z, x.w)), a = s_q + row * C::Q_STRIDE;
            if (KIND == Q4K_Q8) {
                /* lane t feeds dims 4 t .. 4 t + 3 of 16, as it gets the codes */
                asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(a + d * 2u), "r"(lo), "r"(hi) : "memory");
            } else {
                /* lane t feeds dims 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of 16: one behind the other */
                const uint32_t in = d & 15u, p = a + (d & ~15u) * 2u + (in & 7u) / 2u * 8u + (in >> 3) * 4u;
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(p), "r"(lo) : "memory");
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(p + 8u), "r"(hi) : "memory");
            }
        }
        __syncthreads();


        float o[MT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int i = 0; i < NT; i++) {
            m[i][0] = m[i][1] = -CUDART_INF_F;
            l[i][0] = l[i][1] = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < MT; k++) o[k][i][0] = o[k][i][1] = o[k][i][2] = o[k][i][3] = 0.f;
        }
        /* codes enter K Q^T raised by 1152: the product starts from -1152 times the sum of the queries over the block (exact
         * codes to fp32 sums; two subtractions per word less).  More columns take the subtractions. */
        constexpr bool RAISED = KIND == Q4K_Q8 && NT == 1;
        float below[RAISED ? HD / 32 : 1][2];
        if constexpr (RAISED) {
#pragma unroll
            for (uint32_t b = 0; b < HD / 32u; b++)
#pragma unroll
                for (uint32_t e = 0; e < 2; e++) {
                    /* lane (g, t) sums dims 4 g .. 4 g + 3 of column 2 t + e, the eight lanes of a column then one another's */
                    const uint2 w = lds64(s_q + (2u * t + e) * C::Q_STRIDE + b * 64u + g * 8u);
                    const float2 f0 = __half22float2(u2h(w.x)), f1 = __half22float2(u2h(w.y));
                    float x = (f0.x + f0.y) + (f1.x + f1.y);
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    below[b][e] = -1152.f * x;
                }
        }
        const uint32_t mrow = (lane & 7u) + ((lane >> 3) & 1u) * 8u, mchunk = lane >> 4;   /* of ldmatrix: the row and 16-byte piece this lane addresses */
        uint32_t slot = taken % DEPTH, phase = (taken / DEPTH) & 1u;                       /* of the next tile to wait for */
        auto landed = [&]() -> uint32_t {   /* waits for it, and goes on */
            const uint32_t sb = ring + slot * TILE;
            for (uint32_t spin = 0; !bar_test(bars + 8u * slot, phase); spin++)
                if (spin >= PG_SPIN_LIMIT) { ok = false; break; }
            ok = __all_sync(0xffffffffu, ok);
            if (++slot == DEPTH) { slot = 0u; phase ^= 1u; }
            taken++;
            return sb;
        };
        /* scores of the tile at sb: c0, c1 of position g, c2, c3 of position g + 8, columns 2 t and 2 t + 1 */
        auto scores = [&](uint32_t sb, float (&sc)[NT][4]) {
#pragma unroll
            for (int n = 0; n < NT; n++) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
            if constexpr (KIND == Q4K_Q8) {
                constexpr uint32_t NB = HD / 32u;
                uint32_t k0[NB / 2], k1[NB / 2];   /* K scales of positions g and g + 8 */
                const uint32_t ka = sb + g * (TILE / 16u) + 2u * HD, kb = ka + 8u * (TILE / 16u);
#pragma unroll
                for (uint32_t b = 0; b < NB / 2; b++) { k0[b] = lds32(ka + 4u * b); k1[b] = lds32(kb + 4u * b); }
#pragma unroll
                for (uint32_t b = 0; b < NB; b++) {
                    uint32_t w[4], a0[4], a1[4];
                    ldmatrix_x4(w, sb + mrow * (TILE / 16u) + (2u * b + mchunk) * 16u);
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] ^= 0x80808080u;
                    if constexpr (RAISED) {
                        a0[0] = raised2<0x4140>(w[0]); a0[2] = raised2<0x4342>(w[0]); a0[1] = raised2<0x4140>(w[1]); a0[3] = raised2<0x4342>(w[1]);
                        a1[0] = raised2<0x4140>(w[2]); a1[2] = raised2<0x4342>(w[2]); a1[1] = raised2<0x4140>(w[3]); a1[3] = raised2<0x4342>(w[3]);
                    } else {
                        a0[0] = codes2<0x4140>(w[0]); a0[2] = codes2<0x4342>(w[0]); a0[1] = codes2<0x4140>(w[1]); a0[3] = codes2<0x4342>(w[1]);
                        a1[0] = codes2<0x4140>(w[2]); a1[2] = codes2<0x4342>(w[2]); a1[1] = codes2<0x4140>(w[3]); a1[3] = codes2<0x4342>(w[3]);
                    }
                    const float2 f0 = __half22float2(u2h(k0[b / 2])), f1 = __half22float2(u2h(k1[b / 2]));
                    const float e0 = b & 1u ? f0.y : f0.x, e1 = b & 1u ? f1.y : f1.x;
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const uint32_t qa = s_q + (8u * n + g) * C::Q_STRIDE + b * 64u + t * 8u;
                        const uint2 qx = lds64(qa), qy = lds64(qa + 32u);
                        float c[4];
                        if constexpr (RAISED) mma16816_from(c, a0, qx.x, qx.y, below[b][0], below[b][1]);
                        else mma16816_from(c, a0, qx.x, qx.y, 0.f, 0.f);
                        mma16816(c, a1, qy.x, qy.y);
                        sc[n][0] = fmaf(c[0], e0, sc[n][0]); sc[n][1] = fmaf(c[1], e0, sc[n][1]);
                        sc[n][2] = fmaf(c[2], e1, sc[n][2]); sc[n][3] = fmaf(c[3], e1, sc[n][3]);
                    }
                }
            } else {
#pragma unroll
                for (uint32_t ks = 0; ks < MT; ks++) {
                    uint32_t a[4];
                    const uint32_t c = 2u * ks + mchunk;
                    ldmatrix_x4(a, sb + (c >> 3) * 2048u + mrow * 128u + (((c & 7u) ^ (mrow & 7u)) << 4));
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const uint2 qx = lds64(s_q + (8u * n + g) * C::Q_STRIDE + ks * 32u + t * 8u);
                        mma16816(sc[n], a, qx.x, qx.y);
                    }
                }
            }
        };
        /* Tile i at sb, whose scores are in sc.  The scores of the next one are computed beside its P V: neither needs the other, and a
         * warp's chain of one tile alone (4000 cycles) left a third of the issue slots empty. */
        float sc[NT][4];
        uint32_t sb = 0;
        auto step = [&](uint32_t i, auto more) {
            const uint32_t p0 = ((st + i) * WARPS + warp) * 16u;
            uint32_t sb_next = 0;
            if constexpr (decltype(more)::value) {
                sb_next = landed();
                if (!ok) return;
            }
            const bool gone = (dead >> (i & 31u)) & 1u;   /* its page is not the pool's: all masked */
            if ((i & 31u) == 31u) dead = dead_nxt;
            /* Rows whose V is taken: a weight of 0 does not keep one that is not finite from a sum.  Those behind the last position hold
             * anything; one that some columns attend and some do not is left out too, and makes the former NaN by their scores.
             * Both can be in a warp's last tile only: the positions from lim_min on lie in consecutive tiles of different warps. */
            uint32_t live16 = gone ? 0u : 0xffffu;
            if (gone) {
#pragma unroll
                for (int n = 0; n < NT; n++) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = -CUDART_INF_F;
            }
            if constexpr (!decltype(more)::value) {
                if (p0 + 16u > lim_min && !gone) {
                    if (p0 + 16u > n_kv) live16 = (1u << (n_kv - p0)) - 1u;
                    if (lim_min < n_kv) {
                        const uint32_t bad = not_finite<KIND, HD>(sb, lane);
                        if (bad) {
#pragma unroll
                            for (int n = 0; n < NT; n++)
#pragma unroll
                                for (int k = 0; k < 4; k++)
                                    if ((bad >> (g + (k >> 1) * 8u)) & 1u) sc[n][k] = CUDART_NAN_F;
                            live16 &= ~bad;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            if (p0 + g + (k >> 1) * 8u >= lim[n][k & 1]) sc[n][k] = -CUDART_INF_F;
                }
            }
            /* the maxima (of scores times scale_log2e) move only where a score is above them: seldom, after the first tiles */
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) sc[n][k] *= P.scale_log2e;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) grow = grow || fmaxf(sc[n][e], sc[n][e + 2]) > m[n][e];
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float x = fmaxf(sc[n][e], sc[n][e + 2]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        if (x > m[n][e]) {
                            const float f = ex2(m[n][e] - x);
                            m[n][e] = x;
                            l[n][e] *= f;
#pragma unroll
                            for (uint32_t k = 0; k < MT; k++) { o[k][n][e] *= f; o[k][n][e + 2] *= f; }
                        }
                    }
            }
            uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
            if (live16 != 0xffffu) {
                const uint32_t rows = live16 >> (2u * t);
                keep0 = (rows & 1u ? 0xffffu : 0u) | (rows & 2u ? 0xffff0000u : 0u);
                keep1 = (rows & 0x100u ? 0xffffu : 0u) | (rows & 0x200u ? 0xffff0000u : 0u);
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float m0 = m[n][0] == -CUDART_INF_F ? 0.f : m[n][0], m1 = m[n][1] == -CUDART_INF_F ? 0.f : m[n][1];
                const float x0 = ex2(sc[n][0] - m0), x1 = ex2(sc[n][1] - m1), x2 = ex2(sc[n][2] - m0), x3 = ex2(sc[n][3] - m1);
                l[n][0] += x0 + x2;
                l[n][1] += x1 + x3;
                pb[n][0] = movmatrix_t(h2u(__floats2half2_rn(x0, x1)));
                pb[n][1] = movmatrix_t(h2u(__floats2half2_rn(x2, x3)));
            }
            if constexpr (decltype(more)::value) scores(sb_next, sc);
            /* ---- O^T += V^T P^T */
            if constexpr (KIND == Q4K_Q8) {
                constexpr uint32_t NB = HD / 32u;
                uint32_t v0[NB / 2], v1[NB / 2], v2[NB / 2], v3[NB / 2];   /* V scales of positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9 */
                const uint32_t va = sb + 2u * t * (TILE / 16u) + 2u * HD + NB * 2u;
#pragma unroll
                for (uint32_t b = 0; b < NB / 2; b++) {
                    v0[b] = lds32(va + 4u * b); v1[b] = lds32(va + TILE / 16u + 4u * b);
                    v2[b] = lds32(va + 8u * (TILE / 16u) + 4u * b); v3[b] = lds32(va + 9u * (TILE / 16u) + 4u * b);
                }
#pragma unroll
                for (uint32_t b = 0; b < NB; b++) {
                    const uint32_t sel = b & 1u ? 0x7632u : 0x5410u;
                    const __half2 f0 = u2h(__byte_perm(v0[b / 2], v1[b / 2], sel) & keep0), f1 = u2h(__byte_perm(v2[b / 2], v3[b / 2], sel) & keep1);
                    uint32_t w[4];
                    ldmatrix_x4_trans(w, sb + mrow * (TILE / 16u) + HD + (2u * b + mchunk) * 16u);
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] ^= 0x80808080u;
#pragma unroll
                    for (uint32_t c = 0; c < 2; c++) {
                        /* dims 2 g (rows g) and 2 g + 1 (rows g + 8) of 16; fp16(code x scale): 2^-12 of a value on average, as P is rounded */
                        uint32_t a[4] = {h2u(__hmul2(u2h(codes2<0x4240>(w[2 * c])), f0)), h2u(__hmul2(u2h(codes2<0x4341>(w[2 * c])), f0)),
                                         h2u(__hmul2(u2h(codes2<0x4240>(w[2 * c + 1])), f1)), h2u(__hmul2(u2h(codes2<0x4341>(w[2 * c + 1])), f1))};
#pragma unroll
                        for (int n = 0; n < NT; n++) mma16816(o[2 * b + c][n], a, pb[n][0], pb[n][1]);
                    }
                }
            } else {
#pragma unroll
                for (uint32_t k = 0; k < MT; k++) {
                    uint32_t w[4];
                    const uint32_t c = 2u * k + mchunk;
                    ldmatrix_x4_trans(w, sb + TILE / 2u + (c >> 3) * 2048u + mrow * 128u + (((c & 7u) ^ (mrow & 7u)) << 4));
                    uint32_t a[4] = {w[0], w[2], w[1], w[3]};
                    if (live16 != 0xffffu) { a[0] &= keep0; a[1] &= keep0; a[2] &= keep1; a[3] &= keep1; }
#pragma unroll
                    for (int n = 0; n < NT; n++) mma16816(o[k][n], a, pb[n][0], pb[n][1]);
                }
            }
            __syncwarp();   /* all lanes have read the slot */
            if (ahead < n_my) issue();
            sb = sb_next;
        };
        if (n_my) {
            sb = landed();
            if (ok) scores(sb, sc);
            for (uint32_t i = 0; ok && i + 1u < n_my; i++) step(i, std::true_type());
            if (ok) step(n_my - 1u, std::false_type());
        }

        /* ---- the warps' results are joined through shared memory (the rings are empty: all that was issued was taken) */
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
                l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
                l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
            }
        float *xch = reinterpret_cast<float *>(base);
        if constexpr (C::PARTS < WARPS) {
            constexpr uint32_t half = WARPS / 2u;
            __syncthreads();
            if (warp >= half) {
                float *to = xch + (warp - half) * (C::FRAG / 4u) + lane;
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) { to[(n * 4 + e) * 32] = m[n][e]; to[(n * 4 + 2 + e) * 32] = l[n][e]; }
#pragma unroll
                    for (uint32_t k = 0; k < MT; k++)
#pragma unroll
                        for (int e = 0; e < 4; e++) to[(NT * 4 + (n * MT + k) * 4 + e) * 32] = o[k][n][e];
                }
            }
            __syncthreads();
            if (warp < half) {
                const float *from = xch + warp * (C::FRAG / 4u) + lane;
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float mo = from[(n * 4 + e) * 32], lo = from[(n * 4 + 2 + e) * 32];
                        const float M = fmaxf(m[n][e], mo), Mu = M == -CUDART_INF_F ? 0.f : M;
                        const float fa = ex2(m[n][e] - Mu), fb = ex2(mo - Mu);
                        m[n][e] = M;
                        l[n][e] = l[n][e] * fa + lo * fb;
#pragma unroll
                        for (uint32_t k = 0; k < MT; k++) {
                            o[k][n][e] = o[k][n][e] * fa + from[(NT * 4 + (n * MT + k) * 4 + e) * 32] * fb;
                            o[k][n][e + 2] = o[k][n][e + 2] * fa + from[(NT * 4 + (n * MT + k) * 4 + e + 2) * 32] * fb;
                        }
                    }
            }
        }
        __syncthreads();
        if (warp < C::PARTS) {   /* [warp][row][hd + 4]: acc, m, l */
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float *rec = xch + (warp * C::ROWS + 8u * n + 2u * t + e) * C::REC;
#pragma unroll
                    for (uint32_t k = 0; k < MT; k++) {
                        if (KIND == Q4K_Q8) {
                            *reinterpret_cast<float2 *>(rec + 16u * k + 2u * g) = make_float2(o[k][n][e], o[k][n][e + 2]);
                        } else {
                            rec[16u * k + g] = o[k][n][e];
                            rec[16u * k + g + 8u] = o[k][n][e + 2];
                        }
                    }
                    if (g == 0) *reinterpret_cast<float2 *>(rec + HD) = make_float2(m[n][e], l[n][e]);
                }
        }
        __syncthreads();
        const bool whole = st == 0u && here == n_steps;
        const uint32_t first = whole ? 0u : s_shares.first(s - at, s - at + steps), last = whole ? 0u : s_shares.last(s - at, s - at + steps), n_recs = last - first + 1u;
        float M, L;
        float4 A;
        auto join = [&](float m1, float l1, float4 x) {
            const float Mn = fmaxf(M, m1), Mu = Mn == -CUDART_INF_F ? 0.f : Mn, fa = ex2(M - Mu), fb = ex2(m1 - Mu);
            M = Mn;
            L = L * fa + l1 * fb;
            A.x = A.x * fa + x.x * fb; A.y = A.y * fa + x.y * fb; A.z = A.z * fa + x.z * fb; A.w = A.w * fa + x.w * fb;
        };
        auto gate_of = [&](uint32_t row, uint32_t d) -> const float * {
            return P.gate ? P.gate + ((size_t)(tok0 + row / P.gqa) * P.n_head + kh * P.gqa + row % P.gqa) * HD + d : nullptr;
        };
        float *part = P.part + ((size_t)blockIdx.x * 2u + (st == 0u ? 1u : 0u)) * C::ROWS * C::REC;
        for (uint32_t i = tid; i < live_rows * (HD / 4u); i += C::THREADS) {
            const uint32_t row = i / (HD / 4u), d = i % (HD / 4u) * 4u;
            const float *rec = xch + row * C::REC;
            const float2 ml0 = *reinterpret_cast<const float2 *>(rec + HD);
            M = ml0.x; L = ml0.y;
            A = *reinterpret_cast<const float4 *>(rec + d);
#pragma unroll
            for (uint32_t w = 1; w < C::PARTS; w++) {
                const float *r2 = rec + w * (C::ROWS * C::REC);
                const float2 ml = *reinterpret_cast<const float2 *>(r2 + HD);
                join(ml.x, ml.y, *reinterpret_cast<const float4 *>(r2 + d));
            }
            if (whole) {
                pg_store<HD, true>(P, tok0 + row / P.gqa, kh * P.gqa + row % P.gqa, d, A, L, gate_of(row, d));
            } else {
                *reinterpret_cast<float4 *>(part + row * C::REC + d) = A;
                if (d == 0u) *reinterpret_cast<float2 *>(part + row * C::REC + HD) = make_float2(M, L);
            }
        }
        if (!whole) {
            if (n_recs <= C::DIRECT) {   /* few records: the block that comes last joins them, the others go on */
                __syncthreads();
                if (tid == 0) {
                    __threadfence();
                    s_last = atomicAdd(P.meet + first, 1u) == n_recs - 1u;
                    if (s_last) P.meet[first] = 0u;
                }
                __syncthreads();
                if (s_last) {
                    __threadfence();
                    for (uint32_t i = tid; i < live_rows * (HD / 4u); i += C::THREADS) {
                        const uint32_t row = i / (HD / 4u), d = i % (HD / 4u) * 4u;
                        constexpr uint32_t BATCH = 4u;
                        M = -CUDART_INF_F; L = 0.f;
                        A = make_float4(0.f, 0.f, 0.f, 0.f);
                        for (uint32_t c0 = first; c0 <= last; c0 += BATCH) {
                            float2 ml[BATCH];
                            float4 x[BATCH];
#pragma unroll
                            for (uint32_t b = 0; b < BATCH; b++) {
                                const uint32_t c = min(c0 + b, last);
                                const float *rec = P.part + (((size_t)c * 2u + (c == first ? 1u : 0u)) * C::ROWS + row) * C::REC;
                                ml[b] = __ldcg(reinterpret_cast<const float2 *>(rec + HD));
                                x[b] = __ldcg(reinterpret_cast<const float4 *>(rec + d));
                            }
#pragma unroll
                            for (uint32_t b = 0; b < BATCH; b++)
                                if (c0 + b <= last) join(ml[b].x, ml[b].y, x[b]);
                        }
                        pg_store<HD, true>(P, tok0 + row / P.gqa, kh * P.gqa + row % P.gqa, d, A, L, gate_of(row, d));
                    }
                }
            } else if (tid == 0) {
                s_split[st == 0u] = {first, last, tok0, n_here, kh};
            }
        }
        s += take;
        off += take;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   /* the next bulk copies overwrite what was stored here */
    }
    /* ---- units of many records: their blocks meet, and each joins slices of 32 dims of a row: eight lanes to a slice, the records
     * shared out over the block's groups of eight lanes.  (All of a row by one block: 2 us more.) */
    __syncthreads();
    if (tid == 0) {
        pg_arrive(P, s_split[0], true);
        pg_arrive(P, s_split[1], false);
    }
    if (s_split[0].last >= s_split[0].first) {
        const PgSplit u = s_split[0];
        const uint32_t k = u.last - u.first + 1u, joiners = pg_joiners(k, false), mine_no = blockIdx.x - u.first - 1u;
        constexpr uint32_t GROUPS = C::THREADS / 8u, BATCH = 5u;
        float4 *s_a = reinterpret_cast<float4 *>(base);
        float2 *s_ml = reinterpret_cast<float2 *>(base + C::THREADS * 16u);
        const uint32_t slices = u.n_here * P.gqa * (HD / 32u), per_joiner = (slices + joiners - 1u) / joiners, x0 = min(mine_no * per_joiner, slices), x1 = min(x0 + per_joiner, slices);
        if (x0 < x1) pg_wait(P, u, k);
        for (uint32_t x = x0; x < x1; x++) {
            const uint32_t row = x / (HD / 32u), d = x % (HD / 32u) * 32u + (lane & 7u) * 4u, group = tid >> 3;
            const float *gate = P.gate ? P.gate + ((size_t)(u.tok0 + row / P.gqa) * P.n_head + u.kh * P.gqa + row % P.gqa) * HD + d : nullptr;
            float M = -CUDART_INF_F, L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
            auto join = [&](float m1, float l1, float4 v) {
                const float Mn = fmaxf(M, m1), Mu = Mn == -CUDART_INF_F ? 0.f : Mn, fa = ex2(M - Mu), fb = ex2(m1 - Mu);
                M = Mn;
                L = L * fa + l1 * fb;
                A.x = A.x * fa + v.x * fb; A.y = A.y * fa + v.y * fb; A.z = A.z * fa + v.z * fb; A.w = A.w * fa + v.w * fb;
            };
            for (uint32_t c0 = u.first + group; c0 <= u.last; c0 += GROUPS * BATCH) {
                float2 ml[BATCH];
                float4 v[BATCH];
#pragma unroll
                for (uint32_t b = 0; b < BATCH; b++) {
                    const uint32_t c = min(c0 + b * GROUPS, u.last);
                    const float *rec = P.part + (((size_t)c * 2u + (c == u.first ? 1u : 0u)) * C::ROWS + row) * C::REC;
                    ml[b] = __ldcg(reinterpret_cast<const float2 *>(rec + HD));
                    v[b] = __ldcg(reinterpret_cast<const float4 *>(rec + d));
                }
#pragma unroll
                for (uint32_t b = 0; b < BATCH; b++)
                    if (c0 + b * GROUPS <= u.last) join(ml[b].x, ml[b].y, v[b]);
            }
#pragma unroll
            for (int o2 = 8; o2 < 32; o2 <<= 1) {
                const float m1 = __shfl_xor_sync(0xffffffffu, M, o2), l1 = __shfl_xor_sync(0xffffffffu, L, o2);
                const float4 v = make_float4(__shfl_xor_sync(0xffffffffu, A.x, o2), __shfl_xor_sync(0xffffffffu, A.y, o2), __shfl_xor_sync(0xffffffffu, A.z, o2), __shfl_xor_sync(0xffffffffu, A.w, o2));
                join(m1, l1, v);
            }
            __syncthreads();   /* the slice before has been joined */
            if (lane < 8u) {
                s_a[warp * 8u + lane] = A;
                s_ml[warp * 8u + lane] = make_float2(M, L);
            }
            __syncthreads();
            if (tid < 8u) {
                for (uint32_t w = 1; w < WARPS; w++) join(s_ml[w * 8u + tid].x, s_ml[w * 8u + tid].y, s_a[w * 8u + tid]);
                pg_store<HD, true>(P, u.tok0 + row / P.gqa, u.kh * P.gqa + row % P.gqa, d, A, L, gate);
            }
        }
        pg_leave(P, u);
    }
    if (!ok) {   /* gave up on a copy: those behind it land before the block's shared memory is another's (bounded as well) */
        if (lane == 0) atomicOr(P.err, (uint32_t)Q4E_CUDA);
        for (; taken < issued; taken++)
            for (uint32_t i = 0; i < 4096u && !bar_test(bars + 8u * (taken % DEPTH), (taken / DEPTH) & 1u); i++) {}
    }
    if (P.beside) q4d_pdl_wait();
}

template <int KIND, int HD, int NT>
bool few(PagedParams &p, float *scratch) {
    using C = FewCfg<KIND, HD, NT>;
    static int per_sm = 0;
    if (!per_sm && (!q4i_check(cudaFuncSetAttribute(q4_pg_few_k<KIND, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM), "pages_attend smem attribute") ||
                    !q4i_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, q4_pg_few_k<KIND, HD, NT>, (int)C::THREADS, C::SMEM), "pages_attend occupancy")))
        return false;
    const uint32_t blocks = (uint32_t)g_q4.sm_count * ((uint32_t)per_sm < C::CTAS ? (uint32_t)per_sm : C::CTAS);   /* all resident: they meet */
    if (!blocks) return q4i_fail(Q4E_CUDA, "pages_attend: no block fits an SM");
    if (blocks > PG_MAX_BLOCKS) return q4i_fail(Q4E_CUDA, "pages_attend: more SMs than the counters are for");
    const size_t recs = (size_t)blocks * 2u * C::ROWS * C::REC;
    if (!scratch) {
        if (!q4i_scratch(recs, 0)) return false;
        scratch = g_q4.part;
    }
    p.part = scratch;
    p.tpg = C::ROWS / p.gqa;
    static uint32_t *meet = nullptr;
    if (!meet && !q4i_check(cudaGetSymbolAddress((void **)&meet, g_few_meet), "pages_attend counters")) return false;
    p.meet = meet;
    return q4i_launch_pdl("pages_attend launch", q4_pg_few_k<KIND, HD, NT>, dim3(blocks), C::THREADS, C::SMEM, p);
}
template <int KIND, int HD>
bool few_by_rows(PagedParams &p, uint32_t rows, float *scratch) {
    if (rows <= 8u) return few<KIND, HD, 1>(p, scratch);
    if (rows <= 16u || HD == 256) return few<KIND, HD, 2>(p, scratch);
    return few<KIND, HD, HD == 256 ? 2 : 4>(p, scratch);
}
bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0u; }

}  // namespace

extern "C" bool q4_gpu_pages_attend(const q4_gpu_pages *pg, uint32_t layer, const void *q, int q_bf16, const float *gate, void *out, int out_bf16,
                                    uint32_t n_head, const int32_t *rows, const int32_t *start, uint32_t n_req, uint32_t n_tok, const int32_t *table,
                                    uint32_t table_stride, uint32_t max_add, float scale) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "pages_attend: library not initialised");
    Q4_REQUIRE(q4i_pages_ok(pg) && pg->mem && aligned16(pg->mem) && layer < pg->n_layers, "pages_attend: bad pool or layer");
    Q4_REQUIRE(q && out && rows && start && table && n_req && n_tok && table_stride && n_head, "pages_attend: bad argument");
    Q4_REQUIRE(n_head % pg->n_kvh == 0 && n_head / pg->n_kvh <= 16, "pages_attend: n_head/n_kvh must be 1..16");
    Q4_REQUIRE(aligned16(q) && aligned16(gate) && aligned16(out), "pages_attend: q, gate and out must be 16-byte aligned");
    Q4_REQUIRE(scale > 0.f, "pages_attend: scale must be positive");
    Q4_REQUIRE(n_tok <= 0x7fffffffu && (uint64_t)table_stride * pg->page_rows <= 0x7fffffffu, "pages_attend: a block table's rows pass 2^31 - 1");
    PagedParams p = {};
    const uint32_t row = q4i_pages_row_bytes(pg->hd, pg->kind);
    p.part_bytes = row * pg->page_rows;
    p.page_bytes = (uint64_t)p.part_bytes * pg->n_kvh;
    p.mem = (const uint8_t *)pg->mem + (uint64_t)layer * p.page_bytes * pg->n_pages;
    p.n_pages = pg->n_pages; p.page_shift = (uint32_t)__builtin_ctz(pg->page_rows);
    p.n_kvh = pg->n_kvh; p.n_head = n_head; p.gqa = n_head / pg->n_kvh;
    p.rows = rows; p.start = start; p.table = table; p.table_stride = table_stride; p.n_req = n_req; p.n_tok = n_tok;
    p.q = q; p.q_bf16 = q_bf16; p.gate = gate; p.out = out; p.out_bf16 = out_bf16;
    p.scale_log2e = scale * 1.4426950408889634f;
    p.err = g_q4.err_d;
    const uint32_t most = max_add && max_add < n_tok ? max_add : n_tok;
    uint32_t few_rows = (uint32_t)(most * (uint64_t)p.gqa < 64u ? most * p.gqa : 64u);   /* (token, head) pairs that q4_pg_few_k takes at once */
    float *scratch = nullptr;
    p.add_split = 0xffffffffu;
    if (few_rows > (pg->hd == 256 ? 16u : 32u)) {
        /* requests that bring more than fits the smallest tile go to the tensor cores; a single request in any case */
        few_rows = p.gqa <= 8u ? 8u : 16u;
        p.add_split = n_req == 1u ? 0u : few_rows / p.gqa;
        /* Many units per request read its rows from a copy in fp16 (q4_paged_stage.cu), if it is not too large: on average 12 per request
         * at hd 256, 32 at 64 and 128, and 1024 tokens in all.  Without and with, us: at hd 256 8192 tokens over 16 384 (820 units) 5700
         * and 3350, three prompts (130) 201 and 132, 128 tokens each over 4000 rows (13) 99 and 90, 60 (6) 66 and 69, one prompt of
         * 320 tokens 29 and 38; at hd 128 8192 over 16 384 (256) 1390 and 1225, 2048 over 16 001 (64) 323 and 302, 1024 (32) 192 and
         * 184, 512 (16) 106 and 106; three prompts (40) 73 and 75. */
        const uint32_t per_unit = 128u / p.gqa * (pg->hd == 256 ? 1u : 2u);
        const uint64_t img_page = (uint64_t)pg->page_rows * pg->n_kvh * pg->hd * 4u, places = (uint64_t)n_req * table_stride, most_pages = (512ull << 20) / img_page;
        bool stage = pg->kind == Q4K_Q8 && n_req <= PG_STAGE_REQ && places <= 1u << 24 && most_pages && n_tok >= 1024u && n_tok >= (uint64_t)n_req * per_unit * (pg->hd == 256 ? 12u : 32u);
        const uint32_t cap = stage ? (uint32_t)(places < most_pages ? places : most_pages) : 0u;
        /* records of both kernels: the second's must not fall on the first's while those are joined */
        const size_t chunk = (q4i_paged_chunk_floats(pg->hd) + 63u) / 64u * 64u, rest = (size_t)g_q4.sm_count * 2u * 2u * 32u * (256u + 4u), img = cap * (size_t)(img_page / 4u);
        if (stage) stage = q4i_scratch_spare(chunk + rest + img + (size_t)places + 1u);   /* no room, or a capture before it was made: the pages as they are */
        if (!q4i_scratch(chunk + rest, 0)) return false;
        if (stage) {
            PagedParams c = p;
            uint8_t *to = (uint8_t *)(g_q4.part + chunk + rest);
            int32_t *img_table = (int32_t *)(to + cap * img_page);
            uint32_t *fits = (uint32_t *)(img_table + places);
            if (!q4i_paged_stage(p, pg->hd, to, img_table, cap, fits)) return false;
            c.mem = to; c.part_bytes = pg->hd * 4u * pg->page_rows; c.page_bytes = img_page; c.n_pages = cap; c.table = img_table;
            c.fits = fits; c.fits_is = 1u;
            if (!q4i_paged_chunk(c, Q4K_F16, pg->hd, g_q4.part)) return false;
            if (places > cap) {   /* they may be more than fit: then as they are */
                c = p;
                c.fits = fits; c.fits_is = 0u;
                if (!q4i_paged_chunk(c, Q4K_Q8, pg->hd, g_q4.part)) return false;
            }
        } else if (!q4i_paged_chunk(p, pg->kind, pg->hd, g_q4.part)) {
            return false;
        }
        if (n_req == 1u) return true;
        p.beside = 1u;
        scratch = g_q4.part + chunk;
    }
    if (pg->kind == Q4K_Q8)
        return pg->hd == 64 ? few_by_rows<Q4K_Q8, 64>(p, few_rows, scratch) : pg->hd == 128 ? few_by_rows<Q4K_Q8, 128>(p, few_rows, scratch) : few_by_rows<Q4K_Q8, 256>(p, few_rows, scratch);
    return pg->hd == 64 ? few_by_rows<Q4K_F16, 64>(p, few_rows, scratch) : pg->hd == 128 ? few_by_rows<Q4K_F16, 128>(p, few_rows, scratch) : few_by_rows<Q4K_F16, 256>(p, few_rows, scratch);
}
