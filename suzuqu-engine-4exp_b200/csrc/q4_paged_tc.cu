/*
 * Attention of chunks of new tokens over a pool of pages on the tensor cores (tcgen05.mma, accumulators in tensor memory): the
 * requests that bring more tokens than q4_pg_few_k takes at once.  Token j of request r attends [0, rows[r] + j].
 *
 * One block per SM, each with an equal share of the step's work: the tiles of 128 positions of all units (request, kv head, group of
 * tokens) one behind the other, cut into as many shares as there are blocks.  Lengths are read from the device.  A unit's
 * tokens fill the rows of the products: 2 x 128 (token, head) pairs at hd 64 and 128, 128 at hd 256 (whose outputs take half
 * of tensor memory).  What a share holds of a unit is a piece; a piece that is not the whole unit leaves (acc, m, l) records.
 *
 *   warps 0 - 7    softmax: thread r owns row r (hd 256: two threads, half of a unit's positions each): its scores out of tensor
 *                  memory, causal mask, running maximum with lazy rescale, weights as fp16 back into the columns they came from
 *   producers      (one team of four warps, or three of two) K and V of a tile into a ring of operand slots.  fp16 pages hold tiles as the tensor core reads them: bulk copies.
 *                  q8_0: codes and scales by asynchronous copies, then fp16(code x scale) into the slot (7 instructions
 *                  per 4 values).  Scales on the scores instead, as for few tokens, would need a product and an accumulator per 32 dims, and
 *                  their sums on the softmax warps, which set the pace
 *   issuer         the products: O += P V of a unit of positions as its weights appear, then the scores that take over the buffer
 *   walker         the share's pieces, and where the rows of their tiles lie, ahead of the others
 * V stays as it lies in the page, positions by dims: the product takes it as an operand whose dims are contiguous.
 *
 * A weight of 0 does not keep a V that is not finite from a sum.  Rows behind the last position are zeros in the slot.  Of the
 * unit's own tokens, which earlier ones do not attend, the walker looks through the rows before it hands their tile on; where
 * there is a V that is not finite the producers take the tile's rows by a slower way, with zeros in its place, and a row that
 * attends the first of them is NaN, by its sum.  (What lies before the unit's tokens is attended by every row.)
 *
 * Every wait is bounded: on expiry the block's waits all end, Q4E_CUDA is set, and tensor memory is freed.
 */
#include <cuda_bf16.h>
#include <math_constants.h>
#include <string.h>
#include <type_traits>

#include "q4_paged.h"
#include "q4_tc.h"

using namespace q4tc;

namespace {

__device__ uint32_t g_chunk_meet[PG_MAX_BLOCKS];
constexpr uint32_t CK_BN = 128;
constexpr uint32_t CK_SPIN_LIMIT = 1u << 22;
constexpr unsigned long long CK_LIMIT_NS = 2000000000ull;
constexpr uint32_t PIECES = 4, TILES = 4;   /* pieces that are walked ahead, tiles whose pages are found ahead */
constexpr float CK_RESCALE_TAU = 8.f;   /* weights reach 2^8 before the reference moves */

template <int KIND, int HD>
struct ChunkCfg {
    static constexpr uint32_t NQ = HD == 256 ? 1u : 2u, ROWS = NQ * 128u;
    static constexpr uint32_t SLOT = HD == 64 ? 16384u : 32768u, SLOTS = HD == 64 ? 10u : KIND == Q4K_Q8 ? 3u : 5u;
    static constexpr uint32_t ISSUER = 8u, WALKER = 9u, PRODUCER = 10u, THREADS = 512u;   /* first warps of the roles */
    /* Producer warps: TEAMS x WPT, a slot is one team's.  At hd 256 three slots are worked at at once, or the fixed part of a slot (900
     * of 1640 cycles) is not hidden: 8192 tokens over 16 384 5060 -> 3600 us; where the scores set the pace short slots leave more of
     * the ring free: 512 tokens over 16 001 at hd 128 98 us, by two teams of two warps 110. */
    static constexpr uint32_t TEAMS = HD == 256 ? 3u : 1u, WPT = HD == 256 ? 2u : 4u;
    static constexpr uint32_t RPS = HD == 256 ? 2u : 1u;          /* rounds of a slot */
    static constexpr uint32_t ITEMS = SLOT / 32u / (WPT * 32u * RPS);   /* of 16 codes, per producer thread and round */
    static constexpr uint32_t ROUNDS = HD == 256 ? 2u : 3u;       /* rounds of codes on their way to a warp */
    static constexpr uint32_t RAW = KIND == Q4K_Q8 ? ITEMS * 544u : 0u;   /* codes and scales of a warp's round */
    /* A piece takes 7.7 us (hd 256: 8.7) besides its tiles (queries in, the first scores, outputs out), a tile 2.2 (hd 256: 1.4 in fp16, 3.2
     * in q8_0): a unit counts as EXTRA more steps when the work is shared out.  Only tiles are walked.  512 tokens over 16 001 rows
     * 109 us with EXTRA 2, 98 with 3. */
    static constexpr uint32_t EXTRA = HD == 256 && KIND == Q4K_F16 ? 6u : 3u;
    static constexpr uint32_t LITTLE = HD == 256 ? 4u * EXTRA : 16u;
    /* registers of a thread: the block's 512 x 128 are 256 threads x (softmax + the others) */
    static constexpr uint32_t R_SOFTMAX = 168u, R_OTHERS = 88u;
    static_assert(R_SOFTMAX + R_OTHERS <= 256u, "register split");
    static constexpr uint32_t PARTS = HD == 256 ? 2u : 1u;        /* slots of a K or a V tile: K by 128 dims, V by 64 positions */
    static constexpr uint32_t QG = 128u * HD * 2u;                /* one group's queries */
    static constexpr uint32_t REC = HD + 4u;
    static constexpr uint32_t BARS = 1024u + (NQ == 1u ? 1024u : 0u);
    static constexpr uint32_t SMEM = NQ * QG + SLOTS * SLOT + TEAMS * WPT * ROUNDS * RAW + BARS + 1024u;
    static constexpr uint32_t UN = NQ == 2u ? 64u : 128u;         /* positions of a unit of scores */
    static_assert(SMEM <= 232448u, "shared memory");
};

__device__ __forceinline__ uint64_t v_desc(uint32_t saddr, uint32_t block_bytes) {
    /* dims contiguous: blocks of 64 dims (block_bytes apart), in them rows of 128 bytes per position, swizzled in groups of eight
     * (1024 bytes apart) */
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(block_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
/* fp16 1024 + 128 + code has (code ^ 0x80) in its low byte: two bytes picked out of word x (its codes ^ 0x80) become the exact codes */
template <uint32_t SEL>
__device__ __forceinline__ __half2 codes2(uint32_t x) {
    const uint32_t u = __byte_perm(x, 0x64646464u, SEL), off = 0x64806480u;
    return __hsub2(*reinterpret_cast<const __half2 *>(&u), *reinterpret_cast<const __half2 *>(&off));
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, bool there) {   /* zeros where there is nothing */
    if (there) {
        if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < BYTES; i += 4) asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + i), "r"(0u) : "memory");
    }
}
constexpr uint32_t TILE_BAD = 0x100u;   /* beside the eight bits of a tile's places without a page: new rows whose V is not finite */
/* whether the V of a record is not finite as fp16(code x scale): the largest code is 127, which reaches 65520 from 516 on */
template <int HD>
__device__ __forceinline__ bool not_finite_q8(const uint8_t *rec) {
    bool bad = false;
#pragma unroll
    for (uint32_t b = 0; b < HD / 64u; b++) {
        const uint32_t x = __ldcg(reinterpret_cast<const uint32_t *>(rec + 2u * HD + HD / 16u) + b);
        bad |= (x & 0x7fffu) > 0x6007u || (x >> 16 & 0x7fffu) > 0x6007u;
    }
    return bad;
}
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) {   /* all ones for a half whose exponent is */
    return ((x & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((x & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}
/* the rest of a wait whose first test found the phase incomplete (in line: ptxas does not allocate calls beside setmaxnreg) */
__device__ __forceinline__ bool ck_wait_on(uint32_t bar, uint32_t parity, uint32_t s_abort) {
    const unsigned long long t0 = global_ns();
    for (uint32_t i = 0; i < CK_SPIN_LIMIT; i++) {
        if (mbar_test<OWN>(bar, parity)) return true;
        if ((i & 63u) == 63u) {
            uint32_t a;
            asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(a) : "r"(s_abort) : "memory");
            if (a) return false;
            if (global_ns() - t0 > CK_LIMIT_NS) break;
        }
    }
    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(s_abort), "r"(1u) : "memory");
    return false;
}
/* by a whole warp, which goes on as one */
__device__ __forceinline__ bool ck_all_wait(uint32_t bar, uint32_t parity, uint32_t s_abort) {
    if (__builtin_expect(__all_sync(0xffffffffu, mbar_test<OWN>(bar, parity)), 1)) return true;
    return __all_sync(0xffffffffu, ck_wait_on(bar, parity, s_abort));
}

/* sum of floor((a i + b) / 128) over i < n, a up to 256 and a n + b below 2^32: whole multiples are taken out of a and b, what is left is counted
 * along the other axis of the lattice triangle, which swaps a and 128 (the reciprocity of floor sums, Graham, Knuth, Patashnik,
 * Concrete Mathematics, section 3.5), as in Euclid's algorithm */
__device__ __forceinline__ uint64_t floor_sum(uint32_t n, uint32_t a, uint32_t b) {
    uint64_t r = 0;
    uint32_t m = 128u;
    while (n) {
        if (a >= m) { r += (uint64_t)n * (n - 1u) / 2u * (a / m); a %= m; }
        if (b >= m) { r += (uint64_t)n * (b / m); b %= m; }
        const uint32_t y = a * n + b;
        if (y < m) break;
        n = y / m;
        b = y % m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
    return r;
}
/* tiles of a unit, and of the first g of a request's units on one kv head */
__device__ __forceinline__ uint32_t unit_tiles(const PgReq &R, uint32_t tpu, uint32_t g) {
    return (R.held + min((uint32_t)min((uint64_t)(g + 1u) * tpu, (uint64_t)R.add), R.add) + CK_BN - 1u) / CK_BN;
}
__device__ __forceinline__ uint64_t tiles_before(const PgReq &R, uint32_t tpu, uint32_t g) { return floor_sum(g, tpu, R.held + tpu + CK_BN - 1u); }   /* g below the last */
__device__ __forceinline__ PgReq chunk_request(const PagedParams &P, uint32_t r, bool &bad) {
    PgReq q = pg_request(P, r, bad);
    if (q.add <= P.add_split) q.add = 0u;
    return q;
}
template <uint32_t CK_EXTRA>
__device__ __forceinline__ uint64_t request_steps(const PagedParams &P, const PgReq &R, uint32_t tpu) {
    if (!R.add) return 0u;
    const uint32_t groups = (R.add + tpu - 1u) / tpu;
    return (tiles_before(R, tpu, groups - 1u) + unit_tiles(R, tpu, groups - 1u) + (uint64_t)CK_EXTRA * groups) * P.n_kvh;
}

/* A share's pieces, one after the other: one warp walks them ahead of the others and leaves them in shared memory */
struct Piece {
    uint32_t before;             /* rows of the request before the unit's first token: it attends those and itself */
    uint32_t tok0, n_here, kh;   /* the unit's first token, its tokens, its kv head */
    uint32_t req, st, here;      /* the piece: tiles [st, st + here) of the unit; here = 0: there are no more */
                                 /* (in the ring the first new position whose V is not finite has the place of req, which only the walker uses) */
    uint32_t tiles;              /* of the unit */
    bool gone;                   /* some of its positions are on pages that are not the pool's */
};
template <uint32_t CK_EXTRA>
struct Walk {
    uint64_t left;               /* steps of the share still to come */
    uint64_t now;                /* of all steps, the next one */
    uint64_t unit_at;            /* of all steps, the first of the unit of the last piece */
    uint32_t req, kh, g, st;
    PgReq R;
    __device__ __forceinline__ void begin(const PagedParams &P, uint64_t s0, uint64_t n, uint32_t r, uint32_t kh_, uint32_t g_, uint32_t st_) {
        bool bad;
        left = n; now = s0; req = r; kh = kh_; g = g_; st = st_;
        R = chunk_request(P, r, bad);
    }
    __device__ __forceinline__ bool next(const PagedParams &P, uint32_t tpu, Piece &p) {
        while (left) {
            bool bad;
            while (!R.add) R = chunk_request(P, ++req, bad);   /* `left` steps lie ahead: there is one with tokens */
            p.tiles = unit_tiles(R, tpu, g);
            p.n_here = min(tpu, R.add - g * tpu);
            p.before = R.held + g * tpu; p.tok0 = R.tok0 + g * tpu; p.kh = kh; p.req = req;
            const uint32_t here = (uint32_t)min((uint64_t)(p.tiles + CK_EXTRA - st), left), end = st + here;
            unit_at = now - st;
            p.st = max(st, CK_EXTRA) - CK_EXTRA;
            p.here = max(end, CK_EXTRA) - CK_EXTRA - p.st;
            left -= here;
            now += here;
            st = end;
            if (st == p.tiles + CK_EXTRA) {
                st = 0;
                if (++g * (uint64_t)tpu >= R.add) {
                    g = 0;
                    if (++kh == P.n_kvh) {
                        kh = 0;
                        R.add = 0;
                    }
                }
            }
            if (p.here) return true;
        }
        p.here = 0;
        return false;
    }
};

template <int KIND, int HD>
__global__ void __launch_bounds__(ChunkCfg<KIND, HD>::THREADS, 1) q4_pg_chunk_k(const PagedParams P) {
    using C = ChunkCfg<KIND, HD>;
    constexpr uint32_t CK_THREADS = C::THREADS, TEAMS = C::TEAMS, WPT = C::WPT, NQ = C::NQ, SLOT = C::SLOT, SLOTS = C::SLOTS, PARTS = C::PARTS, UN = C::UN, TU = 64;
    constexpr uint32_t CK_EXTRA = C::EXTRA, O_COL = 256, TMEM_COLS = 512, TILE = PgTile<KIND, HD>::BYTES, ROW = PgTile<KIND, HD>::ROW;
    extern __shared__ uint8_t smem_dyn[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t sQ = (smem_u32(smem_dyn) + 1023u) & ~1023u, sR = sQ + NQ * C::QG, bars = sR + SLOTS * SLOT + TEAMS * WPT * C::ROUNDS * C::RAW;
    const uint32_t full = bars, empty = bars + 80, bar_s = bars + 160, bar_p = bars + 192, bar_o = bars + 224, bar_q = bars + 240,
                   s_tmem = bars + 248, s_abort = bars + 252, s_gone = bars + 256, s_at = bars + 320, s_sum = bars + 352, w_full = bars + 480,
                   w_empty = bars + 512, t_full = bars + 544, t_empty = bars + 576, s_piece = bars + 608, s_tile = bars + 736, s_split = bars + 928, checks = bars + 968, s_xch = bars + 1024;
    uint8_t *base = smem_dyn + (sQ - smem_u32(smem_dyn));
    const uint32_t tpu = P.tpg * NQ;

    if (warp == C::ISSUER) {
        if (lane == 0) {
            for (uint32_t s = 0; s < SLOTS; s++) {
                mbar_init(full + 8 * s, WPT);
                mbar_init(empty + 8 * s, 1);
            }
            for (uint32_t s = 0; s < 4; s++) {
                mbar_init(bar_s + 8 * s, 1);
                mbar_init(bar_p + 8 * s, NQ == 2u ? 128u : 256u);
            }
            mbar_init(bar_o, 1);
            mbar_init(bar_o + 8, 1);
            mbar_init(bar_q, 256);
            for (uint32_t s = 0; s < PIECES; s++) {
                mbar_init(w_full + 8 * s, 1);
                mbar_init(w_empty + 8 * s, 9u + TEAMS * WPT);   /* a warp each of softmax, issuer and producers */
            }
            for (uint32_t s = 0; s < TILES; s++) {
                mbar_init(t_full + 8 * s, 1);
                mbar_init(t_empty + 8 * s, WPT * PARTS * 2u);   /* the warps of every slot of its K and V */
            }
            for (uint32_t s = 0; s < TEAMS * WPT; s++) mbar_init(checks + 8 * s, 1);
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(s_abort), "r"(0u) : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_tmem), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    q4d_pdl_wait();

    /* ---- this block's share: the steps of all requests by one scan, the two places where it is cut by two warps */
    PgShares shares;
    {
        const uint32_t n_req = P.fits && *P.fits != P.fits_is ? 0u : P.n_req, per = (n_req + CK_THREADS - 1u) / CK_THREADS, r0 = min(tid * per, n_req), r1 = min(r0 + per, n_req);
        uint64_t mine = 0, before = 0, total = 0;
        bool bad, any_bad = false;
        PgReq R = {0u, 0u, 0u};
        for (uint32_t r = r0; r < r1; r++) {
            R = chunk_request(P, r, bad);
            mine += request_steps<CK_EXTRA>(P, R, tpu);
            any_bad |= bad;
        }
        uint64_t x = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= (uint32_t)d) x += y;
        }
        uint64_t *sums = reinterpret_cast<uint64_t *>(base + (s_sum - sQ));
        if (lane == 31u) sums[warp] = x;
        __syncthreads();
        for (uint32_t w = 0; w < CK_THREADS / 32u; w++) {
            if (w < warp) before += sums[w];
            total += sums[w];
        }
        before += x - mine;
        if (blockIdx.x == 0 && any_bad) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        shares.set(total, CK_EXTRA, C::LITTLE, CK_EXTRA + 2u);
        if (tid < 2u) asm volatile("st.shared.v2.u64 [%0], {%1, %1};" ::"r"(s_at + 16u), "l"(total) : "memory");   /* begin and end: none yet, the last share's end */
        __syncthreads();
        if (mine && blockIdx.x < shares.blocks) {
#pragma unroll 1
            for (uint32_t i = 0; i < 2u; i++) {
                if (blockIdx.x + i >= shares.blocks) break;
                const uint64_t s = shares.cut(blockIdx.x + i);
                if (s < before || s >= before + mine) continue;
                uint64_t at = before;
                for (uint32_t r = r0; r < r1; r++) {
                    if (per > 1u) R = chunk_request(P, r, bad);
                    const uint64_t n = per > 1u ? request_steps<CK_EXTRA>(P, R, tpu) : mine;
                    if (s < at + n) {
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(s_piece + 64u * i), "r"(r), "r"(R.held), "r"(R.add), "r"(R.tok0) : "memory");
                        asm volatile("st.shared.v2.u64 [%0], {%1, %2};" ::"r"(s_piece + 64u * i + 16u), "l"(s), "l"(s - at) : "memory");
                        asm volatile("st.shared.u64 [%0], %1;" ::"r"(s_piece + 64u * i + 32u), "l"(n) : "memory");
                        break;
                    }
                    at += n;
                }
            }
        }
        __syncthreads();
        const uint32_t which = warp - C::WALKER;
        if (which < 2u && blockIdx.x + which < shares.blocks) {   /* the last group that begins at or before the cut: 32 places at a time */
            uint32_t r;
            uint64_t s, in, n_all;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r), "=r"(R.held), "=r"(R.add), "=r"(R.tok0) : "r"(s_piece + 64u * which));
            asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(s), "=l"(in) : "r"(s_piece + 64u * which + 16u));
            asm volatile("ld.shared.u64 %0, [%1];" : "=l"(n_all) : "r"(s_piece + 64u * which + 32u));
            uint32_t kh;
            if (n_all >> 32) {
                const uint64_t per_kh = n_all / P.n_kvh;
                kh = (uint32_t)(in / per_kh);
                in -= kh * per_kh;
            } else {
                const uint32_t per_kh = (uint32_t)n_all / P.n_kvh;
                kh = (uint32_t)in / per_kh;
                in -= kh * per_kh;
            }
            uint32_t lo = 0, n = (R.add + tpu - 1u) / tpu;   /* it is lo or one of the n - 1 behind it */
            uint64_t at = 0;
            while (true) {
                const uint32_t step = (n + 31u) / 32u, g = lo + lane * step;
                const uint64_t x2 = tiles_before(R, tpu, g) + (uint64_t)CK_EXTRA * g;
                const uint32_t below = __ballot_sync(0xffffffffu, lane * step < n && x2 <= in);   /* lane 0 always */
                const uint32_t last = 31u - (uint32_t)__clz((int)below);
                at = __shfl_sync(0xffffffffu, x2, (int)last);
                n = min(step, n - last * step);
                lo += last * step;
                if (step == 1u) break;
            }
            const uint32_t st = (uint32_t)(in - at), to = (uint32_t)shares.snap(st, unit_tiles(R, tpu, lo) + CK_EXTRA);
            if (lane == 0) {
                if (which == 0u) asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(s_at), "r"(r), "r"(kh), "r"(lo), "r"(to) : "memory");
                asm volatile("st.shared.u64 [%0], %1;" ::"r"(s_at + 16u + 8u * which), "l"(s - st + to) : "memory");
            }
        }
    }
    tc_fence_before();
    __syncthreads();   /* barriers initialised, tensor memory allocated, the share's place found */
    tc_fence_after();
    uint32_t tmem, w_req, w_kh, w_g, w_st;
    uint64_t s_begin, s_end;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(s_tmem));
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w_req), "=r"(w_kh), "=r"(w_g), "=r"(w_st) : "r"(s_at));
    asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(s_begin), "=l"(s_end) : "r"(s_at + 16u));
    bool ok = true;
    /* the next piece, by a whole warp; its place is given back with piece_done */
    uint32_t n_piece = 0;
    auto next_piece = [&](Piece &p) -> bool {
        const uint32_t e = n_piece % PIECES, a = s_piece + e * 32u;
        if (!ck_all_wait(w_full + 8 * e, (n_piece / PIECES) & 1u, s_abort)) {
            ok = false;
            return false;
        }
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(p.before), "=r"(p.tok0), "=r"(p.n_here), "=r"(p.kh) : "r"(a) : "memory");
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(p.req), "=r"(p.st), "=r"(p.here), "=r"(p.tiles) : "r"(a + 16u) : "memory");
        p.gone = p.n_here >> 31;
        p.n_here &= 0x7fffffffu;
        return p.here != 0u;
    };
    auto piece_done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(w_empty + 8 * (n_piece % PIECES));
        n_piece++;
    };
    Piece p;

    if (warp >= 8u) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::R_OTHERS));
        if (warp == C::ISSUER) {
            /* ================= issuer: a converged warp, one elected lane ================= */
            constexpr uint32_t IDESC_QK = (1u << 4) | ((uint32_t)(UN >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            const uint32_t el = elect_one();
            uint32_t slot = 0, phase = 0, use0 = 0, use1 = 0;   /* two groups: phase of their score buffers; one: units so far */
            auto take = [&]() -> uint32_t {
                const uint32_t s = slot;
                ok = ok && ck_all_wait(full + 8 * s, phase, s_abort);
                if (++slot == SLOTS) { slot = 0; phase ^= 1u; }
                return s;
            };
            const uint64_t q_desc = umma_desc(sQ), k_desc = umma_desc(sR), vt_desc = v_desc(sR, HD == 256 ? 64u * 128u : 128u * 128u);
            /* scores of a unit (row0: its first position in the tile) of group g from K slot s, dims 128 c .. */
            auto qk = [&](uint32_t col, uint32_t g, uint32_t c, uint32_t s, uint32_t row0) {
                const uint64_t qd = q_desc + ((g * C::QG + c * (2u * 16384u)) >> 4), kd = k_desc + ((s * SLOT + row0 * 128u) >> 4);
#pragma unroll
                for (uint32_t kk = 0; kk < (HD == 64 ? 4u : 8u); kk++)
                    umma_f16<false>(el, tmem + col, qd + (((kk >> 2) * 16384u + (kk & 3u) * 32u) >> 4), kd + (((kk >> 2) * 16384u + (kk & 3u) * 32u) >> 4), IDESC_QK, (c | kk) > 0u);
            };
            /* 64 positions, from byte `at` of V slot s */
            auto pv = [&](uint32_t col, uint32_t g, uint32_t s, uint32_t at, bool first) {
                const uint64_t vd = vt_desc + ((s * SLOT + at) >> 4);
#pragma unroll
                for (uint32_t kk = 0; kk < 4; kk++)
                    umma_f16_ta<false>(el, tmem + O_COL + g * 128u, tmem + col + kk * 8u, vd + kk * (2048u >> 4), IDESC_PV, (first && kk == 0u) ? 0u : 1u);
            };
            while (ok && next_piece(p)) {
                const uint32_t groups = NQ == 2u && p.n_here > P.tpg ? 2u : 1u;
                ok = ck_all_wait(bar_q, n_piece & 1u, s_abort);
                piece_done();
                if (NQ == 2u) {
                    uint32_t ks = take();
                    tc_fence_after();
                    if (!ok) break;
                    const bool two = groups == 2u;
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++)   /* half e >> 1 of the tile, group e & 1 */
                        if (two || !(e & 1u)) {
                            qk((e & 1u) * 128u + (e >> 1) * 64u, e & 1u, 0u, ks, (e >> 1) * 64u);
                            umma_commit<false>(el, bar_s + 8 * ((e & 1u) * 2u + (e >> 1)));
                        }
                    umma_commit<false>(el, empty + 8 * ks);
                    for (uint32_t j = 0; j < p.here && ok; j++) {
                        const uint32_t sv = take();
                        const bool more = j + 1u < p.here;
                        if (more) ks = take();
                        tc_fence_after();
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++) {
                            if (!two && (e & 1u)) continue;
                            const uint32_t b = (e & 1u) * 2u + (e >> 1), col = (e & 1u) * 128u + (e >> 1) * 64u;
                            ok = ok && ck_all_wait(bar_p + 8 * b, e & 1u ? use1 : use0, s_abort);
                            tc_fence_after();
                            if (!ok) break;
                            pv(col, e & 1u, sv, (e >> 1) * (64u * 128u), j == 0u && e < 2u);
                            umma_commit<false>(el, bar_o + 8 * (e & 1u));
                            if (e == (two ? 3u : 2u)) umma_commit<false>(el, empty + 8 * sv);
                            if (more) {
                                qk(col, e & 1u, 0u, ks, (e >> 1) * 64u);
                                umma_commit<false>(el, bar_s + 8 * b);
                            }
                        }
                        use0 ^= 1u;
                        use1 ^= two ? 1u : 0u;
                        if (more && ok) umma_commit<false>(el, empty + 8 * ks);
                    }
                } else {
                    uint32_t issued = use0;
                    auto issue_qk = [&]() {
                        const uint32_t b = issued & 1u;
                        for (uint32_t c = 0; c < PARTS; c++) {
                            const uint32_t s = take();
                            tc_fence_after();
                            if (!ok) return;
                            qk(b * 128u, 0u, c, s, 0u);
                            umma_commit<false>(el, empty + 8 * s);
                        }
                        umma_commit<false>(el, bar_s + 8 * b);
                        issued++;
                    };
                    issue_qk();
                    if (ok && p.here > 1u) issue_qk();
                    for (uint32_t j = 0; j < p.here && ok; j++) {
                        const uint32_t b = use0 & 1u;
#pragma unroll
                        for (uint32_t h = 0; h < 2; h++) {
                            const uint32_t sv = take();
                            if (h == 0u) ok = ok && ck_all_wait(bar_p + 8 * b, (use0 >> 1) & 1u, s_abort);
                            tc_fence_after();
                            if (!ok) break;
                            pv(b * 128u + h * 64u, 0u, sv, 0u, j == 0u && h == 0u);
                            umma_commit<false>(el, empty + 8 * sv);
                        }
                        if (!ok) break;
                        use0++;
                        umma_commit<false>(el, bar_o);
                        if (j + 2u < p.here) issue_qk();
                    }
                }
            }
        }
        if (warp == C::WALKER) {
            /* ================= walker: the share's pieces, where their tiles lie, and the units that are not this block's alone ================= */
            uint32_t n_tile = 0;
            const uint32_t per_page = P.part_bytes / TILE;
            PgSplit split[2] = {{1u, 0u, 0u, 0u, 0u}, {1u, 0u, 0u, 0u, 0u}};   /* that began before this block; that go on behind it */
            /* the first of rows r0 .. r1 - 1 of a tile of 128 positions whose V is not finite (none: all ones); lane i knows where its rows
             * from 16 i on lie */
            auto look = [&](uint32_t at, uint32_t gone8, uint32_t r0, uint32_t r1) -> uint32_t {
                uint32_t bad = 0xffffffffu;
                if constexpr (KIND == Q4K_Q8) {
#pragma unroll 1
                    for (uint32_t i = r0; i < r1; i += 32u) {
                        const uint32_t row = min(i + lane, r1 - 1u), lies = __shfl_sync(0xffffffffu, at, (int)(row >> 4));
                        if (not_finite_q8<HD>(P.mem + (uint64_t)lies * TILE + (row & 15u) * ROW) && !((gone8 >> (row >> 4)) & 1u)) bad = min(bad, row);
                    }
                } else {   /* 16 bytes of a row per lane, four loads on their way */
                    constexpr uint32_t LANES = HD / 8u, RPL = 32u / LANES, BATCH = 4u;   /* lanes of a row, rows of a load */
                    const uint32_t x = lane % LANES, in_row = TILE / 2u + (x >> 3) * 2048u + (x & 7u) * 16u;
#pragma unroll 1
                    for (uint32_t i = r0; i < r1; i += RPL * BATCH) {
                        uint4 w[BATCH];
#pragma unroll
                        for (uint32_t k = 0; k < BATCH; k++) {
                            const uint32_t row = min(i + k * RPL + lane / LANES, r1 - 1u), lies = __shfl_sync(0xffffffffu, at, (int)(row >> 4));
                            w[k] = __ldcg(reinterpret_cast<const uint4 *>(P.mem + (uint64_t)lies * TILE + in_row + (row & 15u) * 128u));
                        }
#pragma unroll
                        for (uint32_t k = 0; k < BATCH; k++) {
                            const uint32_t row = min(i + k * RPL + lane / LANES, r1 - 1u);
                            if ((not_finite2(w[k].x) | not_finite2(w[k].y) | not_finite2(w[k].z) | not_finite2(w[k].w)) && !((gone8 >> (row >> 4)) & 1u)) bad = min(bad, row);
                        }
                    }
                }
                return __reduce_min_sync(0xffffffffu, bad);
            };
            Walk<CK_EXTRA> W;
            W.left = 0;
            if (s_begin < s_end) W.begin(P, s_begin, s_end - s_begin, w_req, w_kh, w_g, w_st);
            for (uint32_t n = 0;; n++) {   /* to the end also where the others gave up: who meets whom does not change */
                const uint32_t e = n % PIECES, a = s_piece + e * 32u;
                const bool more = W.next(P, tpu, p);
                const int32_t *tab = P.table + (size_t)p.req * P.table_stride;
                const uint32_t n_kv = p.before + p.n_here, q0 = p.st * CK_BN + (lane & 7u) * 16u;
                auto entry = [&](uint32_t tile) -> int32_t { return tile < p.here && q0 + tile * CK_BN < n_kv ? tab[(q0 + tile * CK_BN) >> P.page_shift] : 0; };
                int32_t next = entry(0);
                bool gone = false;
                if (more) {   /* the softmax looks for missing pages only where there are any */
                    const uint32_t last = min((p.st + p.here) * CK_BN, n_kv) - 1u;
#pragma unroll 4
                    for (uint32_t i = (p.st * CK_BN >> P.page_shift) + lane; i <= last >> P.page_shift; i += 32u) gone |= (uint32_t)tab[i] >= P.n_pages;
                    gone = __any_sync(0xffffffffu, gone);
                    if (gone && lane == 0) atomicOr(P.err, (uint32_t)Q4E_RANGE);
                }
                if (n >= PIECES) ok = ok && ck_all_wait(w_empty + 8 * e, (n / PIECES - 1u) & 1u, s_abort);
                if (ok && lane == 0) {
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(p.before), "r"(p.tok0), "r"(p.n_here | (gone ? 0x80000000u : 0u)), "r"(p.kh) : "memory");
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a + 16u), "r"(0xffffffffu), "r"(p.st), "r"(p.here), "r"(p.tiles) : "memory");
                    mbar_arrive(w_full + 8 * e);
                }
                if (!more) break;
                if (n) {   /* its queries, and the gates if it is a whole unit, are on their way when it begins (the first piece begins at once) */
                    const bool whole = p.st == 0u && p.here == p.tiles;
                    const uint32_t q_line = P.gqa * HD * (P.q_bf16 ? 2u : 4u) / 128u, g_line = whole && P.gate ? P.gqa * HD / 32u : 0u;   /* lines of 128 bytes per token */
                    for (uint32_t i = lane; i < p.n_here * (q_line + g_line); i += 32u) {
                        const uint32_t t = i / (q_line + g_line), x = i - t * (q_line + g_line);
                        const size_t at = ((size_t)(p.tok0 + t) * P.n_head + (size_t)p.kh * P.gqa) * HD;
                        const uint8_t *line = x < q_line ? (const uint8_t *)P.q + at * (P.q_bf16 ? 2u : 4u) + x * 128u : (const uint8_t *)(P.gate + at) + (x - q_line) * 128u;
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
                    }
                }
                const uint32_t first_new = p.n_here > 1u ? p.before + 1u : 0xffffffffu;   /* from here on some rows attend a position and some do not */
                bool bad_yet = false;
                /* tile by tile: where its eight tiles of 16 positions lie, in units of such tiles; its live positions; those without a page */
                for (uint32_t tile = 0; tile < p.here && ok; tile++, n_tile++) {
                    const int32_t page = next;
                    next = entry(tile + 1u);
                    const uint32_t q = q0 + tile * CK_BN, te = n_tile % TILES, ta = s_tile + te * 48u;
                    const bool there = (uint32_t)page < P.n_pages;
                    const uint32_t at = there ? ((uint32_t)page * P.n_kvh + p.kh) * per_page + ((q & ((1u << P.page_shift) - 1u)) >> 4) : 0u;
                    uint32_t gone8 = __ballot_sync(0xffffffffu, !there) & 0xffu;
                    if ((p.st + tile + 1u) * CK_BN > first_new) {   /* new rows whose V is not finite */
                        const uint32_t t0 = (p.st + tile) * CK_BN, r0 = max(first_new, t0) - t0, r1 = min(n_kv - t0, CK_BN), bad = look(at, gone8, r0, r1);
                        if (bad != 0xffffffffu) {
                            gone8 |= TILE_BAD;
                            if (!bad_yet && ok && lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(a + 16u), "r"(t0 + bad) : "memory");
                            bad_yet = true;
                        }
                    }
                    if (n_tile >= TILES) ok = ok && ck_all_wait(t_empty + 8 * te, (n_tile / TILES - 1u) & 1u, s_abort);
                    if (!ok) break;
                    if (lane < 8u) asm volatile("st.shared.u32 [%0], %1;" ::"r"(ta + lane * 4u), "r"(at) : "memory");
                    if (lane == 8u) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(ta + 32u), "r"(n_kv - (p.st + tile) * CK_BN), "r"(gone8) : "memory");
                    if (lane == 9u) asm volatile("st.shared.u32 [%0], %1;" ::"r"(s_gone + 4u * (n_tile & 15u)), "r"(gone8 & 0xffu) : "memory");   /* for the softmax, once the tile's scores are there */
                    __syncwarp();
                    if (lane == 0) mbar_arrive(t_full + 8 * te);
                }
                if (p.st > 0u || p.here < p.tiles) {
                    const uint64_t u1 = W.unit_at + p.tiles + CK_EXTRA;
                    split[p.st == 0u] = {shares.first(W.unit_at, u1), shares.last(W.unit_at, u1), p.tok0, p.n_here, p.kh};
                }
            }
            if (lane < 2u) *reinterpret_cast<PgSplit *>(base + (s_split - sQ) + lane * sizeof(PgSplit)) = lane ? split[1] : split[0];
        }
        if (warp >= C::PRODUCER && warp < C::PRODUCER + TEAMS * WPT) {
        /* ================= producers ================= */
        const uint32_t team = (warp - C::PRODUCER) / WPT, share = (warp - C::PRODUCER) % WPT;   /* its share of every slot of the team */
        uint32_t at = team, in_piece = team, tiles_before = 0;   /* the team's next slot: of all, in the piece; tiles of earlier pieces */
        bool have = false;
        struct Job { uint32_t tile, part; bool v; };             /* tile: its place in the ring of tiles found */
        /* The slots of a piece in the order of their use.  Two groups: K0 V0 K1 V1 ..; one: K0 K1 V0 K2 V1 .. V(n-1), two slots each (the
         * scores run a tile and two tiles ahead of the outputs) */
        auto next_job = [&](Job &job) -> bool {
            while (!have || in_piece >= 2u * PARTS * p.here) {
                if (have) {
                    in_piece -= 2u * PARTS * p.here;
                    tiles_before += p.here;
                }
                if (!ok || !next_piece(p)) return false;
                piece_done();
                have = true;
            }
            const uint32_t m = in_piece / PARTS;
            uint32_t tile;
            if (NQ == 2u) {
                job.v = m & 1u;
                tile = m >> 1;
            } else {
                const bool last = m == 2u * p.here - 1u;
                job.v = last || (m && !(m & 1u));
                tile = last ? p.here - 1u : m == 0u ? 0u : m & 1u ? (m + 1u) >> 1 : (m >> 1) - 1u;
            }
            job.part = in_piece % PARTS;
            tile += tiles_before;
            job.tile = tile % TILES;
            ok = ck_all_wait(t_full + 8 * job.tile, (tile / TILES) & 1u, s_abort);
            in_piece += TEAMS;
            return ok;
        };
        auto tile_read = [&](const Job &job) {                   /* its place is not needed any more */
            __syncwarp();
            if (lane == 0) mbar_arrive(t_empty + 8 * job.tile);
        };
        auto wait_empty = [&]() {
            const uint32_t s = at % SLOTS, n = at / SLOTS;
            if (n > 0u) ok = ok && ck_all_wait(empty + 8 * s, (n - 1u) & 1u, s_abort);
        };
        auto lds = [&](uint32_t a) -> uint32_t {
            uint32_t v;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
            return v;
        };
        if constexpr (KIND == Q4K_Q8) {
            /* An item is 16 codes: 16 bytes that come in, two 16-byte pieces of fp16 that go out.  A pass of a warp is 8 rows x 64 dims:
             * four lanes to a row, so that the eight lanes whose stores go together (two rows) meet no bank twice.  A warp's share of a
             * slot is RPS rounds of RG groups of 8 rows x NB blocks of 64 dims (passes) each; the codes and scales of the next rounds
             * arrive by asynchronous copies meanwhile, in places that this warp alone uses.  A warp here issues once in three to five
             * cycles, beside two of the softmax: where things lie is found for it. */
            constexpr uint32_t ITEMS = C::ITEMS, NBK = HD == 64 ? 1u : 2u, NBV = HD / 64u;
            const uint32_t r8 = lane >> 2, c4 = lane & 3u;
            const uint32_t raw0 = sR + SLOTS * SLOT + (warp - C::PRODUCER) * C::ROUNDS * C::RAW;
            auto request = [&](const Job &job, uint32_t round, uint32_t raw, auto nb) {
                constexpr uint32_t NB = decltype(nb)::value, RG = ITEMS / NB, T = RG > 2u ? 2u : 1u;
                static_assert(RG <= 4u, "a lane brings the scales of one row");   /* T: tiles of 16 rows of a round */
                const uint32_t place = s_tile + job.tile * 48u;
                const uint32_t g0 = (HD == 256 && job.v ? job.part * 8u : 0u) + (share * C::RPS + round) * RG;   /* the first group of 8 rows, in the tile of 128 */
                const uint32_t col = (job.v ? HD : 0u) + (HD == 256 && !job.v ? job.part * 128u : 0u) + c4 * 16u;
                const uint32_t sc = 2u * HD + (job.v ? HD / 16u : 0u) + (HD == 256 && !job.v ? job.part * 8u : 0u);
                const uint32_t live = lds(place + 32u), gone = lds(place + 36u);
                const uint8_t *rec[T];
#pragma unroll
                for (uint32_t i = 0; i < T; i++) rec[i] = P.mem + (uint64_t)lds(place + ((g0 >> 1) + i) * 4u) * TILE;
                const uint8_t *srec = (T == 2u && lane >= 16u ? rec[T - 1] : rec[0]) + (lane & 15u) * ROW + sc;   /* of the row whose scales this lane brings */
                if (live >= CK_BN && !gone) {
#pragma unroll
                    for (uint32_t i = 0; i < RG; i++)
#pragma unroll
                        for (uint32_t b = 0; b < NB; b++) copy_async<16>(raw + (i * NB + b) * 512u + lane * 16u, rec[i / 2u] + ((i & 1u) * 8u + r8) * ROW + col + b * 64u, true);
                    if (lane < RG * 8u) copy_async<NB * 4>(raw + ITEMS * 512u + lane * (NB * 4u), srec, true);
                } else {   /* zeros for rows that are not there, and V that is not finite, where that matters */
                    uint32_t bad = 0;   /* of the round's rows */
                    if (gone & TILE_BAD && job.v) {
                        const uint32_t row = min(g0 * 8u + lane, CK_BN - 1u);
                        bad = __ballot_sync(0xffffffffu, not_finite_q8<HD>(P.mem + (uint64_t)lds(place + (row >> 4) * 4u) * TILE + (row & 15u) * ROW));
                    }
                    auto there = [&](uint32_t row) -> bool { return row < live && !((gone >> (row >> 4)) & 1u) && !((bad >> (row - g0 * 8u)) & 1u); };
#pragma unroll 1
                    for (uint32_t i = 0; i < RG; i++)
#pragma unroll
                        for (uint32_t b = 0; b < NB; b++)
                            copy_async<16>(raw + (i * NB + b) * 512u + lane * 16u, (T == 2u && i >= 2u ? rec[T - 1] : rec[0]) + ((i & 1u) * 8u + r8) * ROW + col + b * 64u, there((g0 + i) * 8u + r8));
                    if (lane < RG * 8u) copy_async<NB * 4>(raw + ITEMS * 512u + lane * (NB * 4u), srec, there(g0 * 8u + lane));
                }
                if (round + 1u == C::RPS) tile_read(job);
            };
            const uint32_t scale_sel = c4 & 2u ? 0x3232u : 0x1010u;
            auto convert = [&](uint32_t round, uint32_t raw, auto nb) {
                constexpr uint32_t NB = decltype(nb)::value, RG = ITEMS / NB, BLOCK = NB == 4u ? 64u * 128u : 128u * 128u;
                uint4 w[ITEMS];
                uint32_t sc[ITEMS];
#pragma unroll
                for (uint32_t k = 0; k < ITEMS; k++)
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[k].x), "=r"(w[k].y), "=r"(w[k].z), "=r"(w[k].w) : "r"(raw + k * 512u + lane * 16u) : "memory");
#pragma unroll
                for (uint32_t i = 0; i < RG; i++) {   /* all scales of the row's part */
                    const uint32_t a = raw + ITEMS * 512u + (i * 8u + r8) * (NB * 4u);
                    if constexpr (NB == 1u) sc[i] = lds(a);
                    else if constexpr (NB == 2u) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(sc[2 * i]), "=r"(sc[2 * i + 1]) : "r"(a) : "memory");
                    else asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(sc[4 * i]), "=r"(sc[4 * i + 1]), "=r"(sc[4 * i + 2]), "=r"(sc[4 * i + 3]) : "r"(a) : "memory");
                }
                if (round == 0u) wait_empty();
                if (!ok) return;
                const uint32_t dst = sR + (at % SLOTS) * SLOT + ((share * C::RPS + round) * RG * 8u + r8) * 128u;
                const uint32_t a0 = dst + (((2u * c4) ^ r8) << 4), a1 = dst + (((2u * c4 + 1u) ^ r8) << 4);
#pragma unroll
                for (uint32_t k = 0; k < ITEMS; k++) {
                    const uint32_t s2 = __byte_perm(sc[k], 0u, scale_sel), off = k / NB * 1024u + k % NB * BLOCK;
                    const uint32_t u[4] = {w[k].x ^ 0x80808080u, w[k].y ^ 0x80808080u, w[k].z ^ 0x80808080u, w[k].w ^ 0x80808080u};
                    uint32_t o[8];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        o[2 * e] = h2u(__hmul2(codes2<0x4140>(u[e]), *reinterpret_cast<const __half2 *>(&s2)));
                        o[2 * e + 1] = h2u(__hmul2(codes2<0x4342>(u[e]), *reinterpret_cast<const __half2 *>(&s2)));
                    }
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a0 + off), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a1 + off), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
                }
            };
            Job job;
            bool more = true;
            uint32_t asked = 0, is_v = 0, done = 0;              /* rounds asked for; bit i: slot i of the team's last 32 is of V; rounds converted */
            auto request_next = [&]() {                          /* a group per call in any case, so that they can be counted */
                const uint32_t slot = asked / C::RPS & 31u, round = asked % C::RPS, raw = raw0 + asked % C::ROUNDS * C::RAW;
                if (round == 0u) {
                    more = more && next_job(job);
                    is_v = (is_v & ~(1u << slot)) | (job.v ? 1u : 0u) << slot;
                }
                if (more) {
                    if (NBK != NBV && job.v) request(job, round, raw, std::integral_constant<uint32_t, NBV>());
                    else request(job, round, raw, std::integral_constant<uint32_t, NBK>());
                    asked++;
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll 1
            for (uint32_t d = 0; d < C::ROUNDS; d++) request_next();
            while (ok && done < asked) {
                asm volatile("cp.async.wait_group %0;" ::"n"(C::ROUNDS - 1u) : "memory");
                __syncwarp();
                const uint32_t round = done % C::RPS, raw = raw0 + done % C::ROUNDS * C::RAW;
                if (NBK != NBV && (is_v >> (done / C::RPS & 31u)) & 1u) convert(round, raw, std::integral_constant<uint32_t, NBV>());
                else convert(round, raw, std::integral_constant<uint32_t, NBK>());
                if (!ok) break;
                done++;
                if (round + 1u == C::RPS) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + 8 * (at % SLOTS));
                    at += TEAMS;
                }
                __syncwarp();       /* the round's codes have been read by all lanes */
                request_next();
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            /* a slot is 16 units of 2 KB (8 at hd 64): 16 rows of a block of 64 dims.  One bulk copy each, shared out over the warps: a
             * warp issues one in about 100 cycles */
            constexpr uint32_t UNITS = SLOT / 2048u / WPT;
            const uint32_t check_bar = checks + 8u * (warp - C::PRODUCER);
            uint32_t n_check = 0;
            Job job;
            while (ok && next_job(job)) {
                const uint32_t nblk = HD == 256 ? (job.v ? 4u : 2u) : HD / 64u, rows = HD == 256 && job.v ? 64u : 128u, place = s_tile + job.tile * 48u;
                const uint32_t unit = share * UNITS + (lane & (UNITS - 1u)), tile = unit / nblk, b = unit - tile * nblk;
                const uint32_t in = (HD == 256 && job.v ? job.part * 4u : 0u) + tile;
                const uint32_t lies = lds(place + in * 4u), left = lds(place + 32u), gone = lds(place + 36u);
                const uint32_t live = (gone >> in) & 1u || left <= in * 16u ? 0u : min(16u, left - in * 16u);
                tile_read(job);
                wait_empty();
                if (!ok) break;
                const bool check = job.v && gone & TILE_BAD;
                const uint32_t s = at % SLOTS, bar = check ? check_bar : full + 8 * s, to = sR + s * SLOT + b * rows * 128u + tile * 2048u;
                const uint32_t all = __reduce_add_sync(0xffffffffu, lane < UNITS ? live : 0u);
                if (job.v && all < 16u * UNITS) {   /* what is not copied has to be 0: weights there are 0, and 0 x NaN is not */
                    for (uint32_t u = 0; u < UNITS; u++) {
                        const uint32_t there = __shfl_sync(0xffffffffu, live, (int)u), a = __shfl_sync(0xffffffffu, to, (int)u);
#pragma unroll
                        for (uint32_t i = 0; i < 4; i++)
                            if (i * 4u + (lane >> 3) >= there) asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(a + i * 512u + lane * 16u), "r"(0u) : "memory");
                    }
                    fence_async_smem();
                    __syncwarp();
                }
                if (lane == 0) {
                    if (all) mbar_expect_tx(bar, all * 128u);
                    else mbar_arrive(bar);
                }
                __syncwarp();
                if (lane < UNITS && live)
                    bulk_load(to, P.mem + (uint64_t)lies * TILE + (job.v ? TILE / 2u : 0u) + ((HD == 256 && !job.v ? job.part * 2u : 0u) + b) * 2048u, live * 128u, bar);
                if (__builtin_expect(check, 0)) {   /* zeros for what is not finite, before the slot is handed on */
                    n_check++;
                    ok = ck_all_wait(check_bar, (n_check - 1u) & 1u, s_abort);
                    if (!ok) {   /* its copies land all the same (bounded) */
                        for (uint32_t i = 0; i < 4096u && !mbar_test<OWN>(check_bar, (n_check - 1u) & 1u); i++) {}
                        break;
                    }
#pragma unroll 1
                    for (uint32_t u = 0; u < UNITS * 4u; u++) {
                        const uint32_t a = __shfl_sync(0xffffffffu, to, (int)(u >> 2)) + (u & 3u) * 512u + lane * 16u;
                        uint4 w;
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(a) : "memory");
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(w.x & ~not_finite2(w.x)), "r"(w.y & ~not_finite2(w.y)), "r"(w.z & ~not_finite2(w.z)), "r"(w.w & ~not_finite2(w.w)) : "memory");
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + 8 * s);
                }
                at += TEAMS;
            }
            /* gave up: copies in flight land before the block's shared memory is another's (bounded) */
            if (!ok)
                for (uint32_t t = at; t >= TEAMS && at - t < SLOTS;) {
                    t -= TEAMS;
                    for (uint32_t i = 0; i < 4096u && !mbar_test<OWN>(full + 8 * (t % SLOTS), (t / SLOTS) & 1u); i++) {}
                }
        }
        }
    } else {
        /* ================= softmax ================= */
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::R_SOFTMAX));
        const uint32_t g = NQ == 2u ? warp >> 2 : 0u, h = NQ == 2u ? 0u : warp >> 2, r = tid & 127u, t_lane = tmem + (((warp & 3u) * 32u) << 16);
        const uint32_t inv_gqa = 65536u / P.gqa + 1u;   /* row / gqa = row * inv_gqa >> 16 for rows below 128, gqa up to 16 */
        const uint32_t tl = r * inv_gqa >> 16;
        auto pair_sync = [&]() {   /* the two warps of the same 32 rows (hd 256) */
            __syncwarp();
            asm volatile("bar.sync %0, 64;" ::"r"(1u + (warp & 3u)) : "memory");
        };
        auto pair_any = [&](bool x) -> bool {
            uint32_t any;
            __syncwarp();
            asm volatile("{ .reg .pred p, q; setp.ne.u32 q, %1, 0; bar.red.or.pred p, %2, 64, q; selp.u32 %0, 1, 0, p; }"
                         : "=r"(any) : "r"((uint32_t)x), "r"(1u + (warp & 3u)) : "memory");
            return any != 0u;
        };
        auto partner = [&](float x) -> float {   /* the other half's value of this row; a meeting lies between two calls */
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(s_xch + 4u * tid), "f"(x) : "memory");
            pair_sync();
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(s_xch + 4u * (tid ^ 128u)) : "memory");
            return x;
        };
        /* whether x holds for all warps of the group (hd 256: all eight): they take up and leave pieces together, whichever of them gave up */
        auto agree = [&](bool x) -> bool {
            uint32_t all;
            __syncwarp();
            asm volatile("{ .reg .pred p, q; setp.ne.u32 q, %1, 0; bar.red.and.pred p, %2, %3, q; selp.u32 %0, 1, 0, p; }"
                         : "=r"(all) : "r"((uint32_t)x), "r"(NQ == 2u ? 5u + g : 5u), "n"(NQ == 2u ? 128 : 256) : "memory");
            return all != 0u;
        };
        uint32_t use = 0, tiles_seen = 0;   /* units of this group so far; K tiles so far */
        while (ok) {
            if (!agree(next_piece(p))) break;
            const bool active = g == 0u || p.n_here > P.tpg;
            /* ---- queries as fp16, swizzled rows of 64 dims: the products of the piece before have read theirs (its last scores are here) */
            {
                /* a thread keeps its 8 dims and goes down the rows, 8 or 16 at a time: its places in the swizzled tiles lie in line */
                constexpr uint32_t PER = HD / 8u, T = NQ == 2u ? 128u : 256u, DOWN = T / PER, STEPS = 128u / DOWN, BATCH = 8u;   /* loads in flight before the first store */
                static_assert(DOWN % 8u == 0u && STEPS % BATCH == 0u, "queries by rows");
                const uint32_t qt = NQ == 2u ? r : tid, c = qt % PER, row0 = qt / PER, elem = P.q_bf16 ? 2u : 4u;
                if (active) {
                    const uint8_t *src = reinterpret_cast<const uint8_t *>(P.q) + (((size_t)(p.tok0 + g * P.tpg) * P.n_head + (size_t)p.kh * P.gqa) * HD + c * 8u) * elem;
                    const uint32_t a = sQ + g * C::QG + (c >> 3) * 16384u + row0 * 128u + (((c & 7u) ^ (row0 & 7u)) << 4), n_q = min(P.tpg, p.n_here - g * P.tpg), skip = P.n_head - P.gqa;
#pragma unroll 1
                    for (uint32_t k0 = 0; k0 < STEPS; k0 += BATCH) {
                        uint4 w[BATCH][2];
#pragma unroll
                        for (uint32_t k = 0; k < BATCH; k++) {
                            const uint32_t row = row0 + (k0 + k) * DOWN, ql = row * inv_gqa >> 16;
                            w[k][0] = w[k][1] = make_uint4(0u, 0u, 0u, 0u);
                            if (ql < n_q) {
                                const uint4 *x = reinterpret_cast<const uint4 *>(src + (uint64_t)(ql * skip + row) * (HD * elem));   /* ql whole tokens and the row's head */
                                w[k][0] = *x;
                                if (!P.q_bf16) w[k][1] = x[1];
                            }
                        }
#pragma unroll
                        for (uint32_t k = 0; k < BATCH; k++) {
                            const uint32_t in[8] = {w[k][0].x, w[k][0].y, w[k][0].z, w[k][0].w, w[k][1].x, w[k][1].y, w[k][1].z, w[k][1].w};
                            uint32_t o[4];
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                o[e] = P.q_bf16 ? h2u(__floats2half2_rn(__uint_as_float(in[e] << 16), __uint_as_float(in[e] & 0xffff0000u)))
                                                : h2u(__floats2half2_rn(__uint_as_float(in[2 * e]), __uint_as_float(in[2 * e + 1])));
                            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a + (k0 + k) * (DOWN * 128u)), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
                        }
                    }
                }
                fence_async_smem();
                mbar_arrive(bar_q);
                /* a group without tokens would run ahead, and its next arrival count for this piece */
                if (!active) ok = ck_all_wait(bar_q, n_piece & 1u, s_abort);
            }
            const uint32_t tok = g * P.tpg + tl;
            const bool row_live = tl < P.tpg && tok < p.n_here;
            /* this row attends positions [0, row_nkv); padding rows (queries of zeros, never stored) need no mask */
            const uint32_t row_nkv = row_live ? p.before + tok + 1u : 0xffffffffu;
            const uint32_t warp_min = __reduce_min_sync(0xffffffffu, row_nkv);
            const uint32_t n_seq = active ? (NQ == 2u ? 2u * p.here : p.here) : 0u;
            float m_ref = -CUDART_INF_F, l_run = 0.f;
            for (uint32_t u = 0; u < n_seq && (NQ == 1u || ok); u++, use++) {
                const uint32_t b = g * 2u + (use & 1u), p0 = p.st * CK_BN + u * UN + h * TU;
                const uint32_t t_s = t_lane + (NQ == 2u ? g * 128u + (use & 1u) * 64u : (use & 1u) * 128u + h * TU);
                ok = ok && ck_all_wait(bar_s + 8 * b, (use >> 1) & 1u, s_abort);
                if (NQ == 1u && !ok) {   /* the other warp of the rows may have gone on: its meetings are kept */
                    if (pair_any(false)) partner(0.f);
                    continue;
                }
                tc_fence_after();
                float s[TU];
#pragma unroll
                for (int c = 0; c < (int)TU / 32; c++) tmem_ld32(t_s + 32 * c, *reinterpret_cast<float(*)[32]>(&s[32 * c]));
                tmem_wait_ld();
                if (__builtin_expect(p0 + TU > warp_min || p.gone, 0)) {
                    uint32_t keep[2];   /* of 32 positions each */
#pragma unroll
                    for (uint32_t k = 0; k < 2; k++) keep[k] = row_nkv >= p0 + 32u * k + 32u ? 0xffffffffu : row_nkv > p0 + 32u * k ? (1u << (row_nkv - (p0 + 32u * k))) - 1u : 0u;
                    if (p.gone) {   /* positions on pages that are not the pool's */
                        uint32_t gone;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(gone) : "r"(s_gone + 4u * ((tiles_seen + (NQ == 2u ? u >> 1 : u)) & 15u)) : "memory");
                        gone >>= (p0 & 127u) >> 4;
#pragma unroll
                        for (uint32_t k = 0; k < 2; k++) keep[k] &= ~((gone >> (2u * k) & 1u ? 0xffffu : 0u) | (gone >> (2u * k + 1u) & 1u ? 0xffff0000u : 0u));
                    }
#pragma unroll
                    for (int k = 0; k < (int)TU; k++)
                        if (!((keep[k / 32] >> (k & 31)) & 1u)) s[k] = -CUDART_INF_F;
                }
                uint32_t pk[TU / 2];
                uint64_t ls[2];
                /* The exponentials start against the maximum of the units before, while this unit's own is being formed; where that
                 * is not within 2^8 the reference moves and they are taken again (by the same code: instructions that do not fit
                 * the SM's cache together cost the roles more than this loop). */
                for (bool again = false;; again = true) {
                    const float mneg = m_ref == -CUDART_INF_F ? 0.f : -m_ref;
                    const uint64_t sc2 = pack2(P.scale_log2e, P.scale_log2e), mn2 = pack2(mneg, mneg);
                    ls[0] = ls[1] = 0ull;
#pragma unroll
                    for (int k = 0; k < (int)TU / 2; k++) {
                        const float2 x = unpack2(fma2(pack2(s[2 * k], s[2 * k + 1]), sc2, mn2));
                        const float e0 = ex2f(x.x), e1 = ex2f(x.y);
                        ls[k & 1] = add2(ls[k & 1], pack2(e0, e1));
                        pk[k] = h2u(__floats2half2_rn(e0, e1));
                    }
                    if (__builtin_expect(again, 0)) break;
                    float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
                    for (int k = 0; k < (int)TU; k += 8) {
                        mx[0] = fmaxf(fmaxf(mx[0], s[k]), s[k + 1]); mx[1] = fmaxf(fmaxf(mx[1], s[k + 2]), s[k + 3]);
                        mx[2] = fmaxf(fmaxf(mx[2], s[k + 4]), s[k + 5]); mx[3] = fmaxf(fmaxf(mx[3], s[k + 6]), s[k + 7]);
                    }
                    float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * P.scale_log2e;   /* scale > 0 */
                    bool grow = m_new > m_ref + CK_RESCALE_TAU;   /* also true on the first live unit (m_ref = -inf) */
                    if (__builtin_expect(!(NQ == 2u ? __any_sync(0xffffffffu, grow) : pair_any(grow)), 1)) break;
                    if (NQ == 1u) {   /* both halves of a row keep one reference: they share its O */
                        m_new = fmaxf(m_new, partner(m_new));
                        grow = m_new > m_ref + CK_RESCALE_TAU;
                    }
                    float alpha = 1.f;
                    if (grow) {
                        alpha = ex2f(m_ref - m_new);
                        m_ref = m_new;
                        l_run *= alpha;
                    }
                    if (u > 0u) {   /* O is rescaled only here; the group's last product must have drained */
                        ok = ck_all_wait(bar_o + 8 * g, (use - 1u) & 1u, s_abort) && ok;
                        tc_fence_after();
#pragma unroll 1
                        for (uint32_t c = h * (HD / 64); c < (NQ == 2u ? HD / 32 : (h + 1u) * (HD / 64)); c++) {
                            float o[32];
                            tmem_ld32(t_lane + O_COL + g * 128u + 32 * c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; k++) o[k] *= alpha;
                            tmem_st32(t_lane + O_COL + g * 128u + 32 * c, o);
                        }
                    }
                }
                tmem_st32(t_s, *reinterpret_cast<const float(*)[32]>(&pk[0]));
                tmem_wait_st();
                /* a parity wait can tell the present phase from the one before it, no further, and bar_o's are not followed unit by
                 * unit: the phase before the last is waited for here, while the last cannot complete without this thread */
                if (u > 0u && u + 1u == n_seq) ok = ck_all_wait(bar_o + 8 * g, (use - 1u) & 1u, s_abort) && ok;
                tc_fence_before();
                mbar_arrive(bar_p + 8 * b);
                const float2 l0 = unpack2(ls[0]), l1 = unpack2(ls[1]);
                l_run += (l0.x + l0.y) + (l1.x + l1.y);
            }
            tiles_seen += p.here;
            if (NQ == 1u) {
                pair_sync();
                l_run += partner(l_run);
                pair_sync();   /* before the next piece's first exchange */
            }
            /* ---- the piece's outputs.  32 columns at a time go through the warp's share of the query tiles (read by no product any
             * more), so that rows leave in whole lines: step q of a column block is 4 rows of 32 columns, 8 lanes each.  (From
             * the threads that hold the rows a piece took 8000 cycles.) */
            const bool whole = p.st == 0u && p.here == p.tiles;
            const uint32_t w_row0 = (warp & 3u) * 32u;
            uint32_t off[8], live = 0;   /* in 16-byte units from the unit's first token */
#pragma unroll
            for (uint32_t q = 0; q < 8; q++) {
                const uint32_t row = w_row0 + 4u * q + (lane >> 3), ti = row * inv_gqa >> 16;
                if (ti < P.tpg && g * P.tpg + ti < p.n_here) live |= 1u << q;
                off[q] = whole ? ((g * P.tpg + ti) * P.n_head + p.kh * P.gqa + (row - ti * P.gqa)) * (HD / 4u) + (lane & 7u) : (g * 128u + row) * (C::REC / 4u) + (lane & 7u);
            }
            const size_t first = (size_t)p.tok0 * P.n_head * (HD / 4u);
            float *rec = P.part + ((size_t)blockIdx.x * 2u + (p.st == 0u ? 1u : 0u)) * C::ROWS * C::REC;
            if (active && ok) ok = ck_all_wait(bar_o + 8 * g, (use - 1u) & 1u, s_abort);
            tc_fence_after();
            {
                uint32_t bad;   /* the first position whose V is not finite */
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(bad) : "r"(s_piece + n_piece % PIECES * 32u + 16u) : "memory");
                if (row_live && row_nkv > bad) l_run = CUDART_NAN_F;
            }
            if (active && ok) {
                const float inv = whole ? (l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f) : 1.f;
                const uint32_t buf = sQ + warp * (NQ * C::QG / 8u);   /* [32 rows][8 x 16 bytes], piece k of row r at k ^ (r & 7) */
                if (!whole && row_live && h == 0u) *reinterpret_cast<float2 *>(rec + (size_t)(g * 128u + r) * C::REC + HD) = make_float2(m_ref, l_run);
#pragma unroll 1
                for (uint32_t c = h * (HD / 64); c < (NQ == 2u ? HD / 32 : (h + 1u) * (HD / 64)); c++) {
                    float o[32];
                    float4 x[8], gt[8];
                    tmem_ld32(t_lane + O_COL + g * 128u + 32 * c, o);
                    if (whole && P.gate) {
#pragma unroll
                        for (int q = 0; q < 8; q++)
                            if ((live >> q) & 1u) gt[q] = reinterpret_cast<const float4 *>(P.gate)[first + off[q] + 8u * c];
                    }
                    tmem_wait_ld();
                    __syncwarp();
#pragma unroll
                    for (uint32_t k = 0; k < 8; k++)
                        asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(buf + lane * 128u + ((k ^ (lane & 7u)) << 4)), "f"(o[4 * k] * inv), "f"(o[4 * k + 1] * inv), "f"(o[4 * k + 2] * inv), "f"(o[4 * k + 3] * inv) : "memory");
                    __syncwarp();
#pragma unroll
                    for (uint32_t q = 0; q < 8; q++) {
                        const uint32_t row = 4u * q + (lane >> 3);
                        asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(x[q].x), "=f"(x[q].y), "=f"(x[q].z), "=f"(x[q].w) : "r"(buf + row * 128u + (((lane & 7u) ^ (row & 7u)) << 4)) : "memory");
                    }
                    if (!whole) {
#pragma unroll
                        for (int q = 0; q < 8; q++)
                            if ((live >> q) & 1u) reinterpret_cast<float4 *>(rec)[off[q] + 8u * c] = x[q];
                        continue;
                    }
                    if (P.gate) {
#pragma unroll
                        for (int q = 0; q < 8; q++)
                            if ((live >> q) & 1u) {
                                x[q].x = gated(x[q].x, gt[q].x); x[q].y = gated(x[q].y, gt[q].y);
                                x[q].z = gated(x[q].z, gt[q].z); x[q].w = gated(x[q].w, gt[q].w);
                            }
                    }
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        if (!((live >> q) & 1u)) continue;
                        if (P.out_bf16) {
                            const __nv_bfloat162 b0 = __floats2bfloat162_rn(x[q].x, x[q].y), b1 = __floats2bfloat162_rn(x[q].z, x[q].w);
                            reinterpret_cast<uint2 *>(P.out)[first + off[q] + 8u * c] = make_uint2(*reinterpret_cast<const uint32_t *>(&b0), *reinterpret_cast<const uint32_t *>(&b1));
                        } else {
                            reinterpret_cast<float4 *>(P.out)[first + off[q] + 8u * c] = x[q];
                        }
                    }
                }
            }
            tc_fence_before();   /* the next piece's first product overwrites O behind this thread's next arrival */
            ok = agree(ok);   /* and the next piece's queries may come where the outputs were */
            piece_done();
        }
    }
    if (!ok && lane == 0) atomicOr(P.err, (uint32_t)Q4E_CUDA);
    asm volatile("fence.proxy.async;" ::: "memory");   /* this thread's records, which others read by bulk copies */
    __threadfence();
    tc_fence_before();
    __syncthreads();
    if (warp == C::ISSUER) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    const PgSplit *split = reinterpret_cast<const PgSplit *>(base + (s_split - sQ));
    if (tid == 0) {
        pg_arrive(P, split[0], true);
        pg_arrive(P, split[1], pg_first_joins(split[1].last - split[1].first + 1u));
    }
    const PgSplit ends = split[0], begins = split[1];   /* what follows uses the shared memory */
    bool joining = true;
    pg_join<HD, CK_THREADS>(P, ends, C::ROWS, base, NQ * C::QG + SLOTS * SLOT, s_sum, joining);
    if (begins.last >= begins.first && pg_first_joins(begins.last - begins.first + 1u)) pg_join<HD, CK_THREADS>(P, begins, C::ROWS, base, NQ * C::QG + SLOTS * SLOT, s_sum, joining);
}

template <int KIND, int HD>
bool chunk(PagedParams p, float *scratch) {
    using C = ChunkCfg<KIND, HD>;
    static bool attr = false;
    if (!attr && !q4i_check(cudaFuncSetAttribute(q4_pg_chunk_k<KIND, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM), "pages_attend smem attribute")) return false;
    attr = true;
    const uint32_t blocks = (uint32_t)g_q4.sm_count;
    if (blocks > PG_MAX_BLOCKS) return q4i_fail(Q4E_CUDA, "pages_attend: more SMs than the counters are for");
    p.part = scratch;
    p.tpg = 128u / p.gqa;
    static uint32_t *meet = nullptr;
    if (!meet && !q4i_check(cudaGetSymbolAddress((void **)&meet, g_chunk_meet), "pages_attend counters")) return false;
    p.meet = meet;
    return q4i_launch_pdl("pages_attend launch", q4_pg_chunk_k<KIND, HD>, dim3(blocks), C::THREADS, C::SMEM, p);
}

}  // namespace

size_t q4i_paged_chunk_floats(uint32_t hd) {
    const size_t rows = hd == 256 ? 128u : 256u;
    return (size_t)g_q4.sm_count * 2u * rows * (hd + 4u);
}
bool q4i_paged_chunk(const PagedParams &p, int kind, uint32_t hd, float *scratch) {
    if (kind == Q4K_Q8) return hd == 64 ? chunk<Q4K_Q8, 64>(p, scratch) : hd == 128 ? chunk<Q4K_Q8, 128>(p, scratch) : chunk<Q4K_Q8, 256>(p, scratch);
    return hd == 64 ? chunk<Q4K_F16, 64>(p, scratch) : hd == 128 ? chunk<Q4K_F16, 128>(p, scratch) : chunk<Q4K_F16, 256>(p, scratch);
}
