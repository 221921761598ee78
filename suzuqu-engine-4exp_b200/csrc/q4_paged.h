/* Shared by the kernels over a pool of pages (q4_pages.cu, q4_paged.cu, q4_paged_tc.cu, q4_paged_stage.cu; not installed). */
#ifndef Q4_PAGED_H
#define Q4_PAGED_H

#include <cuda_bf16.h>
#include <math_constants.h>

#include "q4_internal.h"

struct PagedParams {
    const uint8_t *mem;          /* of the layer */
    uint64_t page_bytes;         /* of all kv heads */
    uint32_t part_bytes;         /* of one kv head */
    uint32_t n_pages, page_shift, n_kvh, n_head, gqa;
    uint32_t tpg;                /* tokens of a group of rows (128 in q4_pg_chunk_k, of which the last ones may be empty) */
    uint32_t add_split;          /* requests that bring at most so many tokens are q4_pg_few_k's, the others q4_pg_chunk_k's */
    const int32_t *rows, *start, *table;
    uint32_t table_stride, n_req, n_tok;
    const void *q;
    const float *gate;
    void *out;
    int q_bf16, out_bf16;
    float scale_log2e;
    float *part;                 /* [block][2][rows of a unit][hd + 4]: acc, m (log2 units, scale folded in), l */
    uint32_t *meet;              /* [block]: the word at which the blocks of the unit that begins in the block meet; zero between launches */
    uint32_t *err;
    const uint32_t *fits;        /* not NULL: the launch has work only if this word is `fits_is` (q4i_paged_stage's) */
    uint32_t fits_is;
    uint32_t beside;             /* q4_pg_few_k behind q4_pg_chunk_k of the same call: it need not wait for that one's end */
};

/* of 16 rows of a kv head, K and V; of one row */
template <int KIND, int HD>
struct PgTile {
    static constexpr uint32_t ROW = KIND == Q4K_Q8 ? (2u * HD + HD / 8u + 15u) / 16u * 16u : 4u * HD, BYTES = 16u * ROW;
};

constexpr uint32_t PG_MAX_BLOCKS = 1024;

/* The tokens of requests that bring more than P.add_split, on the tensor cores (q4_paged_tc.cu), with its records in `scratch`, of
 * at least q4i_paged_chunk_floats floats.  hd 64, 128 or 256, kind fp16 or q8_0. */
size_t q4i_paged_chunk_floats(uint32_t hd);
bool q4i_paged_chunk(const PagedParams &p, int kind, uint32_t hd, float *scratch);

/* A copy in fp16 of the pages of those requests (pool of q8_0): at most cap pages of page_rows rows and all kv heads, their table, and
 * whether they were that few (q4_paged_stage.cu).  n_req up to PG_STAGE_REQ. */
constexpr uint32_t PG_STAGE_REQ = 8192;
bool q4i_paged_stage(const PagedParams &p, uint32_t hd, uint8_t *to, int32_t *table, uint32_t cap, uint32_t *fits);

/* The word at which the blocks of a split unit meet counts in its lower half the blocks that have arrived, in its upper half those that
 * will not look at it any more.  Every block counts once in each, whatever happened before, one that joins nothing in both at once, and
 * whoever completes the upper half leaves zero: nothing comes to the word after that. */
constexpr uint32_t PG_HERE = 1u, PG_GONE = 1u << 16;
__host__ __device__ inline uint32_t pg_arrival(bool joins) { return joins ? PG_HERE : PG_HERE + PG_GONE; }
__host__ __device__ inline bool pg_all_here(uint32_t word, uint32_t blocks) { return (word & (PG_GONE - 1u)) >= blocks; }
__host__ __device__ inline bool pg_last_gone(uint32_t before, uint32_t blocks) { return before >> 16 == blocks - 1u; }   /* before the addition */
/* the blocks of a unit that join its records; the first, which may have the end of another unit to see to, only where that is said */
__host__ __device__ inline uint32_t pg_joiners(uint32_t blocks, bool first_too) { return first_too ? blocks : blocks - 1u; }
__host__ __device__ inline bool pg_first_joins(uint32_t blocks) { return blocks <= 3u; }                               /* in q4_pg_chunk_k */
/* a wait: whether one of at most so many probes says yes */
template <typename Probe>
__host__ __device__ inline bool pg_within(uint32_t probes, Probe probe) {
    for (uint32_t i = 0; i < probes; i++)
        if (probe()) return true;
    return false;
}

#ifdef __CUDACC__
/* what the host or the device gave for request r: tokens (0: none of this launch's), rows before them */
struct PgReq { uint32_t held, add, tok0; };
__device__ __forceinline__ PgReq pg_request(const PagedParams &P, uint32_t r, bool &bad) {
    const int32_t s0 = __ldcg(P.start + r), s1 = __ldcg(P.start + r + 1u), h = __ldcg(P.rows + r);
    PgReq q = {0u, 0u, 0u};
    bad = false;
    if (s1 <= s0) return q;
    if (h < 0 || s0 < 0 || (uint32_t)s1 > P.n_tok || (uint64_t)(uint32_t)h + (uint32_t)(s1 - s0) > ((uint64_t)P.table_stride << P.page_shift)) {
        bad = true;
        return q;
    }
    q.held = (uint32_t)h; q.add = (uint32_t)(s1 - s0); q.tok0 = (uint32_t)s0;
    return q;
}
__device__ __forceinline__ float pg_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
/* four dims of a row: acc / l * sigmoid(gate), where there are gates (LDCG: in global memory).  A row that attended nothing is 0, one with a NaN among its scores stays NaN */
template <int HD, bool LDCG = false>
__device__ __forceinline__ void pg_store(const PagedParams &P, uint32_t tok, uint32_t head, uint32_t d, float4 x, float L, const float *gate) {
    const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
    const size_t at = ((size_t)tok * P.n_head + head) * HD + d;
    x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
    if (gate) {
        const float4 gt = LDCG ? __ldcg(reinterpret_cast<const float4 *>(gate)) : *reinterpret_cast<const float4 *>(gate);
        x.x *= 1.f / (1.f + __expf(-gt.x)); x.y *= 1.f / (1.f + __expf(-gt.y));
        x.z *= 1.f / (1.f + __expf(-gt.z)); x.w *= 1.f / (1.f + __expf(-gt.w));
    }
    if (P.out_bf16) {
        const __nv_bfloat162 b0 = __floats2bfloat162_rn(x.x, x.y), b1 = __floats2bfloat162_rn(x.z, x.w);
        *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(P.out) + at) = make_uint2(*reinterpret_cast<const uint32_t *>(&b0), *reinterpret_cast<const uint32_t *>(&b1));
    } else {
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(P.out) + at) = x;
    }
}

/* ---- shares.  `total` steps in `blocks` shares: share c begins at cut(c).  A cut that falls into a unit of at most `little` steps, or
 * within `near` steps of the end of a longer one, goes to the unit's nearer end: that costs less than another piece and records
 * that have to be joined.  near is at least what a unit counts besides its own steps (a cut among those would be of no use). */
struct PgShares {
    uint64_t total;
    uint32_t blocks, near, little;
    /* as many shares as there are blocks, but none of fewer than `least` steps */
    __device__ __forceinline__ void set(uint64_t n, uint32_t near_, uint32_t little_, uint32_t least) {
        total = n; near = near_; little = little_;
        blocks = (uint32_t)min((uint64_t)gridDim.x, n >> 32 ? n : max((uint32_t)n / least, n ? 1u : 0u));
    }
    __device__ __forceinline__ uint64_t cut(uint32_t c) const {
        return total >> 22 ? total * c / blocks : (uint32_t)total * c / blocks;   /* up to 1024 blocks */
    }
    __device__ __forceinline__ uint32_t of(uint64_t step) const {   /* the share that step would be in if no cut moved */
        return total >> 21 ? (uint32_t)(((step + 1u) * blocks - 1u) / total) : (((uint32_t)step + 1u) * blocks - 1u) / (uint32_t)total;
    }
    /* where in a unit of `steps` steps a cut that falls on its step st lies */
    __device__ __forceinline__ uint64_t snap(uint64_t st, uint64_t steps) const {
        const uint64_t left = steps - st;
        return steps > little && st > near && left > near ? st : st <= left ? 0u : steps;
    }
    /* the shares that the first and the last step of the unit [u0, u1) are in */
    __device__ __forceinline__ uint32_t first(uint64_t u0, uint64_t u1) const {
        uint32_t c = of(u0);
        while (c + 1u < blocks) {
            const uint64_t b = cut(c + 1u);
            if (b > u1 || snap(b - u0, u1 - u0) != 0u) break;
            c++;
        }
        return c;
    }
    __device__ __forceinline__ uint32_t last(uint64_t u0, uint64_t u1) const {
        uint32_t c = of(u1 - 1u);
        while (c > 0u) {
            const uint64_t b = cut(c);
            if (b <= u0 || snap(b - u0, u1 - u0) != u1 - u0) break;
            c--;
        }
        return c;
    }
};
/* A unit that lies in several blocks, first to last; last < first: none */
struct PgSplit { uint32_t first, last, tok0, n_here, kh; };
/* The blocks of a split unit meet at a word and join its records, each an equal part (the first of many records not at all: one block
 * alone takes 15 us for it): some of the rows, or, where there are more blocks than rows, a half, a quarter .. of one.  All blocks
 * of the launch are resident in the end (the grid is what the SMs hold) and none waits for another before its share is done; a
 * launch of its own for this took 8 to 12 us (one request over 262 144 rows 44 us with it).  They end their shares within a few
 * microseconds of one another, but for q4_pg_few_k beside q4_pg_chunk_k, whose blocks come in as the chunks' leave: there a wait is up to
 * the spread of those.  The wait is bounded (2 s).
 */
__device__ __forceinline__ void pg_meet(const PagedParams &P, const PgSplit &u, uint32_t what) {   /* one thread */
    const uint32_t k = u.last - u.first + 1u, before = atomicAdd(P.meet + u.first, what);
    if (what >= PG_GONE && pg_last_gone(before, k)) P.meet[u.first] = 0u;
}
__device__ __forceinline__ void pg_arrive(const PagedParams &P, const PgSplit &u, bool joins) {    /* one thread, behind the block's records and a barrier */
    if (u.last < u.first) return;
    __threadfence();
    pg_meet(P, u, pg_arrival(joins));
}
/* the whole block, until k have arrived */
__device__ __forceinline__ void pg_wait(const PagedParams &P, const PgSplit &u, uint32_t k) {
    if (threadIdx.x == 0) {
        unsigned long long t0, t;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
        for (uint32_t i = 0;; i++) {
            uint32_t n;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(P.meet + u.first) : "memory");
            if (pg_all_here(n, k)) break;
            if ((i & 63u) == 63u) {
                asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
                if (t - t0 > 2000000000ull) {
                    atomicOr(P.err, (uint32_t)Q4E_CUDA);
                    break;
                }
            }
        }
        __threadfence();
    }
    __syncthreads();
}
__device__ __forceinline__ void pg_leave(const PagedParams &P, const PgSplit &u) {
    __syncthreads();
    if (threadIdx.x == 0) pg_meet(P, u, PG_GONE);
}
/* What a block joins, and its gates, come to shared memory by bulk copies, all at once; then a thread has four dims of a row, or
 * shares them with others that take the other records.  bar: 8 bytes of shared memory for a barrier, not in use by anything.  ok: false
 * once a wait for copies has run out (Q4E_CUDA): nothing more is brought or stored, by a later call neither */
template <int HD, uint32_t THREADS>
__device__ __forceinline__ void pg_join(const PagedParams &P, const PgSplit &u, uint32_t unit_rows, uint8_t *smem, uint32_t smem_bytes, uint32_t bar, bool &ok) {
    constexpr uint32_t REC = HD + 4u;
    if (u.last < u.first) return;
    const uint32_t tid = threadIdx.x, k = u.last - u.first + 1u, joiners = pg_joiners(k, pg_first_joins(k)), mine = blockIdx.x - u.last + joiners - 1u;   /* the last ones */
    if (mine >= joiners) return;   /* the first of many: it arrived as one that joins nothing */
    uint32_t cut = 0;   /* a row is 1 << cut slices of at least 32 dims */
    while (cut < (HD == 64 ? 1u : HD == 128 ? 2u : 3u) && unit_rows << cut < joiners) cut++;
    const uint32_t wide = (uint32_t)HD >> cut, slices = unit_rows << cut;
    const uint32_t s_begin = slices * mine / joiners, s_end = slices * (mine + 1u) / joiners;
    const bool works = ok && s_begin < s_end;
    if (works) {
        if (tid == 0) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory");
        pg_wait(P, u, k);
        float4 *s_a = reinterpret_cast<float4 *>(smem);                      /* [thread] */
        float2 *s_ml = reinterpret_cast<float2 *>(smem + THREADS * 16u);     /* [thread] */
        float *s_gate = reinterpret_cast<float *>(smem + THREADS * 24u);     /* [slice][its dims] */
        /* as many slices at once as fit with all their records; or one, and its records in turn */
        const uint32_t stride = wide + 4u, room = smem_bytes - THREADS * 24u, gate_bytes = P.gate ? wide * 4u : 0u, fit = room / (k * stride * 4u + gate_bytes);
        const uint32_t at_once = fit ? fit : 1u, recs_at_once = fit ? k : (room - gate_bytes) / (stride * 4u);
        uint32_t phase = 0;
        auto there = [&]() -> bool {
            uint32_t done;
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(done) : "r"(bar), "r"(phase) : "memory");
            return done != 0u;
        };
        const uint32_t inv_gqa = 65536u / P.gqa + 1u, per_slice = (HD == 64 ? 4u : HD == 128 ? 5u : 6u) - cut;   /* in / gqa = in * inv_gqa >> 16 for in below 128, gqa up to 16; log2 of a slice's items */
        for (uint32_t s0 = s_begin; s0 < s_end && ok; s0 += at_once) {
            const uint32_t n_s = min(at_once, s_end - s0), items = n_s * (wide / 4u), padded = (items + 31u) & ~31u, groups = padded < THREADS ? THREADS / padded : 1u;
            float *s_rec = s_gate + (P.gate ? n_s * wide : 0u);              /* [record][slice][its dims, m, l, -, -] */
            /* token and head of a slice's row; false: a row without a token */
            auto place = [&](uint32_t s, uint32_t &tok, uint32_t &head) -> bool {
                const uint32_t row = (s0 + s) >> cut, tg = row >> 7, in = row & 127u, tl = in * inv_gqa >> 16;
                tok = tg * P.tpg + tl;
                head = u.kh * P.gqa + in - tl * P.gqa;
                const bool live = tl < P.tpg && tok < u.n_here;
                tok += u.tok0;
                return live;
            };
            auto copy = [&](float *to, const float *from, uint32_t bytes) {
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(bytes), "r"(bar) : "memory");
            };
            auto bring = [&](uint32_t c0, uint32_t n, bool gates) {
                asm volatile("fence.proxy.async;" ::: "memory");             /* what lies there was used by ordinary accesses, and the records were written by such */
                __syncthreads();
                if (tid == 0) {
                    uint32_t bytes = n * n_s * stride * 4u;
                    if (gates) bytes += n_s * wide * 4u;
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
                }
                __syncthreads();
                if (cut == 0u) {                                             /* whole rows lie one behind the other */
                    for (uint32_t c = tid; c < n; c += THREADS) {
                        const uint32_t b = u.first + c0 + c;
                        copy(s_rec + (size_t)c * n_s * REC, P.part + (((size_t)b * 2u + (b == u.first ? 1u : 0u)) * unit_rows + s0) * REC, n_s * REC * 4u);
                    }
                } else {
                    for (uint32_t i = tid; i < n * n_s; i += THREADS) {
                        const uint32_t c = i / n_s, s = i - c * n_s, b = u.first + c0 + c, row = (s0 + s) >> cut, part = (s0 + s) & ((1u << cut) - 1u);
                        const float *rec = P.part + (((size_t)b * 2u + (b == u.first ? 1u : 0u)) * unit_rows + row) * REC;
                        copy(s_rec + (size_t)i * stride, rec + part * wide, wide * 4u);
                        copy(s_rec + (size_t)i * stride + wide, rec + HD, 16u);
                    }
                }
                if (gates)
                    for (uint32_t s = tid; s < n_s; s += THREADS) {
                        uint32_t tok, head;
                        if (!place(s, tok, head)) tok = u.tok0, head = u.kh * P.gqa;   /* any gate: not used */
                        copy(s_gate + s * wide, P.gate + ((size_t)tok * P.n_head + head) * HD + ((s0 + s) & ((1u << cut) - 1u)) * wide, wide * 4u);
                    }
                ok = __syncthreads_and(pg_within(1u << 20, there));
                if (ok) phase ^= 1u;
            };
            bring(0u, recs_at_once < k ? recs_at_once : k, P.gate != nullptr);
            for (uint32_t item0 = 0; item0 < items && ok; item0 += groups > 1u ? padded : THREADS) {
                const uint32_t group = groups > 1u ? tid / padded : 0u, item = item0 + (groups > 1u ? tid - group * padded : tid);
                const uint32_t s = item >> per_slice, d = (item & ((1u << per_slice) - 1u)) * 4u;
                uint32_t tok, head;
                const bool live = item < items && group < groups && place(s, tok, head);
                float M = -CUDART_INF_F, L = 0.f;
                float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
                auto join = [&](float m, float l, float4 x) {
                    const float Mn = fmaxf(M, m), Mu = Mn == -CUDART_INF_F ? 0.f : Mn, fa = pg_ex2(M - Mu), fb = pg_ex2(m - Mu);
                    M = Mn;
                    L = L * fa + l * fb;
                    A.x = A.x * fa + x.x * fb; A.y = A.y * fa + x.y * fb; A.z = A.z * fa + x.z * fb; A.w = A.w * fa + x.w * fb;
                };
                for (uint32_t c0 = 0; c0 < k; c0 += recs_at_once) {          /* more than one turn: one slice, and at most a thread per item */
                    const uint32_t n = min(recs_at_once, k - c0);
                    if (c0) bring(c0, n, false);
                    if (!ok) break;
                    if (live)
                        for (uint32_t c = group; c < n; c += groups) {
                            const float *rec = s_rec + ((size_t)c * n_s + s) * stride;
                            const float2 ml = *reinterpret_cast<const float2 *>(rec + wide);
                            join(ml.x, ml.y, *reinterpret_cast<const float4 *>(rec + d));
                        }
                }
                if (!ok) break;
                if (groups > 1u) {
                    s_a[tid] = A;
                    s_ml[tid] = make_float2(M, L);
                    __syncthreads();
                    if (live && group == 0u)
                        for (uint32_t o = 1; o < groups; o++) join(s_ml[o * padded + tid].x, s_ml[o * padded + tid].y, s_a[o * padded + tid]);
                }
                if (live && group == 0u) pg_store<HD>(P, tok, head, ((s0 + s) & ((1u << cut) - 1u)) * wide + d, A, L, P.gate ? s_gate + s * wide + d : nullptr);
            }
        }
        __syncthreads();
        if (ok) {
            if (tid == 0) asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
        } else {
            if (tid == 0) atomicOr(P.err, (uint32_t)Q4E_CUDA);
            (void)pg_within(4096u, there);   /* those on their way land before the block's shared memory is another's */
        }
    }
    pg_leave(P, u);
}
#endif

#endif
