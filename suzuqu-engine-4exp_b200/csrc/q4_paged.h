/* Shared by the two attention kernels over a pool of pages (q4_paged.cu, q4_paged_tc.cu; not installed). */
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
    uint32_t tpg, group_rows;    /* tokens of a group, rows that a group takes (the last ones may be empty) */
    uint32_t add_split;          /* requests that bring at most so many tokens are q4_pg_few_k's, the others q4_pg_chunk_k's */
    const int32_t *rows, *start, *table;
    uint32_t table_stride, n_req, n_tok;
    const void *q;
    const float *gate;
    void *out;
    int q_bf16, out_bf16;
    float scale_log2e;
    float *part;                 /* [block][2][rows of a unit][hd + 4]: acc, m (log2 units, scale folded in), l */
    uint32_t *meet;              /* [block][2]: arrived, gone, of the blocks of the unit that begins in the block; zero between launches */
    uint32_t *err;
};

template <int KIND, int HD>
struct PgTile {
    static constexpr uint32_t ROW = KIND == Q4K_Q8 ? (2u * HD + HD / 8u + 15u) / 16u * 16u : 4u * HD, BYTES = 16u * ROW;
};

constexpr uint32_t PG_MAX_BLOCKS = 1024;

/* The tokens of requests that bring more than P.add_split, on the tensor cores (q4_paged_tc.cu), with its records in `scratch`, of
 * at least q4i_paged_chunk_floats floats.  hd 64, 128 or 256, kind fp16 or q8_0. */
size_t q4i_paged_chunk_floats(uint32_t hd);
bool q4i_paged_chunk(const PagedParams &p, int kind, uint32_t hd, float *scratch);

#ifdef __CUDACC__
/* what the host or the device gave for request r: tokens (0: none of this launch's), rows before them */
struct PgReq { uint32_t held, add, tok0; };
__device__ __forceinline__ PgReq pg_request(const PagedParams &P, uint32_t r, bool &bad) {
    const int32_t s0 = P.start[r], s1 = P.start[r + 1u], h = P.rows[r];
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
/* four dims of a row: acc / l * sigmoid(gate), where there are gates.  A row that attended nothing is 0, one with a NaN among its scores stays NaN */
template <int HD>
__device__ __forceinline__ void pg_store(const PagedParams &P, uint32_t tok, uint32_t head, uint32_t d, float4 x, float L, const float *gate) {
    const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
    const size_t at = ((size_t)tok * P.n_head + head) * HD + d;
    x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
    if (gate) {
        const float4 gt = *reinterpret_cast<const float4 *>(gate);
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

/* A unit that lies in several blocks, first to last; last < first: none */
struct PgSplit { uint32_t first, last, tok0, n_here, kh; };
/* The blocks of a split unit meet at a counter, and all but the first, which has the end of another unit to see to, join its
 * records, each an equal part of the rows.  All blocks of the launch are resident (the grid is what the SMs hold), and end their
 * shares within a few microseconds of one another; a launch of its own for this took 8 to 12 us (one request over 262 144 rows
 * 44 us with it).  The wait is bounded.  Every block arrives and goes once, whatever happened before, and the last to go leaves
 * the counters at zero.
 * What a block joins, and its gates, come to shared memory by asynchronous copies, all at once; then a thread has four dims of a
 * row, or shares them with others that take the other records. */
__device__ __forceinline__ void pg_arrive(const PagedParams &P, const PgSplit &u) {   /* one thread, behind the block's records and a barrier */
    if (u.last < u.first) return;
    __threadfence();
    atomicAdd(P.meet + 2u * u.first, 1u);
}
template <int HD, uint32_t THREADS>
__device__ __forceinline__ void pg_join(const PagedParams &P, const PgSplit &u, uint32_t unit_rows, uint8_t *smem, uint32_t smem_bytes) {
    constexpr uint32_t REC = HD + 4u, PIECES = REC / 4u, WARPS = THREADS / 32u;   /* of 16 bytes */
    if (u.last < u.first) return;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, k = u.last - u.first + 1u, mine = blockIdx.x - u.first - 1u;
    const uint32_t r_begin = unit_rows * mine / (k - 1u), r_end = unit_rows * (mine + 1u) / (k - 1u);
    if (r_begin < r_end) {
        if (tid == 0) {
            unsigned long long t0, t;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
            for (uint32_t i = 0;; i++) {
                uint32_t n;
                asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(P.meet + 2u * u.first) : "memory");
                if (n >= k) break;
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
        float4 *s_a = reinterpret_cast<float4 *>(smem);                      /* [thread] */
        float2 *s_ml = reinterpret_cast<float2 *>(smem + THREADS * 16u);     /* [thread] */
        float *s_gate = reinterpret_cast<float *>(smem + THREADS * 24u);     /* [row][hd] */
        /* as many rows at once as fit with all their records; or one row, and its records in turn */
        const uint32_t room = smem_bytes - THREADS * 24u, gate_bytes = P.gate ? HD * 4u : 0u, fit = room / (k * REC * 4u + gate_bytes);
        const uint32_t rows_at_once = fit ? fit : 1u, recs_at_once = fit ? k : (room - gate_bytes) / (REC * 4u);
        for (uint32_t r0 = r_begin; r0 < r_end; r0 += rows_at_once) {
        const uint32_t rows = min(rows_at_once, r_end - r0), items = rows * (HD / 4u), padded = (items + 31u) & ~31u, groups = padded < THREADS ? THREADS / padded : 1u;
        float *s_rec = s_gate + (P.gate ? rows * HD : 0u);                   /* [record][row][hd + 4] */
        /* token and head of a row of these; false: a row without a token */
        auto place = [&](uint32_t rl, uint32_t &tok, uint32_t &head) -> bool {
            const uint32_t row = r0 + rl, tg = row / P.group_rows, in = row - tg * P.group_rows, tl = in / P.gqa;
            tok = tg * P.tpg + tl;
            head = u.kh * P.gqa + in - tl * P.gqa;
            const bool live = tl < P.tpg && tok < u.n_here;
            tok += u.tok0;
            return live;
        };
        auto copy = [&](float *to, const float *from) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
        };
        auto bring = [&](uint32_t c0, uint32_t n) {   /* a row of a record per warp and step */
            for (uint32_t pair = warp; pair < n * rows; pair += WARPS) {
                const uint32_t c = pair / rows, rl = pair - c * rows, b = u.first + c0 + c;
                const float *src = P.part + (((size_t)b * 2u + (b == u.first ? 1u : 0u)) * unit_rows + r0 + rl) * REC;
                for (uint32_t x = lane; x < PIECES; x += 32u) copy(s_rec + (size_t)pair * REC + x * 4u, src + x * 4u);
            }
            if (P.gate && c0 == 0u)
                for (uint32_t rl = warp; rl < rows; rl += WARPS) {
                    uint32_t tok, head;
                    if (place(rl, tok, head))
                        for (uint32_t x = lane; x < HD / 4u; x += 32u) copy(s_gate + rl * HD + x * 4u, P.gate + ((size_t)tok * P.n_head + head) * HD + x * 4u);
                }
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
            __syncthreads();
        };
        __syncthreads();   /* the rows before have been read */
        bring(0u, recs_at_once);
        for (uint32_t item0 = 0; item0 < items; item0 += groups > 1u ? padded : THREADS) {
            const uint32_t group = groups > 1u ? tid / padded : 0u, item = item0 + (groups > 1u ? tid - group * padded : tid);
            const uint32_t rl = item / (HD / 4u), d = item % (HD / 4u) * 4u;
            uint32_t tok, head;
            const bool live = item < items && group < groups && place(rl, tok, head);
            float M = -CUDART_INF_F, L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
            auto join = [&](float m, float l, float4 x) {
                const float Mn = fmaxf(M, m), Mu = Mn == -CUDART_INF_F ? 0.f : Mn, fa = pg_ex2(M - Mu), fb = pg_ex2(m - Mu);
                M = Mn;
                L = L * fa + l * fb;
                A.x = A.x * fa + x.x * fb; A.y = A.y * fa + x.y * fb; A.z = A.z * fa + x.z * fb; A.w = A.w * fa + x.w * fb;
            };
            for (uint32_t c0 = 0; c0 < k; c0 += recs_at_once) {   /* more than one turn: one row, and at most a thread per item */
                const uint32_t n = min(recs_at_once, k - c0);
                if (c0) {
                    __syncthreads();   /* the records before have been read */
                    bring(c0, n);
                }
                if (live)
                    for (uint32_t c = group; c < n; c += groups) {
                        const float *rec = s_rec + ((size_t)c * rows + rl) * REC;
                        const float2 ml = *reinterpret_cast<const float2 *>(rec + HD);
                        join(ml.x, ml.y, *reinterpret_cast<const float4 *>(rec + d));
                    }
            }
            if (groups > 1u) {
                s_a[tid] = A;
                s_ml[tid] = make_float2(M, L);
                __syncthreads();
                if (live && group == 0u)
                    for (uint32_t o = 1; o < groups; o++) join(s_ml[o * padded + tid].x, s_ml[o * padded + tid].y, s_a[o * padded + tid]);
            }
            if (live && group == 0u) pg_store<HD>(P, tok, head, d, A, L, P.gate ? s_gate + rl * HD + d : nullptr);
        }
        }
    }
    __syncthreads();
    if (tid == 0 && atomicAdd(P.meet + 2u * u.first + 1u, 1u) == k - 2u) {
        P.meet[2u * u.first] = 0u;
        P.meet[2u * u.first + 1u] = 0u;
    }
}
#endif

#endif
