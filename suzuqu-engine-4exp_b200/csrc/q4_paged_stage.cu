/*
 * The pages of requests that bring many tokens, from q8_0 to fp16: a copy in the layout of an fp16 pool (K and V as fp16(code x scale),
 * the values that the attention itself forms), read by q4_pg_chunk_k's fp16 form with a table of its own.
 *
 * That kernel takes 128 to 256 (token, head) pairs at a time and converts every tile of the request for each such unit: at hd 256,
 * where the conversion sets its pace, a tile costs 3.3 us instead of 1.3.  A request of 2000 tokens with 12 heads per kv head is 200
 * units.  Here every row is converted once, at the rate of memory: 1.06 bytes read and 2 written per value, mostly from and to L2.
 */
#include "q4_paged.h"

namespace {

constexpr uint32_t ST_THREADS = 256, ST_WARPS = ST_THREADS / 32u;

__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
/* fp16 1024 + 128 + code has (code ^ 0x80) in its low byte: two bytes picked out of word x (its codes ^ 0x80), the exact codes, times s */
template <uint32_t SEL>
__device__ __forceinline__ uint32_t scaled2(uint32_t x, __half2 s) {
    const uint32_t u = __byte_perm(x, 0x64646464u, SEL), off = 0x64806480u;
    return h2u(__hmul2(__hsub2(*reinterpret_cast<const __half2 *>(&u), *reinterpret_cast<const __half2 *>(&off)), s));
}

/* A warp takes a tile of 16 rows of one kv head.  `to`: pages in the order of the requests; table: which of them lies where (as wide
 * as the pool's).  fits: whether there are `cap` of them at most; else nothing is done. */
template <int HD>
__global__ void __launch_bounds__(ST_THREADS) q4_pg_stage_k(const PagedParams P, uint8_t *to, int32_t *table, uint32_t cap, uint32_t *fits) {
    extern __shared__ uint32_t s_end[];   /* pages up to and with request r */
    __shared__ uint64_t s_sum[ST_WARPS];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, mask = (1u << P.page_shift) - 1u;
    q4d_pdl_wait();
    auto pages_of = [&](uint32_t r) -> uint32_t {
        bool bad;
        const PgReq R = pg_request(P, r, bad);
        return R.add > P.add_split ? (R.held + R.add + mask) >> P.page_shift : 0u;
    };
    const uint32_t per = (P.n_req + ST_THREADS - 1u) / ST_THREADS, r0 = min(tid * per, P.n_req), r1 = min(r0 + per, P.n_req);
    uint64_t sum = 0, total = 0;
    for (uint32_t r = r0; r < r1; r++) sum += pages_of(r);
    const uint64_t mine = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= (uint32_t)d) sum += x;
    }
    if (lane == 31u) s_sum[warp] = sum;
    __syncthreads();
    uint64_t at = sum - mine;
#pragma unroll
    for (uint32_t w = 0; w < ST_WARPS; w++) {
        if (w < warp) at += s_sum[w];
        total += s_sum[w];
    }
    if (blockIdx.x == 0 && tid == 0) *fits = total <= cap ? 1u : 0u;
    if (total > cap) return;
    for (uint32_t r = r0; r < r1; r++) {
        at += pages_of(r);
        s_end[r] = (uint32_t)at;
    }
    __syncthreads();
    constexpr uint32_t ROW = PgTile<Q4K_Q8, HD>::ROW, OUT = PgTile<Q4K_F16, HD>::BYTES, NB = HD / 64u;
    const uint32_t per_page = 1u << (P.page_shift - 4u), r8 = lane >> 2, c4 = lane & 3u;
    const uint64_t items = total * P.n_kvh * per_page;
    for (uint64_t i = (uint64_t)blockIdx.x * ST_WARPS + warp; i < items; i += (uint64_t)gridDim.x * ST_WARPS) {
        const uint64_t part = i >> (P.page_shift - 4u);   /* page of the copy, kv head */
        const uint32_t tile = (uint32_t)i & (per_page - 1u), sp = (uint32_t)(part / P.n_kvh), kh = (uint32_t)(part - (uint64_t)sp * P.n_kvh);
        uint32_t lo = 0, hi = P.n_req - 1u;               /* the first request whose pages end behind it */
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (s_end[mid] > sp) hi = mid;
            else lo = mid + 1u;
        }
        bool bad;
        const PgReq R = pg_request(P, lo, bad);
        const uint32_t pg = sp - (lo ? s_end[lo - 1u] : 0u);
        const size_t entry = (size_t)lo * P.table_stride + pg;
        const uint32_t page = (uint32_t)P.table[entry];
        const bool there = page < P.n_pages;
        if (lane == 0 && tile == 0u && kh == 0u) table[entry] = there ? (int32_t)sp : -1;
        if (!there || (pg << P.page_shift) + tile * 16u >= R.held + R.add) continue;   /* rows behind the last are not read */
        const uint8_t *src = P.mem + (((uint64_t)page * P.n_kvh + kh) * per_page + tile) * PgTile<Q4K_Q8, HD>::BYTES;
        uint8_t *dst = to + i * OUT;
#pragma unroll
        for (uint32_t w = 0; w < 2; w++) {
            uint4 x[2 * NB];
            uint32_t s[2 * NB];
#pragma unroll
            for (uint32_t k = 0; k < 2u * NB; k++) {
                const uint8_t *rec = src + ((k & 1u) * 8u + r8) * ROW;
                x[k] = __ldcg(reinterpret_cast<const uint4 *>(rec + w * HD + (k >> 1) * 64u + c4 * 16u));
                s[k] = __ldcg(reinterpret_cast<const uint32_t *>(rec + 2u * HD + w * (HD / 16u)) + (k >> 1));
            }
#pragma unroll
            for (uint32_t k = 0; k < 2u * NB; k++) {
                const uint32_t row = (k & 1u) * 8u + r8, s2 = __byte_perm(s[k], 0u, c4 & 2u ? 0x3232u : 0x1010u);
                const __half2 sc = *reinterpret_cast<const __half2 *>(&s2);
                const uint32_t u[4] = {x[k].x ^ 0x80808080u, x[k].y ^ 0x80808080u, x[k].z ^ 0x80808080u, x[k].w ^ 0x80808080u};
                uint32_t o[8];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    o[2 * e] = scaled2<0x4140>(u[e], sc);
                    o[2 * e + 1] = scaled2<0x4342>(u[e], sc);
                }
                uint8_t *d = dst + w * (OUT / 2u) + (k >> 1) * 2048u + row * 128u;
                *reinterpret_cast<uint4 *>(d + (((2u * c4) ^ (row & 7u)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4 *>(d + (((2u * c4 + 1u) ^ (row & 7u)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
            }
        }
    }
}

template <int HD>
bool stage(const PagedParams &p, uint8_t *to, int32_t *table, uint32_t cap, uint32_t *fits) {
    const uint64_t most = (uint64_t)cap * p.n_kvh << (p.page_shift - 4u), want = (most + ST_WARPS - 1u) / ST_WARPS, all = (uint64_t)g_q4.sm_count * 4u;
    /* not a dependent launch: with its blocks resident ahead of time three prompts of heads of 256 took 148 us back to back, so 129 */
    q4_pg_stage_k<HD><<<dim3((unsigned)(want < all ? want : all)), ST_THREADS, p.n_req * sizeof(uint32_t), g_q4.stream>>>(p, to, table, cap, fits);
    return q4i_launched(q4i_check(cudaGetLastError(), "pages_attend stage launch"));
}

}  // namespace

bool q4i_paged_stage(const PagedParams &p, uint32_t hd, uint8_t *to, int32_t *table, uint32_t cap, uint32_t *fits) {
    return hd == 64 ? stage<64>(p, to, table, cap, fits) : hd == 128 ? stage<128>(p, to, table, cap, fits) : stage<256>(p, to, table, cap, fits);
}
