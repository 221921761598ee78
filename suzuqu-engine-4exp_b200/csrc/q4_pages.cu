/*
 * A paged KV cache: pages handed out and taken back on the device, block tables and slot maps from the requests' lengths,
 * rows appended to and read back from their slots.  (Its attention is in q4_paged.cu.)  No counterpart in the reference,
 * which holds one contiguous cache per session (src/q4_fwd.c:1944-1950).
 *
 * Memory of a pool: [layer][page][kv head][page_rows / 16 tiles of 16 rows].  A tile is what the attention brings in at once:
 *   q8_0  16 records {K codes hd | V codes hd | K scales hd/32 fp16 | V scales}, padded to 16 bytes: the record of the library's
 *         store, whose odd number of 16-byte pieces (hd 64, 128) puts the rows of a matrix fragment on different banks
 *   fp16  K, then V, each hd / 64 blocks of 16 rows x 128 bytes; piece c (16 bytes) of row r lies at c ^ (r & 7): 8 or 16 such
 *         tiles one behind the other are the swizzled operand that the tensor core reads
 * Either way a tile is contiguous and arrives by bulk copies as it is used.
 */
#include "q4_paged.h"

namespace {

constexpr uint32_t PLAN_THREADS = 512, PLAN_MAX_REQ = 8192;

/* blocks of a launch that have finished, in the upper half those that want the stack left alone; zero between launches */
__device__ uint32_t g_plan_arrived;

struct PlanParams {
    const int32_t *rows, *more;  /* plan: rows held, new tokens; trim: rows held, rows kept */
    uint32_t n_req, table_stride, page_shift, n_pages, max_tok;
    int32_t *table, *start, *slot, *pos, *req;
    int32_t *free_list, *n_free;
    uint32_t vec;                /* the token arrays take 16-byte stores */
    uint32_t *err;
};

/* exclusive sums over the block's threads of (a, b), and their totals */
__device__ __forceinline__ void block_scan2(uint64_t &a, uint64_t &b, uint64_t &ta, uint64_t &tb) {
    __shared__ uint64_t s_a[PLAN_THREADS / 32], s_b[PLAN_THREADS / 32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint64_t a0 = a, b0 = b;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, a, d), y = __shfl_up_sync(0xffffffffu, b, d);
        if (lane >= (uint32_t)d) { a += x; b += y; }
    }
    if (lane == 31u) { s_a[warp] = a; s_b[warp] = b; }
    __syncthreads();
    uint64_t pa = 0, pb = 0;
    ta = tb = 0;
#pragma unroll
    for (uint32_t w = 0; w < PLAN_THREADS / 32; w++) {
        if (w < warp) { pa += s_a[w]; pb += s_b[w]; }
        ta += s_a[w]; tb += s_b[w];
    }
    a += pa - a0;
    b += pb - b0;
}

/* the last block to finish moves the stack's top, unless a thread of any block says no: all of them have read it by then */
__device__ __forceinline__ void move_top(int32_t *n_free, int32_t to, uint32_t *err, bool no = false) {
    const bool stays = __syncthreads_or(no);
    if (threadIdx.x == 0) {
        __threadfence();
        const uint32_t mine = stays ? 0x10001u : 1u, all = atomicAdd(&g_plan_arrived, mine) + mine;
        if ((all & 0xffffu) == gridDim.x) {
            g_plan_arrived = 0u;
            if (all >> 16) atomicOr(err, (uint32_t)Q4E_RANGE);
            else *n_free = to;
        }
    }
}

/*
 * Plan.  With h rows held and n new tokens request r takes need = ceil((h + n) / P) - ceil(h / P) pages; page i of all of them,
 * in the order of the requests, is the i-th from the top of the stack.  Requests are served up to the first one that the
 * sums show not to fit (pages left, tokens of the step).
 * Every block forms the sums over all requests itself: 8 bytes per request from L2 and one scan are less than a meeting of
 * the blocks.  Then a thread takes four tokens, finds the request of the first by bisection, and stores 16 bytes of each map;
 * the token on a new page's first row stores its table entry (every new page has one).
 */
__global__ void __launch_bounds__(PLAN_THREADS) q4_pg_plan_k(const PlanParams P) {
    extern __shared__ uint32_t s_plan[];
    __shared__ uint64_t s_total, s_pages;
    uint32_t *tok_end = s_plan, *page_at = s_plan + P.n_req;   /* tokens up to and with request r; pages before it */
    const uint32_t tid = threadIdx.x, mask = (1u << P.page_shift) - 1u;
    const uint64_t room = (uint64_t)P.table_stride << P.page_shift;
    if (tid == 0) s_total = s_pages = 0;
    q4d_pdl_wait();
    const int32_t top = *P.n_free;
    const uint64_t n_free = top < 0 ? 0u : min((uint32_t)top, P.n_pages);
    const uint32_t per = (P.n_req + PLAN_THREADS - 1u) / PLAN_THREADS, r0 = min(tid * per, P.n_req), r1 = min(r0 + per, P.n_req);
    auto one = [&](uint32_t r, uint64_t &n, uint64_t &need, bool &bad) {
        const int32_t h = __ldcg(P.rows + r), a = __ldcg(P.more + r);
        n = a > 0 ? (uint64_t)a : 0u;
        bad = n && (h < 0 || (uint64_t)h + n > room);
        if (bad) n = 0;
        need = n ? (((uint64_t)h + n + mask) >> P.page_shift) - (((uint64_t)h + mask) >> P.page_shift) : 0u;
    };
    uint64_t n_sum = 0, need_sum = 0, n_all, need_all, n, need;
    bool bad, any_bad = false;
    for (uint32_t r = r0; r < r1; r++) {
        one(r, n, need, bad);
        n_sum += n; need_sum += need;
        any_bad |= bad;
    }
    block_scan2(n_sum, need_sum, n_all, need_all);
    uint64_t fit_n = 0, fit_pages = 0;   /* sums up to this thread's last served request */
    for (uint32_t r = r0; r < r1; r++) {
        one(r, n, need, bad);
        const uint64_t before = need_sum;
        n_sum += n; need_sum += need;
        const bool fits = n_sum <= P.max_tok && need_sum <= n_free;
        if (fits) { fit_n = n_sum; fit_pages = need_sum; }
        tok_end[r] = fits ? (uint32_t)n_sum : 0xffffffffu;   /* 0xffffffff: not served */
        page_at[r] = (uint32_t)before;
    }
    if (fit_n) atomicMax((unsigned long long *)&s_total, (unsigned long long)fit_n);
    if (fit_pages) atomicMax((unsigned long long *)&s_pages, (unsigned long long)fit_pages);
    __syncthreads();
    const uint32_t total = (uint32_t)s_total, pages = (uint32_t)s_pages;
    if (blockIdx.x == 0) {
        for (uint32_t r = tid; r < P.n_req; r += PLAN_THREADS) P.start[r + 1u] = (int32_t)min(tok_end[r], total);
        if (tid == 0) P.start[0] = 0;
        if (any_bad) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        if (tid == 0 && (n_all > total || need_all > pages)) atomicOr(P.err, (uint32_t)Q4E_SCRATCH);
    }
    for (uint64_t t0 = ((uint64_t)blockIdx.x * PLAN_THREADS + tid) * 4u; t0 < P.max_tok; t0 += (uint64_t)gridDim.x * PLAN_THREADS * 4u) {
        int32_t slot[4], pos[4], req[4];
        uint32_t r = 0, first_page = 0, begin = 0, end = 0;
        int32_t h = 0;
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) {
            const uint32_t t = (uint32_t)t0 + k;
            slot[k] = pos[k] = req[k] = -1;
            if (t >= total) continue;
            if (t >= end) {
                uint32_t lo = end ? r + 1u : 0u, hi = P.n_req - 1u;   /* the first request whose tokens end behind t */
                while (lo < hi) {
                    const uint32_t mid = (lo + hi) >> 1;
                    if (tok_end[mid] > t) hi = mid;
                    else lo = mid + 1u;
                }
                r = lo;
                begin = r ? tok_end[r - 1u] : 0u;
                end = tok_end[r];
                h = __ldcg(P.rows + r);
                first_page = ((uint32_t)h + mask) >> P.page_shift;
            }
            const uint32_t p = (uint32_t)h + (t - begin), pg = p >> P.page_shift;
            int32_t *entry = P.table + (size_t)r * P.table_stride + pg;
            int32_t page;
            if (pg < first_page) {
                page = *entry;
            } else {
                page = __ldcg(P.free_list + (n_free - 1u - (page_at[r] + (pg - first_page))));
                if ((p & mask) == 0u) *entry = page;
            }
            slot[k] = page < 0 || (uint32_t)page >= P.n_pages ? -1 : (int32_t)(((uint32_t)page << P.page_shift) | (p & mask));
            if (slot[k] < 0) atomicOr(P.err, (uint32_t)Q4E_RANGE);
            pos[k] = (int32_t)p;
            req[k] = (int32_t)r;
        }
        if (P.vec && t0 + 4u <= P.max_tok) {
            *reinterpret_cast<int4 *>(P.slot + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4 *>(P.pos + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
            *reinterpret_cast<int4 *>(P.req + t0) = make_int4(req[0], req[1], req[2], req[3]);
        } else {
            for (uint32_t k = 0; k < 4u && t0 + k < P.max_tok; k++) {
                P.slot[t0 + k] = slot[k]; P.pos[t0 + k] = pos[k]; P.req[t0 + k] = req[k];
            }
        }
    }
    move_top(P.n_free, (int32_t)(n_free - pages), P.err);
}

/* Trim: pages ceil(kept / P) .. ceil(held / P) of every request go back, the last one of all lowest, so that a plan that is
 * taken back leaves the stack as it was.  An entry that is no page of the pool (rows that no plan served) leaves all of them out: on the
 * stack it would be handed out in place of a page. */
__global__ void __launch_bounds__(PLAN_THREADS) q4_pg_trim_k(const PlanParams P) {
    extern __shared__ uint32_t s_plan[];
    uint32_t *page_end = s_plan;
    const uint32_t tid = threadIdx.x, mask = (1u << P.page_shift) - 1u;
    const uint64_t room = (uint64_t)P.table_stride << P.page_shift;
    q4d_pdl_wait();
    const int32_t top = *P.n_free;
    const uint64_t n_free = top < 0 ? 0u : (uint32_t)top;
    const uint32_t per = (P.n_req + PLAN_THREADS - 1u) / PLAN_THREADS, r0 = min(tid * per, P.n_req), r1 = min(r0 + per, P.n_req);
    auto one = [&](uint32_t r, bool &bad) -> uint32_t {
        const int32_t h = __ldcg(P.rows + r), k = __ldcg(P.more + r);
        bad = h > 0 && (uint64_t)h > room;
        if (bad || h <= 0 || k >= h) return 0u;
        return (((uint32_t)h + mask) >> P.page_shift) - ((k > 0 ? (uint32_t)k + mask : 0u) >> P.page_shift);
    };
    uint64_t sum = 0, all, none = 0, none_all;
    bool bad, any_bad = false;
    for (uint32_t r = r0; r < r1; r++) {
        sum += one(r, bad);
        any_bad |= bad;
    }
    block_scan2(sum, none, all, none_all);
    for (uint32_t r = r0; r < r1; r++) {
        sum += one(r, bad);
        page_end[r] = (uint32_t)min(sum, (uint64_t)0xffffffffu);
    }
    const bool fits = n_free + all <= P.n_pages;   /* else a page would come back twice */
    if (blockIdx.x == 0 && (any_bad || (tid == 0 && !fits))) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    __syncthreads();
    bool no_page = false;
    if (fits) {
        for (uint64_t i = (uint64_t)blockIdx.x * PLAN_THREADS + tid; i < all; i += (uint64_t)gridDim.x * PLAN_THREADS) {
            uint32_t lo = 0, hi = P.n_req - 1u;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) >> 1;
                if (page_end[mid] > i) hi = mid;
                else lo = mid + 1u;
            }
            const int32_t h = __ldcg(P.rows + lo);
            /* counted from the request's end */
            const uint32_t pg = (((uint32_t)h + mask) >> P.page_shift) - (page_end[lo] - (uint32_t)i);
            const int32_t page = P.table[(size_t)lo * P.table_stride + pg];
            no_page |= (uint32_t)page >= P.n_pages;
            P.free_list[n_free + all - 1u - i] = page;   /* above the top: of no meaning until that moves */
        }
    }
    move_top(P.n_free, fits ? (int32_t)(n_free + all) : top, P.err, no_page);
}

struct RowParams {
    uint8_t *mem;                /* of the layer */
    uint32_t n_kvh, page_shift, n_tok;
    uint32_t slots;              /* n_pages << page_shift */
    const int32_t *slot;
    const float *k, *v;          /* append: [token][kv head][hd] */
    float *k_out, *v_out;        /* gather */
    uint32_t *err;
};
/* of the slot: its page's part of the kv head, its tile, its row of the tile */
template <int KIND, int HD>
__device__ __forceinline__ uint8_t *slot_tile(const RowParams &P, uint32_t slot, uint32_t kh) {
    const uint32_t page = slot >> P.page_shift, in = slot & ((1u << P.page_shift) - 1u);
    const uint64_t part = ((uint64_t)page * P.n_kvh + kh) << (P.page_shift - 4u);
    return P.mem + (part + (in >> 4)) * PgTile<KIND, HD>::BYTES;
}

/*
 * Append and gather: 8 dims per thread (two 16-byte loads of fp32; 8 codes or one 16-byte piece of fp16), K and V of them, so
 * that a thread has 64 bytes in flight.  Both are bound by memory: 4 bytes read per value for 1 or 2 written, or the reverse.
 * The quantiser is the store's (q4d_scale, q4d_quant4), with four lanes to a block of 32 instead of eight.
 */
template <int KIND, int HD>
__global__ void __launch_bounds__(256) q4_pg_append_k(const RowParams P) {
    constexpr uint32_t PER = HD / 8u;
    q4d_pdl_wait();
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint32_t c = (uint32_t)i % PER;
    const uint64_t row = i / PER;
    const uint32_t tok = (uint32_t)(row / P.n_kvh), kh = (uint32_t)(row % P.n_kvh);
    const bool live = tok < P.n_tok;
    float4 x[2][2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const float4 *src = reinterpret_cast<const float4 *>((w ? P.v : P.k) + (size_t)row * HD + c * 8u);
        x[w][0] = live ? __ldcs(src) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[w][1] = live ? __ldcs(src + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int32_t slot = live ? __ldcg(P.slot + tok) : -1;
    const bool store = slot >= 0 && (uint32_t)slot < P.slots;
    if (slot >= 0 && !store && c == 0u) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    uint8_t *tile = slot_tile<KIND, HD>(P, store ? (uint32_t)slot : 0u, kh);
    const uint32_t in = (uint32_t)slot & 15u;
#pragma unroll
    for (uint32_t w = 0; w < 2; w++) {
        const float4 a = x[w][0], b = x[w][1];
        if constexpr (KIND == Q4K_Q8) {
            float m = fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))),
                            fmaxf(fmaxf(fabsf(b.x), fabsf(b.y)), fmaxf(fabsf(b.z), fabsf(b.w))));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            float d, id;
            q4d_scale(m, d, id);
            if (store) {
                uint8_t *rec = tile + in * PgTile<KIND, HD>::ROW;
                *reinterpret_cast<uint2 *>(rec + w * HD + c * 8u) = make_uint2(q4d_quant4(a, id), q4d_quant4(b, id));
                if ((c & 3u) == 0u) reinterpret_cast<__half *>(rec + 2u * HD)[w * (HD / 32u) + (c >> 2)] = __float2half_rn(d);
            }
        } else if (store) {
            const __half2 h[4] = {__floats2half2_rn(a.x, a.y), __floats2half2_rn(a.z, a.w), __floats2half2_rn(b.x, b.y), __floats2half2_rn(b.z, b.w)};
            uint8_t *dst = tile + w * (PgTile<KIND, HD>::BYTES / 2u) + (c >> 3) * 2048u + in * 128u + (((c & 7u) ^ (in & 7u)) << 4);
            *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(h);
        }
    }
}

template <int KIND, int HD>
__global__ void __launch_bounds__(256) q4_pg_gather_k(const RowParams P) {
    constexpr uint32_t PER = HD / 8u;
    q4d_pdl_wait();
    const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint32_t c = (uint32_t)i % PER;
    const uint64_t row = i / PER;
    const uint32_t tok = (uint32_t)(row / P.n_kvh), kh = (uint32_t)(row % P.n_kvh);
    if (tok >= P.n_tok) return;
    const int32_t slot = __ldcg(P.slot + tok);
    const bool there = slot >= 0 && (uint32_t)slot < P.slots;
    if (slot >= 0 && !there && c == 0u) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    const uint8_t *tile = slot_tile<KIND, HD>(P, there ? (uint32_t)slot : 0u, kh);
    const uint32_t in = (uint32_t)slot & 15u;
    float x[2][8];
#pragma unroll
    for (uint32_t w = 0; w < 2; w++) {
        if constexpr (KIND == Q4K_Q8) {
            const uint8_t *rec = tile + in * PgTile<KIND, HD>::ROW;
            const uint2 q = there ? __ldcg(reinterpret_cast<const uint2 *>(rec + w * HD + c * 8u)) : make_uint2(0u, 0u);
            const float s = there ? __half2float(__ushort_as_half(__ldcg(reinterpret_cast<const unsigned short *>(rec + 2u * HD) + w * (HD / 32u) + (c >> 2)))) : 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) x[w][j] = (float)(int8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3))) * s;
        } else {
            const uint8_t *src = tile + w * (PgTile<KIND, HD>::BYTES / 2u) + (c >> 3) * 2048u + in * 128u + (((c & 7u) ^ (in & 7u)) << 4);
            const uint4 q = there ? __ldcg(reinterpret_cast<const uint4 *>(src)) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
                x[w][2 * j] = f.x; x[w][2 * j + 1] = f.y;
            }
        }
    }
#pragma unroll
    for (uint32_t w = 0; w < 2; w++) {
        float *out = w ? P.v_out : P.k_out;
        if (!out) continue;
        float4 *dst = reinterpret_cast<float4 *>(out + (size_t)row * HD + c * 8u);
        __stcs(dst, make_float4(x[w][0], x[w][1], x[w][2], x[w][3]));
        __stcs(dst + 1, make_float4(x[w][4], x[w][5], x[w][6], x[w][7]));
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0u; }

bool rows_launch(const char *what, const q4_gpu_pages *pg, RowParams &p, uint32_t layer, bool append) {
    p.mem = (uint8_t *)pg->mem + (uint64_t)layer * (q4i_pages_row_bytes(pg->hd, pg->kind) * pg->page_rows * pg->n_kvh) * pg->n_pages;
    p.n_kvh = pg->n_kvh;
    p.page_shift = (uint32_t)__builtin_ctz(pg->page_rows);
    p.slots = pg->n_pages << p.page_shift;
    p.err = g_q4.err_d;
    const uint64_t blocks = ((uint64_t)p.n_tok * pg->n_kvh * (pg->hd / 8u) + 255u) / 256u;
    if (blocks > 0x7fffffffu) return q4i_fail(Q4E_ARG, "pages: too many tokens for one call");
    const dim3 grid((unsigned)blocks);
#define PG_ROWS(KIND, HD)                                                                                  \
    if (pg->kind == KIND && pg->hd == HD)                                                                  \
        return append ? q4i_launch_pdl(what, q4_pg_append_k<KIND, HD>, grid, 256u, 0, p)                   \
                      : q4i_launch_pdl(what, q4_pg_gather_k<KIND, HD>, grid, 256u, 0, p);
    PG_ROWS(Q4K_Q8, 64) PG_ROWS(Q4K_Q8, 128) PG_ROWS(Q4K_Q8, 256) PG_ROWS(Q4K_F16, 64) PG_ROWS(Q4K_F16, 128) PG_ROWS(Q4K_F16, 256)
#undef PG_ROWS
    return q4i_fail(Q4E_ARG, what);
}

}  // namespace

/* K and V of one position and kv head */
uint32_t q4i_pages_row_bytes(uint32_t hd, int kind) { return kind == Q4K_Q8 ? (2u * hd + hd / 8u + 15u) / 16u * 16u : 4u * hd; }
bool q4i_pages_ok(const q4_gpu_pages *pg) {
    return pg && (pg->kind == Q4K_Q8 || pg->kind == Q4K_F16) && (pg->hd == 64 || pg->hd == 128 || pg->hd == 256) && pg->n_layers && pg->n_kvh &&
           pg->n_kvh <= 4096 && pg->n_pages && pg->page_rows >= 16 && pg->page_rows <= 256 && (pg->page_rows & (pg->page_rows - 1u)) == 0 &&
           (uint64_t)pg->n_pages * pg->page_rows <= 0x7fffffffu;
}

extern "C" uint64_t q4_gpu_pages_bytes(uint32_t n_layers, uint32_t n_kvh, uint32_t hd, uint32_t n_pages, uint32_t page_rows, int kind) {
    q4_gpu_pages pg = {};
    pg.n_layers = n_layers; pg.n_kvh = n_kvh; pg.hd = hd; pg.n_pages = n_pages; pg.page_rows = page_rows; pg.kind = kind;
    if (!q4i_pages_ok(&pg)) return 0;
    return (uint64_t)q4i_pages_row_bytes(hd, kind) * page_rows * n_kvh * n_pages * n_layers;
}

extern "C" bool q4_gpu_pages_plan(const q4_gpu_pages *pg, const int32_t *rows, const int32_t *add, uint32_t n_req, int32_t *table,
                                  uint32_t table_stride, int32_t *start, int32_t *slot, int32_t *pos, int32_t *req, uint32_t max_tok) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "pages_plan: library not initialised");
    Q4_REQUIRE(q4i_pages_ok(pg) && pg->free_list && pg->n_free, "pages_plan: bad pool");
    Q4_REQUIRE(rows && add && table && start && slot && pos && req && n_req && table_stride && max_tok, "pages_plan: bad argument");
    Q4_REQUIRE(n_req <= PLAN_MAX_REQ && max_tok <= 0x7fffffffu, "pages_plan: at most 8192 requests and 2^31 - 1 tokens");
    Q4_REQUIRE((uint64_t)table_stride * pg->page_rows <= 0x7fffffffu, "pages_plan: a block table's rows pass 2^31 - 1");
    PlanParams p = {};
    p.rows = rows; p.more = add; p.n_req = n_req; p.table = table; p.table_stride = table_stride;
    p.start = start; p.slot = slot; p.pos = pos; p.req = req; p.max_tok = max_tok;
    p.free_list = pg->free_list; p.n_free = pg->n_free; p.n_pages = pg->n_pages;
    p.page_shift = (uint32_t)__builtin_ctz(pg->page_rows);
    p.vec = aligned16(slot) && aligned16(pos) && aligned16(req);
    p.err = g_q4.err_d;
    /* one round of four tokens per thread, while that is at most four blocks per SM */
    const uint32_t want = (max_tok + PLAN_THREADS * 4u - 1u) / (PLAN_THREADS * 4u), cap = (uint32_t)g_q4.sm_count * 4u;
    const size_t smem = 2u * n_req * sizeof(uint32_t);
    static bool attr = false;
    if (!attr && !q4i_check(cudaFuncSetAttribute(q4_pg_plan_k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(2u * PLAN_MAX_REQ * sizeof(uint32_t))), "pages_plan smem attribute")) return false;
    attr = true;
    return q4i_launch_pdl("pages_plan launch", q4_pg_plan_k, dim3(want < cap ? want : cap), PLAN_THREADS, smem, p);
}

extern "C" bool q4_gpu_pages_trim(const q4_gpu_pages *pg, const int32_t *rows, const int32_t *keep, uint32_t n_req, const int32_t *table, uint32_t table_stride) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "pages_trim: library not initialised");
    Q4_REQUIRE(q4i_pages_ok(pg) && pg->free_list && pg->n_free, "pages_trim: bad pool");
    Q4_REQUIRE(rows && keep && table && n_req && table_stride, "pages_trim: bad argument");
    Q4_REQUIRE(n_req <= PLAN_MAX_REQ, "pages_trim: at most 8192 requests");
    Q4_REQUIRE((uint64_t)table_stride * pg->page_rows <= 0x7fffffffu, "pages_trim: a block table's rows pass 2^31 - 1");
    PlanParams p = {};
    p.rows = rows; p.more = keep; p.n_req = n_req; p.table = (int32_t *)table; p.table_stride = table_stride;
    p.free_list = pg->free_list; p.n_free = pg->n_free; p.n_pages = pg->n_pages;
    p.page_shift = (uint32_t)__builtin_ctz(pg->page_rows);
    p.err = g_q4.err_d;
    const uint64_t most = (uint64_t)n_req * table_stride < pg->n_pages ? (uint64_t)n_req * table_stride : pg->n_pages;
    const uint64_t want = (most + PLAN_THREADS - 1u) / PLAN_THREADS, cap = (uint64_t)g_q4.sm_count;
    return q4i_launch_pdl("pages_trim launch", q4_pg_trim_k, dim3((unsigned)(want < cap ? want : cap)), PLAN_THREADS, n_req * sizeof(uint32_t), p);
}

extern "C" bool q4_gpu_pages_append(const q4_gpu_pages *pg, uint32_t layer, const float *k, const float *v, const int32_t *slot, uint32_t n_tok) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "pages_append: library not initialised");
    Q4_REQUIRE(q4i_pages_ok(pg) && pg->mem && aligned16(pg->mem) && layer < pg->n_layers, "pages_append: bad pool or layer");
    Q4_REQUIRE(k && v && slot && n_tok, "pages_append: bad argument");
    Q4_REQUIRE(aligned16(k) && aligned16(v), "pages_append: rows must be 16-byte aligned");
    RowParams p = {};
    p.k = k; p.v = v; p.slot = slot; p.n_tok = n_tok;
    return rows_launch("pages_append launch", pg, p, layer, true);
}

extern "C" bool q4_gpu_pages_gather(const q4_gpu_pages *pg, uint32_t layer, const int32_t *slot, uint32_t n_tok, float *k, float *v) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "pages_gather: library not initialised");
    Q4_REQUIRE(q4i_pages_ok(pg) && pg->mem && aligned16(pg->mem) && layer < pg->n_layers, "pages_gather: bad pool or layer");
    Q4_REQUIRE((k || v) && slot && n_tok, "pages_gather: bad argument");
    Q4_REQUIRE(aligned16(k) && aligned16(v), "pages_gather: rows must be 16-byte aligned");
    RowParams p = {};
    p.k_out = k; p.v_out = v; p.slot = slot; p.n_tok = n_tok;
    return rows_launch("pages_gather launch", pg, p, layer, false);
}
