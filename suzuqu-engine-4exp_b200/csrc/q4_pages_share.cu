/*
 * Pages with several holders, and pools that are cut: fork (a prefix is taken over), release (pages go back with their last holder),
 * compact (the pages in use are moved to the low end).  No counterpart in the reference, whose session holds its one cache alone.
 *
 * shares[p] counts the holders of page p besides the first, so that pages which plan hands out need no count and those of a pool
 * without forks stay at zero.  Behind the counts lie two words per page that are the calls' own and zero between them.
 */
#include "q4_paged.h"
#include "q4_pages_scan.h"

namespace {

/* blocks of a launch that have finished, as in q4_pages.cu; of fork, of release */
__device__ uint32_t g_fork_arrived, g_rel_arrived;

/* 16 bytes, by copies that go past L1 and are not wanted again */
__device__ __forceinline__ uint4 load16(const uint8_t *p) { return __ldcs(reinterpret_cast<const uint4 *>(p)); }
__device__ __forceinline__ void store16(uint8_t *p, uint4 x) { __stcs(reinterpret_cast<uint4 *>(p), x); }
/* n bytes (a multiple of 16) by a warp, 16 * BATCH per lane on their way */
template <uint32_t BATCH>
__device__ __forceinline__ void warp_copy(uint8_t *to, const uint8_t *from, uint32_t n) {
    const uint32_t lane = threadIdx.x & 31u;
    for (uint32_t at = lane * 16u; at < n; at += 512u * BATCH) {
        uint4 x[BATCH];
#pragma unroll
        for (uint32_t i = 0; i < BATCH; i++)
            if (at + i * 512u < n) x[i] = load16(from + at + i * 512u);
#pragma unroll
        for (uint32_t i = 0; i < BATCH; i++)
            if (at + i * 512u < n) store16(to + at + i * 512u, x[i]);
    }
}

struct ForkParams {
    uint8_t *mem;
    uint64_t layer_bytes;        /* of all pages */
    uint32_t n_layers, n_kvh, tile_bytes, tiles;   /* tiles: of a page and kv head */
    uint32_t n_req, n_fork, table_stride, page_shift, n_pages;
    const int32_t *src, *dst, *len;
    int32_t *rows, *table, *free_list, *n_free, *shares;
    uint32_t *err;
};

/*
 * Fork.  Every block forms the sums over all forks itself, as plan does, and looks up the pages that are copied; then the table entries of whole pages are shared out
 * by threads, the tiles to copy (fork, layer, kv head, 16 rows) by warps.  The last block to finish writes what the others have read: the
 * stack's top and the children's rows.  Under the profiler 256 forks with 104 MB to copy, most of it out of and into L2, take 25 us, four of
 * one prompt 9: sums, look-ups that follow one another and a fence, where the bytes are worth nothing.
 */
constexpr uint32_t NOT_SERVED = 0xffffffffu, NO_PAGE = 0xfffffffeu;
__global__ void __launch_bounds__(PLAN_THREADS) q4_pg_fork_k(const ForkParams P) {
    extern __shared__ uint32_t s_fork[];
    __shared__ uint32_t s_entries, s_tiles, s_pages, s_last;
    /* of places: the fork that fills each; of forks: entries and tiles up to and with each; source and place; the page that is copied and the one that it is copied to */
    uint32_t *owner = s_fork, *entry_end = owner + P.n_req, *tile_end = entry_end + P.n_fork, *places = tile_end + P.n_fork, *old_page = places + P.n_fork, *new_page = old_page + P.n_fork;
    const uint32_t tid = threadIdx.x, mask = (1u << P.page_shift) - 1u;
    const uint64_t room = (uint64_t)P.table_stride << P.page_shift;
    for (uint32_t r = tid; r < P.n_req; r += PLAN_THREADS) owner[r] = 0xffffffffu;
    if (tid == 0) s_entries = s_tiles = s_pages = s_last = 0;
    __syncthreads();
    q4d_pdl_wait();
    const int32_t top = __ldcg(P.n_free);
    const uint32_t per = (P.n_fork + PLAN_THREADS - 1u) / PLAN_THREADS, i0 = min(tid * per, P.n_fork), i1 = min(i0 + per, P.n_fork);
    for (uint32_t i = i0; i < i1; i++) {   /* a place is the first fork's that names it */
        const uint32_t s = (uint32_t)__ldcg(P.src + i), d = (uint32_t)__ldcg(P.dst + i);
        places[i] = s < P.n_req && d < P.n_req ? s | d << 16 : NOT_SERVED;   /* up to 8192 of them */
        if (d < P.n_req) atomicMin(owner + d, i);
    }
    const uint64_t n_free = top < 0 ? 0u : min((uint32_t)top, P.n_pages);
    __syncthreads();
    bool any_bad = false;
    uint64_t e_sum = 0, tp_sum = 0, e_all, tp_all;   /* tp: tiles, and above them pages */
    auto one = [&](uint32_t i, uint64_t &e, uint64_t &tp) {
        e = entry_end[i];
        tp = tile_end[i];
        if (tp) tp |= 1ull << 32;
    };
    for (uint32_t i = i0; i < i1; i++) {
        const uint32_t where = places[i], s = where & 0xffffu, d = where >> 16;
        bool good = where != NOT_SERVED && owner[d] == i;
        const int32_t n = good ? __ldcg(P.len + i) : 0, held = good ? __ldcg(P.rows + s) : 0;
        good = good && n >= 0 && n <= max(held, 0) && (uint64_t)max(held, 0) <= room && __ldcg(P.rows + d) <= 0;
        any_bad |= !good;
        places[i] = good ? where : NOT_SERVED;
        entry_end[i] = good ? (uint32_t)n >> P.page_shift : 0u;
        tile_end[i] = good ? (((uint32_t)n & mask) + 15u) >> 4 : 0u;
        old_page[i] = (uint32_t)n;   /* the thread's own until below */
        uint64_t e, tp;
        one(i, e, tp);
        e_sum += e; tp_sum += tp;
    }
    block_scan2(e_sum, tp_sum, e_all, tp_all);
    uint64_t fit_e = 0, fit_tp = 0;
    uint32_t served = i0;        /* behind the thread's last fork that is */
    bool no_page = false;
    for (uint32_t i = i0; i < i1; i++) {
        uint64_t e, tp;
        one(i, e, tp);
        const uint32_t before = (uint32_t)(tp_sum >> 32);
        e_sum += e; tp_sum += tp;
        const bool fits = (tp_sum >> 32) <= n_free && e_sum < NOT_SERVED;
        if (fits && places[i] != NOT_SERVED) owner[places[i] >> 16] = old_page[i];   /* from now on the rows of the place: P.len may be P.rows */
        old_page[i] = new_page[i] = NO_PAGE;
        if (fits && tp) {
            const uint32_t where = places[i];
            old_page[i] = (uint32_t)P.table[(size_t)(where & 0xffffu) * P.table_stride + e];   /* behind the whole pages */
            new_page[i] = (uint32_t)__ldcg(P.free_list + (n_free - 1u - before));
        }
        if (fits) { fit_e = e_sum; fit_tp = tp_sum; served = i + 1u; }
        else places[i] = NOT_SERVED;
        entry_end[i] = fits ? (uint32_t)e_sum : NOT_SERVED;
        tile_end[i] = fits ? (uint32_t)tp_sum : NOT_SERVED;
    }
    __syncthreads();
    if (served > i0 && (served == P.n_fork || entry_end[served] == NOT_SERVED)) {   /* the last one that is served */
        s_entries = (uint32_t)fit_e;
        s_tiles = (uint32_t)fit_tp;
        s_pages = (uint32_t)(fit_tp >> 32);
    }
    __syncthreads();
    const uint32_t entries = s_entries, tiles = s_tiles, pages = s_pages;
    if (blockIdx.x == 0) {
        if (any_bad) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        if (tid == 0 && ((tp_all >> 32) > pages || e_all > entries)) atomicOr(P.err, (uint32_t)Q4E_SCRATCH);
        for (uint32_t i = tid; i < P.n_fork; i += PLAN_THREADS)   /* the entry of the page that was copied */
            if (places[i] != NOT_SERVED && new_page[i] != NO_PAGE) P.table[(size_t)(places[i] >> 16) * P.table_stride + (entry_end[i] - (i ? entry_end[i - 1u] : 0u))] = (int32_t)new_page[i];
    }
    /* a unit is a tile of all kv heads; of one where there are warps for that (one long prompt's four beams: 2 us less a call) */
    const uint32_t warps = gridDim.x * (PLAN_THREADS / 32u), at_once = (uint64_t)tiles * P.n_layers * P.n_kvh <= warps ? 1u : P.n_kvh, parts = P.n_kvh / at_once, units = tiles * P.n_layers * parts;
    const uint64_t page_bytes = (uint64_t)P.n_kvh * P.tiles * P.tile_bytes;
    for (uint32_t u = blockIdx.x + (tid >> 5) * gridDim.x; u < units; u += warps) {   /* neighbours on different SMs */
        const uint32_t lk = u / tiles, x = u - lk * tiles, layer = lk / parts, kh0 = lk - layer * parts, i = first_above(tile_end, P.n_fork, x), tile = x - (i ? tile_end[i - 1u] : 0u), from = old_page[i], to = new_page[i];
        if (from >= P.n_pages || to >= P.n_pages) {
            no_page = true;
            continue;
        }
        uint8_t *at = P.mem + layer * P.layer_bytes + (uint64_t)(kh0 * P.tiles + tile) * P.tile_bytes;
        const uint8_t *old = at + from * page_bytes;
        at += to * page_bytes;
        for (uint32_t k = 0; k < at_once; k++, at += P.tiles * P.tile_bytes, old += P.tiles * P.tile_bytes) warp_copy<9>(at, old, P.tile_bytes);   /* a tile of q8_0 rows of 128 dims at once */
    }
    for (uint64_t x = (uint64_t)blockIdx.x * PLAN_THREADS + tid; x < entries; x += (uint64_t)gridDim.x * PLAN_THREADS) {
        const uint32_t i = first_above(entry_end, P.n_fork, (uint32_t)x), col = (uint32_t)x - (i ? entry_end[i - 1u] : 0u), where = places[i];
        const int32_t page = P.table[(size_t)(where & 0xffffu) * P.table_stride + col];
        P.table[(size_t)(where >> 16) * P.table_stride + col] = page;
        if ((uint32_t)page < P.n_pages) atomicAdd(P.shares + page, 1);
        else no_page = true;
    }
    if (no_page) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    bool no;
    if (last_arrives(&g_fork_arrived, false, no)) {
        *P.n_free = (int32_t)(n_free - pages);
        s_last = 1u;
    }
    __syncthreads();
    if (s_last)
        for (uint32_t i = tid; i < P.n_fork; i += PLAN_THREADS)
            if (places[i] != NOT_SERVED) P.rows[places[i] >> 16] = (int32_t)owner[places[i] >> 16];
}

struct ReleaseParams {
    int32_t *rows;
    const int32_t *keep, *table;
    uint32_t n_req, table_stride, page_shift, n_pages;
    int32_t *free_list, *n_free, *shares;
    uint32_t *err;
};
constexpr uint32_t REL_MAX_BLOCKS = 1024, REL_PROBES = 1u << 22;
static_assert(REL_MAX_BLOCKS * 2u < MEET_BAD, "arrivals stay below the flags");
__device__ uint32_t g_rel_count[REL_MAX_BLOCKS];   /* of a call's blocks: pages that go back */
__device__ uint32_t g_rel_meet;                    /* where they meet; zero between calls */

/* All blocks of the launch (at most one per SM, none of which waits for anything before) have come so many times; bounded by 2 s.  What they go by: the word, with bad said by any
 * thread.  The same for all of a block's threads, and behind the second meeting meet_good is the same for all blocks */
__device__ __forceinline__ uint32_t rel_meet(uint32_t times, bool bad, uint32_t *err) {
    __shared__ uint32_t s_word;
    const bool any = __syncthreads_or(bad);
    if (gridDim.x == 1u) return times * MEET_HERE | (any ? MEET_BAD : 0u);
    if (threadIdx.x == 0) {
        __threadfence();
        if (any) atomicOr(&g_rel_meet, MEET_BAD);
        atomicAdd(&g_rel_meet, MEET_HERE);
        uint32_t word = 0;
        unsigned long long t0, t1;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
        const bool over = pg_within(REL_PROBES, [&]() {
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(word) : "l"(&g_rel_meet) : "memory");
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
            return meet_over(word, gridDim.x, times) || t1 - t0 > 2000000000ull;
        });
        if (!over || !meet_over(word, gridDim.x, times))
            pg_within(4u * REL_MAX_BLOCKS, [&]() {   /* whoever is in between has come, found something bad or given up: three times a block at most */
                const uint32_t late = meet_given_up(word, gridDim.x, times), seen = late == word ? word : atomicCAS(&g_rel_meet, word, late);
                const bool done = seen == word;
                if (done && late != word) atomicOr(err, (uint32_t)Q4E_CUDA);
                word = done ? late : seen;
                return done || (word & MEET_LATE);
            });
        __threadfence();
        s_word = word;
    }
    __syncthreads();
    return s_word;
}

/*
 * Release.  The entries that requests give up are numbered in the requests' order, a block has an equal part of them.  A page goes back with the last of its
 * entries, if there are as many as it has holders: first every page's entries are counted and the largest number kept, then the blocks
 * count the pages that go back, then they put them on the stack; between these they meet.  Which entry is a page's last does not depend on the
 * order of the atomics.  Bound by those trips to L2.  (Under the profiler 7 us for four beams, 11 to 12 for 256 answers;
 * as three launches 14 and 21.)
 */
__global__ void __launch_bounds__(PLAN_THREADS) q4_pg_release_k(const ReleaseParams P) {
    extern __shared__ uint32_t s_rel[];
    __shared__ uint32_t s_count, s_before, s_all, s_warp[PLAN_THREADS / 32u], s_last;
    /* of requests: entries up to and with each, the column of the first, rows afterwards */
    uint32_t *ends = s_rel, *first = ends + P.n_req;
    int32_t *rows_after = (int32_t *)(first + P.n_req);
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, mask = (1u << P.page_shift) - 1u;
    const uint64_t room = (uint64_t)P.table_stride << P.page_shift;
    if (tid == 0) s_count = s_before = s_all = s_last = 0;
    q4d_pdl_wait();
    const int32_t top = __ldcg(P.n_free);
    const uint32_t per = (P.n_req + PLAN_THREADS - 1u) / PLAN_THREADS, r0 = min(tid * per, P.n_req), r1 = min(r0 + per, P.n_req);
    uint64_t sum = 0, all_entries, none = 0, none_all;
    bool any_bad = false;
    for (uint32_t r = r0; r < r1; r++) {
        const int32_t h = __ldcg(P.rows + r), k = max(__ldcg(P.keep + r), 0);
        bool bad = h > 0 && (uint64_t)h > room, gives = !bad && h > 0 && k < h;
        if (gives && ((uint32_t)k & mask)) {   /* its next rows go where others' may be */
            const int32_t page = P.table[(size_t)r * P.table_stride + ((uint32_t)k >> P.page_shift)];
            bad = (uint32_t)page < P.n_pages && __ldcg(P.shares + page) > 0;
            gives = !bad;
        }
        first[r] = ((uint32_t)k + mask) >> P.page_shift;
        ends[r] = gives ? (((uint32_t)h + mask) >> P.page_shift) - first[r] : 0u;
        rows_after[r] = gives ? k : h;
        sum += ends[r];
        any_bad |= bad;
    }
    block_scan2(sum, none, all_entries, none_all);
    const bool too_many = all_entries > 0x7fffffffu;
    for (uint32_t r = r0; r < r1; r++) {
        sum += ends[r];
        ends[r] = too_many ? 0u : (uint32_t)sum;
    }
    if (blockIdx.x == 0 && any_bad) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    __syncthreads();
    const uint32_t total = too_many ? 0u : (uint32_t)all_entries, share = (total + gridDim.x - 1u) / gridDim.x;
    const uint64_t x0 = (uint64_t)blockIdx.x * share, x1 = min(x0 + share, (uint64_t)total);
    int32_t *times = P.shares + P.n_pages, *last = times + P.n_pages;
    auto page_of = [&](uint32_t x) -> uint32_t {
        const uint32_t r = first_above(ends, P.n_req, x);
        return (uint32_t)P.table[(size_t)r * P.table_stride + first[r] + (x - (r ? ends[r - 1u] : 0u))];
    };
    /* the thread's first entry is looked up once */
    const uint32_t page0 = x0 + tid < x1 ? page_of((uint32_t)(x0 + tid)) : NO_PAGE;
    bool bad = too_many;
    for (uint64_t x = x0 + tid; x < x1; x += PLAN_THREADS) {
        const uint32_t page = x == x0 + tid ? page0 : page_of((uint32_t)x);
        if (page < P.n_pages) {
            atomicAdd(times + page, 1);
            atomicMax(last + page, (int32_t)x + 1);
        } else {
            bad = true;          /* an entry that is no page */
        }
    }
    rel_meet(1u, bad, P.err);

    uint32_t n = 0;
    bool mine0 = false;
    int32_t held0 = 0, given0 = 0;
    for (uint64_t x = x0 + tid; x < x1; x += PLAN_THREADS) {
        const bool is0 = x == x0 + tid;
        const uint32_t page = is0 ? page0 : page_of((uint32_t)x);
        if (page >= P.n_pages) continue;
        const int32_t held = __ldcg(P.shares + page) + 1, given = __ldcg(times + page);
        const bool mine = __ldcg(last + page) == (int32_t)x + 1;
        if (is0) { mine0 = mine; held0 = held; given0 = given; }
        n += mine && given == held;
        bad |= mine && given > held;
    }
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0u && n) atomicAdd(&s_count, n);
    __syncthreads();
    if (tid == 0) __stcg(g_rel_count + blockIdx.x, s_count);
    const bool stays = !meet_good(rel_meet(2u, bad, P.err), gridDim.x);

    for (uint32_t b = tid; b < gridDim.x; b += PLAN_THREADS) {
        const uint32_t k = __ldcg(g_rel_count + b);
        if (k) atomicAdd(&s_all, k);
        if (k && b < blockIdx.x) atomicAdd(&s_before, k);
    }
    const uint64_t n_free = top < 0 ? 0u : (uint32_t)top;
    __syncthreads();
    const uint32_t all = s_all;
    const bool good = !stays && n_free + all <= P.n_pages;
    uint32_t before = s_before;
    for (uint64_t x = x0; x < x1; x += PLAN_THREADS) {   /* the block stays together */
        uint32_t page = NO_PAGE;
        bool goes = false;
        if (x + tid < x1) {
            page = x == x0 ? page0 : page_of((uint32_t)(x + tid));
            if (page < P.n_pages) {
                bool mine = mine0;
                int32_t held = held0, given = given0;
                if (x != x0) {
                    mine = __ldcg(last + page) == (int32_t)(x + tid) + 1;
                    held = __ldcg(P.shares + page) + 1;
                    given = __ldcg(times + page);
                }
                if (!good) {
                    times[page] = last[page] = 0;
                } else if (mine) {
                    goes = given == held;
                    P.shares[page] = goes ? 0 : held - given - 1;
                    times[page] = last[page] = 0;   /* the others of its entries find that they are not the last, whichever value they read */
                }
            }
        }
        const uint32_t votes = __ballot_sync(0xffffffffu, goes);
        if (lane == 0) s_warp[warp] = __popc(votes);
        __syncthreads();
        uint32_t at = before;
        for (uint32_t w = 0; w < PLAN_THREADS / 32u; w++) {
            if (w < warp) at += s_warp[w];
            before += s_warp[w];
        }
        if (goes) P.free_list[n_free + all - 1u - (at + __popc(votes & ((1u << lane) - 1u)))] = (int32_t)page;
        __syncthreads();
    }
    bool no;
    if (last_arrives(&g_rel_arrived, !good, no)) {
        if (no) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        else *P.n_free = (int32_t)(n_free + all);
        g_rel_meet = 0u;
        s_last = no ? 0u : 1u;
    }
    __syncthreads();
    if (s_last)
        for (uint32_t r = tid; r < P.n_req; r += PLAN_THREADS) P.rows[r] = rows_after[r];
}

struct CompactParams {
    uint8_t *mem;
    uint64_t layer_bytes, page_bytes;
    uint32_t n_layers, n_req, table_stride, page_shift, n_pages;
    const int32_t *rows;
    int32_t *table, *free_list, *n_free, *shares, *map;
    int32_t *hole;               /* pages to fill, and behind as many of them as there are pages in use those to move, in ascending order */
    uint32_t *err;
};
constexpr uint32_t CMP_THREADS = 1024, CMP_WORDS = 40960;   /* 160 KB: 1.3 M pages at once */
__device__ uint32_t g_cmp_moves, g_cmp_good;

/*
 * Compact.  Which pages go where follows from the stack alone: one block marks the free pages as bits in shared memory and counts them off
 * (65 536 pages: 8 KB of bits; larger pools in windows).  Then all copy: 4096 pages, 1013 of 417 KB to move, 7 and 140 us, 92 % of a copy's rate.
 */
__global__ void __launch_bounds__(CMP_THREADS) q4_pg_cmp_plan_k(const CompactParams P) {
    extern __shared__ uint32_t s_bits[];
    __shared__ uint32_t s_hole[32], s_move[32];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    q4d_pdl_wait();
    const int32_t top = *P.n_free;
    const bool fits = top >= 0 && (uint32_t)top <= P.n_pages;
    const uint32_t n_free = fits ? (uint32_t)top : 0u, live = P.n_pages - n_free;
    int32_t *const moving = P.hole + live;
    bool bad = !fits;
    uint32_t n_hole = 0, n_move = 0;
    for (uint32_t w0 = 0; w0 < P.n_pages; w0 += CMP_WORDS * 32u) {   /* below 2^31 - 2^21: no wrap */
        const uint32_t pages = min(P.n_pages - w0, CMP_WORDS * 32u), words = (pages + 31u) / 32u;
        for (uint32_t w = tid; w < words; w += CMP_THREADS) s_bits[w] = 0u;
        __syncthreads();
        for (uint32_t i = tid; i < n_free; i += CMP_THREADS) {
            const uint32_t p = (uint32_t)__ldcg(P.free_list + i);
            if (p >= P.n_pages) bad = true;
            else if (p - w0 < pages) bad |= (atomicOr(s_bits + ((p - w0) >> 5), 1u << (p & 31u)) >> (p & 31u)) & 1u;
        }
        __syncthreads();
        const uint32_t per = (words + CMP_THREADS - 1u) / CMP_THREADS, a = min(tid * per, words), b = min(a + per, words);
        auto of = [&](uint32_t w, uint32_t &hole, uint32_t &move) {
            const uint32_t p = w0 + w * 32u, bits = s_bits[w];
            const uint32_t there = P.n_pages - p >= 32u ? 0xffffffffu : (1u << (P.n_pages - p)) - 1u;
            const uint32_t low = p >= live ? 0u : live - p >= 32u ? 0xffffffffu : (1u << (live - p)) - 1u;
            hole = bits & low;
            move = ~bits & ~low & there;
        };
        uint32_t h = 0, m = 0, hole, move;
        for (uint32_t w = a; w < b; w++) {
            of(w, hole, move);
            h += __popc(hole);
            m += __popc(move);
        }
        uint32_t hs = h, ms = m;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, hs, d), y = __shfl_up_sync(0xffffffffu, ms, d);
            if (lane >= (uint32_t)d) { hs += x; ms += y; }
        }
        if (lane == 31u) { s_hole[warp] = hs; s_move[warp] = ms; }
        __syncthreads();
        uint32_t hb = n_hole + hs - h, mb = n_move + ms - m;
        for (uint32_t w = 0; w < 32u; w++) {
            if (w < warp) { hb += s_hole[w]; mb += s_move[w]; }
            n_hole += s_hole[w]; n_move += s_move[w];
        }
        for (uint32_t w = a; w < b; w++) {
            of(w, hole, move);
            for (; hole; hole &= hole - 1u) P.hole[hb++] = (int32_t)(w0 + w * 32u + (uint32_t)__ffs((int)hole) - 1u);
            for (; move; move &= move - 1u) moving[mb++] = (int32_t)(w0 + w * 32u + (uint32_t)__ffs((int)move) - 1u);
        }
        for (uint32_t i = tid; i < pages; i += CMP_THREADS) P.map[w0 + i] = (s_bits[i >> 5] >> (i & 31u)) & 1u ? -1 : (int32_t)(w0 + i);
        __syncthreads();
    }
    const bool good = !__syncthreads_or(bad) && n_hole == n_move;
    if (good)
        for (uint32_t k = tid; k < n_move; k += CMP_THREADS) P.map[moving[k]] = P.hole[k];
    else
        for (uint32_t p = tid; p < P.n_pages; p += CMP_THREADS) P.map[p] = (int32_t)p;
    if (tid == 0) {
        g_cmp_moves = good ? n_move : 0u;
        g_cmp_good = good;
        if (!good) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    }
}
constexpr uint32_t CMP_UNIT = 4096;   /* bytes that a warp moves at once */
__global__ void __launch_bounds__(PLAN_THREADS) q4_pg_cmp_move_k(const CompactParams P) {
    const uint32_t tid = threadIdx.x, threads = gridDim.x * PLAN_THREADS, me = blockIdx.x * PLAN_THREADS + tid;
    q4d_pdl_wait();
    if (!__ldcg(&g_cmp_good)) return;
    const uint32_t n_move = __ldcg(&g_cmp_moves), n_free = (uint32_t)__ldcg(P.n_free);
    const int32_t *const moving = P.hole + (P.n_pages - n_free);
    for (uint32_t i = me; i < n_free; i += threads) P.free_list[i] = (int32_t)(P.n_pages - 1u - i);
    if (P.shares)
        for (uint32_t k = me; k < n_move; k += threads) {
            const int32_t from = __ldcg(moving + k);
            P.shares[__ldcg(P.hole + k)] = P.shares[from];
            P.shares[from] = 0;
        }
    bool bad = false;
    for (uint32_t r = blockIdx.x; r < P.n_req; r += gridDim.x) {
        const int32_t h = __ldcg(P.rows + r);
        uint64_t n = h > 0 ? ((uint64_t)(uint32_t)h + (1u << P.page_shift) - 1u) >> P.page_shift : 0u;
        if (n > P.table_stride) { n = P.table_stride; bad = true; }
        for (uint32_t c = tid; c < n; c += PLAN_THREADS) {
            int32_t *entry = P.table + (size_t)r * P.table_stride + c;
            const uint32_t page = (uint32_t)*entry;
            const int32_t to = page < P.n_pages ? __ldcg(P.map + page) : -1;
            if (to < 0) bad = true;
            else if ((uint32_t)to != page) *entry = to;
        }
    }
    if (bad) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    const uint32_t parts = (uint32_t)((P.page_bytes + CMP_UNIT - 1u) / CMP_UNIT);
    const uint64_t units = (uint64_t)n_move * P.n_layers * parts;
    for (uint64_t u = me >> 5; u < units; u += threads >> 5) {
        const uint64_t pl = u / parts;
        const uint32_t at = (uint32_t)(u - pl * parts) * CMP_UNIT, k = (uint32_t)(pl / P.n_layers), layer = (uint32_t)(pl - (uint64_t)k * P.n_layers);
        uint8_t *base = P.mem + layer * P.layer_bytes + at;
        warp_copy<8>(base + (uint32_t)__ldcg(P.hole + k) * P.page_bytes, base + (uint32_t)__ldcg(moving + k) * P.page_bytes, (uint32_t)min((uint64_t)CMP_UNIT, P.page_bytes - at));
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0u; }
uint64_t page_bytes_of(const q4_gpu_pages *pg) { return (uint64_t)q4i_pages_row_bytes(pg->hd, pg->kind) * pg->page_rows * pg->n_kvh; }
/* blocks for so many items of a thread each, one per SM at most */
uint32_t blocks_for(uint64_t items) {
    const uint64_t want = (items + PLAN_THREADS - 1u) / PLAN_THREADS, cap = (uint64_t)g_q4.sm_count;
    return (uint32_t)(want < 1u ? 1u : want < cap ? want : cap);
}

}  // namespace

extern "C" bool q4_gpu_pages_fork(const q4_gpu_pages *pg, int32_t *shares, int32_t *rows, uint32_t n_req, const int32_t *src, const int32_t *dst, const int32_t *len,
                                  uint32_t n_fork, int32_t *table, uint32_t table_stride) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "pages_fork: library not initialised");
    Q4_REQUIRE(q4i_pages_ok(pg) && pg->mem && aligned16(pg->mem) && pg->free_list && pg->n_free, "pages_fork: bad pool");
    Q4_REQUIRE(shares && rows && src && dst && len && table && n_req && n_fork && table_stride, "pages_fork: bad argument");
    Q4_REQUIRE(n_req <= PLAN_MAX_REQ && n_fork <= PLAN_MAX_REQ, "pages_fork: at most 8192 requests and forks");
    Q4_REQUIRE((uint64_t)table_stride * pg->page_rows <= 0x7fffffffu, "pages_fork: a block table's rows pass 2^31 - 1");
    Q4_REQUIRE((uint64_t)n_fork * (pg->page_rows / 16u) * pg->n_layers <= 0x7fffffffu, "pages_fork: too many layers for so many forks");
    ForkParams p = {};
    p.mem = (uint8_t *)pg->mem;
    p.layer_bytes = page_bytes_of(pg) * pg->n_pages;
    p.n_layers = pg->n_layers; p.n_kvh = pg->n_kvh;
    p.tile_bytes = 16u * q4i_pages_row_bytes(pg->hd, pg->kind); p.tiles = pg->page_rows / 16u;
    p.n_req = n_req; p.n_fork = n_fork; p.table_stride = table_stride; p.n_pages = pg->n_pages;
    p.page_shift = (uint32_t)__builtin_ctz(pg->page_rows);
    p.src = src; p.dst = dst; p.len = len; p.rows = rows; p.table = table;
    p.free_list = pg->free_list; p.n_free = pg->n_free; p.shares = shares;
    p.err = g_q4.err_d;
    static bool attr = false;
    if (!attr && !q4i_check(cudaFuncSetAttribute(q4_pg_fork_k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(6u * PLAN_MAX_REQ * sizeof(uint32_t))), "pages_fork smem attribute")) return false;
    attr = true;
    /* a warp per tile to copy, or a thread per entry, up to a block per SM: each forms the sums (256 answers there and back 53 us, with one and a half 57, with two 61) */
    const uint64_t tiles = (uint64_t)n_fork * p.tiles * p.n_layers * p.n_kvh, items = tiles * 32u + (uint64_t)n_fork * table_stride, want = (items + PLAN_THREADS - 1u) / PLAN_THREADS, cap = (uint64_t)g_q4.sm_count;
    return q4i_launch_pdl("pages_fork launch", q4_pg_fork_k, dim3((unsigned)(want < cap ? want : cap)), PLAN_THREADS, (n_req + 5u * (size_t)n_fork) * sizeof(uint32_t), p);
}

extern "C" bool q4_gpu_pages_release(const q4_gpu_pages *pg, int32_t *shares, int32_t *rows, const int32_t *keep, uint32_t n_req, const int32_t *table, uint32_t table_stride) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "pages_release: library not initialised");
    Q4_REQUIRE(q4i_pages_ok(pg) && pg->free_list && pg->n_free, "pages_release: bad pool");
    Q4_REQUIRE(shares && rows && keep && table && n_req && table_stride, "pages_release: bad argument");
    Q4_REQUIRE(n_req <= PLAN_MAX_REQ, "pages_release: at most 8192 requests");
    Q4_REQUIRE((uint64_t)table_stride * pg->page_rows <= 0x7fffffffu, "pages_release: a block table's rows pass 2^31 - 1");
    ReleaseParams p = {};
    p.rows = rows; p.keep = keep; p.n_req = n_req; p.table = table; p.table_stride = table_stride; p.n_pages = pg->n_pages;
    p.page_shift = (uint32_t)__builtin_ctz(pg->page_rows);
    p.free_list = pg->free_list; p.n_free = pg->n_free; p.shares = shares;
    p.err = g_q4.err_d;
    const dim3 grid(blocks_for((uint64_t)n_req * table_stride));
    if (grid.x > REL_MAX_BLOCKS) return q4i_fail(Q4E_CUDA, "pages_release: more SMs than the counts are for");
    static bool attr = false;
    if (!attr && !q4i_check(cudaFuncSetAttribute(q4_pg_release_k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(3u * PLAN_MAX_REQ * sizeof(uint32_t))), "pages_release smem attribute")) return false;
    attr = true;
    return q4i_launch_pdl("pages_release launch", q4_pg_release_k, grid, PLAN_THREADS, 3u * n_req * sizeof(uint32_t), p);
}

extern "C" bool q4_gpu_pages_compact(const q4_gpu_pages *pg, int32_t *shares, const int32_t *rows, uint32_t n_req, int32_t *table, uint32_t table_stride, int32_t *map) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "pages_compact: library not initialised");
    Q4_REQUIRE(q4i_pages_ok(pg) && pg->mem && aligned16(pg->mem) && pg->free_list && pg->n_free, "pages_compact: bad pool");
    Q4_REQUIRE(map && (!n_req || (rows && table && table_stride)), "pages_compact: bad argument");
    Q4_REQUIRE((uint64_t)table_stride * pg->page_rows <= 0x7fffffffu, "pages_compact: a block table's rows pass 2^31 - 1");
    if (!q4i_scratch(pg->n_pages, 0)) return false;
    CompactParams p = {};
    p.mem = (uint8_t *)pg->mem;
    p.page_bytes = page_bytes_of(pg);
    p.layer_bytes = p.page_bytes * pg->n_pages;
    p.n_layers = pg->n_layers; p.n_req = n_req; p.table_stride = table_stride; p.n_pages = pg->n_pages;
    p.page_shift = (uint32_t)__builtin_ctz(pg->page_rows);
    p.rows = rows; p.table = table; p.free_list = pg->free_list; p.n_free = pg->n_free; p.shares = shares; p.map = map;
    p.hole = (int32_t *)g_q4.part;
    p.err = g_q4.err_d;
    const uint32_t words = (pg->n_pages + 31u) / 32u;
    static bool attr = false;
    if (!attr && !q4i_check(cudaFuncSetAttribute(q4_pg_cmp_plan_k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(CMP_WORDS * sizeof(uint32_t))), "pages_compact smem attribute")) return false;
    attr = true;
    return q4i_launch_pdl("pages_compact launch", q4_pg_cmp_plan_k, dim3(1), CMP_THREADS, (words < CMP_WORDS ? words : CMP_WORDS) * sizeof(uint32_t), p) &&
           q4i_launch_pdl("pages_compact launch", q4_pg_cmp_move_k, dim3(2u * (unsigned)g_q4.sm_count), PLAN_THREADS, 0, p);
}
