/* Shared by the two attention kernels over a pool of pages (q4_paged.cu, q4_paged_tc.cu; not installed). */
#ifndef Q4_PAGED_H
#define Q4_PAGED_H

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
    int4 *ends;                  /* [block] {first block of the unit that ends here, or -1; its first token; its tokens; its kv head} */
    uint32_t *err;
};

template <int KIND, int HD>
struct PgTile {
    static constexpr uint32_t ROW = KIND == Q4K_Q8 ? (2u * HD + HD / 8u + 15u) / 16u * 16u : 4u * HD, BYTES = 16u * ROW;
};

/* The tokens of requests that bring more than P.add_split, on the tensor cores (q4_paged_tc.cu): launched with its records in
 * `scratch`, of at least q4i_paged_chunk_floats floats.  hd 64, 128 or 256, kind fp16 or q8_0. */
size_t q4i_paged_chunk_floats(uint32_t hd);
bool q4i_paged_chunk(const PagedParams &p, int kind, uint32_t hd, float *scratch);
/* joins the records that `blocks` blocks left (q4_paged.cu) */
bool q4i_paged_merge(const PagedParams &p, uint32_t hd, uint32_t blocks, uint32_t unit_rows);

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
#endif

#endif
