/* Shared by the kernels that plan over all requests of a call (q4_pages.cu, q4_pages_share.cu; not installed). */
#ifndef Q4_PAGES_SCAN_H
#define Q4_PAGES_SCAN_H

#include "q4_internal.h"

constexpr uint32_t PLAN_THREADS = 512, PLAN_MAX_REQ = 8192;

/* The word at which the blocks of a launch meet twice: in its lower half the arrivals, above them whether a block found that nothing may come of the call, and whether
 * one gave up waiting.  That it does only while not all have come, in one step with looking.  So a word in which all have come twice does not
 * change any more, one that somebody gave up never becomes good, and all blocks decide alike whenever they look. */
constexpr uint32_t MEET_HERE = 1u, MEET_BAD = 1u << 16, MEET_LATE = 1u << 17;   /* up to 32767 blocks */
__host__ __device__ inline bool meet_came(uint32_t word, uint32_t blocks, uint32_t times) { return (word & (MEET_BAD - 1u)) >= times * blocks; }
__host__ __device__ inline bool meet_over(uint32_t word, uint32_t blocks, uint32_t times) { return meet_came(word, blocks, times) || (word & MEET_LATE); }
__host__ __device__ inline uint32_t meet_given_up(uint32_t word, uint32_t blocks, uint32_t times) { return meet_came(word, blocks, times) ? word : word | MEET_LATE; }
__host__ __device__ inline bool meet_good(uint32_t word, uint32_t blocks) { return meet_came(word, blocks, 2u) && !(word & (MEET_BAD | MEET_LATE)); }

#ifdef __CUDACC__
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

/* Counts a block that has finished with the stack; for thread 0 of the last one true, with `no` whether a thread of any block wants it left alone.
 * arrived: blocks in its lower half, those in its upper; zero between launches */
__device__ __forceinline__ bool last_arrives(uint32_t *arrived, bool mine_no, bool &no) {
    const bool stays = __syncthreads_or(mine_no);
    if (threadIdx.x != 0) return false;
    __threadfence();
    const uint32_t mine = stays ? 0x10001u : 1u, all = atomicAdd(arrived, mine) + mine;
    if ((all & 0xffffu) != gridDim.x) return false;
    *arrived = 0u;
    __threadfence();
    no = all >> 16;
    return true;
}
/* the last block to finish moves the stack's top, unless a thread of any block says no: all of them have read it by then */
__device__ __forceinline__ void move_top(uint32_t *arrived, int32_t *n_free, int32_t to, uint32_t *err, bool mine_no = false) {
    bool no;
    if (last_arrives(arrived, mine_no, no)) {
        if (no) atomicOr(err, (uint32_t)Q4E_RANGE);
        else *n_free = to;
    }
}
/* of n ascending ends (inclusive), the first above i */
__device__ __forceinline__ uint32_t first_above(const uint32_t *ends, uint32_t n, uint32_t i) {
    uint32_t lo = 0, hi = n - 1u;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (ends[mid] > i) hi = mid;
        else lo = mid + 1u;
    }
    return lo;
}
#endif

#endif
