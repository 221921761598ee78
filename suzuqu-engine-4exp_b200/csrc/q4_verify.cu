/*
 * Drafted tokens held against the target's distributions, and the token behind the last one that is kept.  No counterpart in the reference.
 *
 *     p_i = exp((x_i - M) / T) / S,  S = sum exp((x_i - M) / T),  M the largest logit;  q likewise from the draft's logits
 *     draft d is kept while u q_d < p_d;  next = the first i with sum_{j <= i} w_j > u sum w,  w = max(p - q, 0), or p
 *
 * Two launches.  The first goes once through all rows, a block per row and CHUNK logits, and leaves (M, S) per chunk, relative to the chunk's own
 * largest logit: bound by memory, and by the 64-bit pipe, in which the exponentials and sums are taken (a token's border in the running sum may lie
 * anywhere; with 32 bits a draw over a flat distribution of 10^5 tokens falls on the wrong side once in some thousands).  The second decides per
 * request; the sums of the chunks tell in which one the next token lies, and only that one is looked through.  Where a draft was refused the
 * request's blocks go through that row of p and q once more for max(p - q, 0), and the last of them to finish looks.
 */
#include <math_constants.h>

#include "q4_internal.h"
#include "q4_pages_scan.h"

namespace {

constexpr uint32_t CHUNK = 8192, VF_THREADS = 256, EACH = CHUNK / VF_THREADS;

struct VfStat { double s; float m; int32_t at; };   /* of a chunk: sum relative to the largest logit, that logit (NaN or +inf: the row is no distribution), its first place (greedy) */

struct VerifyParams {
    const void *logits, *draft;
    int bf16;
    uint64_t ld, draft_ld;
    uint32_t vocab, chunks, n_req, n_tok;
    const int32_t *token, *start;
    const float *temp, *u_accept, *u_next;
    int32_t *accepted, *next;
    float *logp;
    const int32_t *rows;
    int32_t *keep;
    VfStat *stat;                /* [target's rows, draft's rows][chunk] */
    double *rest;                /* [request][chunk]: sums of max(p - q, 0) */
    uint32_t *err;
};
__device__ uint32_t g_vf_arrived[PLAN_MAX_REQ];   /* zero between launches */

__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
template <bool BF16>
__device__ __forceinline__ float logit(const void *row, uint64_t at) {
    if constexpr (BF16) return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(row) + at) << 16);
    else return __ldcg(reinterpret_cast<const float *>(row) + at);
}
/* the request of token t: the last one that begins at or before it; by a whole warp */
__device__ __forceinline__ uint32_t request_of(const int32_t *start, uint32_t n_req, uint32_t t) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t lo = 0, n = n_req;
    while (n > 1u) {
        const uint32_t step = (n + 31u) / 32u, i = lane * step;
        const uint32_t below = __ballot_sync(0xffffffffu, i < n && __ldcg(start + lo + i) <= (int32_t)t);
        const uint32_t last = below ? 31u - (uint32_t)__clz((int)below) : 0u;
        n = min(step, n - last * step);
        lo += last * step;
    }
    return lo;
}
__device__ __forceinline__ float temperature(const VerifyParams &P, uint32_t r) { return P.temp ? __ldcg(P.temp + r) : 1.f; }
__device__ __forceinline__ bool temperature_ok(float t) { return t >= 0.f && t <= 3.402823466e38f; }

template <bool BF16>
__global__ void __launch_bounds__(VF_THREADS) q4_vf_stat_k(const VerifyParams P) {
    __shared__ float s_max[VF_THREADS / 32u];
    __shared__ double s_sum[VF_THREADS / 32u];
    __shared__ uint32_t s_at;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    q4d_pdl_wait();
    const uint32_t chunk = blockIdx.x % P.chunks, row = blockIdx.x / P.chunks;
    const bool drafts = row >= P.n_tok;
    const uint32_t t = drafts ? row - P.n_tok : row;
    const uint32_t r = request_of(P.start, P.n_req, t);
    const int32_t a = __ldcg(P.start + r), b = __ldcg(P.start + r + 1u);
    const float T = temperature(P, r);
    if ((int32_t)t < a || (int32_t)t >= b || !temperature_ok(T)) return;
    if (drafts && ((int32_t)t + 1 == b || T == 0.f)) return;
    const uint8_t *base = (const uint8_t *)(drafts ? P.draft : P.logits) + (uint64_t)t * (drafts ? P.draft_ld : P.ld) * (BF16 ? 2u : 4u);
    const uint32_t i0 = chunk * CHUNK, n = min(CHUNK, P.vocab - i0);
    float x[EACH];
    float m = -CUDART_INF_F;
#pragma unroll
    for (uint32_t k = 0; k < EACH; k++) {
        const uint32_t i = k * VF_THREADS + tid;
        x[k] = i < n ? logit<BF16>(base, i0 + i) : -CUDART_INF_F;
        m = max_nan(m, x[k]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s_max[warp] = m;
    if (tid == 0) s_at = 0xffffffffu;
    __syncthreads();
    m = s_max[0];
#pragma unroll
    for (uint32_t w = 1; w < VF_THREADS / 32u; w++) m = max_nan(m, s_max[w]);
    VfStat *out = P.stat + (uint64_t)row * P.chunks + chunk;
    if (T == 0.f) {
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (uint32_t k = 0; k < EACH; k++)
            if (x[k] == m) at = min(at, k * VF_THREADS + tid);
        if (at < n) atomicMin(&s_at, at);
        __syncthreads();
        if (tid == 0) *out = {1.0, m, (int32_t)(i0 + s_at)};
        return;
    }
    double s = 0.0;
    if (fabsf(m) <= 3.402823466e38f) {
        const double inv = 1.0 / (double)T;
#pragma unroll
        for (uint32_t k = 0; k < EACH; k++) s += exp(((double)x[k] - (double)m) * inv);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) s_sum[warp] = s;
    __syncthreads();
    if (tid == 0) {
        for (uint32_t w = 1; w < VF_THREADS / 32u; w++) s += s_sum[w];
        *out = {s, m, 0};
    }
}

/* a row's M and S from its chunks', by a whole warp; false: no distribution */
struct Row { double m, s; };
__device__ __forceinline__ bool row_of(const VfStat *stat, uint32_t chunks, double inv, Row &R) {
    const uint32_t lane = threadIdx.x & 31u;
    float m = -CUDART_INF_F;
    for (uint32_t c = lane; c < chunks; c += 32u) m = max_nan(m, __ldcg(&stat[c].m));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    R.m = m;
    R.s = 0.0;
    if (!(fabsf(m) <= 3.402823466e38f)) return false;
    for (uint32_t c = lane; c < chunks; c += 32u) {
        const double s = __ldcg(&stat[c].s);
        if (s > 0.0) R.s += s * exp(((double)__ldcg(&stat[c].m) - R.m) * inv);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) R.s += __shfl_xor_sync(0xffffffffu, R.s, o);
    return true;
}
/* the row's largest logit and its first place, by a whole warp */
__device__ __forceinline__ bool best_of(const VfStat *stat, uint32_t chunks, int32_t &at) {
    const uint32_t lane = threadIdx.x & 31u;
    float m = -CUDART_INF_F;
    for (uint32_t c = lane; c < chunks; c += 32u) m = max_nan(m, __ldcg(&stat[c].m));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    at = 0x7fffffff;
    for (uint32_t c = lane; c < chunks; c += 32u)
        if (__ldcg(&stat[c].m) == m) at = min(at, __ldcg(&stat[c].at));
    at = __reduce_min_sync(0xffffffffu, at);
    return fabsf(m) <= 3.402823466e38f;
}

/* what a request's blocks agree on */
struct Decision {
    Row p, q;
    double inv;
    uint32_t stop;               /* the row that decides next */
    int32_t refused;             /* the draft there, if one was refused */
    int32_t best;                /* greedy: next */
    bool ok, greedy;
};

template <bool BF16>
__global__ void __launch_bounds__(VF_THREADS) q4_vf_pick_k(const VerifyParams P) {
    constexpr uint32_t WARPS = VF_THREADS / 32u;
    __shared__ Decision s_d;
    __shared__ uint32_t s_kept[WARPS];    /* 0: refused, 1: kept, 2: no distribution */
    __shared__ double s_scan[WARPS];
    __shared__ int32_t s_best[WARPS];
    __shared__ uint32_t s_chunk, s_found, s_last, s_over;
    __shared__ double s_left;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, chunk = blockIdx.x, r = blockIdx.y;
    const bool first = chunk == 0u;
    q4d_pdl_wait();
    const int32_t a = __ldcg(P.start + r), b = __ldcg(P.start + r + 1u);
    const bool bounds = a >= 0 && b >= a && (uint32_t)b <= P.n_tok;
    if (!bounds || a == b) {
        if (first && tid == 0) {
            P.accepted[r] = 0;
            P.next[r] = -1;
            if (P.keep) P.keep[r] = __ldcg(P.rows + r);
            if (!bounds) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        }
        return;
    }
    const float T = temperature(P, r);
    const bool greedy = T == 0.f;
    const double inv = greedy ? 1.0 : 1.0 / (double)T;
    const VfStat *stat_p = P.stat, *stat_q = P.stat + (uint64_t)P.n_tok * P.chunks;
    auto p_row = [&](uint32_t t) -> const uint8_t * { return (const uint8_t *)P.logits + (uint64_t)t * P.ld * (BF16 ? 2u : 4u); };
    auto q_row = [&](uint32_t t) -> const uint8_t * { return (const uint8_t *)P.draft + (uint64_t)t * P.draft_ld * (BF16 ? 2u : 4u); };
    auto log_p = [&](uint32_t t, const Row &R, int32_t i) -> float { return (float)(((double)logit<BF16>(p_row(t), (uint32_t)i) - R.m) * inv - log(R.s)); };

    /* ---- the drafts, a warp each, eight at a time */
    uint32_t stop = (uint32_t)b - 1u;
    bool ok = temperature_ok(T), out_of_vocab = false;
    if (!ok) stop = (uint32_t)a;
    for (uint32_t t0 = (uint32_t)a; ok && t0 < (uint32_t)b - 1u; t0 += WARPS) {
        const uint32_t t = t0 + warp;
        uint32_t kept = 1u;
        float lp = 0.f;
        if (t < (uint32_t)b - 1u) {
            const int32_t d = __ldcg(P.token + t + 1u);
            const bool in = (uint32_t)d < P.vocab;
            Row p, q;
            if (greedy) {
                int32_t best;
                kept = best_of(stat_p + (uint64_t)t * P.chunks, P.chunks, best) ? best == d : 2u;
            } else if (!row_of(stat_p + (uint64_t)t * P.chunks, P.chunks, inv, p) || (P.draft && !row_of(stat_q + (uint64_t)t * P.chunks, P.chunks, inv, q))) {
                kept = 2u;
            } else if (in) {
                const double pd = exp(((double)logit<BF16>(p_row(t), (uint32_t)d) - p.m) * inv) / p.s;
                const double qd = P.draft ? exp(((double)logit<BF16>(q_row(t), (uint32_t)d) - q.m) * inv) / q.s : 1.0;
                kept = (double)__ldcg(P.u_accept + t) * qd < pd;
                if (kept && lane == 0) lp = log_p(t, p, d);
            } else {
                kept = 0u;
            }
            out_of_vocab = !in;
        }
        __syncthreads();
        if (lane == 0) s_kept[warp] = kept;
        __syncthreads();
        uint32_t n = 0;
        while (n < WARPS && s_kept[n] == 1u) n++;
        if (first && lane == 0 && t < (uint32_t)b - 1u) {
            if (P.logp && warp < n) P.logp[t] = lp;
            if (out_of_vocab && warp <= n) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        }
        if (n < WARPS) {
            stop = t0 + n;
            ok = s_kept[n] != 2u;
            break;
        }
    }
    if (first && P.logp)
        for (uint32_t t = stop + 1u + tid; t < (uint32_t)b; t += VF_THREADS) P.logp[t] = 0.f;
    /* ---- the row that decides */
    const bool some_refused = ok && stop + 1u < (uint32_t)b;
    __syncthreads();
    if (warp == 0) {
        Decision D = {};
        D.inv = inv; D.stop = stop; D.greedy = greedy; D.ok = ok;
        if (some_refused) D.refused = __ldcg(P.token + stop + 1u);
        if (ok && greedy) D.ok = best_of(stat_p + (uint64_t)stop * P.chunks, P.chunks, D.best);
        if (ok && !greedy) {
            D.ok = row_of(stat_p + (uint64_t)stop * P.chunks, P.chunks, inv, D.p);
            if (some_refused && P.draft) D.ok = row_of(stat_q + (uint64_t)stop * P.chunks, P.chunks, inv, D.q) && D.ok;
        }
        if (lane == 0) s_d = D;
    }
    if (tid == 0) s_last = s_found = 0u;
    __syncthreads();
    const Decision D = s_d;
    const bool was_refused = some_refused && D.ok && !D.greedy;
    const bool with_q = was_refused && P.draft != nullptr;
    if (!first && !with_q) return;
    if (first && tid == 0) {
        P.accepted[r] = (int32_t)(stop - (uint32_t)a);
        if (P.keep) P.keep[r] = __ldcg(P.rows + r) + (int32_t)(stop - (uint32_t)a) + 1;
        if (!D.ok || D.greedy) {
            P.next[r] = D.ok ? D.best : -1;
            if (P.logp) P.logp[stop] = 0.f;
            if (!D.ok) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        }
    }
    if (!D.ok || D.greedy) return;

    /* weight of token i: p (without the refused one, where drafts are certain), or what p has over q */
    auto weight = [&](uint32_t i, bool over_q) -> double {
        const double p = exp(((double)logit<BF16>(p_row(stop), i) - D.p.m) * inv) / D.p.s;
        if (over_q) return fmax(p - exp(((double)logit<BF16>(q_row(stop), i) - D.q.m) * inv) / D.q.s, 0.0);
        return was_refused && !P.draft && (int32_t)i == D.refused ? 0.0 : p;
    };
    auto block_sum = [&](double x) -> double {   /* over the block, in every thread */
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        __syncthreads();
        if (lane == 0) s_scan[warp] = x;
        __syncthreads();
        x = s_scan[0];
        for (uint32_t w = 1; w < WARPS; w++) x += s_scan[w];
        return x;
    };
    auto chunk_sum = [&](uint32_t c, bool over_q) -> double {
        const uint32_t i0 = c * CHUNK, n = min(CHUNK, P.vocab - i0);
        double x = 0.0;
        for (uint32_t i = tid; i < n; i += VF_THREADS) x += weight(i0 + i, over_q);
        return block_sum(x);
    };
    double *rest = P.rest + (uint64_t)r * P.chunks;
    bool over_q = with_q;
    if (with_q) {
        const double x = chunk_sum(chunk, true);
        if (tid == 0) {
            __stcg(rest + chunk, x);
            __threadfence();
            s_last = atomicAdd(&g_vf_arrived[r], 1u) == P.chunks - 1u;
            if (s_last) g_vf_arrived[r] = 0u;
            __threadfence();
        }
        __syncthreads();
        if (!s_last) return;
    }
    /* ---- the chunk in which the running sum passes u times the whole, by one warp; then the place in it */
    double special = 0.0;
    const uint32_t special_at = was_refused && !P.draft && (uint32_t)D.refused < P.vocab ? (uint32_t)D.refused / CHUNK : 0xffffffffu;
    if (special_at != 0xffffffffu) special = chunk_sum(special_at, false);
    const VfStat *sp = stat_p + (uint64_t)stop * P.chunks;
    const double u = (double)__ldcg(P.u_next + r);
    auto of_chunk = [&](uint32_t c, bool q) -> double {
        if (q) return __ldcg(rest + c);
        if (c == special_at) return special;
        const double s = __ldcg(&sp[c].s);
        return s > 0.0 ? s * exp(((double)__ldcg(&sp[c].m) - D.p.m) * inv) / D.p.s : 0.0;
    };
    if (tid == 0) {
        double all = 0.0;
        for (uint32_t c = 0; c < P.chunks; c++) all += of_chunk(c, over_q);
        if (over_q && !(all > 0.0)) {   /* p nowhere above q: as if none was refused */
            over_q = false;
            for (uint32_t c = 0; c < P.chunks; c++) all += of_chunk(c, false);
        }
        s_over = over_q;
        const double want = u * all;
        double sum = 0.0;
        uint32_t at = 0xffffffffu, some = 0;
        for (uint32_t c = 0; c < P.chunks; c++) {
            const double x = of_chunk(c, over_q);
            if (x > 0.0) some = c;
            if (sum + x > want) { at = c; break; }
            sum += x;
        }
        s_chunk = at == 0xffffffffu ? some : at;   /* rounding: the last with anything in it */
        s_left = at == 0xffffffffu ? CUDART_INF : want - sum;
    }
    __syncthreads();
    over_q = s_over;
    const double want = s_left;
    const uint32_t i0 = s_chunk * CHUNK, n = min(CHUNK, P.vocab - i0), mine0 = min(tid * EACH, n), mine1 = min(mine0 + EACH, n);
    double sum = 0.0;
    int32_t some = -1;
    for (uint32_t i = mine0; i < mine1; i++) {
        const double x = weight(i0 + i, over_q);
        if (x > 0.0) some = (int32_t)(i0 + i);
        sum += x;
    }
    double before = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= (uint32_t)d) before += x;
    }
    __syncthreads();
    if (lane == 31u) s_scan[warp] = before;
    some = (int32_t)__reduce_max_sync(0xffffffffu, (uint32_t)(some + 1)) - 1;
    if (lane == 0) s_best[warp] = some;
    if (tid == 0) s_found = 0xffffffffu;
    __syncthreads();
    before -= sum;
    for (uint32_t w = 0; w < warp; w++) before += s_scan[w];
    if (before + sum > want)   /* the first token above it; threads behind find later ones */
        for (uint32_t i = mine0; i < mine1; i++) {
            before += weight(i0 + i, over_q);
            if (before > want) {
                atomicMin(&s_found, i0 + i);
                break;
            }
        }
    __syncthreads();
    if (tid == 0) {
        int32_t found = (int32_t)s_found;
        if (s_found == 0xffffffffu)   /* rounding: the last that can be */
            for (uint32_t w = 0; w < WARPS; w++) found = max(found, s_best[w]);
        P.next[r] = found;
        if (P.logp) P.logp[stop] = found >= 0 ? log_p(stop, D.p, found) : 0.f;
    }
}

template <bool BF16>
bool verify_launch(const VerifyParams &p) {
    const uint64_t blocks = (uint64_t)p.n_tok * (p.draft ? 2u : 1u) * p.chunks;
    if (blocks > 0x7fffffffu) return q4i_fail(Q4E_ARG, "verify: too many rows for one call");
    return q4i_launch_pdl("verify launch", q4_vf_stat_k<BF16>, dim3((unsigned)blocks), VF_THREADS, 0, p) &&
           q4i_launch_pdl("verify launch", q4_vf_pick_k<BF16>, dim3(p.chunks, p.n_req), VF_THREADS, 0, p);
}

}  // namespace

extern "C" bool q4_gpu_verify(const void *logits, int bf16, uint64_t ld, const void *draft, uint64_t draft_ld, uint32_t vocab, const int32_t *token, const int32_t *start,
                              uint32_t n_req, uint32_t n_tok, const float *temp, const float *u_accept, const float *u_next, int32_t *accepted, int32_t *next, float *logp,
                              const int32_t *rows, int32_t *keep) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "verify: library not initialised");
    Q4_REQUIRE(logits && token && start && u_accept && u_next && accepted && next && vocab && n_req && n_tok, "verify: bad argument");
    Q4_REQUIRE(!rows == !keep, "verify: rows and keep go together");
    Q4_REQUIRE(n_req <= PLAN_MAX_REQ && n_tok <= 0x7fffffffu && vocab <= 0x7fffffffu, "verify: at most 8192 requests, 2^31 - 1 rows and tokens");
    Q4_REQUIRE(n_tok == 1u || (ld >= vocab && (!draft || draft_ld >= vocab)), "verify: rows are closer than the vocabulary is wide");
    Q4_REQUIRE(((uintptr_t)logits & (bf16 ? 1u : 3u)) == 0 && ((uintptr_t)draft & (bf16 ? 1u : 3u)) == 0, "verify: logits are not aligned to their type");
    VerifyParams p = {};
    p.logits = logits; p.draft = draft; p.bf16 = bf16 != 0; p.ld = ld; p.draft_ld = draft_ld; p.vocab = vocab;
    p.chunks = (vocab + CHUNK - 1u) / CHUNK;
    p.n_req = n_req; p.n_tok = n_tok; p.token = token; p.start = start; p.temp = temp; p.u_accept = u_accept; p.u_next = u_next;
    p.accepted = accepted; p.next = next; p.logp = logp; p.rows = rows; p.keep = keep;
    p.err = g_q4.err_d;
    const uint64_t stats = (uint64_t)n_tok * (draft ? 2u : 1u) * p.chunks, rests = draft ? (uint64_t)n_req * p.chunks : 0u;
    if (!q4i_scratch((size_t)(stats * 4u + rests * 2u), 0)) return false;
    p.stat = (VfStat *)g_q4.part;
    p.rest = (double *)(p.stat + stats);
    return bf16 ? verify_launch<true>(p) : verify_launch<false>(p);
}
