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
 *
 * The exponential: x log2(e) / T in steps of 1/32 is an integer K and a rest |r| <= 1/2; 2^((K + r) / 32) = 2^(K >> 5) 2^((K & 31) / 32) e^(r ln 2 / 32),
 * the second factor from a table of which each lane holds one entry, the third by its Taylor series up to r^5 (what is left out is below 2.3e-15):
 * 10 operations of the 64-bit pipe, the sum's among them, where a library exponential takes some 20 (48 x 5 drafts over 131 072 tokens 206 us with those).
 */
#include <math_constants.h>

#include "q4_internal.h"
#include "q4_pages_scan.h"

namespace {

constexpr uint32_t CHUNK = 4096, VF_THREADS = 128, EACH = CHUNK / VF_THREADS, PICK_THREADS = 512, PICK_EACH = CHUNK / PICK_THREADS;
constexpr float LARGEST = 3.402823466e38f;

struct __align__(16) VfStat { double s; float m; int32_t at; };   /* of a chunk: sum relative to the largest logit, that logit (NaN or +inf: the row is no distribution), its first place (greedy) */

struct VerifyParams {
    const uint8_t *logits, *draft;
    uint64_t ld, draft_ld;       /* bytes */
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
__device__ const double g_vf_pow[32] = {          /* 2^(j / 32) */
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332, 1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
constexpr double LN2 = 0.69314718055994530942, STEPS = 32.0 * 1.44269504088896340736;   /* of 1/32 of a power of two, per unit of the exponent */

__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
__device__ __forceinline__ float warp_max_nan(float m) {
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= LARGEST; }

/* exp((x - M) / T) for the logits of a row whose largest is M.  fast: in steps of c per unit of x from the whole one e next to M, as above; it needs steps below
 * 2^50 and a logit 1000 powers of two below M that is still a number.  Else by the library's function. */
struct VfExp {
    double c, e, inv, m;
    float low;                   /* what is below is nothing (2^-1000) */
    bool fast;
    __device__ __forceinline__ void set(float largest, double inv_t, float T) {
        m = largest;
        inv = inv_t;
        c = inv_t * STEPS;
        const double at = m * c, far = m - 1000.0 * LN2 * (double)T;
        fast = fabs(at) < 1099511627776.0 && far > -1e38;
        e = rint(at);
        low = (float)far;
    }
    /* the steps from e back to M, as a factor */
    __device__ __forceinline__ double to_m() const { return fast ? exp2(fma(m, c, -e) * (-1.0 / 32.0)) : 1.0; }
    /* relative to e where fast; pow: the lane's entry of the table.  By whole warps */
    __device__ __forceinline__ double steps(float x, double pow) const {
        constexpr double MAGIC = 6755399441055744.0;   /* 1.5 * 2^52: the sum's low word is the rounded integer */
        constexpr double L = LN2 / 32.0;
        const double xd = (double)x, t = fma(xd, c, MAGIC - e);
        const double r = fma(xd, c, -(t - (MAGIC - e)));
        const int32_t k = __double2loint(t);
        const int32_t hi = __shfl_sync(0xffffffffu, __double2hiint(pow), k), lo = __shfl_sync(0xffffffffu, __double2loint(pow), k);
        const double p = fma(r, fma(r, fma(r, fma(r, L * L * L * L * L / 120.0, L * L * L * L / 24.0), L * L * L / 6.0), L * L / 2.0), L);
        const double f = __hiloint2double(hi + ((k & ~31) << 15), lo);
        return fma(f * r, p, f);
    }
    __device__ __forceinline__ double of(float x, double pow) const {
        if (!fast) return exp(((double)x - m) * inv);
        const double y = steps(fmaxf(x, low), pow);
        return x < low ? 0.0 : y;
    }
};

template <bool BF16>
__device__ __forceinline__ float logit(const uint8_t *row, uint64_t at) {
    if constexpr (BF16) return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(row) + at) << 16);
    else return __ldcg(reinterpret_cast<const float *>(row) + at);
}
/* Rows begin anywhere: chunks are counted from the 16-byte piece that a row begins in */
template <bool BF16>
__device__ __forceinline__ uint32_t row_begins(const uint8_t *row) { return ((uint32_t)(uintptr_t)row & 15u) / (BF16 ? 2u : 4u); }

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
__device__ __forceinline__ bool temperature_ok(float t) { return t >= 0.f && t <= LARGEST; }

template <bool BF16>
__global__ void __launch_bounds__(VF_THREADS) q4_vf_stat_k(const VerifyParams P) {
    constexpr uint32_t PER = BF16 ? 8u : 4u, WARPS = VF_THREADS / 32u;
    __shared__ float s_max[WARPS];
    __shared__ double s_sum[WARPS], s_inv;
    __shared__ uint32_t s_at;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    q4d_pdl_wait();
    const uint32_t row = blockIdx.x / P.chunks, chunk = blockIdx.x - row * P.chunks;
    const bool drafts = row >= P.n_tok;
    const uint32_t t = drafts ? row - P.n_tok : row;
    const uint8_t *base = drafts ? P.draft + t * P.draft_ld : P.logits + t * P.ld;
    const uint32_t off = row_begins<BF16>(base);
    float x[EACH];
#pragma unroll
    for (uint32_t k = 0; k < EACH / PER; k++) {
        const int64_t i = (int64_t)chunk * CHUNK + (k * VF_THREADS + tid) * PER - off;
        if (i >= 0 && i + PER <= P.vocab) {
            const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(base + i * (BF16 ? 2 : 4)));
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (uint32_t j = 0; j < PER; j++) x[k * PER + j] = __uint_as_float(!BF16 ? u[j & 3u] : j & 1u ? u[j / 2u] & 0xffff0000u : u[j / 2u] << 16);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < PER; j++) x[k * PER + j] = i + j >= 0 && i + j < P.vocab ? logit<BF16>(base, (uint64_t)(i + j)) : -CUDART_INF_F;
        }
    }
    /* whose row it is, while the logits come */
    const uint32_t r = request_of(P.start, P.n_req, t);
    const int32_t a = __ldcg(P.start + r), b = __ldcg(P.start + r + 1u);
    const float T = temperature(P, r);
    if ((int32_t)t < a || (int32_t)t >= b || !temperature_ok(T)) return;
    if (drafts && ((int32_t)t + 1 == b || T == 0.f)) return;
    const double pow = __ldg(g_vf_pow + lane);
    float m = x[0];
#pragma unroll
    for (uint32_t k = 1; k < EACH; k++) m = max_nan(m, x[k]);
    m = warp_max_nan(m);
    if (lane == 0) s_max[warp] = m;
    if (tid == 0) {
        s_at = 0xffffffffu;
        s_inv = 1.0 / (double)T;
    }
    __syncthreads();
    m = s_max[0];
#pragma unroll
    for (uint32_t w = 1; w < WARPS; w++) m = max_nan(m, s_max[w]);
    VfStat *out = P.stat + (uint64_t)row * P.chunks + chunk;
    if (T == 0.f) {
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (uint32_t k = 0; k < EACH; k++)
            if (x[k] == m) at = min(at, (k / PER * VF_THREADS + tid) * PER + k % PER);
        atomicMin(&s_at, at);
        __syncthreads();
        if (tid == 0) *out = {1.0, m, (int32_t)(chunk * CHUNK + s_at - off)};
        return;
    }
    double s = 0.0;
    VfExp E;
    E.set(m, s_inv, T);
    if (!finite(m)) {   /* nothing in it, or no distribution */
    } else if (E.fast) {
        double s1 = 0.0;
#pragma unroll
        for (uint32_t k = 0; k < EACH; k += 2u) {
            s += E.steps(fmaxf(x[k], E.low), pow);
            s1 += E.steps(fmaxf(x[k + 1u], E.low), pow);
        }
        s += s1;
    } else {
#pragma unroll 1
        for (uint32_t k = 0; k < EACH; k++) {
            float y = x[0];
#pragma unroll
            for (uint32_t j = 1; j < EACH; j++) y = j == k ? x[j] : y;
            s += exp(((double)y - E.m) * E.inv);
        }
    }
    s = warp_sum(s);
    if (lane == 0) s_sum[warp] = s;
    __syncthreads();
    if (tid == 0) {
        for (uint32_t w = 1; w < WARPS; w++) s += s_sum[w];
        *out = {finite(m) ? s * E.to_m() : 0.0, m, 0};
    }
}

/* a row's M and S from its chunks', by a whole warp; false: no distribution */
struct Row { float m; double s; };
__device__ __forceinline__ bool row_of(const VfStat *stat, uint32_t chunks, double inv, Row &R) {
    const uint32_t lane = threadIdx.x & 31u;
    float m = -CUDART_INF_F, m0 = -CUDART_INF_F;
    double s0 = 0.0;
    for (uint32_t c = lane; c < chunks; c += 32u) {
        const int4 x = __ldcg(reinterpret_cast<const int4 *>(stat + c));
        if (c == lane) {
            s0 = __hiloint2double(x.y, x.x);
            m0 = __int_as_float(x.z);
        }
        m = max_nan(m, __int_as_float(x.z));
    }
    R.m = m = warp_max_nan(m);
    R.s = 0.0;
    if (!finite(m)) return false;
    if (s0 > 0.0) R.s = s0 * exp(((double)m0 - (double)m) * inv);
    for (uint32_t c = lane + 32u; c < chunks; c += 32u) {
        const double s = __ldcg(&stat[c].s);
        if (s > 0.0) R.s += s * exp(((double)__ldcg(&stat[c].m) - (double)m) * inv);
    }
    R.s = warp_sum(R.s);
    return true;
}
/* the first place of a row's largest logit, by a whole warp */
__device__ __forceinline__ bool best_of(const VfStat *stat, uint32_t chunks, int32_t &at) {
    const uint32_t lane = threadIdx.x & 31u;
    float m = -CUDART_INF_F;
    for (uint32_t c = lane; c < chunks; c += 32u) m = max_nan(m, __ldcg(&stat[c].m));
    m = warp_max_nan(m);
    at = 0x7fffffff;
    for (uint32_t c = lane; c < chunks; c += 32u)
        if (__ldcg(&stat[c].m) == m) at = min(at, __ldcg(&stat[c].at));
    at = __reduce_min_sync(0xffffffffu, at);
    return finite(m);
}

enum { VF_REFUSED = 0, VF_KEPT = 1, VF_NONE = 2 /* no distribution */, VF_LAST = 3 };

template <bool BF16>
__global__ void __launch_bounds__(PICK_THREADS) q4_vf_pick_k(const VerifyParams P) {
    constexpr uint32_t WARPS = PICK_THREADS / 32u;
    __shared__ Row s_p[WARPS], s_q[WARPS];
    __shared__ uint32_t s_said[WARPS];
    __shared__ int32_t s_best[WARPS], s_some[WARPS];
    __shared__ double s_scan[WARPS], s_left, s_special;
    __shared__ uint32_t s_chunk, s_found, s_last, s_over;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, chunk = blockIdx.x, r = blockIdx.y;
    const bool first = chunk == 0u;
    q4d_pdl_wait();
    const int32_t a = __ldcg(P.start + r), b = __ldcg(P.start + r + 1u);
    const float T = temperature(P, r);
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
    const bool greedy = T == 0.f;
    const double inv = greedy ? 1.0 : 1.0 / (double)T, pow = __ldg(g_vf_pow + lane);
    const VfStat *stat_p = P.stat, *stat_q = P.stat + (uint64_t)P.n_tok * P.chunks;
    const uint32_t last = (uint32_t)b - 1u;

    /* ---- the request's rows, a warp each: whether the draft behind a row is kept.  The first that is not, or the last row, decides */
    uint32_t stop = (uint32_t)a, said = VF_NONE;
    Row p = {}, q = {};
    int32_t best = -1;
    bool out_of_vocab = false;
    for (uint32_t t0 = (uint32_t)a; temperature_ok(T); t0 += WARPS) {
        const uint32_t t = t0 + warp;
        uint32_t mine = VF_KEPT;
        float lp = 0.f;
        if (t <= last) {
            const int32_t d = t < last ? __ldcg(P.token + t + 1u) : -1;
            const bool in = (uint32_t)d < P.vocab, with_q = t < last && P.draft;
            /* asked for ahead of the sums */
            const float xp = !greedy && in ? logit<BF16>(P.logits + t * P.ld, (uint32_t)d) : 0.f, xq = !greedy && in && with_q ? logit<BF16>(P.draft + t * P.draft_ld, (uint32_t)d) : 0.f;
            const float u = !greedy && t < last ? __ldcg(P.u_accept + t) : 0.f;
            if (greedy) {
                mine = !best_of(stat_p + (uint64_t)t * P.chunks, P.chunks, best) ? VF_NONE : t == last ? VF_LAST : best == d ? VF_KEPT : VF_REFUSED;
            } else if (!row_of(stat_p + (uint64_t)t * P.chunks, P.chunks, inv, p) || (with_q && !row_of(stat_q + (uint64_t)t * P.chunks, P.chunks, inv, q))) {
                mine = VF_NONE;
            } else if (t == last) {
                mine = VF_LAST;
            } else if (in) {
                const double pd = exp(((double)xp - (double)p.m) * inv) / p.s, qd = P.draft ? exp(((double)xq - (double)q.m) * inv) / q.s : 1.0;
                mine = (double)u * qd < pd ? VF_KEPT : VF_REFUSED;
                if (P.logp && first) lp = (float)(((double)xp - (double)p.m) * inv - log(p.s));
            } else {
                mine = VF_REFUSED;
            }
            out_of_vocab = t < last && !in;
        }
        __syncthreads();
        if (lane == 0) {
            s_said[warp] = mine;
            s_p[warp] = p;
            s_q[warp] = q;
            s_best[warp] = best;
        }
        __syncthreads();
        const uint32_t others = __ballot_sync(0xffffffffu, lane < WARPS && s_said[lane & (WARPS - 1u)] != VF_KEPT);
        const uint32_t n = others ? (uint32_t)__ffs((int)others) - 1u : WARPS;
        if (first && lane == 0 && t < last) {
            if (P.logp && warp < n) P.logp[t] = greedy ? 0.f : lp;
            if (out_of_vocab && warp <= n) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        }
        if (others) {
            stop = t0 + n;
            said = s_said[n];
            p = s_p[n];
            q = s_q[n];
            best = s_best[n];
            break;
        }
    }
    if (first) {
        if (P.logp)
            for (uint32_t t = stop + 1u + tid; t <= last; t += PICK_THREADS) P.logp[t] = 0.f;
        if (tid == 0) {
            P.accepted[r] = (int32_t)(stop - (uint32_t)a);
            if (P.keep) P.keep[r] = __ldcg(P.rows + r) + (int32_t)(stop - (uint32_t)a) + 1;
            if (said == VF_NONE || greedy) {
                P.next[r] = said == VF_NONE ? -1 : best;
                if (P.logp) P.logp[stop] = 0.f;
                if (said == VF_NONE) atomicOr(P.err, (uint32_t)Q4E_RANGE);
            }
        }
    }
    if (said == VF_NONE || greedy) return;
    const bool refused = said == VF_REFUSED, with_q = refused && P.draft;
    if (!first && !with_q) return;

    /* ---- weights of the row's tokens: p without the refused one where drafts are certain, or what p has over q */
    const uint8_t *row_p = P.logits + stop * P.ld, *row_q = with_q ? P.draft + stop * P.draft_ld : nullptr;
    const int64_t off = row_begins<BF16>(row_p);
    const int32_t d = refused ? __ldcg(P.token + stop + 1u) : -1, certain = refused && !with_q ? d : -1;
    VfExp Ep, Eq;
    Ep.set(p.m, inv, T);
    Eq.set(with_q ? q.m : 0.f, inv, T);
    const double scale_p = Ep.to_m() / p.s, scale_q = with_q ? Eq.to_m() / q.s : 0.0;
    auto begin_of = [&](uint32_t c) -> uint32_t { return (uint32_t)max((int64_t)c * CHUNK - off, (int64_t)0); };
    auto end_of = [&](uint32_t c) -> uint32_t { return (uint32_t)min((int64_t)(c + 1u) * CHUNK - off, (int64_t)P.vocab); };
    auto weight = [&](float xp, float xq, bool skip, bool over_q) -> double {   /* by whole warps; minus infinity: nothing */
        const double x = __dmul_rn(Ep.of(xp, pow), scale_p);
        if (!over_q) return skip ? 0.0 : x;
        return fmax(__dsub_rn(x, __dmul_rn(Eq.of(xq, pow), scale_q)), 0.0);   /* both rounded: equal ones leave nothing */
    };
    auto block_sum = [&](double x) -> double {
        x = warp_sum(x);
        __syncthreads();
        if (lane == 0) s_scan[warp] = x;
        __syncthreads();
        x = s_scan[0];
#pragma unroll
        for (uint32_t w = 1; w < WARPS; w++) x += s_scan[w];
        return x;
    };
    auto chunk_sum = [&](uint32_t c, bool over_q) -> double {
        const uint32_t i0 = begin_of(c), i1 = end_of(c);
        float xp[PICK_EACH], xq[PICK_EACH];
#pragma unroll
        for (uint32_t k = 0; k < PICK_EACH; k++) {
            const uint64_t i = (uint64_t)i0 + k * PICK_THREADS + tid;
            xp[k] = i < i1 ? logit<BF16>(row_p, i) : -CUDART_INF_F;
            xq[k] = over_q && i < i1 ? logit<BF16>(row_q, i) : -CUDART_INF_F;
        }
        double x = 0.0;
#pragma unroll
        for (uint32_t k = 0; k < PICK_EACH; k++) x += weight(xp[k], xq[k], (int32_t)(i0 + k * PICK_THREADS + tid) == certain, over_q);
        return block_sum(x);
    };
    double *rest = P.rest + (uint64_t)r * P.chunks;
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
    /* ---- the chunk in which the running sum passes u times the whole, by a warp with a chunk per lane; then the place in it */
    const uint32_t special_at = (uint32_t)certain < P.vocab ? (uint32_t)((certain + off) / CHUNK) : 0xffffffffu;
    if (special_at != 0xffffffffu) {
        const double x = chunk_sum(special_at, false);
        if (tid == 0) s_special = x;
        __syncthreads();
    }
    const VfStat *sp = stat_p + (uint64_t)stop * P.chunks;
    if (warp == 0) {
        const double u = (double)__ldcg(P.u_next + r);
        auto of_chunk = [&](uint32_t c, bool over_q) -> double {
            if (c >= P.chunks) return 0.0;
            if (over_q) return __ldcg(rest + c);
            if (c == special_at) return s_special;
            const int4 x = __ldcg(reinterpret_cast<const int4 *>(sp + c));
            const double s = __hiloint2double(x.y, x.x);
            return s > 0.0 ? s * exp(((double)__int_as_float(x.z) - (double)p.m) * inv) / p.s : 0.0;
        };
        /* sums up to and with every lane's chunk, from chunk c0 on; they are formed in one order for the whole and for the place */
        auto scan = [&](uint32_t c0, double before, bool over_q, double &own) -> double {
            double x = own = of_chunk(c0 + lane, over_q);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= (uint32_t)o) x += y;
            }
            return x + before;
        };
        bool over_q = with_q;
        double all, own, x = 0.0;
        for (;;) {
            all = 0.0;
            for (uint32_t c0 = 0; c0 < P.chunks; c0 += 32u) all = __shfl_sync(0xffffffffu, x = scan(c0, all, over_q, own), 31);
            if (all > 0.0 || !over_q) break;
            over_q = false;      /* p nowhere above q: as if none was refused */
        }
        const double want = u * all;
        double before = 0.0, left = CUDART_INF;
        uint32_t at = 0xffffffffu, some = 0;
        for (uint32_t c0 = 0; c0 < P.chunks && at == 0xffffffffu; c0 += 32u) {
            if (P.chunks > 32u) x = scan(c0, before, over_q, own);
            const uint32_t above = __ballot_sync(0xffffffffu, x > want && own > 0.0), any = __ballot_sync(0xffffffffu, own > 0.0);
            if (any) some = c0 + 31u - (uint32_t)__clz((int)any);
            const double below = __shfl_up_sync(0xffffffffu, x, 1);
            if (above) {
                const uint32_t l = (uint32_t)__ffs((int)above) - 1u;
                at = c0 + l;
                left = want - __shfl_sync(0xffffffffu, lane ? below : before, (int)l);
            }
            before = __shfl_sync(0xffffffffu, x, 31);
        }
        if (lane == 0) {
            s_chunk = at == 0xffffffffu ? some : at;   /* rounding, or u not below 1: the last with anything in it */
            s_left = left;
            s_over = over_q;
            s_found = 0xffffffffu;
        }
    }
    __syncthreads();
    const bool over_q = s_over;
    const double want = s_left;
    const uint32_t i0 = begin_of(s_chunk) + tid * PICK_EACH, i1 = end_of(s_chunk);
    float xp[PICK_EACH], xq[PICK_EACH];
#pragma unroll
    for (uint32_t k = 0; k < PICK_EACH; k++) {
        const uint64_t i = (uint64_t)i0 + k;
        xp[k] = i < i1 ? logit<BF16>(row_p, i) : -CUDART_INF_F;
        xq[k] = over_q && i < i1 ? logit<BF16>(row_q, i) : -CUDART_INF_F;
    }
    double w[PICK_EACH], sum = 0.0;
    int32_t some = -1;
#pragma unroll
    for (uint32_t k = 0; k < PICK_EACH; k++) {
        w[k] = weight(xp[k], xq[k], (int32_t)(i0 + k) == certain, over_q);
        sum += w[k];
        if (w[k] > 0.0) some = (int32_t)(i0 + k);
    }
    double before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= (uint32_t)o) before += x;
    }
    some = (int32_t)__reduce_max_sync(0xffffffffu, (uint32_t)(some + 1)) - 1;
    __syncthreads();
    if (lane == 31u) s_scan[warp] = before;
    if (lane == 0) s_some[warp] = some;
    __syncthreads();
    before -= sum;
    for (uint32_t k = 0; k < warp; k++) before += s_scan[k];
    if (before + sum > want && sum > 0.0) {   /* the first token above it; threads behind find later ones */
        uint32_t found = 0xffffffffu;
#pragma unroll
        for (uint32_t k = 0; k < PICK_EACH; k++) {
            before += w[k];
            if (before > want && w[k] > 0.0 && found == 0xffffffffu) found = i0 + k;
        }
        if (found != 0xffffffffu) atomicMin(&s_found, found);
    }
    __syncthreads();
    if (tid == 0) {
        int32_t found = (int32_t)s_found;
        if (s_found == 0xffffffffu)   /* rounding: the last that can be */
            for (uint32_t k = 0; k < WARPS; k++) found = max(found, s_some[k]);
        P.next[r] = found;
        if (P.logp) P.logp[stop] = found >= 0 ? (float)(((double)logit<BF16>(row_p, (uint32_t)found) - (double)p.m) * inv - log(p.s)) : 0.f;
    }
}

template <bool BF16>
bool verify_launch(const VerifyParams &p) {
    const uint64_t blocks = (uint64_t)p.n_tok * (p.draft ? 2u : 1u) * p.chunks;
    if (blocks > 0x7fffffffu) return q4i_fail(Q4E_ARG, "verify: too many rows for one call");
    return q4i_launch_pdl("verify launch", q4_vf_stat_k<BF16>, dim3((unsigned)blocks), VF_THREADS, 0, p) &&
           q4i_launch_pdl("verify launch", q4_vf_pick_k<BF16>, dim3(p.draft ? p.chunks : 1u, p.n_req), PICK_THREADS, 0, p);
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
    Q4_REQUIRE(ld < 1ull << 40 && draft_ld < 1ull << 40, "verify: rows are too far apart");
    Q4_REQUIRE(((uintptr_t)logits & (bf16 ? 1u : 3u)) == 0 && ((uintptr_t)draft & (bf16 ? 1u : 3u)) == 0, "verify: logits are not aligned to their type");
    VerifyParams p = {};
    const uint64_t size = bf16 ? 2u : 4u;
    p.logits = (const uint8_t *)logits; p.draft = (const uint8_t *)draft; p.ld = ld * size; p.draft_ld = draft_ld * size; p.vocab = vocab;
    p.chunks = (uint32_t)((vocab + 16u / size - 1u + CHUNK - 1u) / CHUNK);   /* wherever in a 16-byte piece a row begins */
    p.n_req = n_req; p.n_tok = n_tok; p.token = token; p.start = start; p.temp = temp; p.u_accept = u_accept; p.u_next = u_next;
    p.accepted = accepted; p.next = next; p.logp = logp; p.rows = rows; p.keep = keep;
    p.err = g_q4.err_d;
    const uint64_t stats = (uint64_t)n_tok * (draft ? 2u : 1u) * p.chunks, rests = draft ? (uint64_t)n_req * p.chunks : 0u;
    if (!q4i_scratch((size_t)(stats * 4u + rests * 2u), 0)) return false;
    p.stat = (VfStat *)g_q4.part;
    p.rest = (double *)(p.stat + stats);
    return bf16 ? verify_launch<true>(p) : verify_launch<false>(p);
}
