/*
 * Drafted tokens held against the target's distributions, and the token behind the last one that is kept.  No counterpart in the reference.
 *
 *     p_i = exp((x_i - M) / T) / S,  S = sum exp((x_i - M) / T),  M the largest logit;  q likewise from the draft's logits
 *     draft d is kept while u q_d < p_d;  next = the first i with sum_{j <= i} w_j > u sum w,  w = max(p - q, 0), or p
 *
 * The first launch goes once through all rows, a warp per row and up to SPAN chunks of CHUNK logits, and leaves the largest logit and the sum of every chunk. The second
 * decides, a block per request: the chunks' sums tell in which one the next token lies, and only that one is looked through.  Where a
 * draft was refused and has logits, the blocks of the third go through that row of p and q once more for the sums of max(p - q, 0), and the last of the
 * request's to finish looks.
 *
 * A token's border in the running sum may lie anywhere: sums in 32 bits put a draw over a flat distribution of 10^5 tokens on the wrong side of one once in some
 * thousands.  So they are in 64 bits.  x log2(e) / T in steps of 1/32 is an integer K and a rest |r| <= 1/2;
 * 2^((K + r) / 32) = 2^(K >> 5) 2^((K & 31) / 32) e^(r ln 2 / 32), the second factor from a table of which each lane holds one entry, the third by its Taylor
 * series.  Where single tokens count (the last two launches) that is in 64 bits up to r^5 (what is left out is below 2.3e-15), for the sums of the first, which
 * see every logit, in two parts of 32 bits (VfFast): two additions of 64 bits per logit, and two logits to an instruction in most of the rest.
 *
 * The first launch is bound by its instructions, 18 per logit where the bytes alone are worth 10: 48 requests with 5 drafts over 131 072 tokens,
 * 280 MB, take 95 us in all, 69 in this launch and 43 of memory's; with all of it in 64 bits 206.
 */
#include <math_constants.h>
#include <type_traits>

#include "q4_internal.h"
#include "q4_pages_scan.h"

namespace {

constexpr uint32_t EACH = 32, CHUNK = 32u * EACH, VF_THREADS = 128, VF_WARPS = VF_THREADS / 32u, PICK_THREADS = 256, PICK_WARPS = PICK_THREADS / 32u, PICK_EACH = CHUNK / PICK_THREADS;
/* of the first launch: chunks of a warp at most, blocks per SM (80 registers, 8 to 36 bytes spilled; with 64, which spill more, it is slower), 16-byte pieces on their way to a lane, chunks that are brought to L2 ahead */
constexpr uint32_t SPAN = 6, STAT_BLOCKS = 6, VF_RING = 4, VF_AHEAD = 2;
constexpr float LARGEST = 3.402823466e38f;

/* of a chunk: its largest logit m (NaN or +inf: the row is no distribution), the sum of exponentials relative to a whole step, whose bits as a float at is (NaN:
 * relative to m); greedy: at is m's first place */
struct __align__(16) VfStat { double s; float m; int32_t at; };
constexpr int32_t NO_STEP = 0x7fffffff;
struct Row { float m; double s; };   /* s relative to VfExp's place */
/* of a request: which row decides next (and how), for the launch that looks where p is over q; none: it has been decided */
struct __align__(16) VfChoice { double c, drop, scale_p, scale_q, sum_p; float m_p, m_q; uint32_t stop, open; };

struct VerifyParams {
    const uint8_t *logits, *draft;
    uint64_t ld, draft_ld;       /* bytes */
    uint32_t vocab, n_req, n_tok;
    uint32_t chunks, span, spans;   /* of a row: chunks, those of a warp, warps */
    uint32_t levels, across;     /* the order of rows: every levels-th one, then those behind them; levels x across covers n_tok */
    uint32_t early;              /* rows, in that order, whose drafts are decided on at once; 0: none, and nobody looks */
    const int32_t *token, *start;
    const float *temp, *u_accept, *u_next;
    int32_t *accepted, *next;
    float *logp;
    const int32_t *rows;
    int32_t *keep;
    VfStat *stat;                /* [target's rows, draft's rows][chunk] */
    VfChoice *choice;            /* [request] */
    double *rest;                /* [request][chunk]: sums of max(p - q, 0) */
    uint32_t *err;
};
__device__ uint32_t g_vf_arrived[PLAN_MAX_REQ];   /* zero between launches */
/* of rows with a draft behind them: the warps that have finished, and what became of the draft; zero between calls */
constexpr uint32_t EARLY_MAX = 1u << 16, EARLY_STOP = 1u << 31, EARLY_NONE = 1u << 30, EARLY_KEPT = 1u << 29;
__device__ uint32_t g_vf_early[EARLY_MAX];
__device__ uint32_t g_vf_stop[PLAN_MAX_REQ];      /* of a request: EARLY_MAX less the first row whose draft is not kept; zero: none yet, and between calls */
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
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float warp_max_nan(float m) {
    float all;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(all) : "f"(m));
    return all;
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
/* sums up to and with each lane's */
__device__ __forceinline__ double warp_scan(double x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, x, o);
        if ((threadIdx.x & 31u) >= (uint32_t)o) x += y;
    }
    return x;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= LARGEST; }

/* steps per unit of a logit, and 1000 powers of two in logits */
struct VfScale {
    double c, drop;
    __device__ __forceinline__ explicit VfScale(float T) : c(STEPS / (double)T), drop(1000.0 * LN2 * (double)T) {}
    __device__ __forceinline__ VfScale(double c_, double drop_) : c(c_), drop(drop_) {}
};
/* exp((x - M) / T) for logits x up to some hundred powers of two above M.  fast: relative to the whole step e next to M, as above, where that is a number of 21 bits
 * and a logit 1000 powers of two below M is still a number.  Else relative to M, by the library's function. */
struct VfExp {
    double c, e, m;              /* e: 0 where not fast */
    float low;                   /* what is below is nothing (2^-1000), token or chunk: a chunk that counts has a token that does */
    bool fast;
    __device__ __forceinline__ void set(float largest, const VfScale &S) {
        m = largest;
        c = S.c;
        const double at = m * c;
        fast = fabs(at) < 2.0e6 && S.drop < 1e35;
        e = fast ? rint(at) : 0.0;
        low = (float)(m - S.drop);
    }
    __device__ __forceinline__ double slow(float x) const { return exp2(((double)x - m) * c * (1.0 / 32.0)); }
    /* table: the lane's entry, less its number at the exponent's lowest bits, which the whole step brings along.  By whole warps, x not below low.  The value is f * (what is returned) */
    __device__ __forceinline__ double steps(float x, int2 table, double &f) const {
        constexpr double MAGIC = 6755399441055744.0;   /* 1.5 * 2^52: the sum's low word is the rounded integer */
        constexpr double L = LN2 / 32.0;
        const double xd = (double)x, base = MAGIC - e, t = fma(xd, c, base), r = fma(xd, c, base - t);
        const int32_t k = __double2loint(t);
        const int32_t hi = __shfl_sync(0xffffffffu, table.y, k), lo = __shfl_sync(0xffffffffu, table.x, k);
        f = __hiloint2double(hi + (k << 15), lo);
        return fma(r, fma(r, fma(r, fma(r, fma(r, L * L * L * L * L / 120.0, L * L * L * L / 24.0), L * L * L / 6.0), L * L / 2.0), L), 1.0);
    }
    /* of several at once: a chain of operations of this kind takes 500 cycles, in which others can be at theirs */
    template <uint32_t N>
    __device__ __forceinline__ void of(const float (&x)[N], int2 table, double (&w)[N]) const {
        if (fast) {
#pragma unroll
            for (uint32_t k = 0; k < N; k++) {
                double f;
                const double y = steps(fmaxf(x[k], low), table, f);
                w[k] = x[k] < low ? 0.0 : f * y;
            }
        } else {
#pragma unroll
            for (uint32_t k = 0; k < N; k++) w[k] = x[k] < low ? 0.0 : slow(x[k]);
        }
    }
    /* A chunk's sum as one relative to this, its row's; pow: the table.  One that counts is above 0, although the logit that it is relative to may lie up to 100 powers of two below its
     * largest: that is taken as 2^-1000 at least, where it makes no difference beside the row's sum */
    __device__ __forceinline__ double chunk_fast(const VfStat &x, const double *pow) const {   /* both by whole steps */
        const int32_t k = (int32_t)fminf(fmaxf(__int_as_float(x.at) - (float)e, -32000.f), 32000.f);
        const double f = pow[k & 31];
        return x.m < low ? 0.0 : x.s * __hiloint2double(__double2hiint(f) + (k >> 5) * 1048576, __double2loint(f));
    }
    __device__ __forceinline__ double chunk(const VfStat &x, const double *pow) const {
        const float at = __int_as_float(x.at);
        if (fast && x.at != NO_STEP) return chunk_fast(x, pow);
        if (!(x.s > 0.0) || x.m < low) return 0.0;
        if (x.at == NO_STEP && !fast) return x.s * slow(x.m);
        return x.s * exp2(fmax(((x.at == NO_STEP ? (double)x.m * c : (double)at) - (fast ? e : m * c)) * (1.0 / 32.0), -1000.0));
    }
    /* log p of logit x, log_s being the logarithm of its row's sum relative to this */
    __device__ __forceinline__ float log_p(float x, double log_s) const { return (float)((fast ? fma((double)x, c, -e) : ((double)x - m) * c) * (LN2 / 32.0) - log_s); }
};
__device__ __forceinline__ int2 lane_table() {
    const uint32_t lane = threadIdx.x & 31u;
    const double x = __ldg(g_vf_pow + lane);
    return make_int2(__double2loint(x), __double2hiint(x) - (int32_t)(lane << 15));
}

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

/* 16 bytes of a row from its logit i on, around its ends: what is not its own is minus infinity */
template <bool BF16>
__device__ __noinline__ uint4 at_the_end(const uint8_t *base, int32_t i, uint32_t vocab) {
    uint32_t u[4];
#pragma unroll
    for (uint32_t j = 0; j < 4u; j++) {
        if constexpr (BF16) {
            const uint32_t a = i + 2 * j, b = a + 1;   /* below 0: beyond any vocabulary */
            u[j] = (a < vocab ? __ldcg(reinterpret_cast<const unsigned short *>(base) + a) : 0xff80u) | (b < vocab ? (uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(base) + b) : 0xff80u) << 16;
        } else {
            u[j] = i + j < vocab ? __ldcg(reinterpret_cast<const uint32_t *>(base) + (i + j)) : 0xff800000u;
        }
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}
/* 16 bytes of a row, a lane's: ring of them */
template <bool BF16>
struct Piece {
    static constexpr uint32_t PER = BF16 ? 8u : 4u, PIECES = EACH / PER, RING = VF_RING;   /* logits; of a chunk and lane; on their way to a lane */
    uint4 v;
    __device__ __forceinline__ void load(const uint8_t *base, int32_t i, uint32_t vocab) {   /* from logit i on, below 0 where the row begins in it */
        if (i >= 0 && i + (int32_t)PER <= (int32_t)vocab) v = __ldcs(reinterpret_cast<const uint4 *>(base + (uint64_t)(uint32_t)i * (BF16 ? 2u : 4u)));
        else v = at_the_end<BF16>(base, i, vocab);
    }
    __device__ __forceinline__ void get(float (&x)[PER]) const {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (uint32_t j = 0; j < PER; j++) x[j] = __uint_as_float(!BF16 ? u[j & 3u] : j & 1u ? u[j / 2u] & 0xffff0000u : u[j / 2u] << 16);
    }
};

/* two floats in a pair of registers */
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float a, float b) {
    Two x;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
    return x;
}
__device__ __forceinline__ void apart(Two x, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two x;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x) : "l"(a), "l"(b), "l"(c));
    return x;
}

/* Exponentials for sums, relative to a whole step e of which all that counts lies within 100 powers of two: as VfExp's, but in 32 bits and in two parts.
 * x c comes to whole steps and a rest by a product in two words.  The step is rounded by c's first word alone: the second, up to 2^-24 of c, adds to the rest, which is
 * 1/2 at small x c and up to 1/2 + 2e6 x 2^-24 = 0.62 at the largest.  The table's entry is 2^(j / 32) rounded, its error goes into the rest's exponential less 1,
 * q: the value is w + w q, where w is exact and q below 0.0135.  The sums are in 64 bits, but for up to eight w q at a time.  Errors, of the sum: steps 2.25 x 2^-25
 * (two roundings, and c's second word over 2^21 steps), times ln 2 / 32: 1.5e-9;  q's series, up to r^3: 0.0135^4 / 24 = 1.4e-9, its last roundings 1.5 x 2^-25 x 0.0135: 6e-10;
 * seven additions 7 x 2^-25 x 0.0135: 2.8e-9.  Below 7e-9 in all (5e-9 at |x| below 5000 T, where q is below 0.0112), and for many tokens far below, as they are not all one way. */
struct VfFast {
    float c_hi, c_lo, base, low, high, step;
    bool ok;
    double sum[2];
    __device__ __forceinline__ void set(const VfExp &E, const VfScale &S) {
        constexpr double MAGIC = 12582912.0;   /* 1.5 * 2^23: the sum's low bits are the rounded integer */
        ok = E.fast && S.c < 1e30;   /* it and its products are fp32 numbers: else (T below 1e-28) every chunk is summed again */
        c_hi = (float)S.c;
        c_lo = (float)(S.c - (double)c_hi);
        base = (float)(MAGIC - E.e);
        step = (float)E.e;
        low = (float)(E.m - 0.1 * S.drop);
        high = (float)(E.m + 0.1 * S.drop);
    }
    /* table: the lane's entry, less its number at the exponent's lowest bits; its error.  By whole warps.  Two logits to an instruction, where there is one for that */
    template <uint32_t N>
    __device__ __forceinline__ void add(const float (&x)[N], uint32_t table, float error) {
        constexpr float L = (float)(LN2 / 32.0);
        const Two ch = two(c_hi, c_hi), cl = two(c_lo, c_lo), b = two(base, base);
        Two rest = two(0.f, 0.f);
#pragma unroll
        for (uint32_t j = 0; j < N; j += 2u) {
            const Two y = two(fmaxf(x[j], low), fmaxf(x[j + 1u], low)), t = fma2(y, ch, b), r = fma2(y, cl, fma2(y, ch, fma2(t, two(-1.f, -1.f), b)));
            float t0, t1, rest0, rest1;
            apart(t, t0, t1);
            const uint32_t k0 = __float_as_uint(t0), k1 = __float_as_uint(t1);
            const float w0 = __uint_as_float(__shfl_sync(0xffffffffu, table, k0) + (k0 << 18)), w1 = __uint_as_float(__shfl_sync(0xffffffffu, table, k1) + (k1 << 18));
            const Two d = two(__shfl_sync(0xffffffffu, error, k0), __shfl_sync(0xffffffffu, error, k1));
            const Two q = fma2(r, fma2(r, fma2(r, two(L * L * L / 6.f, L * L * L / 6.f), two(L * L / 2.f, L * L / 2.f)), two(L, L)), d);
            rest = fma2(two(w0, w1), q, rest);
            sum[0] += (double)w0;
            sum[1] += (double)w1;
            if (j + 2u == N) {
                apart(rest, rest0, rest1);
                sum[0] += (double)(rest0 + rest1);
            }
        }
    }
};
/* a lane's part of a chunk's sum relative to its largest logit */
template <bool BF16>
__device__ __noinline__ double sum_again(const uint8_t *base, int32_t i0, uint32_t vocab, float largest, float T) {
    VfExp E;
    E.set(largest, VfScale(T));
    const int2 table = lane_table();
    double s = 0.0;
#pragma unroll 1
    for (uint32_t k = 0; k < EACH; k++) {
        const uint32_t i = i0 + k * 32u + (threadIdx.x & 31u);   /* below 0: beyond any vocabulary */
        const float x[1] = {i < vocab ? logit<BF16>(base, i) : -CUDART_INF_F};
        double w[1];
        E.of(x, table, w);
        s += w[0];
    }
    return E.fast ? s * exp2(fma(-E.m, E.c, E.e) * (1.0 / 32.0)) : s;
}
/* greedy rows: a chunk's largest logit and its first place */
template <bool BF16>
__device__ __noinline__ void best_in(const uint8_t *base, int32_t i0, uint32_t vocab, VfStat *out) {
    using V = Piece<BF16>;
    const uint32_t lane = threadIdx.x & 31u;
    float m = -CUDART_INF_F;
    uint32_t at = 0xffffffffu;
#pragma unroll 1
    for (uint32_t k0 = 0; k0 < V::PIECES; k0 += V::RING) {
        V ring[V::RING];
#pragma unroll
        for (uint32_t k = 0; k < V::RING; k++) ring[k].load(base, i0 + (int32_t)((k0 + k) * 32u + lane) * (int32_t)V::PER, vocab);
#pragma unroll
        for (uint32_t k = 0; k < V::RING; k++) {
            float x[V::PER];
            ring[k].get(x);
#pragma unroll
            for (uint32_t j = 0; j < V::PER; j++) {
                if (x[j] > m || (at == 0xffffffffu && x[j] == m)) at = ((k0 + k) * 32u + lane) * V::PER + j;   /* the lane's first of the largest */
                m = max_nan(m, x[j]);
            }
        }
    }
    const float all = warp_max_nan(m);
    at = __reduce_min_sync(0xffffffffu, m == all ? at : 0xffffffffu);
    if (lane == 0) *out = {1.0, all, (int32_t)(i0 + at)};
}

enum { VF_REFUSED = 0, VF_KEPT = 1, VF_NONE = 2 /* no distribution */, VF_LAST = 3 };
__device__ __forceinline__ uint32_t said_of(float xp, float xq, float u, const Row &p, const Row &q, bool with_q, const VfScale &S, int2 table);
template <bool BF16>
__device__ __noinline__ void decide_early(const VerifyParams &P, uint32_t r, uint32_t t, float T);
/* a warp has finished with its part of row t; the last of `arrive` of them (0: nobody asks) decides on the draft behind it */
template <bool BF16>
__device__ __forceinline__ void row_done(const VerifyParams &P, uint32_t r, uint32_t t, float T, uint32_t arrive) {
    if (!arrive) return;
    uint32_t n = 0;
    if ((threadIdx.x & 31u) == 0u) {   /* who has written its chunks' sums */
        __threadfence();
        n = atomicAdd(g_vf_early + t, 1u) + 1u;
        __threadfence();
    }
    if (__shfl_sync(0xffffffffu, n, 0) != arrive) return;
    __syncwarp();                /* a shuffle orders no memory: what the lanes read from here on lies behind the first one's fence */
    decide_early<BF16>(P, r, t, T);
}

/*
 * A warp has `span` chunks of a row.  The sums need not be relative to the largest logit but to any within 100 powers of two of it: the largest of the first
 * that the warp sees.  So every logit is taken up once, and its place in the ring is refilled at once from the pieces to come.  Where a
 * chunk's largest logit turns out to lie farther off, it is summed again.
 *
 * Rows behind a refused draft are not needed.  EARLY: the last warp of a row decides on the draft behind it, rows are taken in an order in which the requests'
 * first ones come first (if they bring about as many tokens each), and warps whose row is not needed any more leave.  What such rows leave unwritten is
 * read, but decides nothing.
 */
template <bool BF16, bool EARLY>
__global__ void __launch_bounds__(VF_THREADS, STAT_BLOCKS) q4_vf_stat_k(const __grid_constant__ VerifyParams P) {
    using V = Piece<BF16>;
    constexpr uint32_t PER = V::PER, RING = V::RING, HALF = RING * 32u * PER;   /* logits of a ring */
    static_assert(CHUNK % HALF == 0u, "a chunk is whole rings");
    const uint32_t lane = threadIdx.x & 31u, unit = blockIdx.x * VF_WARPS + (threadIdx.x >> 5), turn = unit / P.spans, c0 = (unit - turn * P.spans) * P.span, c1 = min(c0 + P.span, P.chunks);
    q4d_pdl_wait();
    bool drafts = false;
    uint32_t t;
    bool decides = false;
    if constexpr (EARLY) {       /* a row and the draft's, one behind the other */
        const uint32_t nth = P.draft ? turn >> 1 : turn, level = nth / P.across;
        drafts = P.draft && turn & 1u;
        t = (nth - level * P.across) * P.levels + level;
        decides = nth < P.early;
        if (level >= P.levels || t >= P.n_tok) return;   /* warps behind the last row */
    } else {
        if (turn >= P.n_tok * (P.draft ? 2u : 1u)) return;
        drafts = turn >= P.n_tok;
        t = drafts ? turn - P.n_tok : turn;
    }
    const uint32_t row = drafts ? P.n_tok + t : t, vocab = P.vocab;
    const uint8_t *base = drafts ? P.draft + t * P.draft_ld : P.logits + t * P.ld;
    int32_t i0 = (int32_t)(c0 * CHUNK) - (int32_t)row_begins<BF16>(base);   /* the chunk's first logit */
    V ring[RING];
#pragma unroll
    for (uint32_t k = 0; k < RING; k++) ring[k].load(base, i0 + (int32_t)((k * 32u + lane) * PER), vocab);
    /* whose row it is, while the logits come */
    float T;
    uint32_t arrive = 0, r;      /* warps of this row and the draft's, if there is a draft to decide on */
    {
        r = request_of(P.start, P.n_req, t);
        const int32_t a = __ldcg(P.start + r), b = __ldcg(P.start + r + 1u);
        T = temperature(P, r);
        if ((int32_t)t < a || (int32_t)t >= b || !temperature_ok(T)) return;
        if (drafts && ((int32_t)t + 1 == b || T == 0.f)) return;
        if (EARLY && a >= 0 && (uint32_t)b <= P.n_tok) {
            if (decides && (int32_t)t + 1 < b) arrive = P.spans * (P.draft && T != 0.f ? 2u : 1u);
            if (__ldcg(g_vf_stop + r) > EARLY_MAX - t) return;
        }
    }
    VfStat *out = P.stat + (uint64_t)row * P.chunks + c0;
    const uint32_t chunks = c1 - c0;
    if (T == 0.f) {
        for (uint32_t c = 0; c < chunks; c++, i0 += CHUNK) best_in<BF16>(base, i0, vocab, out + c);
        if constexpr (EARLY) row_done<BF16>(P, r, t, T, arrive);
        return;
    }
    const double pow = __ldg(g_vf_pow + lane);
    const float near = (float)pow, error = (float)((pow - (double)near) / (double)near);
    const uint32_t table = __float_as_uint(near) - (lane << 18);
    /* The lines of the chunks behind the next ones to L2: the ring alone keeps too little on its way */
    constexpr uint32_t AHEAD = VF_AHEAD;
    auto fetch = [&](int32_t i) {
        constexpr uint32_t SIZE = BF16 ? 2u : 4u, LINE = 128u / SIZE;
        i += (int32_t)(lane * LINE);
        if (lane * LINE < CHUNK && i >= 0 && i < (int32_t)vocab) asm volatile("prefetch.global.L2 [%0];" ::"l"(base + (uint64_t)(uint32_t)i * SIZE));
    };
    static_assert(CHUNK * 4u <= 32u * 128u, "a line per lane");
    for (uint32_t c = 1; c < AHEAD && c < chunks; c++) fetch(i0 + (int32_t)(c * CHUNK));
    VfFast F;
    F.ok = false;
    F.c_hi = F.c_lo = F.base = F.low = F.high = F.step = 0.f;
    float ref = -CUDART_INF_F;
    for (uint32_t c = 0; c < chunks; c++, i0 += CHUNK) {
        float m = -CUDART_INF_F;
        uint32_t word = 0;           /* looked at behind the chunk */
        if (EARLY) word = __ldcg(g_vf_stop + r);
        if (!finite(ref)) {          /* of what is there: by and large the row's size */
#pragma unroll
            for (uint32_t k = 0; k < RING; k++) {
                float x[PER];
                ring[k].get(x);
#pragma unroll
                for (uint32_t j = 0; j < PER; j++) ref = fmaxf(ref, x[j]);
            }
            ref = warp_max_nan(ref);
            if (finite(ref)) {
                const VfScale S(T);
                VfExp E;
                E.set(ref, S);
                F.set(E, S);
            }
        }
        F.sum[0] = F.sum[1] = 0.0;
        if (c + AHEAD < chunks) fetch(i0 + (int32_t)(AHEAD * CHUNK));
#pragma unroll 1
        for (uint32_t k0 = 0; k0 < CHUNK; k0 += HALF) {
            const int32_t next = i0 + (int32_t)(k0 + HALF);   /* of the next chunk, which lies behind, at last */
            const bool more = k0 + HALF < CHUNK || c + 1u < chunks, inside = more && next >= 0 && next + HALF <= vocab;
            const uint4 *p = reinterpret_cast<const uint4 *>(base + (int64_t)next * (BF16 ? 2 : 4)) + lane;
            auto take = [&](auto refill) {
#pragma unroll
                for (uint32_t k = 0; k < RING; k++) {
                    float x[PER];
                    ring[k].get(x);
#pragma unroll
                    for (uint32_t j = 0; j < PER; j += 2u) m = max_nan(m, x[j], x[j + 1u]);
                    F.add(x, table, error);
                    if constexpr (decltype(refill)::value) ring[k].v = __ldcs(p + k * 32u);   /* behind the use: ahead of it the logits are moved about (48 x 5 drafts 97.1 us, 95.4 so) */
                }
            };
            if (inside) {
                take(std::true_type());
            } else {
                take(std::false_type());
                if (more)
#pragma unroll
                    for (uint32_t k = 0; k < RING; k++) ring[k].load(base, next + (int32_t)((k * 32u + lane) * PER), vocab);
            }
        }
        const float all = warp_max_nan(m);
        double s = F.sum[0] + F.sum[1];
        int32_t to = __float_as_int(F.step);
        if (finite(all) && (!F.ok || all > F.high || all < F.low)) {
            to = NO_STEP;
            s = sum_again<BF16>(base, i0, vocab, all, T);
        }
        s = warp_sum(s);
        if (lane == 0) out[c] = {finite(all) ? s : 0.0, all, to};
        if (EARLY && word > EARLY_MAX - t) return;
    }
    if constexpr (EARLY) row_done<BF16>(P, r, t, T, arrive);
}

__device__ __forceinline__ VfStat stat_at(const VfStat *p) {
    const int4 x = __ldcg(reinterpret_cast<const int4 *>(p));
    return {__hiloint2double(x.y, x.x), __int_as_float(x.z), x.w};
}
__device__ __noinline__ double chunk_any(double c, double e, double m, float low, bool fast, double s, float x_m, int32_t at, const double *pow) {
    VfExp E;
    E.c = c; E.e = e; E.m = m; E.low = low; E.fast = fast;
    return E.chunk({s, x_m, at}, pow);
}
/* a row's M and S from its chunks', by a whole warp: what is asked for first, so that two rows are on their way at once */
struct RowOf {
    static constexpr uint32_t AT_ONCE = 4;   /* chunks of a lane */
    VfStat x[AT_ONCE];
    const VfStat *stat;
    uint32_t chunks;
    __device__ __forceinline__ void load(const VfStat *stat_, uint32_t chunks_) {
        const uint32_t lane = threadIdx.x & 31u;
        stat = stat_;
        chunks = chunks_;
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; k++) {
            x[k] = {0.0, -CUDART_INF_F, __float_as_int(0.f)};
            if (lane + 32u * k < chunks) x[k] = stat_at(stat + lane + 32u * k);
        }
    }
    __device__ __forceinline__ float largest() const {
        float m = -CUDART_INF_F;
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; k++) m = max_nan(m, x[k].m);
#pragma unroll 1
        for (uint32_t i = (threadIdx.x & 31u) + 32u * AT_ONCE; i < chunks; i += 32u) m = max_nan(m, __ldcg(&stat[i].m));
        return warp_max_nan(m);
    }
    __device__ __forceinline__ double own(const VfExp &E, const double *pow) const {   /* the lane's part of S */
        double s = 0.0;
        bool steps = E.fast;
#pragma unroll
        for (uint32_t k = 0; k < AT_ONCE; k++) steps = steps && x[k].at != NO_STEP;
        const bool all = __all_sync(0xffffffffu, steps);
        if (all) {
#pragma unroll
            for (uint32_t k = 0; k < AT_ONCE; k++) s += E.chunk_fast(x[k], pow);
        }
#pragma unroll 1
        for (uint32_t i = (threadIdx.x & 31u) + (all ? 32u * AT_ONCE : 0u); i < chunks; i += 32u) {
            const VfStat y = stat_at(stat + i);
            s += chunk_any(E.c, E.e, E.m, E.low, E.fast, y.s, y.m, y.at, pow);
        }
        return s;
    }
};
/* of p's row, and q's where it has chunks; false: one of them is no distribution */
__device__ __forceinline__ bool rows_of(const RowOf (&rows)[2], const VfScale &S, const double *pow, Row &p, Row &q) {
    const bool with_q = rows[1].chunks != 0u;
    p.m = rows[0].largest();
    q.m = with_q ? rows[1].largest() : 0.f;
    p.s = q.s = 0.0;
    if (!finite(p.m) || !finite(q.m)) return false;
    VfExp E, F;
    E.set(p.m, S);
    F.set(q.m, S);
    double a = rows[0].own(E, pow), b = with_q ? rows[1].own(F, pow) : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) {   /* side by side */
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    p.s = a;
    q.s = b;
    return true;
}
/* the first place of a row's largest logit, by a whole warp */
__device__ __forceinline__ bool best_of(const VfStat *stat, uint32_t chunks, int32_t &at) {
    const uint32_t lane = threadIdx.x & 31u;
    float m = -CUDART_INF_F;
    at = 0x7fffffff;
    for (uint32_t c = lane; c < chunks; c += 32u) {
        const VfStat x = stat_at(stat + c);
        const float top = max_nan(m, x.m);
        if (x.m == top && (m < top || x.at < at)) at = x.at;
        m = top;
    }
    const float all = warp_max_nan(m);
    at = __reduce_min_sync(0xffffffffu, m == all ? at : 0x7fffffff);
    return finite(all);
}

/* whether the draft with logits xp and xq is kept: u q < p, by both sums; by a whole warp */
__device__ __forceinline__ uint32_t said_of(float xp, float xq, float u, const Row &p, const Row &q, bool with_q, const VfScale &S, int2 table) {
    VfExp E, F;
    double pd, qd = 1.0, f, g;
    E.set(p.m, S);
    F.set(q.m, S);
    if (E.fast && F.fast) {      /* side by side */
        const double y = E.steps(fmaxf(xp, E.low), table, f), z = F.steps(fmaxf(xq, F.low), table, g);
        pd = xp < E.low ? 0.0 : f * y;
        if (with_q) qd = xq < F.low ? 0.0 : g * z;
    } else {
        const float one_p[1] = {xp}, one_q[1] = {xq};
        double one[1];
        E.of(one_p, table, one);
        pd = one[0];
        F.of(one_q, table, one);
        if (with_q) qd = one[0];
    }
    return (double)u * qd * p.s < pd * (with_q ? q.s : 1.0) ? VF_KEPT : VF_REFUSED;
}
/* row t and the draft's are done: what becomes of the draft behind t, by a warp */
template <bool BF16>
__device__ __noinline__ void decide_early(const VerifyParams &P, uint32_t r, uint32_t t, float T) {
    const int32_t d = __ldcg(P.token + t + 1u);
    const bool in = (uint32_t)d < P.vocab, with_q = P.draft != nullptr;
    const VfStat *stat_p = P.stat + (uint64_t)t * P.chunks;
    uint32_t said = VF_NONE;
    if (T == 0.f) {
        int32_t best;
        if (best_of(stat_p, P.chunks, best)) said = best == d ? VF_KEPT : VF_REFUSED;
    } else {
        float xp = 0.f, xq = 0.f;
        if (in) xp = logit<BF16>(P.logits + t * P.ld, (uint32_t)d);
        if (in && with_q) xq = logit<BF16>(P.draft + t * P.draft_ld, (uint32_t)d);
        const float u = __ldcg(P.u_accept + t);
        const VfScale S(T);
        RowOf rows[2];
        Row p = {}, q = {};
        rows[0].load(stat_p, P.chunks);
        rows[1].load(stat_p + (uint64_t)P.n_tok * P.chunks, with_q ? P.chunks : 0u);
        if (rows_of(rows, S, g_vf_pow, p, q)) said = in ? said_of(xp, xq, u, p, q, with_q, S, lane_table()) : (uint32_t)VF_REFUSED;
    }
    if ((threadIdx.x & 31u) == 0u && said != VF_KEPT) atomicMax(g_vf_stop + r, EARLY_MAX - t);
    if ((threadIdx.x & 31u) == 0u) atomicOr(g_vf_early + t, said == VF_KEPT ? EARLY_KEPT : said == VF_NONE ? EARLY_STOP | EARLY_NONE : EARLY_STOP);
}

/* The chunk of w_0 w_1 .. w_(n - 1) at which the running sum passes u times the whole, and what is left for it; by a whole warp.  A lane sums n / 32 of them (of(i0, i1, w): w_i0
 * up to w_i1, 0 behind them; N at a time), then all look through those of the lane in whose sum it lies.  Where rounding leaves none: the last one with
 * anything in it.  whole: the sum (0: nothing there) */
template <uint32_t N, typename F>
__device__ __forceinline__ uint32_t place_in(uint32_t n, double u, double &left, double &whole, F of) {
    const uint32_t lane = threadIdx.x & 31u, step = (n + 31u) / 32u, i0 = min(lane * step, n), i1 = min(i0 + step, n);
    double w[N], own = 0.0;
#pragma unroll 1
    for (uint32_t i = 0; i < step; i += N) {
        of(min(i0 + i, i1), i1, w);
#pragma unroll
        for (uint32_t k = 0; k < N; k++) own += w[k];
    }
    const double x = warp_scan(own);
    whole = __shfl_sync(0xffffffffu, x, 31);
    left = u * whole;
    if (!(whole > 0.0)) return 0u;
    const uint32_t above = __ballot_sync(0xffffffffu, x > left && own > 0.0), any = __ballot_sync(0xffffffffu, own > 0.0);
    const uint32_t l = above ? (uint32_t)__ffs((int)above) - 1u : any ? 31u - (uint32_t)__clz((int)any) : 0u;
    const double before = __shfl_up_sync(0xffffffffu, x, 1);
    left = above ? left - __shfl_sync(0xffffffffu, lane ? before : 0.0, (int)l) : CUDART_INF;
    if (N == 1u) return l;       /* n <= 32 */
    uint32_t found = 0, last = 0;
    double sum = 0.0, passed = 0.0;
    bool there = false;
#pragma unroll 1
    for (uint32_t i = 0; i < step; i += N) {
        if (step > N) of(min(i0 + i, i1), i1, w);
#pragma unroll
        for (uint32_t k = 0; k < N; k++) {
            const double v = __shfl_sync(0xffffffffu, w[k], (int)l);
            if (v > 0.0) last = i + k;
            if (!there && v > 0.0 && sum + v > left) {
                there = true;
                found = i + k;
                passed = sum;
            }
            sum += v;
        }
    }
    left = there ? left - passed : CUDART_INF;
    return l * step + (there ? found : last);
}
template <typename F>
__device__ __forceinline__ uint32_t place_of(uint32_t n, double u, double &left, double &whole, F of) {
    return n <= 32u ? place_in<1>(n, u, left, whole, of) : place_in<6>(n, u, left, whole, of);
}

/* N of a row's chunks' sums relative to E; of the one called special: another one */
template <uint32_t N>
__device__ __forceinline__ void chunks_of(const VfExp &E, const VfStat *stat, const double *pow, uint32_t special, double other, uint32_t i0, uint32_t i1, double (&w)[N]) {
    VfStat x[N];
    bool steps = E.fast;
#pragma unroll
    for (uint32_t k = 0; k < N; k++) {
        x[k] = {0.0, -CUDART_INF_F, __float_as_int(0.f)};
        if (i0 + k < i1) x[k] = stat_at(stat + i0 + k);
    }
#pragma unroll
    for (uint32_t k = 0; k < N; k++) steps = steps && x[k].at != NO_STEP;
    if (__all_sync(0xffffffffu, steps)) {
#pragma unroll
        for (uint32_t k = 0; k < N; k++) w[k] = E.chunk_fast(x[k], pow);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < N; k++) w[k] = chunk_any(E.c, E.e, E.m, E.low, E.fast, x[k].s, x[k].m, x[k].at, pow);
    }
#pragma unroll
    for (uint32_t k = 0; k < N; k++)
        if (i0 + k == special && i0 + k < i1) w[k] = other;
}

/* a row's tokens by weight: p times its row's sum, without the refused one where drafts are certain, or what p has over q */
template <bool BF16>
struct Weights {
    const uint8_t *row_p, *row_q;
    VfExp p, q;
    double scale_p, scale_q;     /* over q */
    int64_t off;
    uint32_t vocab;
    int32_t certain;             /* the token left out; -1: none */
    bool over_q;
    int2 table;
    __device__ __forceinline__ void set(const VerifyParams &P, uint32_t row, float m_p, float m_q, double scale_p_, double scale_q_, const VfScale &S, bool with_q, int32_t left_out) {
        row_p = P.logits + row * P.ld;
        row_q = with_q ? P.draft + row * P.draft_ld : nullptr;
        off = row_begins<BF16>(row_p);
        vocab = P.vocab;
        certain = left_out;
        over_q = with_q;
        table = lane_table();
        p.set(m_p, S);
        q.set(m_q, S);
        scale_p = scale_p_;
        scale_q = scale_q_;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t c) const { return (uint32_t)max((int64_t)c * CHUNK - off, (int64_t)0); }
    __device__ __forceinline__ uint32_t end(uint32_t c) const { return (uint32_t)min((int64_t)(c + 1u) * CHUNK - off, (int64_t)vocab); }
    __device__ __forceinline__ void load(uint64_t i, uint32_t end, float &xp, float &xq) const {
        xp = i < end ? logit<BF16>(row_p, i) : -CUDART_INF_F;
        xq = over_q && i < end ? logit<BF16>(row_q, i) : -CUDART_INF_F;
    }
    template <uint32_t N>
    __device__ __forceinline__ void of(const float (&xp)[N], const float (&xq)[N], uint32_t i0, uint32_t step, double (&w)[N]) const {   /* of tokens i0, i0 + step ..; by whole warps; minus infinity: nothing */
        p.of(xp, table, w);
        if (over_q) {
            double y[N];
            q.of(xq, table, y);
#pragma unroll
            for (uint32_t k = 0; k < N; k++) w[k] = fmax(__dsub_rn(__dmul_rn(w[k], scale_p), __dmul_rn(y[k], scale_q)), 0.0);   /* both rounded: equal ones leave nothing */
        } else {
#pragma unroll
            for (uint32_t k = 0; k < N; k++)
                if ((int32_t)(i0 + k * step) == certain) w[k] = 0.0;
        }
    }
};
/* by a block: the token of chunk c at which the running sum passes `left`, and its log p */
template <bool BF16>
__device__ __forceinline__ void look(const VerifyParams &P, const Weights<BF16> &W, uint32_t r, uint32_t stop, double sum_p, uint32_t c, double left) {
    __shared__ double s_scan[PICK_WARPS];
    __shared__ int32_t s_some[PICK_WARPS];
    __shared__ unsigned long long s_found;   /* the token, and below it the logit's bits */
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, i0 = W.begin(c) + tid * PICK_EACH, i1 = W.end(c);
    if (tid == 0) s_found = ~0ull;
    float xp[PICK_EACH], xq[PICK_EACH];
#pragma unroll
    for (uint32_t k = 0; k < PICK_EACH; k++) W.load((uint64_t)i0 + k, i1, xp[k], xq[k]);
    const double log_s = log(sum_p);   /* while they come */
    double w[PICK_EACH], sum = 0.0;
    int32_t some = -1;
    W.of(xp, xq, i0, 1u, w);
#pragma unroll
    for (uint32_t k = 0; k < PICK_EACH; k++) {
        sum += w[k];
        if (w[k] > 0.0) some = (int32_t)(i0 + k);
    }
    double before = warp_scan(sum);
    some = (int32_t)__reduce_max_sync(0xffffffffu, (uint32_t)(some + 1)) - 1;
    if (lane == 31u) s_scan[warp] = before;
    if (lane == 0) s_some[warp] = some;
    __syncthreads();
    before -= sum;
    for (uint32_t k = 0; k < warp; k++) before += s_scan[k];
    if (before + sum > left && sum > 0.0) {   /* the first token above it; threads behind find later ones */
        unsigned long long found = ~0ull;
#pragma unroll
        for (uint32_t k = 0; k < PICK_EACH; k++) {
            before += w[k];
            if (before > left && w[k] > 0.0 && found == ~0ull) found = (unsigned long long)(i0 + k) << 32 | __float_as_uint(xp[k]);
        }
        if (found != ~0ull) atomicMin(&s_found, found);
    }
    __syncthreads();
    if (tid == 0) {
        int32_t found = (int32_t)(s_found >> 32);
        float x = __uint_as_float((uint32_t)s_found);
        if (s_found == ~0ull) {  /* rounding, or u not below 1: the last that can be */
            for (uint32_t k = 0; k < PICK_WARPS; k++) found = max(found, s_some[k]);
            if (found >= 0) x = logit<BF16>(W.row_p, (uint32_t)found);
        }
        P.next[r] = found;
        if (P.logp) P.logp[stop] = found >= 0 ? W.p.log_p(x, log_s) : 0.f;
    }
}

template <bool BF16>
__global__ void __launch_bounds__(PICK_THREADS) q4_vf_pick_k(const VerifyParams P) {
    __shared__ Row s_p[PICK_WARPS], s_q[PICK_WARPS];
    __shared__ uint32_t s_said[PICK_WARPS], s_chunk, s_alone;
    __shared__ int32_t s_best[PICK_WARPS], s_draft[PICK_WARPS];
    __shared__ double s_left, s_part[PICK_WARPS], s_pow[32];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, r = blockIdx.x;
    /* The launch before this one began behind everything that its inputs come from: they are there.  What it writes is waited for below. */
    if (tid < 32u) s_pow[tid] = __ldg(g_vf_pow + tid);
    const int32_t a = __ldcg(P.start + r), b = __ldcg(P.start + r + 1u);
    const float T = temperature(P, r);
    const bool bounds = a >= 0 && b >= a && (uint32_t)b <= P.n_tok;
    if (!bounds || a == b) {
        q4d_pdl_wait();
        if (P.early && tid == 0) g_vf_stop[r] = 0u;
        if (P.early)
            for (int64_t t = (int64_t)max(a, 0) + tid; t < b && t < (int64_t)P.n_tok; t += PICK_THREADS) g_vf_early[t] = 0u;
        if (tid == 0) {
            if (P.draft) P.choice[r].open = 0u;
            P.accepted[r] = 0;
            P.next[r] = -1;
            if (P.keep) P.keep[r] = __ldcg(P.rows + r);
            if (!bounds) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        }
        return;
    }
    __syncthreads();             /* s_pow: all warps read what the first has put there */
    const bool greedy = T == 0.f;
    const VfStat *stat_p = P.stat, *stat_q = P.stat + (uint64_t)P.n_tok * P.chunks;
    const uint32_t last = (uint32_t)b - 1u;
    const VfScale S(T);
    const int2 table = lane_table();

    /* ---- the request's rows, a warp each: whether the draft behind a row is kept.  The first that is not, or the last row, decides */
    uint32_t stop = (uint32_t)a, said = VF_NONE;
    Row p = {}, q = {};
    int32_t best = -1, left_out = -1;   /* left_out: the draft behind the row that decides */
    bool out_of_vocab = false, waited = false;
    for (uint32_t t0 = (uint32_t)a; temperature_ok(T); t0 += PICK_WARPS) {
        const uint32_t t = t0 + warp;
        uint32_t mine = VF_KEPT;
        int32_t d = -1;
        float xp = 0.f, xq = 0.f;
        if (t <= last) {
            if (t < last) d = __ldcg(P.token + t + 1u);
            const bool in = (uint32_t)d < P.vocab, with_q = t < last && P.draft;
            /* asked for ahead of the sums */
            if (!greedy && in) xp = logit<BF16>(P.logits + t * P.ld, (uint32_t)d);
            if (!greedy && in && with_q) xq = logit<BF16>(P.draft + t * P.draft_ld, (uint32_t)d);
            const float u = !greedy && t < last ? __ldcg(P.u_accept + t) : 0.f;
            if (!waited) q4d_pdl_wait();
            waited = true;
            if (greedy) {
                mine = !best_of(stat_p + (uint64_t)t * P.chunks, P.chunks, best) ? VF_NONE : t == last ? VF_LAST : best == d ? VF_KEPT : VF_REFUSED;
            } else {
                RowOf rows[2];
                rows[0].load(stat_p + (uint64_t)t * P.chunks, P.chunks);
                rows[1].load(stat_q + (uint64_t)t * P.chunks, with_q ? P.chunks : 0u);
                if (!rows_of(rows, S, s_pow, p, q)) {
                    mine = VF_NONE;
                } else if (t == last) {
                    mine = VF_LAST;
                } else if (in) {
                    mine = said_of(xp, xq, u, p, q, with_q, S, table);
                } else {
                    mine = VF_REFUSED;
                }
                /* what the first launch went by, whichever way the sums are rounded here */
                const uint32_t word = P.early && t < last ? __ldcg(g_vf_early + t) : 0u;
                if (word & (EARLY_STOP | EARLY_KEPT)) mine = word & EARLY_KEPT ? VF_KEPT : word & EARLY_NONE ? VF_NONE : VF_REFUSED;
            }
            out_of_vocab = t < last && !in;
        }
        if (!waited) q4d_pdl_wait();
        waited = true;
        __syncthreads();
        if (lane == 0) {
            s_said[warp] = mine;
            s_p[warp] = p;
            s_q[warp] = q;
            s_best[warp] = best;
            s_draft[warp] = d;
        }
        __syncthreads();
        const uint32_t others = __ballot_sync(0xffffffffu, lane < PICK_WARPS && s_said[lane % PICK_WARPS] != VF_KEPT);
        const uint32_t n = others ? (uint32_t)__ffs((int)others) - 1u : PICK_WARPS;
        if (lane == 0 && t < last) {
            if (P.logp && warp < n) {
                VfExp E;
                E.set(p.m, S);
                P.logp[t] = greedy ? 0.f : E.log_p(xp, log(p.s));
            }
            if (out_of_vocab && warp <= n) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        }
        if (others) {
            stop = t0 + n;
            said = s_said[n];
            p = s_p[n];
            q = s_q[n];
            best = s_best[n];
            left_out = s_draft[n];
            break;
        }
    }
    if (!waited) q4d_pdl_wait();
    if (P.early && tid == 0) g_vf_stop[r] = 0u;
    if (P.early)
        for (uint32_t t = (uint32_t)a + tid; t <= last; t += PICK_THREADS) g_vf_early[t] = 0u;   /* they have been read */
    if (P.logp)
        for (uint32_t t = stop + 1u + tid; t <= last; t += PICK_THREADS) P.logp[t] = 0.f;
    const bool refused = said == VF_REFUSED && !greedy, open = refused && P.draft;
    if (tid == 0) {
        P.accepted[r] = (int32_t)(stop - (uint32_t)a);
        if (P.keep) P.keep[r] = __ldcg(P.rows + r) + (int32_t)(stop - (uint32_t)a) + 1;
        if (said == VF_NONE || greedy) {
            P.next[r] = said == VF_NONE ? -1 : best;
            if (P.logp) P.logp[stop] = 0.f;
            if (said == VF_NONE) atomicOr(P.err, (uint32_t)Q4E_RANGE);
        }
        if (P.draft && !open) P.choice[r].open = 0u;
        if (open) P.choice[r] = {S.c, S.drop, 1.0 / p.s, 1.0 / q.s, p.s, p.m, q.m, stop, 1u};
    }
    if (said == VF_NONE || greedy || open) return;

    /* ---- from p: the chunk, then the place in it.  The chunk with a certain draft that was refused is summed again without that */
    Weights<BF16> W;
    W.set(P, stop, p.m, 0.f, 1.0, 0.0, S, false, left_out);
    const uint32_t special = (uint32_t)W.certain < P.vocab ? (uint32_t)((W.certain + W.off) / CHUNK) : 0xffffffffu;
    double without = 0.0;
    if (special != 0xffffffffu) {
        const uint32_t i0 = W.begin(special) + tid, i1 = W.end(special);
        float xp[PICK_EACH], xq[PICK_EACH];
        double w[PICK_EACH];
#pragma unroll
        for (uint32_t k = 0; k < PICK_EACH; k++) W.load((uint64_t)i0 + k * PICK_THREADS, i1, xp[k], xq[k]);
        W.of(xp, xq, i0, PICK_THREADS, w);
#pragma unroll
        for (uint32_t k = 0; k < PICK_EACH; k++) without += w[k];
        without = warp_sum(without);
        if (lane == 0) s_part[warp] = without;
        __syncthreads();
        without = 0.0;
        for (uint32_t k = 0; k < PICK_WARPS; k++) without += s_part[k];
    }
    if (warp == 0) {
        const VfStat *sp = stat_p + (uint64_t)stop * P.chunks;
        const double u = (double)__ldcg(P.u_next + r);
        double left, whole;
        uint32_t at, apart = special;
        bool alone = false;
#pragma unroll 1
        for (;; apart = 0xffffffffu) {   /* nothing besides the draft: p itself */
            at = place_of(P.chunks, u, left, whole, [&](uint32_t i0, uint32_t i1, auto &w) { chunks_of(W.p, sp, s_pow, apart, without, i0, i1, w); });
            if (whole > 0.0 || apart == 0xffffffffu) break;
            alone = true;
        }
        if (lane == 0) {
            s_chunk = at;
            s_left = left;
            s_alone = alone;
        }
    }
    __syncthreads();
    if (s_alone) W.certain = -1;
    look<BF16>(P, W, r, stop, p.s, s_chunk, s_left);
}

__device__ __forceinline__ VfChoice choice_at(const VfChoice *p) {
    VfChoice D;
    const int4 *from = reinterpret_cast<const int4 *>(p);
    int4 *to = reinterpret_cast<int4 *>(&D);
#pragma unroll
    for (uint32_t i = 0; i < sizeof(VfChoice) / 16u; i++) to[i] = __ldcg(from + i);
    return D;
}
/* What p has over q is a difference of numbers that are off by 7e-9 of themselves.  Where it comes to less than this in all (a draft that p and q all but exclude was refused), both
 * rows are summed again in 64 bits, and chunk by chunk what p has over q by these sums: by a block, 1 over the sums being what comes back.  Above it what p has over q is off by a
 * thousandth of itself at most.  A draft that was drawn from q is refused so once in 65 536 at most; it costs about 230 us over 131 072 tokens (a block for both rows, twice) */
constexpr double REST_LITTLE = 1.0 / 65536.0;
template <bool BF16>
__device__ __noinline__ double2 rest_again(const VerifyParams &P, uint32_t r) {
    __shared__ double s_a[PICK_WARPS], s_b[PICK_WARPS];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const VfChoice D = choice_at(P.choice + r);
    double *rest = P.rest + (uint64_t)r * P.chunks;
    Weights<BF16> W;
    W.set(P, D.stop, D.m_p, D.m_q, 1.0, 1.0, VfScale(D.c, D.drop), true, -1);
    double2 scale = make_double2(1.0, 1.0);
#pragma unroll 1
    for (uint32_t over = 0; over < 2u; over++) {
        double a = 0.0, b = 0.0;
#pragma unroll 1
        for (uint32_t chunk = 0; chunk < P.chunks; chunk++) {
            const uint32_t i0 = W.begin(chunk) + tid, i1 = W.end(chunk);
            float xp[PICK_EACH], xq[PICK_EACH];
            double w[PICK_EACH], y[PICK_EACH];
#pragma unroll
            for (uint32_t k = 0; k < PICK_EACH; k++) W.load((uint64_t)i0 + k * PICK_THREADS, i1, xp[k], xq[k]);
            if (over) {
                W.of(xp, xq, i0, PICK_THREADS, w);
#pragma unroll
                for (uint32_t k = 0; k < PICK_EACH; k++) a += w[k];
            } else {
                W.p.of(xp, W.table, w);
                W.q.of(xq, W.table, y);
#pragma unroll
                for (uint32_t k = 0; k < PICK_EACH; k++) {
                    a += w[k];
                    b += y[k];
                }
            }
            if (!over && chunk + 1u < P.chunks) continue;
            a = warp_sum(a);
            b = warp_sum(b);
            __syncthreads();     /* what was there has been read */
            if (lane == 0) {
                s_a[warp] = a;
                s_b[warp] = b;
            }
            __syncthreads();
            a = b = 0.0;
            for (uint32_t k = 0; k < PICK_WARPS; k++) {
                a += s_a[k];
                b += s_b[k];
            }
            if (!over) {
                scale = make_double2(1.0 / a, 1.0 / b);
                W.scale_p = scale.x;
                W.scale_q = scale.y;
            } else {
                if (tid == 0) __stcg(rest + chunk, a);
                a = 0.0;
            }
        }
    }
    __syncthreads();
    return scale;
}

/* what p has over q, chunk by chunk, the next one's logits on their way meanwhile; the request's last block to finish looks for next */
template <bool BF16>
__global__ void __launch_bounds__(PICK_THREADS, 3) q4_vf_rest_k(const __grid_constant__ VerifyParams P) {
    __shared__ uint32_t s_last, s_chunk, s_over, s_little;
    __shared__ double s_left, s_part[2][PICK_WARPS], s_pow[32];
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, r = blockIdx.y, chunk0 = blockIdx.x;
    if (tid < 32u) s_pow[tid] = __ldg(g_vf_pow + tid);
    q4d_pdl_wait();
    const VfChoice D = choice_at(P.choice + r);
    if (!D.open) return;
    const uint32_t stop = D.stop;
    const VfScale S(D.c, D.drop);
    Weights<BF16> W;
    W.set(P, stop, D.m_p, D.m_q, D.scale_p, D.scale_q, S, true, -1);
    double *rest = P.rest + (uint64_t)r * P.chunks;
    float xp[PICK_EACH], xq[PICK_EACH], xp_next[PICK_EACH], xq_next[PICK_EACH];
    auto load = [&](uint32_t chunk, float (&p)[PICK_EACH], float (&q)[PICK_EACH]) {
        const uint32_t i0 = W.begin(chunk) + tid, i1 = chunk < P.chunks ? W.end(chunk) : 0u;
#pragma unroll
        for (uint32_t k = 0; k < PICK_EACH; k++) W.load((uint64_t)i0 + k * PICK_THREADS, i1, p[k], q[k]);
    };
    load(chunk0, xp, xq);
    uint32_t turn = 0;
    for (uint32_t chunk = chunk0; chunk < P.chunks; chunk += gridDim.x, turn ^= 1u) {
        load(chunk + gridDim.x, xp_next, xq_next);
        double w[PICK_EACH], x = 0.0;
        W.of(xp, xq, W.begin(chunk) + tid, PICK_THREADS, w);
#pragma unroll
        for (uint32_t k = 0; k < PICK_EACH; k++) x += w[k];
        x = warp_sum(x);
        if (lane == 0) s_part[turn][warp] = x;
        __syncthreads();         /* and the parts of two turns before have been read */
        if (warp == 0) {
            x = lane < PICK_WARPS ? s_part[turn][lane] : 0.0;
#pragma unroll
            for (uint32_t o = PICK_WARPS / 2u; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            if (lane == 0) __stcg(rest + chunk, x);
        }
#pragma unroll
        for (uint32_t k = 0; k < PICK_EACH; k++) {
            xp[k] = xp_next[k];
            xq[k] = xq_next[k];
        }
    }
    if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(&g_vf_arrived[r], 1u) == gridDim.x - 1u;
        if (s_last) g_vf_arrived[r] = 0u;
        __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
#pragma unroll 1
    for (uint32_t again = 0; again < 2u; again++) {
        if (warp == 0) {
            const double u = (double)__ldcg(P.u_next + r);
            double left, whole;
            uint32_t at = place_of(P.chunks, u, left, whole, [&](uint32_t i0, uint32_t i1, auto &w) {
#pragma unroll
                for (uint32_t k = 0; k < sizeof(w) / sizeof(w[0]); k++) w[k] = i0 + k < i1 ? __ldcg(rest + i0 + k) : 0.0;
            });
            const bool over_q = whole > 0.0, little = !again && whole < REST_LITTLE;
            if (!over_q && !little) {   /* p nowhere above q: as if none was refused */
                const VfStat *sp = P.stat + (uint64_t)stop * P.chunks;
                at = place_of(P.chunks, u, left, whole, [&](uint32_t i0, uint32_t i1, auto &w) { chunks_of(W.p, sp, s_pow, 0xffffffffu, 0.0, i0, i1, w); });
            }
            if (lane == 0) {
                s_chunk = at;
                s_left = left;
                s_over = over_q;
                s_little = little;
            }
        }
        __syncthreads();
        if (!s_little) break;
        const double2 scale = rest_again<BF16>(P, r);
        W.scale_p = scale.x;
        W.scale_q = scale.y;
    }
    W.over_q = s_over;
    look<BF16>(P, W, r, stop, D.sum_p, s_chunk, s_left);
}

template <bool BF16>
bool verify_launch(const VerifyParams &p) {
    const uint64_t warps = (uint64_t)p.levels * p.across * (p.draft ? 2u : 1u) * p.spans, blocks = (warps + VF_WARPS - 1u) / VF_WARPS;
    if (warps > 0x7fffffffu) return q4i_fail(Q4E_ARG, "verify: too many rows for one call");
    const uint32_t rest_blocks = (8u * (uint32_t)g_q4.sm_count + p.n_req - 1u) / p.n_req;   /* of a request; most have nothing to do where few drafts are refused */
    return (p.early ? q4i_launch_pdl("verify launch", q4_vf_stat_k<BF16, true>, dim3((unsigned)blocks), VF_THREADS, 0, p)
                    : q4i_launch_pdl("verify launch", q4_vf_stat_k<BF16, false>, dim3((unsigned)blocks), VF_THREADS, 0, p)) &&
           q4i_launch_pdl("verify launch", q4_vf_pick_k<BF16>, dim3(p.n_req), PICK_THREADS, 0, p) &&
           (!p.draft || q4i_launch_pdl("verify launch", q4_vf_rest_k<BF16>, dim3(rest_blocks < p.chunks ? rest_blocks : p.chunks, p.n_req), PICK_THREADS, 0, p));
}

}  // namespace

extern "C" bool q4_gpu_verify(const void *logits, int bf16, uint64_t ld, const void *draft, uint64_t draft_ld, uint32_t vocab, const int32_t *token, const int32_t *start,
                              uint32_t n_req, uint32_t n_tok, const float *temp, const float *u_accept, const float *u_next, int32_t *accepted, int32_t *next, float *logp,
                              const int32_t *rows, int32_t *keep) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "verify: library not initialised");
    Q4_REQUIRE(logits && token && start && u_accept && u_next && accepted && next && vocab && n_req && n_tok, "verify: bad argument");
    Q4_REQUIRE(!rows == !keep, "verify: rows and keep go together");
    Q4_REQUIRE(n_req <= PLAN_MAX_REQ && n_tok <= 0x3fffffffu && vocab <= 0x3fffffffu, "verify: at most 8192 requests, 2^30 - 1 rows and tokens");
    Q4_REQUIRE(n_tok == 1u || (ld >= vocab && (!draft || draft_ld >= vocab)), "verify: rows are closer than the vocabulary is wide");
    Q4_REQUIRE(ld < 1ull << 40 && draft_ld < 1ull << 40, "verify: rows are too far apart");
    Q4_REQUIRE(((uintptr_t)logits & (bf16 ? 1u : 3u)) == 0 && ((uintptr_t)draft & (bf16 ? 1u : 3u)) == 0, "verify: logits are not aligned to their type");
    VerifyParams p = {};
    const uint64_t size = bf16 ? 2u : 4u;
    p.logits = (const uint8_t *)logits; p.draft = (const uint8_t *)draft; p.ld = ld * size; p.draft_ld = draft_ld * size; p.vocab = vocab;
    p.chunks = (uint32_t)((vocab + 16u / size - 1u + CHUNK - 1u) / CHUNK);   /* wherever in a 16-byte piece a row begins */
    /* A warp's chunks: as many as leave a round and a half of warps (24 on an SM at once), so that the search for the request and the scale are done once for them: 48 x 5
     * drafts over 131 072 tokens 105 us with three, 101 with six, 103 with nine.  A draft row is counted for every token: those behind a request's last one, which are
     * not read, are known on the device alone.  256 draws over 32 003 tokens come to three with a tensor of draft logits beside them (22.5 us, 26.5 with one; half of the
     * warps leave at once, the others fill 0.8 of a round) and to one without it (22.7). */
    const uint64_t all = (uint64_t)n_tok * (draft ? 2u : 1u) * p.chunks, share = all / (36u * (uint64_t)g_q4.sm_count);
    p.span = share < 1u ? 1u : share < SPAN ? (uint32_t)share : SPAN;
    p.spans = (p.chunks + p.span - 1u) / p.span;
    /* Rows behind refused drafts can be spared where warps come in several rounds; finding out costs a warp a fence and an atomic, and is of no use to the rows of the last two
     * rounds, which are under way by then.  us, without and with: 256 requests with 8 looked-up drafts, most of them refused, over 50 001 tokens (5.8 rounds) 101 and 54,
     * 64 with 8 drafts, most of them kept, over 131 072 (7 rounds) 153 and 140, 48 with 5 (3.6 rounds) 95.4 and 96.0 */
    const uint64_t warps_of = (uint64_t)p.spans * (draft ? 2u : 1u), at_once = STAT_BLOCKS * VF_WARPS * (uint64_t)g_q4.sm_count;
    p.early = n_tok > n_req && n_tok <= EARLY_MAX && n_tok * warps_of > 4u * at_once ? n_tok - (uint32_t)(2u * at_once / warps_of) : 0u;
    p.levels = p.early ? (n_tok + n_req - 1u) / n_req : 1u;
    p.across = (n_tok + p.levels - 1u) / p.levels;
    p.n_req = n_req; p.n_tok = n_tok; p.token = token; p.start = start; p.temp = temp; p.u_accept = u_accept; p.u_next = u_next;
    p.accepted = accepted; p.next = next; p.logp = logp; p.rows = rows; p.keep = keep;
    p.err = g_q4.err_d;
    const uint64_t stats = all, rests = draft ? (uint64_t)n_req * p.chunks : 0u, choices = draft ? n_req : 0u;
    if (!q4i_scratch((size_t)(stats * 4u + rests * 2u + choices * (sizeof(VfChoice) / 4u)), 0)) return false;
    p.stat = (VfStat *)g_q4.part;
    p.choice = (VfChoice *)(p.stat + stats);
    p.rest = (double *)(p.choice + choices);
    return bf16 ? verify_launch<true>(p) : verify_launch<false>(p);
}
