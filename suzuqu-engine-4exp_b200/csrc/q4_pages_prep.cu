/*
 * The projections of a step's tokens made ready for the paged attention: norm of every query and key head, rotation by the token's own
 * position, the gates split off, keys and values into the pages.  (q4_prep.cu does the like for one session, whose tokens lie one
 * behind the other.)
 *
 *     y = x / sqrt(mean x^2 + eps) * w;  (a, b) -> mag (a cos - b sin, a sin + b cos), the angle of pair i being pos * f_i
 *
 * The angle is the part of pos * f_i behind the last whole turn.  f_i is kept in turns as a fraction of 2^64, so that the product with
 * the position, modulo 2^64, is that part exactly: an fp32 angle is off by 0.008 at position 262 144, by half a turn at 2^26.
 *
 * Bound by memory: every value is read once and written once.
 */
#include <math.h>
#include <string.h>

#include "q4_paged.h"

namespace {

constexpr uint32_t PREP_THREADS = 256, PREP_WARPS = PREP_THREADS / 32u;

struct PrepParams {
    uint8_t *mem;                /* of the layer */
    uint32_t n_head, n_kvh, n_tok, page_shift;
    uint32_t slots;              /* n_pages << page_shift */
    uint32_t q_bf16;             /* the type of q_out */
    uint32_t jobs, per;          /* of a token: pairs of rows (query and gate, K and V), in groups of lanes; of a block */
    const void *q, *k, *v;
    uint64_t q_stride, kv_stride;
    const float *wq, *wk;
    float eps;
    const int32_t *pos, *slot;
    void *q_out;
    float *gate;
    uint32_t *err;
    q4_gpu_rope rope;
};

/* four values of a row, as they lie */
template <bool BF16>
struct Four {
    typename std::conditional<BF16, uint2, float4>::type x;
    __device__ __forceinline__ void load(const void *base, uint64_t at) {
        if constexpr (BF16) x = __ldcs(reinterpret_cast<const uint2 *>(reinterpret_cast<const __nv_bfloat16 *>(base) + at));
        else x = __ldcs(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(base) + at));
    }
    __device__ __forceinline__ void none() {
        if constexpr (BF16) x = make_uint2(0u, 0u);
        else x = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __device__ __forceinline__ float4 get() const {
        if constexpr (BF16)
            return make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u));
        else return x;
    }
};
__device__ __forceinline__ uint2 to_bf16(float4 x) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

/* A row lies in LPR lanes, CH groups of four dims each, 128 dims apart: the eight lanes of a q8_0 block are neighbours at every head size, and
 * at hd 64 a warp has two rows.  A job is a query row and its gate, or a K row and its V: both are on their way at once. */
template <int KIND, int HD, bool BF16, uint32_t TOK>
__global__ void __launch_bounds__(PREP_THREADS) q4_pg_prep_k(const __grid_constant__ PrepParams P) {
    constexpr uint32_t LPR = HD == 64 ? 16u : 32u, RPW = 32u / LPR, CH = HD / (4u * LPR);
    __shared__ float4 cs[TOK][64];       /* (cos, sin) of two pairs */
    const uint32_t tid = threadIdx.x, lane = tid & 31u, in = lane % LPR;
    const uint32_t np = P.rope.n_rot / 2u, t0 = blockIdx.x * TOK;
    q4d_pdl_wait();
    for (uint32_t i = tid; i < TOK * np; i += PREP_THREADS) {
        const uint32_t t = TOK == 1u ? 0u : i / np, pair = i - t * np;
        const int32_t pos = t0 + t < P.n_tok ? __ldcg(P.pos + t0 + t) : 0;
        const uint64_t angle = (uint64_t)(uint32_t)pos * P.rope.turn[pair];
        float s, c;
        sincospif((float)(int32_t)(angle >> 32) * 4.656612873077393e-10f, &s, &c);   /* 2^-31: half turns */
        reinterpret_cast<float2 *>(cs[t])[pair] = make_float2(c * P.rope.mag, s * P.rope.mag);
    }
    __syncthreads();
    const uint32_t j0 = blockIdx.y * P.per, j1 = min(j0 + P.per, P.jobs), n_jobs = (j1 - j0) * TOK;
    for (uint32_t g = (tid >> 5) * RPW + lane / LPR; g - lane / LPR < n_jobs; g += PREP_WARPS * RPW) {   /* the lanes of a warp stay together */
        const uint32_t t = TOK == 1u ? 0u : g / (j1 - j0), job = j0 + g - t * (j1 - j0), tok = t0 + t;
        const bool is_q = job < P.n_head, mine = g < n_jobs && tok < P.n_tok;
        const uint32_t head = is_q ? job : job - P.n_head;
        const int32_t pos = mine ? __ldcg(P.pos + tok) : -1;
        const bool live = pos >= 0;
        Four<BF16> a[CH], b[CH];
        const uint64_t at = is_q ? tok * P.q_stride + (uint64_t)head * (P.gate ? 2u * HD : HD) : tok * P.kv_stride + (uint64_t)head * HD;
#pragma unroll
        for (uint32_t c = 0; c < CH; c++) {
            const uint32_t d = c * 128u + in * 4u;
            a[c].none(); b[c].none();
            if (live) {
                a[c].load(is_q ? P.q : P.k, at + d);
                if (!is_q) b[c].load(P.v, at + d);
                else if (P.gate) b[c].load(P.q, at + HD + d);
            }
        }
        const float *wn = is_q ? P.wq : P.wk;
        float4 x[CH];
#pragma unroll
        for (uint32_t c = 0; c < CH; c++) x[c] = a[c].get();
        if (P.eps >= 0.f) {
            float ss = 0.f;
#pragma unroll
            for (uint32_t c = 0; c < CH; c++) ss += x[c].x * x[c].x + x[c].y * x[c].y + x[c].z * x[c].z + x[c].w * x[c].w;
#pragma unroll
            for (uint32_t o = LPR / 2u; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = 1.f / sqrtf(ss * (1.f / HD) + P.eps);
#pragma unroll
            for (uint32_t c = 0; c < CH; c++) {
                const float4 w = wn ? __ldg(reinterpret_cast<const float4 *>(wn + c * 128u) + in) : make_float4(1.f, 1.f, 1.f, 1.f);
                x[c].x *= r * w.x; x[c].y *= r * w.y; x[c].z *= r * w.z; x[c].w *= r * w.w;
            }
        }
        /* the rotation */
        if (!P.rope.half) {
#pragma unroll
            for (uint32_t c = 0; c < CH; c++) {
                const uint32_t grp = c * 32u + in;
                if (grp * 4u < P.rope.n_rot) {
                    const float4 k = cs[t][grp];
                    const float4 y = x[c];
                    const bool both = grp * 4u + 2u < P.rope.n_rot;
                    x[c].x = y.x * k.x - y.y * k.y; x[c].y = y.x * k.y + y.y * k.x;
                    if (both) { x[c].z = y.z * k.z - y.w * k.w; x[c].w = y.z * k.w + y.w * k.z; }
                }
            }
        } else if (np) {
            const uint32_t half = np / 4u;   /* groups of four dims */
            float4 y[CH];
#pragma unroll
            for (uint32_t c = 0; c < CH; c++) {
                const uint32_t grp = c * 32u + in, other = grp < half ? grp + half : grp - half, from = (lane & ~(LPR - 1u)) + (other & (LPR - 1u));
#pragma unroll
                for (uint32_t s = 0; s < CH; s++) {
                    const float4 z = make_float4(__shfl_sync(0xffffffffu, x[s].x, from), __shfl_sync(0xffffffffu, x[s].y, from), __shfl_sync(0xffffffffu, x[s].z, from), __shfl_sync(0xffffffffu, x[s].w, from));
                    if (s == 0u || other / LPR == s) y[c] = z;
                }
            }
#pragma unroll
            for (uint32_t c = 0; c < CH; c++) {
                const uint32_t grp = c * 32u + in;
                if (grp < 2u * half) {
                    const uint32_t i = (grp < half ? grp : grp - half) * 2u;
                    const float4 k0 = cs[t][i], k1 = cs[t][i + 1u];
                    const float sign = grp < half ? -1.f : 1.f;
                    x[c].x = x[c].x * k0.x + sign * (y[c].x * k0.y); x[c].y = x[c].y * k0.z + sign * (y[c].y * k0.w);
                    x[c].z = x[c].z * k1.x + sign * (y[c].z * k1.y); x[c].w = x[c].w * k1.z + sign * (y[c].w * k1.w);
                }
            }
        }
        if (is_q) {
            if (live) {
                const uint64_t to = ((uint64_t)tok * P.n_head + head) * HD + in * 4u;
#pragma unroll
                for (uint32_t c = 0; c < CH; c++) {
                    if (P.q_bf16) *reinterpret_cast<uint2 *>(reinterpret_cast<__nv_bfloat16 *>(P.q_out) + to + c * 128u) = to_bf16(x[c]);
                    else *reinterpret_cast<float4 *>(reinterpret_cast<float *>(P.q_out) + to + c * 128u) = x[c];
                    if (P.gate) *reinterpret_cast<float4 *>(P.gate + to + c * 128u) = b[c].get();
                }
            }
        }
        if (RPW > 1u || !is_q) {
            const int32_t slot = live && !is_q ? __ldcg(P.slot + tok) : -1;
            const bool store = slot >= 0 && (uint32_t)slot < P.slots;
            if (slot >= 0 && !store && in == 0u) atomicOr(P.err, (uint32_t)Q4E_RANGE);
            const uint32_t page = (uint32_t)(store ? slot : 0) >> P.page_shift, row = (uint32_t)(store ? slot : 0) & ((1u << P.page_shift) - 1u), r16 = row & 15u;
            uint8_t *tile = P.mem + ((((uint64_t)page * P.n_kvh + head) << (P.page_shift - 4u)) + (row >> 4)) * PgTile<KIND, HD>::BYTES;
#pragma unroll
            for (uint32_t w = 0; w < 2u; w++)
#pragma unroll
                for (uint32_t c = 0; c < CH; c++) {
                    const float4 y = w ? b[c].get() : x[c];
                    const uint32_t d = c * 128u + in * 4u;
                    if constexpr (KIND == Q4K_Q8) {
                        float s, id;
                        q4d_block_scale(y, s, id);
                        if (store) {
                            uint8_t *rec = tile + r16 * PgTile<KIND, HD>::ROW;
                            *reinterpret_cast<uint32_t *>(rec + w * HD + d) = q4d_quant4(y, id);
                            if ((in & 7u) == 0u) reinterpret_cast<__half *>(rec + 2u * HD)[w * (HD / 32u) + (d >> 5)] = __float2half_rn(s);
                        }
                    } else if (store) {
                        const __half2 h0 = __floats2half2_rn(y.x, y.y), h1 = __floats2half2_rn(y.z, y.w);
                        uint8_t *dst = tile + w * (PgTile<KIND, HD>::BYTES / 2u) + (d >> 6) * 2048u + r16 * 128u + ((((d >> 3) & 7u) ^ (r16 & 7u)) << 4) + (d & 4u) * 2u;
                        *reinterpret_cast<uint2 *>(dst) = make_uint2(*reinterpret_cast<const uint32_t *>(&h0), *reinterpret_cast<const uint32_t *>(&h1));
                    }
                }
        }
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0u; }

template <int KIND, int HD, bool BF16>
bool prep_launch(PrepParams &p) {
    const uint32_t sms = (uint32_t)g_q4.sm_count;
    if (p.n_tok >= 4u * sms) {
        p.per = p.jobs;
        return q4i_launch_pdl("pages_prep launch", q4_pg_prep_k<KIND, HD, BF16, 4>, dim3((p.n_tok + 3u) / 4u), PREP_THREADS, 0, p);
    }
    const uint32_t one = PREP_WARPS * (HD == 64 ? 2u : 1u);   /* few tokens: a job per group of lanes */
    p.per = p.n_tok < sms ? one : p.jobs;
    return q4i_launch_pdl("pages_prep launch", q4_pg_prep_k<KIND, HD, BF16, 1>, dim3(p.n_tok, (p.jobs + p.per - 1u) / p.per), PREP_THREADS, 0, p);
}

}  // namespace

extern "C" bool q4_gpu_rope_set(q4_gpu_rope *r, uint32_t n_rot, int half, double base, int scaling, double factor, double orig, double fast, double slow, double mag) {
    const double two_pi = 6.283185307179586476925286766559;
    const bool scaled = scaling >= 1 && scaling <= 3;
    Q4_REQUIRE(r && n_rot <= 256 && n_rot % 2u == 0 && (!half || n_rot % 8u == 0), "rope_set: n_rot must be even, up to 256, and a multiple of 8 for halves");
    Q4_REQUIRE(base > 0.0 && isfinite(base) && mag > 0.0 && isfinite((float)mag), "rope_set: base and mag must be above 0");
    Q4_REQUIRE(scaling == 0 || scaled, "rope_set: scaling is 0 to 3");
    Q4_REQUIRE(!scaled || (factor > 0.0 && isfinite(factor)), "rope_set: factor must be above 0");
    Q4_REQUIRE(scaling < 2 || (base > 1.0 && orig > 0.0 && isfinite(orig) && slow > 0.0 && fast > slow && isfinite(fast)), "rope_set: base above 1, orig above 0, fast above slow above 0");
    memset(r, 0, sizeof(*r));
    r->n_rot = n_rot;
    r->half = half != 0;
    r->mag = (float)mag;
    const uint32_t np = n_rot / 2u;
    /* the pair that turns so many times in orig positions */
    auto pair_of = [&](double turns) { return np * log(orig / (turns * two_pi)) / log(base); };
    const double lo = scaling == 2 ? fmax(0.0, floor(pair_of(fast))) : 0.0, hi = scaling == 2 ? fmin((double)np - 1.0, ceil(pair_of(slow))) : 0.0;
    for (uint32_t i = 0; i < np; i++) {
        double f = pow(base, -2.0 * i / n_rot);
        double s = 0.0;   /* how far it is slowed down */
        if (scaling == 1) s = 1.0;
        if (scaling == 2) s = fmin(1.0, fmax(0.0, (i - lo) / fmax(hi - lo, 0.001)));
        if (scaling == 3) s = 1.0 - fmin(1.0, fmax(0.0, (f * orig / two_pi - slow) / (fast - slow)));
        f = f * (1.0 - s) + f / factor * s;
        if (scaling == 0) f = pow(base, -2.0 * i / n_rot);
        /* turns per position: whole ones make no difference at whole positions */
        double turns = f / two_pi;
        Q4_REQUIRE(isfinite(turns), "rope_set: a frequency is not finite");
        turns -= floor(turns);
        const double high = floor(turns * 4294967296.0), low = (turns * 4294967296.0 - high) * 4294967296.0;
        r->turn[i] = ((uint64_t)high << 32) + (uint64_t)(low + 0.5);
    }
    return true;
}

extern "C" bool q4_gpu_pages_prep(const q4_gpu_pages *pg, uint32_t layer, const void *q, const void *k, const void *v, int in_bf16, uint64_t q_stride,
                                  uint64_t kv_stride, uint32_t n_head, const float *wq, const float *wk, float eps, const q4_gpu_rope *rope, const int32_t *pos,
                                  const int32_t *slot, uint32_t n_tok, void *q_out, int q_out_bf16, float *gate) {
    if (!g_q4.ok) return q4i_fail(Q4E_INIT, "pages_prep: library not initialised");
    Q4_REQUIRE(q4i_pages_ok(pg) && pg->mem && aligned16(pg->mem) && layer < pg->n_layers, "pages_prep: bad pool or layer");
    Q4_REQUIRE(q && k && v && rope && pos && slot && q_out && n_tok && n_head && n_head <= 65536, "pages_prep: bad argument");
    Q4_REQUIRE(n_tok <= 0x7fffffffu, "pages_prep: at most 2^31 - 1 tokens");
    Q4_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(gate) && aligned16(wq) && aligned16(wk), "pages_prep: rows and weights must be 16-byte aligned");
    const uint64_t per16 = in_bf16 ? 8u : 4u;
    Q4_REQUIRE(q_stride % per16 == 0 && kv_stride % per16 == 0 && q_stride < 1ull << 40 && kv_stride < 1ull << 40, "pages_prep: row strides must be multiples of 16 bytes");
    Q4_REQUIRE(n_tok == 1u || (q_stride >= (uint64_t)n_head * pg->hd * (gate ? 2u : 1u) && kv_stride >= (uint64_t)pg->n_kvh * pg->hd), "pages_prep: row strides are smaller than the rows");
    Q4_REQUIRE(rope->n_rot <= pg->hd && rope->n_rot % 2u == 0 && (!rope->half || rope->n_rot % 8u == 0), "pages_prep: more dims to rotate than a head has");
    Q4_REQUIRE(eps == eps, "pages_prep: eps is not a number");
    PrepParams p = {};
    p.mem = (uint8_t *)pg->mem + (uint64_t)layer * (q4i_pages_row_bytes(pg->hd, pg->kind) * pg->page_rows * pg->n_kvh) * pg->n_pages;
    p.n_head = n_head; p.n_kvh = pg->n_kvh; p.n_tok = n_tok;
    p.page_shift = (uint32_t)__builtin_ctz(pg->page_rows);
    p.slots = pg->n_pages << p.page_shift;
    p.q_bf16 = q_out_bf16 != 0;
    p.jobs = n_head + pg->n_kvh;
    p.q = q; p.k = k; p.v = v; p.q_stride = q_stride; p.kv_stride = kv_stride;
    p.wq = wq; p.wk = wk; p.eps = eps;
    p.pos = pos; p.slot = slot; p.q_out = q_out; p.gate = gate;
    p.err = g_q4.err_d;
    p.rope = *rope;
#define PG_PREP(KIND, HD) \
    if (pg->kind == KIND && pg->hd == HD) return in_bf16 ? prep_launch<KIND, HD, true>(p) : prep_launch<KIND, HD, false>(p);
    PG_PREP(Q4K_Q8, 64) PG_PREP(Q4K_Q8, 128) PG_PREP(Q4K_Q8, 256) PG_PREP(Q4K_F16, 64) PG_PREP(Q4K_F16, 128) PG_PREP(Q4K_F16, 256)
#undef PG_PREP
    return q4i_fail(Q4E_ARG, "pages_prep: bad pool");
}
