/*
 * The projections of a step's tokens made ready for the paged attention: norm of every query and key head, rotation by the token's own
 * position, the gates split off, keys and values into the pages.  (q4_prep.cu does the like for one session, whose tokens lie one
 * behind the other.)
 *
 *     y = x / sqrt(mean x^2 + eps) * w;  (a, b) -> mag (a cos - b sin, a sin + b cos), the angle of pair i being pos * f_i
 *
 * The angle is the part of pos * f_i behind the last whole turn.  f_i is kept in turns as a fraction of 2^64, so that the product with
 * the position, modulo 2^64, is that part exactly; sine and cosine are taken of it rounded to fp32, 2^-26 of a turn off at most at any position.  An angle
 * in fp32 throughout is off by 0.008 at position 262 144, by half a turn at 2^26.
 *
 * Bound by memory: every value is read once and written once.  4096 tokens of 24 gated heads of 256 in fp32, 373 MB, take 62 us (92 % of a copy's rate); 16 001 fused
 * bf16 rows of 32 heads of 128 with 8 kv heads, 394 MB, 75 us (80 %), there beside the issue slots.
 */
#include <math.h>
#include <string.h>

#include "q4_paged.h"
#include "q4_tc.h"

namespace {

using namespace q4tc;

/* Warps differ in their turns: a block of several would keep its place for the longest (16 001 fused rows 78 us, in pairs 99, in eights 115).  28 of them on an SM, by 72 registers (forms
 * that take bf16, and halves of fp32, spill up to 32 bytes, neighbours of fp32 none): 8192 fused rows of 16 heads 31.6 us, 33.5 with up to 96; 32 of them are slower for few tokens (700 tokens of 32 heads 9.2 us, 8.4) */
constexpr uint32_t PREP_THREADS = 32, PREP_BLOCKS = 28;

struct PrepParams {
    uint8_t *mem;                /* of the layer */
    uint32_t n_head, n_kvh, n_tok, page_shift;
    uint32_t slots;              /* n_pages << page_shift */
    uint32_t q_bf16;             /* the type of q_out */
    uint32_t q_units, units;     /* warps of a token: those for its queries (and gates), then those for its keys and values */
    uint32_t q_per, kv_per;      /* turns of each; a turn is a row, and its gate or value, per group of lanes */
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

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

/* eight values of a row, as they lie, the second four of them `apart` bytes behind the first where SPLIT */
template <bool BF16, bool SPLIT>
struct Eight {
    uint4 x[BF16 ? 1 : 2];
    __device__ __forceinline__ void load(const uint8_t *p, uint32_t apart, bool live) {
        if constexpr (BF16 && SPLIT) {
            const uint2 none = make_uint2(0u, 0u), a = live ? __ldcs(reinterpret_cast<const uint2 *>(p)) : none, b = live ? __ldcs(reinterpret_cast<const uint2 *>(p + apart)) : none;
            x[0] = make_uint4(a.x, a.y, b.x, b.y);
        } else {
#pragma unroll
            for (int i = 0; i < (BF16 ? 1 : 2); i++) x[i] = live ? __ldcs(reinterpret_cast<const uint4 *>(p + (i ? SPLIT ? apart : 16u : 0u))) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    __device__ __forceinline__ void get(uint64_t (&f)[4]) const {   /* two by two */
        const uint32_t *u = reinterpret_cast<const uint32_t *>(x);
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = BF16 ? pack2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u)) : pack2(__uint_as_float(u[BF16 ? 0 : 2 * i]), __uint_as_float(u[BF16 ? 0 : 2 * i + 1]));
    }
};
__device__ __forceinline__ float4 four_floats(const float *p) { return __ldg(reinterpret_cast<const float4 *>(p)); }
__device__ __forceinline__ float4 four(uint64_t a, uint64_t b) {
    const float2 x = unpack2(a), y = unpack2(b);
    return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ uint32_t bf16s(uint64_t x) {
    const float2 f = unpack2(x);
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

/* 1 / sqrt(mean x^2 + eps) of a row that LPR lanes hold: 2 units in the last place at most */
template <uint32_t LPR>
__device__ __forceinline__ float norm_of(const uint64_t (&x)[4], float eps) {
    uint64_t s = mul2(x[0], x[0]);
#pragma unroll
    for (int i = 1; i < 4; i++) s = fma2(x[i], x[i], s);
    const float2 two = unpack2(s);
    float ss = two.x + two.y;
#pragma unroll
    for (uint32_t o = LPR / 2u; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return rsqrtf(fmaf(ss, 1.f / (LPR * 8u), eps));
}
/* What dims become: r (x fa + y fb), y the pairs' other dims.  Both hold the weights.  on: the twos that are turned; of the others r x fa alone, as the other dim may be infinite */
template <bool FULL>
__device__ __forceinline__ void turn(uint64_t (&x)[4], const uint64_t (&y)[4], const uint64_t (&fa)[4], const uint64_t (&fb)[4], uint32_t on, float r) {
    const uint64_t rr = pack2(r, r);
    uint64_t out[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint64_t z = mul2(x[i], fa[i]), turned = fma2(y[i], fb[i], z);
        out[i] = mul2(rr, FULL || (on >> i) & 1u ? turned : z);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = out[i];
}

/*
 * A warp has a token's queries, or its keys and values, or a part of them where there are few tokens, and keeps what belongs to the token in registers:
 * sines and cosines, with the weights in them.  Lanes hold eight dims of a row each, so that a warp has 1, 2 or 4 rows at a time (hd 256, 128, 64).  The
 * warps' issue slots set the pace beside memory (16 001 rows of a fused bf16 projection 169 us with four dims per lane).  A turn's rows are requested
 * before the one before them is worked at, the first before the token's position is there.  Where pairs lie in two halves a lane has four dims of a query's each and no
 * other needs them; keys are stored by 16 bytes or quantised by 32 dims, and pass the other dim on between lanes.
 */
template <int KIND, int HD, bool BF16, bool HALF, bool FULL>
__global__ void __launch_bounds__(PREP_THREADS, PREP_BLOCKS) q4_pg_prep_k(const __grid_constant__ PrepParams P) {
    constexpr uint32_t LPR = HD / 8u, RPW = 32u / LPR, U = BF16 ? 2u : 1u, SIZE = BF16 ? 2u : 4u;   /* U: turns at a time, as many bytes on their way in either type */
    const uint32_t lane = threadIdx.x, in = lane % LPR, sub = lane / LPR, unit = blockIdx.x;
    const uint32_t tok = unit / P.units, which = unit - tok * P.units;
    const uint32_t n_rot = P.rope.n_rot, np = n_rot / 2u, quarter = np / 4u;   /* of halves: groups of four dims that have their other ones as many groups behind */
    /* The warp's lanes take the sines and cosines of the head's pairs, C consecutive ones each, for one another */
    constexpr uint32_t C = HD / 64u;
    float cs[C], sn[C];
    auto angles = [&](int32_t pos) {
        const uint64_t *turns;             /* as memory: the lanes' addresses differ, which the constant port takes one by one */
        asm("mov.u64 %0, %1;" : "=l"(turns) : "l"(P.rope.turn));
#pragma unroll
        for (uint32_t i = 0; i < C; i++) {
            const uint64_t angle = (uint64_t)(uint32_t)pos * turns[lane * C + i];
            sincospif((float)(int32_t)(angle >> 32) * 4.656612873077393e-10f, &sn[i], &cs[i]);   /* 2^-31: half turns */
            cs[i] *= P.rope.mag;
            sn[i] *= P.rope.mag;
        }
    };
    auto pair_at = [&](uint32_t pair, uint32_t i, float &c, float &s) {   /* of pair + i, pair a multiple of C; by the whole warp */
        const uint32_t holder = ((pair + i) / C) & 31u;
        c = __shfl_sync(0xffffffffu, cs[i % C], holder);
        s = __shfl_sync(0xffffffffu, sn[i % C], holder);
    };
    uint64_t fa[4], fb[4], x[4];
    uint32_t on = 0;
    auto interleaved = [&](const float *wn) {
        float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        if (wn) {
            *reinterpret_cast<float4 *>(w) = four_floats(wn + in * 8u);
            *reinterpret_cast<float4 *>(w + 4) = four_floats(wn + in * 8u + 4u);
        }
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            float c, s;
            pair_at(in * 4u, i, c, s);
            const bool turns = FULL || in * 4u + i < np;
            fa[i] = turns ? pack2(w[2 * i] * c, w[2 * i + 1] * c) : pack2(w[2 * i], w[2 * i + 1]);
            fb[i] = pack2(w[2 * i + 1] * -s, w[2 * i] * s);
            on |= turns ? 1u << i : 0u;
        }
    };
    auto other_of_two = [&](uint64_t (&y)[4]) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            const float2 f = unpack2(x[i]);
            y[i] = pack2(f.y, f.x);
        }
    };
    q4d_pdl_wait();
    const int32_t pos = __ldcg(P.pos + tok);

    if (which < P.q_units) {
        const uint32_t first = which * P.q_per * RPW + sub, behind = min(first - sub + P.q_per * RPW, P.n_head);
        /* the lane's groups of four dims: both sides of its pairs, and those that are not turned as they lie; else next to one another */
        const uint32_t g0 = HALF && in < quarter ? in : in * 2u, g1 = HALF && in < quarter ? in + quarter : in * 2u + 1u, apart = (g1 - g0) * (4u * SIZE);
        const uint32_t width = HD * (P.gate ? 2u : 1u), step = RPW * width * SIZE;
        const uint8_t *pa = (const uint8_t *)P.q + (tok * P.q_stride + (uint64_t)first * width + g0 * 4u) * SIZE, *pb = (const uint8_t *)P.q + (tok * P.q_stride + (uint64_t)first * width + HD + in * 8u) * SIZE;
        Eight<BF16, HALF> a[U], a_next[U];
        Eight<BF16, false> b[U], b_next[U];
        auto load = [&](uint32_t head, Eight<BF16, HALF> (&x)[U], Eight<BF16, false> (&y)[U]) {
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                const bool live = head + u * RPW < behind;
                x[u].load(pa, apart, live);
                if (P.gate) y[u].load(pb, 0u, live);
                pa += step;
                pb += step;
            }
        };
        load(first, a, b);
        if (pos < 0) return;
        angles(pos);
        const float *wn = P.eps >= 0.f ? P.wq : nullptr;
        if constexpr (HALF) {
            float4 w0 = make_float4(1.f, 1.f, 1.f, 1.f), w1 = w0;
            if (wn) {
                w0 = four_floats(wn + g0 * 4u);
                w1 = four_floats(wn + g1 * 4u);
            }
            const bool turns = FULL || in < quarter;
            float c[4], s[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                pair_at(in * 4u, i, c[i], s[i]);
                if (!turns) c[i] = 1.f;
            }
            fa[0] = pack2(w0.x * c[0], w0.y * c[1]);
            fa[1] = pack2(w0.z * c[2], w0.w * c[3]);
            fa[2] = pack2(w1.x * c[0], w1.y * c[1]);
            fa[3] = pack2(w1.z * c[2], w1.w * c[3]);
            fb[0] = pack2(w1.x * -s[0], w1.y * -s[1]);
            fb[1] = pack2(w1.z * -s[2], w1.w * -s[3]);
            fb[2] = pack2(w0.x * s[0], w0.y * s[1]);
            fb[3] = pack2(w0.z * s[2], w0.w * s[3]);
            on = turns ? 0xfu : 0u;
        } else {
            interleaved(wn);
        }
        for (uint32_t head0 = first; head0 - sub < behind; head0 += RPW * U) {
            load(head0 + RPW * U, a_next, b_next);
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                const uint32_t head = head0 + u * RPW;
                if (head - sub >= behind) break;
                a[u].get(x);
                const float r = P.eps >= 0.f ? norm_of<LPR>(x, P.eps) : 1.f;
                uint64_t y[4];
                if constexpr (HALF) {
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++) y[i] = x[i ^ 2u];
                } else {
                    other_of_two(y);
                }
                turn<FULL>(x, y, fa, fb, on, r);
                if (head >= behind) continue;
                const uint64_t to = ((uint64_t)tok * P.n_head + head) * HD;
                if (P.q_bf16) {
                    __nv_bfloat16 *out = reinterpret_cast<__nv_bfloat16 *>(P.q_out) + to + g0 * 4u;
                    if constexpr (HALF) {
                        *reinterpret_cast<uint2 *>(out) = make_uint2(bf16s(x[0]), bf16s(x[1]));
                        *reinterpret_cast<uint2 *>(out + (g1 - g0) * 4u) = make_uint2(bf16s(x[2]), bf16s(x[3]));
                    } else {
                        *reinterpret_cast<uint4 *>(out) = make_uint4(bf16s(x[0]), bf16s(x[1]), bf16s(x[2]), bf16s(x[3]));
                    }
                } else {
                    float *out = reinterpret_cast<float *>(P.q_out) + to + g0 * 4u;
                    *reinterpret_cast<float4 *>(out) = four(x[0], x[1]);
                    *reinterpret_cast<float4 *>(out + (g1 - g0) * 4u) = four(x[2], x[3]);
                }
                if (P.gate) {
                    b[u].get(x);
                    float *out = P.gate + to + in * 8u;
                    *reinterpret_cast<float4 *>(out) = four(x[0], x[1]);
                    *reinterpret_cast<float4 *>(out + 4) = four(x[2], x[3]);
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                a[u] = a_next[u];
                b[u] = b_next[u];
            }
        }
        return;
    }

    const uint32_t first = (which - P.q_units) * P.kv_per * RPW + sub, behind = min(first - sub + P.kv_per * RPW, P.n_kvh);
    constexpr uint32_t step = RPW * HD * SIZE;
    const uint64_t at = (tok * P.kv_stride + (uint64_t)first * HD + in * 8u) * SIZE;
    const uint8_t *pa = (const uint8_t *)P.k + at, *pb = (const uint8_t *)P.v + at;
    Eight<BF16, false> a[U], b[U], a_next[U], b_next[U];
    auto load = [&](uint32_t head, Eight<BF16, false> (&x)[U], Eight<BF16, false> (&y)[U]) {
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const bool live = head + u * RPW < behind;
            x[u].load(pa, 0u, live);
            y[u].load(pb, 0u, live);
            pa += step;
            pb += step;
        }
    };
    load(first, a, b);
    if (pos < 0) return;
    angles(pos);
    const uint32_t swap = quarter & 1u;
    uint32_t from[2] = {0u, 0u};           /* halves: the lanes where the other dims of the lane's two groups of four lie, in which of its groups is the same for all lanes */
    const float *wn = P.eps >= 0.f ? P.wk : nullptr;
    if constexpr (HALF) {
#pragma unroll
        for (uint32_t s = 0; s < 2u; s++) {
            const uint32_t g = in * 2u + s, other = g < quarter ? g + quarter : g - quarter;
            const bool turns = FULL || g < 2u * quarter;
            from[s] = sub * LPR + ((other >> 1) & (LPR - 1u));
            float4 w = make_float4(1.f, 1.f, 1.f, 1.f), v = w;
            if (wn) {
                w = four_floats(wn + g * 4u);
                if (turns) v = four_floats(wn + other * 4u);
            }
            float c[4], d[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                pair_at((g < quarter ? g : other) * 4u, i, c[i], d[i]);
                if (!turns) c[i] = 1.f;
                if (g < quarter) d[i] = -d[i];
            }
            fa[2 * s] = pack2(w.x * c[0], w.y * c[1]);
            fa[2 * s + 1] = pack2(w.z * c[2], w.w * c[3]);
            fb[2 * s] = pack2(v.x * d[0], v.y * d[1]);
            fb[2 * s + 1] = pack2(v.z * d[2], v.w * d[3]);
            on |= turns ? 3u << (2u * s) : 0u;
        }
    } else {
        interleaved(wn);
    }
    const int32_t slot = __ldcg(P.slot + tok);
    const bool keeps = slot >= 0 && (uint32_t)slot < P.slots;
    if (slot >= 0 && !keeps && lane == 0u) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    const uint32_t row = (uint32_t)(keeps ? slot : 0), page = row >> P.page_shift, in_page = row & ((1u << P.page_shift) - 1u), r16 = row & 15u;

    for (uint32_t head0 = first; head0 - sub < behind; head0 += RPW * U) {
        load(head0 + RPW * U, a_next, b_next);
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint32_t head = head0 + u * RPW;
            if (head - sub >= behind) break;
            const bool live = keeps && head < behind;
            a[u].get(x);
            const float r = P.eps >= 0.f ? norm_of<LPR>(x, P.eps) : 1.f;
            uint64_t y[4];
            if constexpr (HALF) {
                float f[8], g[8];
                *reinterpret_cast<float4 *>(f) = four(x[0], x[1]);
                *reinterpret_cast<float4 *>(f + 4) = four(x[2], x[3]);
                if (swap) {
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++) g[i] = __shfl_sync(0xffffffffu, f[i ^ 4u], from[i >> 2]);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++) g[i] = __shfl_sync(0xffffffffu, f[i], from[i >> 2]);
                }
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) y[i] = pack2(g[2 * i], g[2 * i + 1]);
            } else {
                other_of_two(y);
            }
            turn<FULL>(x, y, fa, fb, on, r);
            uint8_t *tile = P.mem + ((((uint64_t)page * P.n_kvh + head) << (P.page_shift - 4u)) + (in_page >> 4)) * PgTile<KIND, HD>::BYTES;
#pragma unroll
            for (uint32_t v = 0; v < 2u; v++) {
                if (v) b[u].get(x);
                const float4 lo = four(x[0], x[1]), hi = four(x[2], x[3]);
                if constexpr (KIND == Q4K_Q8) {   /* four lanes to a block of 32 */
                    float m = fmaxf(fmaxf(fmaxf(fabsf(lo.x), fabsf(lo.y)), fmaxf(fabsf(lo.z), fabsf(lo.w))), fmaxf(fmaxf(fabsf(hi.x), fabsf(hi.y)), fmaxf(fabsf(hi.z), fabsf(hi.w)))), d, id;
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                    q4d_scale(m, d, id);
                    if (live) {
                        uint8_t *rec = tile + r16 * PgTile<KIND, HD>::ROW;
                        *reinterpret_cast<uint2 *>(rec + v * HD + in * 8u) = make_uint2(q4d_quant4(lo, id), q4d_quant4(hi, id));
                        if ((in & 3u) == 0u) reinterpret_cast<__half *>(rec + 2u * HD)[v * (HD / 32u) + (in >> 2)] = __float2half_rn(d);
                    }
                } else if (live) {
                    const __half2 h[4] = {__floats2half2_rn(lo.x, lo.y), __floats2half2_rn(lo.z, lo.w), __floats2half2_rn(hi.x, hi.y), __floats2half2_rn(hi.z, hi.w)};
                    uint8_t *dst = tile + v * (PgTile<KIND, HD>::BYTES / 2u) + (in >> 3) * 2048u + r16 * 128u + (((in & 7u) ^ (r16 & 7u)) << 4);
                    *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(h);
                }
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            a[u] = a_next[u];
            b[u] = b_next[u];
        }
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0u; }

template <int KIND, int HD, bool BF16>
bool prep_launch(PrepParams &p) {
    constexpr uint32_t RPW = 256u / HD;
    /* A warp's start (sines, factors) is worth some turns: no more warps than the SMs hold at once, and several rounds of them, the last of which may be part empty,
     * only where there are many tokens.  us, with 20 warps per SM and with 54: 300 tokens of 24 heads of 256 6.2 and 8.9, 1000 17.3 and 17.1, 2000 34.4 and 31.9, 3000 47.9 and 46.0,
     * 4000 65.2 and 61.1; 16 of 128 in fp32 500 3.1 and 5.2, 1000 5.6 and 6.3, 2000 12.6 and 12.0, 3000 18.7 and 17.6; 32 of 128 in bf16 2000 12.9 and 15.0, 3000 18.9 and 19.7, 4000
     * 22.8 and 22.6; 8 of 64 2000 4.7 and 6.8, 3000 6.9 and 10.3, 4000 9.0 and 9.0.  The sides meet between 1000 tokens (large rows) and 4000 (small ones): one line between them. */
    const uint32_t most = (p.n_tok < 2048u ? 20u : 54u) * (uint32_t)g_q4.sm_count, want = (most + p.n_tok - 1u) / p.n_tok, q_turns = (p.n_head + RPW - 1u) / RPW, kv_turns = (p.n_kvh + RPW - 1u) / RPW;
    const uint32_t per = (q_turns + kv_turns + want - 1u) / want;
    p.q_per = per < q_turns ? per : q_turns;
    p.kv_per = per < kv_turns ? per : kv_turns;
    p.q_units = (q_turns + p.q_per - 1u) / p.q_per;
    p.units = p.q_units + (kv_turns + p.kv_per - 1u) / p.kv_per;
    const uint64_t blocks = (uint64_t)p.n_tok * p.units;
    if (blocks > 0x7fffffffu) return q4i_fail(Q4E_ARG, "pages_prep: too many tokens for one call");
    const bool full = p.rope.n_rot == HD;
    auto start = [&](auto kernel) { return q4i_launch_pdl("pages_prep launch", kernel, dim3((unsigned)blocks), PREP_THREADS, 0, p); };
    if (p.rope.half) return full ? start(q4_pg_prep_k<KIND, HD, BF16, true, true>) : start(q4_pg_prep_k<KIND, HD, BF16, true, false>);
    return full ? start(q4_pg_prep_k<KIND, HD, BF16, false, true>) : start(q4_pg_prep_k<KIND, HD, BF16, false, false>);
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
    /* the slow end may lie behind the last pair, which then is not slowed down fully */
    const double lo = scaling == 2 ? fmax(0.0, floor(pair_of(fast))) : 0.0, hi = scaling == 2 ? fmin((double)n_rot - 1.0, ceil(pair_of(slow))) : 0.0;
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
