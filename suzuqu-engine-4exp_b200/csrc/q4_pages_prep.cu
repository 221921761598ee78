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
 * Bound by memory: every value is read once and written once.  4096 tokens of 24 gated heads of 256 in fp32, 373 MB, take 63 us (90 % of a copy's rate); 16 001 fused
 * bf16 rows of 32 heads of 128 with 8 kv heads, 394 MB, 78 us (77 %), there beside the issue slots: 63 % busy at the 20 warps that an SM's registers hold.
 */
#include <math.h>
#include <string.h>

#include "q4_paged.h"

namespace {

constexpr uint32_t PREP_THREADS = 32;   /* warps differ in their turns: a block of several would keep its place for the longest (16 001 fused rows 78 us, in pairs 99, in eights 115) */

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

/* eight values of a row, as they lie */
template <bool BF16>
struct Eight {
    uint4 x[BF16 ? 1 : 2];
    __device__ __forceinline__ void load(const uint8_t *p, bool live) {
#pragma unroll
        for (int i = 0; i < (BF16 ? 1 : 2); i++) x[i] = live ? __ldcs(reinterpret_cast<const uint4 *>(p) + i) : make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
        const uint32_t *u = reinterpret_cast<const uint32_t *>(x);
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = __uint_as_float(BF16 ? (i & 1 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16) : u[BF16 ? 0 : i]);
    }
};
__device__ __forceinline__ void eight_floats(const float *p, float (&f)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void store_floats(float *p, const float (&f)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

/*
 * A warp has a token's queries, or its keys and values, or a part of them where there are few tokens, and keeps what belongs to the token in registers:
 * sines and cosines, with the weights in them.  Lanes hold eight dims of a row each, so that a warp has 1, 2 or 4 rows at a time (hd 256, 128, 64).  The
 * warps' issue slots set the pace beside memory (16 001 rows of a fused bf16 projection 169 us with four dims per lane).  A turn's rows are requested
 * before the one before them is worked at, the first before the token's position is there.
 */
template <int KIND, int HD, bool BF16, bool HALF, bool FULL>
__global__ void __launch_bounds__(PREP_THREADS) q4_pg_prep_k(const __grid_constant__ PrepParams P) {
    constexpr uint32_t LPR = HD / 8u, RPW = 32u / LPR, U = BF16 ? 2u : 1u, SIZE = BF16 ? 2u : 4u;   /* U: turns at a time, as many bytes on their way in either type */
    const uint32_t lane = threadIdx.x, in = lane % LPR, sub = lane / LPR, unit = blockIdx.x;
    const uint32_t tok = unit / P.units, which = unit - tok * P.units;
    const bool is_q = which < P.q_units;
    const uint32_t heads = is_q ? P.n_head : P.n_kvh, per = is_q ? P.q_per : P.kv_per, first = (is_q ? which : which - P.q_units) * per * RPW + sub, behind = min(first - sub + per * RPW, heads);
    q4d_pdl_wait();
    const int32_t pos = __ldcg(P.pos + tok);

    /* rows of the group's heads: first, first + RPW .. */
    const bool two = !is_q || P.gate;      /* a second row: gate or value */
    const uint32_t step = RPW * HD * (is_q && P.gate ? 2u : 1u) * SIZE;
    const uint64_t at = (is_q ? tok * P.q_stride : tok * P.kv_stride) + (uint64_t)first * (HD * (is_q && P.gate ? 2u : 1u)) + in * 8u;
    const uint8_t *pa = (const uint8_t *)(is_q ? P.q : P.k) + at * SIZE, *pb = is_q ? pa + HD * SIZE : (const uint8_t *)P.v + at * SIZE;
    Eight<BF16> a[U], b[U], a_next[U], b_next[U];
    auto load = [&](uint32_t head, Eight<BF16> (&x)[U], Eight<BF16> (&y)[U]) {
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const bool live = head + u * RPW < behind;
            x[u].load(pa, live);
            if (two) y[u].load(pb, live);
            pa += step;
            pb += step;
        }
    };
    load(first, a, b);

    if (pos < 0) return;
    /* The warp's lanes take the sines and cosines of the head's pairs, C consecutive ones each, for one another */
    const uint32_t n_rot = P.rope.n_rot, np = n_rot / 2u;
    constexpr uint32_t C = HD / 64u;
    float cs[C], sn[C];
    {
        const uint64_t *turn;              /* as memory: the lanes' addresses differ, which the constant port takes one by one */
        asm("mov.u64 %0, %1;" : "=l"(turn) : "l"(P.rope.turn));
#pragma unroll
        for (uint32_t i = 0; i < C; i++) {
            const uint64_t angle = (uint64_t)(uint32_t)pos * turn[lane * C + i];
            sincospif((float)(int32_t)(angle >> 32) * 4.656612873077393e-10f, &sn[i], &cs[i]);   /* 2^-31: half turns */
            cs[i] *= P.rope.mag;
            sn[i] *= P.rope.mag;
        }
    }
    /* What a dim is made of: x fa + y fb, y the pair's other dim.  Both hold the weights.  Dims that are not turned: x fa */
    float fa[8], fb[8];
    uint32_t on = 0;                       /* dims that are turned */
    const uint32_t quarter = np / 4u, swap = quarter & 1u;
    uint32_t from[2] = {0u, 0u};           /* halves: the lanes where the other dims of the lane's two groups of four lie, in which of its groups is the same for all lanes */
    {
        const float *wn = P.eps >= 0.f ? (is_q ? P.wq : P.wk) : nullptr;
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = 1.f;
        if (wn) eight_floats(wn + in * 8u, w);
        if constexpr (HALF) {
#pragma unroll
            for (uint32_t s = 0; s < 2u; s++) {
                const uint32_t g = in * 2u + s, other = g < quarter ? g + quarter : g - quarter;
                const bool turns = FULL || g < 2u * quarter;
                from[s] = sub * LPR + ((other >> 1) & (LPR - 1u));
                float v[4] = {1.f, 1.f, 1.f, 1.f};
                if (wn && turns) *reinterpret_cast<float4 *>(v) = __ldg(reinterpret_cast<const float4 *>(wn) + other);
                const uint32_t pair = (g < quarter ? g : other) * 4u;   /* of the group's first dim */
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) {
                    const uint32_t k = s * 4u + i, holder = ((pair + i) / C) & 31u;
                    const float c = __shfl_sync(0xffffffffu, cs[i % C], holder), d = __shfl_sync(0xffffffffu, sn[i % C], holder);
                    fa[k] = turns ? w[k] * c : w[k];
                    fb[k] = v[i] * (g < quarter ? -d : d);
                }
                on |= turns ? 0xfu << (4u * s) : 0u;
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                const uint32_t pair = in * 4u + i;
                const float c = __shfl_sync(0xffffffffu, cs[i % C], pair / C), d = __shfl_sync(0xffffffffu, sn[i % C], pair / C);
                const bool turns = FULL || pair < np;
                fa[2 * i] = turns ? w[2 * i] * c : w[2 * i];
                fa[2 * i + 1] = turns ? w[2 * i + 1] * c : w[2 * i + 1];
                fb[2 * i] = w[2 * i + 1] * -d;
                fb[2 * i + 1] = w[2 * i] * d;
                on |= turns ? 3u << (2u * i) : 0u;
            }
        }
    }
    const int32_t slot = is_q ? -1 : __ldcg(P.slot + tok);
    const bool keeps = slot >= 0 && (uint32_t)slot < P.slots;
    if (slot >= 0 && !keeps && lane == 0u) atomicOr(P.err, (uint32_t)Q4E_RANGE);
    const uint32_t row = (uint32_t)(keeps ? slot : 0), page = row >> P.page_shift, in_page = row & ((1u << P.page_shift) - 1u), r16 = row & 15u;

    for (uint32_t head0 = first; head0 - sub < behind; head0 += RPW * U) {
        load(head0 + RPW * U, a_next, b_next);
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint32_t head = head0 + u * RPW;
            if (head - sub >= behind) break;
            const bool live = head < behind;
            float x[8];
            a[u].get(x);
            float r = 1.f;
            if (P.eps >= 0.f) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
                for (uint32_t o = LPR / 2u; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                r = rsqrtf(fmaf(ss, 1.f / HD, P.eps));   /* 2 units in the last place at most */
            }
            float y[8];
            if constexpr (HALF) {
                if (swap) {
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++) y[i] = __shfl_sync(0xffffffffu, x[i ^ 4u], from[i >> 2]);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 8u; i++) y[i] = __shfl_sync(0xffffffffu, x[i], from[i >> 2]);
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8u; i++) y[i] = x[i ^ 1u];
            }
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) {
                const float z = x[i] * fa[i];
                x[i] = r * (FULL || (on >> i) & 1u ? fmaf(y[i], fb[i], z) : z);   /* not turned: the other dim may be infinite */
            }
            if (is_q) {
                if (!live) continue;
                const uint64_t to = ((uint64_t)tok * P.n_head + head) * HD + in * 8u;
                if (P.q_bf16) {
                    __nv_bfloat162 h[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                    *reinterpret_cast<uint4 *>(reinterpret_cast<__nv_bfloat16 *>(P.q_out) + to) = *reinterpret_cast<const uint4 *>(h);
                } else {
                    store_floats(reinterpret_cast<float *>(P.q_out) + to, x);
                }
                if (two) {
                    b[u].get(x);
                    store_floats(P.gate + to, x);
                }
            } else {
                uint8_t *tile = P.mem + ((((uint64_t)page * P.n_kvh + head) << (P.page_shift - 4u)) + (in_page >> 4)) * PgTile<KIND, HD>::BYTES;
#pragma unroll
                for (uint32_t v = 0; v < 2u; v++) {
                    if (v) b[u].get(x);
                    if constexpr (KIND == Q4K_Q8) {   /* four lanes to a block of 32 */
                        float m = 0.f, d, id;
#pragma unroll
                        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(x[i]));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                        q4d_scale(m, d, id);
                        if (keeps && live) {
                            uint8_t *rec = tile + r16 * PgTile<KIND, HD>::ROW;
                            *reinterpret_cast<uint2 *>(rec + v * HD + in * 8u) = make_uint2(q4d_quant4(make_float4(x[0], x[1], x[2], x[3]), id), q4d_quant4(make_float4(x[4], x[5], x[6], x[7]), id));
                            if ((in & 3u) == 0u) reinterpret_cast<__half *>(rec + 2u * HD)[v * (HD / 32u) + (in >> 2)] = __float2half_rn(d);
                        }
                    } else if (keeps && live) {
                        __half2 h[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                        uint8_t *dst = tile + v * (PgTile<KIND, HD>::BYTES / 2u) + (in >> 3) * 2048u + r16 * 128u + (((in & 7u) ^ (r16 & 7u)) << 4);
                        *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(h);
                    }
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
    /* A warp's start (sines, factors) is worth some turns: as many warps as the SMs hold at once, and several rounds of them, the last of which may be part empty,
     * only where there are many tokens.  us, with 20 warps per SM and with 54: 300 tokens of 24 heads of 256 5.9 and 8.9, 500 of 16 of 128 3.3 and 5.4, 4096 of 24 of
     * 256 65.9 and 63.1. */
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
