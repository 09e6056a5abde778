/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_groute.hip -- routing from logits (k3d_route): scores, a selection bias, groups, top-k,
 * renormalised weights, one wave per token.
 *
 *   score = sigmoid(l) or exp(l - max) / sum;  choice = score + bias;  the top_groups groups of
 *   the largest sums of their group_top largest choices;  the topk largest choices among them.
 *
 * Choices are defined in 64 bits, and which of two close experts wins must not depend on how an
 * exponential was rounded to 32; but few experts are close to a border. So lane l holds the choices of experts
 * l + 64 i in fp32, each within a bound E of its definition (the same E for the wave), and what fp32 leaves open is
 * settled in 64 bits:
 *  - groups: their values within 2 E; where the last kept group and the first one left out lie closer, every group's
 *    value is formed again in 64 bits;
 *  - top-k: the k-th largest of the lanes' maxima is at most the k-th largest choice, so only choices of at least
 *    that less 2 E can be selected: about 1.3 topk of them. They are packed, a lane each, computed in 64 bits, and
 *    ranked by counting, equal ones by their order. More than 64 (rows of equal logits): every choice in 64 bits and
 *    topk rounds of wave maxima (route_exact).
 * 8192 tokens of 896 experts, top 16 in 4 of 8 groups: 27.7 us with its logits out of memory, 22.6 out of the last cache, 205 there with every choice
 * in 64 bits and topk rounds of wave maxima; its bytes take 6 us at the rate of a copy. Bound by vector instructions, 1044 a token
 * (14 us of issue slots); one token by the latency of its chain.
 * E covers the largest finite |choice|, so a large finite bias leaves everything of its tokens to 64 bits: with -1e9 on a tenth
 * of the experts the same takes 87 us (with -inf there 26).
 */
#include "k3_common.h"
#include "k3_dev.h"
#include "k3_wave.h"
#include "k3k.h"

namespace {

/* order-preserving bits of a choice; 0 for one that cannot be taken (NaN, -inf) */
__device__ __forceinline__ uint64_t choice_key(double c)
{
    if (!(c > -INFINITY)) return 0ull;
    const uint64_t b = (uint64_t)__double_as_longlong(c == 0.0 ? 0.0 : c);
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

__device__ __forceinline__ double key_value(uint64_t k)
{
    return __longlong_as_double((long long)((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
}

/* order-preserving bits of an fp32 choice, 0 for one that cannot be taken */
__device__ __forceinline__ uint32_t choice_key32(float c)
{
    const uint32_t b = __float_as_uint(c);
    return c > -INFINITY ? ((b >> 31) ? ~b : b | 0x80000000u) : 0u;
}

__device__ __forceinline__ float key32_value(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }

template <int TYPE>
__device__ __forceinline__ float load_logit(const void *p, size_t i)
{
    if (TYPE == K3D_F32) return ((const float *)p)[i];
    return k3_bf16_to_f32(((const uint16_t *)p)[i]);
}

/* e^x in 64 bits, within a unit in the last place: x = n ln 2 + r (ln 2 as a sum of two doubles), the Taylor
 * polynomial to r^13 on |r| <= ln 2 / 2, whose next term is under 2^-57 */
__device__ __forceinline__ double exp64(double x)
{
    const double n = rint(x * 1.44269504088896340736);
    double r = fma(-n, 0.693147180559945286227, x);
    r = fma(-n, 2.31904681384629955842e-17, r);
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double y = ldexp(p, (int)fmin(fmax(n, -1100.0), 1100.0));
    return x > 709.8 ? (double)INFINITY : x < -746.0 ? 0.0 : y;
}

/* exp(l - m) of a present logit; the largest one's is 1, also where it is infinite. (Selections, here and
 * below, of what is computed either way: branches around 40 instructions cost copies of all that lives.) */
__device__ __forceinline__ double soft_term(float l, float m)
{
    const double y = exp64((double)l - (double)m);
    return l == m ? 1.0 : y;
}

template <int SCORE>
__device__ __forceinline__ double score64(float l, float m, double sum)
{
    if constexpr (SCORE == K3D_SCORE_SIGMOID) return 1.0 / (1.0 + exp64(-(double)l));
    else return soft_term(l, m) / sum;
}

/* the key of expert e's choice, from its score s */
__device__ __forceinline__ uint64_t score_key(const K3kRoute &a, double s, float l, int e)
{
    const uint64_t k = choice_key(s + (a.bias ? (double)a.bias[e] : 0.0));
    return l > -INFINITY ? k : 0ull;
}

template <int SCORE>
__device__ __forceinline__ uint64_t key64(const K3kRoute &a, float l, int e, float m, double sum)
{
    return score_key(a, score64<SCORE>(l, m, sum), l, e);
}

template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v)
{
    return __uint_as_float(dpp_u32<CTRL, 0xf, 0u>(__float_as_uint(v)));
}

__device__ __forceinline__ uint64_t lane64(uint64_t v, int l)
{
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}

/* The token's experts with every choice in 64 bits, of those with c > -inf: lane j gets the j-th, or -1. */
template <int TYPE, int P, int SCORE>
__device__ int route_exact(const K3kRoute &a, size_t row, float m, double sum, const float (&c)[P])
{
    const int lane = threadIdx.x & 63, n = a.n;
    /* (the compiler must not keep what the other path formed from these loads: it would be P doubles) */
    asm volatile("" : "+s"(row));
    uint64_t key[P];
#pragma unroll
    for (int i = 0; i < P; i++) {
        const int in = min(lane + 64 * i, n - 1);
        const uint64_t k = key64<SCORE>(a, load_logit<TYPE>(a.logits, row + in), in, m, sum);
        key[i] = c[i] > -INFINITY ? k : 0ull;
        __builtin_amdgcn_sched_barrier(0);      /* (one after another: side by side they take ten registers each) */
    }
    /* topk rounds: the wave's largest key, of equals the lowest expert */
    int mine = -1;
    for (int j = 0; j < a.topk; j++) {
        uint32_t hi = 0;
#pragma unroll
        for (int i = 0; i < P; i++) hi = max(hi, (uint32_t)(key[i] >> 32));
        hi = wave_reduce_u32<true>(hi);
        uint32_t lo = 0;
#pragma unroll
        for (int i = 0; i < P; i++) lo = max(lo, (uint32_t)(key[i] >> 32) == hi ? (uint32_t)key[i] : 0u);
        lo = wave_reduce_u32<true>(lo);
        const uint64_t best = ((uint64_t)hi << 32) | lo;
        uint32_t e = 0xffffffffu;
#pragma unroll
        for (int i = P - 1; i >= 0; i--) e = key[i] == best ? (uint32_t)(lane + 64 * i) : e;
        e = wave_reduce_u32<false>(e);
        if (best == 0ull) break;
#pragma unroll
        for (int i = 0; i < P; i++)
            if (e == (uint32_t)(lane + 64 * i)) key[i] = 0ull;
        if (lane == j) mine = (int)e;
    }
    return mine;
}

/* P: experts per lane. LDS per wave: lds bytes (the wave's choices by expert where there are groups, 64 candidates) */
template <int TYPE, int P, int SCORE>
__global__ __launch_bounds__(256, P <= 14 ? 5 : 1) void route_kernel(K3kRoute a, int lds)
{
    extern __shared__ uint64_t smem[];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x * (blockDim.x >> 6) + wv, n = a.n;
    if (t >= a.T) return;                       /* (nothing below waits for another wave) */
    const size_t row = (size_t)t * a.ld;
    int *const cand = reinterpret_cast<int *>(smem + (size_t)wv * (lds / 8));
    float *const ch = reinterpret_cast<float *>(cand + 64);

    float c[P];                                 /* logits, then choices */
#pragma unroll
    for (int i = 0; i < P; i++) {
        const int e = lane + 64 * i;
        const float l = load_logit<TYPE>(a.logits, row + min(e, n - 1));
        c[i] = e < n ? l : -INFINITY;
    }
    float m = -INFINITY;
    double sum = 0.0;
    if constexpr (SCORE == K3D_SCORE_SOFTMAX) {
#pragma unroll
        for (int i = 0; i < P; i++) m = fmaxf(m, c[i]);         /* (fmaxf passes over NaN) */
        const uint32_t km = wave_reduce_u32<true>(choice_key32(m));
        m = km ? key32_value(km) : -INFINITY;
        float s[P];
#pragma unroll
        for (int i = 0; i < P; i++) {
            const double y = soft_term(c[i], m), q = c[i] > -INFINITY ? y : 0.0;
            sum += q;
            s[i] = (float)q;
            if (i % 2) __builtin_amdgcn_sched_barrier(0);
        }
        sum = wave_total_f64(sum);
        const float inv = (float)(1.0 / sum);
#pragma unroll
        for (int i = 0; i < P; i++) c[i] = c[i] > -INFINITY ? s[i] * inv : -INFINITY;
    } else {
#pragma unroll
        for (int i = 0; i < P; i++) {
            const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * c[i]));
            c[i] = c[i] > -INFINITY ? s : -INFINITY;
        }
    }
    /* The bound E. A sigmoid: the exponent's rounding and the exponential move e^-l by (0.7 |l| + 1) 2^-23 of itself, the
     * score s by s (1 - s) times that, which is at most 0.5 * 2^-23, and the sum's and the reciprocal's roundings by
     * 1.5 * 2^-23 s: under 2^-22 for any l, and where all scores are small, (|l| + 4) 2^-23 of them for |l| up to 64 (past it they are
     * within 2^-90 of 0 or 1). The softmax: three roundings of a score. Twice that, and 2^-22 of the largest choice for
     * the additions of the bias and of a group's two choices. */
    float top_s = 0.0f, top_c = 0.0f;
#pragma unroll
    for (int i = 0; i < P; i++) {
        const int e = lane + 64 * i;
        top_s = fmaxf(top_s, c[i]);
        const float v = a.bias ? c[i] + a.bias[min(e, n - 1)] : c[i];
        c[i] = v > -INFINITY ? v : -INFINITY;                   /* (NaN) */
        top_c = fmaxf(top_c, fabsf(v) < INFINITY ? fabsf(v) : 0.0f);
    }
    /* (positive floats compare as their bits) */
    top_s = __uint_as_float(wave_reduce_u32<true>(__float_as_uint(top_s)));
    top_c = __uint_as_float(wave_reduce_u32<true>(__float_as_uint(top_c)));
    const float Es = SCORE == K3D_SCORE_SIGMOID ? fminf(0x1p-21f, 0x1p-15f * top_s) : 0x1p-21f * top_s;
    const float E = fmaf(0x1p-22f, top_c, Es + 0x1p-80f);

    if (a.top_groups < a.n_groups) {
        /* 64 / n_groups lanes (a power of two of them) take a group: its two largest choices */
#pragma unroll
        for (int i = 0; i < P; i++)
            if (lane + 64 * i < n) ch[lane + 64 * i] = c[i];
        __builtin_amdgcn_wave_barrier();
        const int gs = n / a.n_groups, lsh = 31 - __clz(64 / a.n_groups), LG = 1 << lsh;
        const int g = lane >> lsh;
        float k1 = -INFINITY, k2 = -INFINITY;
        if (g < a.n_groups)
#pragma unroll 4
            for (int j = lane & (LG - 1); j < gs; j += LG) {
                const float v = ch[g * gs + j];
                k2 = fmaxf(k2, fminf(k1, v));
                k1 = fmaxf(k1, v);
            }
        auto meet = [&](float o1, float o2) {
            k2 = fmaxf(fmaxf(k2, o2), fminf(k1, o1));
            k1 = fmaxf(k1, o1);
        };
        /* (neighbours, pairs, quads, eights by mirroring: every lane of a part holds the same) */
        if (LG >= 2) meet(dpp_f32<0xB1>(k1), dpp_f32<0xB1>(k2));
        if (LG >= 4) meet(dpp_f32<0x4E>(k1), dpp_f32<0x4E>(k2));
        if (LG >= 8) meet(dpp_f32<0x141>(k1), dpp_f32<0x141>(k2));
        if (LG >= 16) meet(dpp_f32<0x140>(k1), dpp_f32<0x140>(k2));
        if (LG >= 32) meet(__shfl_xor(k1, 16), __shfl_xor(k2, 16));
        /* (the sum of two finite choices stays finite: two at the lowest value are past fp32, not past 64 bits, and such groups may
         * be taken. Held at the end of the range they compare as equal, which 64 bits then settle.) */
        const float sum2 = __builtin_amdgcn_fmed3f(k1 + k2, -0x1.fffffep127f, 0x1.fffffep127f);
        const float v = a.group_top == 2 && k2 > -INFINITY && k1 < INFINITY ? sum2 : k1;
        int rank = 0;
        for (int q = 0; q < a.n_groups; q++) {
            const float o = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), q << lsh));
            rank += o > v || (o == v && q < g);
        }
        bool keep = g < a.n_groups && v > -INFINITY && rank < a.top_groups;
        /* the least kept and the largest left out (as order-preserving bits; no group: the far end) */
        const uint32_t kv = choice_key32(v);
        const uint32_t in = wave_reduce_u32<false>(keep ? kv : 0xffffffffu);
        const uint32_t out = wave_reduce_u32<true>(keep || g >= a.n_groups ? 0u : kv);
        /* (each within 2 E of its definition; not where both are infinite) */
        if (out && !(key32_value(in) - key32_value(out) > 4.0f * E)) {
            uint64_t x1 = 0ull, x2 = 0ull;
            if (g < a.n_groups)
                for (int j = lane & (LG - 1); j < gs; j += LG) {
                    const int e = g * gs + j;
                    const uint64_t k = key64<SCORE>(a, load_logit<TYPE>(a.logits, row + e), e, m, sum);
                    x2 = k > x1 ? x1 : k > x2 ? k : x2;
                    x1 = k > x1 ? k : x1;
                }
            for (int o = LG >> 1; o; o >>= 1) {
                const uint64_t o1 = __shfl_xor(x1, o), o2 = __shfl_xor(x2, o), less = x1 < o1 ? x1 : o1;
                x1 = x1 > o1 ? x1 : o1;
                x2 = x2 > o2 ? x2 : o2;
                x2 = x2 > less ? x2 : less;
            }
            const uint64_t x = a.group_top == 2 && x2 ? choice_key(key_value(x1) + key_value(x2)) : x1;
            rank = 0;
            for (int q = 0; q < a.n_groups; q++) {
                const uint64_t o = lane64(x, q << lsh);
                rank += o > x || (o == x && q < g);
            }
            keep = g < a.n_groups && x && rank < a.top_groups;
        }
        if (!keep && g < a.n_groups)
            for (int j = lane & (LG - 1); j < gs; j += LG) ch[g * gs + j] = -INFINITY;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < P; i++)
            if (lane + 64 * i < n) c[i] = ch[lane + 64 * i];
    }

    int ncand = 0;
    /* a bound that at least topk lanes' maxima reach (fewer lanes with any: all choices), by halving the keys' range */
    float lm = c[0];
#pragma unroll
    for (int i = 1; i < P; i++) lm = fmaxf(lm, c[i]);
    const uint32_t km = choice_key32(lm);
    uint32_t lo = 0, hi = wave_reduce_u32<true>(km);
    if (__popcll(__ballot(km != 0u)) >= a.topk) {
        lo = wave_reduce_u32<false>(km ? km : 0xffffffffu);
        if (a.topk == 1) lo = hi;
        for (int q = 0; q < 12 && lo < hi; q++) {
            const uint32_t mid = lo + ((hi - lo + 1) >> 1);
            const int above = __popcll(__ballot(km >= mid));
            if (above >= a.topk) lo = mid;
            else hi = mid - 1;
            if (above == a.topk) break;
        }
    }
    const float thr = lo ? key32_value(lo) : -INFINITY;
    const float least = thr < INFINITY ? fmaf(-2.0f, E, thr) : thr;
    /* the candidates, in the experts' order */
#pragma unroll
    for (int i = 0; i < P; i++) {
        const bool in = c[i] >= least && c[i] > -INFINITY;
        const uint64_t who = __ballot(in);
        const int slot = ncand + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
        if (in && slot < 64) cand[slot] = lane + 64 * i;
        ncand += __popcll(who);
    }
    __builtin_amdgcn_wave_barrier();
    int mine = -1, at = lane;                   /* the lane's expert and its place */
    double w = 0.0;                             /* its score */
    if (ncand <= 64) {
        uint64_t key = 0ull;
        if (lane < ncand) {
            mine = cand[lane];
            const float l = load_logit<TYPE>(a.logits, row + mine);
            w = score64<SCORE>(l, m, sum);
            key = score_key(a, w, l, mine);
        }
        int rank = 0;
        for (int q = 0; q < ncand; q++) {
            const uint64_t o = lane64(key, q);
            rank += o > key || (o == key && q < lane);
        }
        at = lane < ncand ? rank : 64;
        if (at >= a.topk) mine = -1;
        /* places that no candidate takes */
        if (lane >= ncand && lane < a.topk) at = lane;
    } else {
        mine = route_exact<TYPE, P, SCORE>(a, row, m, sum, c);
        if (mine >= 0) w = score64<SCORE>(load_logit<TYPE>(a.logits, row + mine), m, sum);
    }
    if (mine < 0) w = 0.0;
    if (a.renorm) {
        const double s = wave_total_f64(w);
        w = s > 0.0 ? w / s : 0.0;
    }
    if (at < a.topk) {
        a.idx[(size_t)t * a.topk + at] = mine;
        a.wt[(size_t)t * a.topk + at] = (float)(w * (double)a.scale);
    }
}

template <int TYPE, int P, int SCORE>
void launch(const K3kRoute *a, hipStream_t st)
{
    const int waves = a->T < 1024 ? 1 : 4;
    const int lds = 256 + (a->top_groups < a->n_groups ? (a->n * 4 + 255) / 256 * 256 : 0);
    route_kernel<TYPE, P, SCORE><<<(a->T + waves - 1) / waves, 64 * waves, (size_t)waves * lds, st>>>(*a, lds);
}

template <int TYPE, int SCORE>
void pick(const K3kRoute *a, hipStream_t st)
{
    const int p = (a->n + 63) / 64;
    if (p <= 2) launch<TYPE, 2, SCORE>(a, st);
    else if (p <= 4) launch<TYPE, 4, SCORE>(a, st);
    else if (p <= 6) launch<TYPE, 6, SCORE>(a, st);
    else if (p <= 10) launch<TYPE, 10, SCORE>(a, st);
    else if (p <= 14) launch<TYPE, 14, SCORE>(a, st);
    else if (p <= 20) launch<TYPE, 20, SCORE>(a, st);
    else launch<TYPE, 32, SCORE>(a, st);
}

template <int TYPE>
void pick_score(const K3kRoute *a, hipStream_t st)
{
    if (a->score == K3D_SCORE_SIGMOID) pick<TYPE, K3D_SCORE_SIGMOID>(a, st);
    else pick<TYPE, K3D_SCORE_SOFTMAX>(a, st);
}

}  // namespace

extern "C" int k3k_route(const K3kRoute *a, void *stream)
{
    if (a->type == K3D_F32) pick_score<K3D_F32>(a, (hipStream_t)stream);
    else pick_score<K3D_BF16>(a, (hipStream_t)stream);
    K3K_LAUNCH_CHECK("route");
    return 0;
}
