/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_groute.hip -- routing from logits (k3d_route): scores, a selection bias, groups, top-k,
 * renormalised weights, one wave per token.
 *
 *   score = sigmoid(l) or exp(l - max) / sum;  choice = score + bias;  the top_groups groups of
 *   the largest sums of their group_top largest choices;  the topk largest choices among them.
 *
 * Lane l of the wave holds experts l + 64 i. Choices are fp64 and are compared as order-preserving
 * 64-bit keys (0: cannot be taken), so which of two close experts wins does not depend on how an
 * exponential was rounded to 32 bits.
 */
#include "k3_common.h"
#include "k3_dev.h"
#include "k3_wave.h"
#include "k3k.h"

namespace {

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

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

template <int TYPE>
__device__ __forceinline__ float load_logit(const void *p, size_t i)
{
    if (TYPE == K3D_F32) return ((const float *)p)[i];
    return k3_bf16_to_f32(((const uint16_t *)p)[i]);
}

/* exp(l - m) of a present logit; the largest one's is 1, also where it is infinite */
__device__ __forceinline__ double soft_term(float l, float m)
{
    return l == m ? 1.0 : exp((double)l - (double)m);
}

__device__ __forceinline__ double score64(int score, float l, float m, double sum)
{
    if (score == K3D_SCORE_SIGMOID) return 1.0 / (1.0 + exp(-(double)l));
    return soft_term(l, m) / sum;
}

/* P: experts per lane */
template <int TYPE, int P>
__global__ __launch_bounds__(256) void route_kernel(K3kRoute a)
{
    extern __shared__ uint64_t smem[];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int t = blockIdx.x * (blockDim.x >> 6) + wv;
    const int n = a.n;
    const bool live = t < a.T;                  /* (waves without a token go along to the barriers) */
    const size_t row = (size_t)(live ? t : 0) * a.ld;
    uint64_t *keys = smem + (size_t)wv * n;     /* this token's keys, when there are groups */

    float lg[P];
#pragma unroll
    for (int i = 0; i < P; i++) {
        const int e = lane + 64 * i;
        lg[i] = e < n ? load_logit<TYPE>(a.logits, row + e) : -INFINITY;
    }
    float m = -INFINITY;
    double sum = 0.0;
    if (a.score == K3D_SCORE_SOFTMAX) {
#pragma unroll
        for (int i = 0; i < P; i++) m = fmaxf(m, lg[i]);        /* (fmaxf passes over NaN) */
#pragma unroll
        for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
#pragma unroll
        for (int i = 0; i < P; i++) sum += lg[i] > -INFINITY ? soft_term(lg[i], m) : 0.0;
        sum = wave_sum_f64(sum);
    }
    uint64_t key[P];
#pragma unroll
    for (int i = 0; i < P; i++) {
        const int e = lane + 64 * i;
        key[i] = 0ull;
        if (lg[i] > -INFINITY) {
            double c = score64(a.score, lg[i], m, sum);
            if (a.bias) c += (double)a.bias[e];
            key[i] = choice_key(c);
        }
    }

    if (a.top_groups < a.n_groups) {
        /* a group per lane: its value; then every lane counts the groups above its own */
#pragma unroll
        for (int i = 0; i < P; i++)
            if (lane + 64 * i < n) keys[lane + 64 * i] = key[i];
        __syncthreads();
        const int gs = n / a.n_groups;
        uint64_t v = 0ull;
        if (lane < a.n_groups) {
            uint64_t k1 = 0ull, k2 = 0ull;
            for (int j = 0; j < gs; j++) {
                const uint64_t k = keys[lane * gs + j];
                k2 = k > k1 ? k1 : k > k2 ? k : k2;
                k1 = k > k1 ? k : k1;
            }
            v = k1;
            if (a.group_top == 2 && k2) v = choice_key(key_value(k1) + key_value(k2));
        }
        int rank = 0;
        for (int g = 0; g < a.n_groups; g++) {
            const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), g) << 32) |
                               (uint32_t)__builtin_amdgcn_readlane((int)v, g);
            rank += o > v || (o == v && g < lane);
        }
        const uint64_t keep = __ballot(lane < a.n_groups && v && rank < a.top_groups);
#pragma unroll
        for (int i = 0; i < P; i++)
            if (!((keep >> ((lane + 64 * i) / gs & 63)) & 1)) key[i] = 0ull;
    }

    /* topk rounds: the wave's largest key, of equals the lowest expert (lowest i, then lane) */
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
    double w = mine >= 0 ? score64(a.score, load_logit<TYPE>(a.logits, row + (mine < 0 ? 0 : mine)), m, sum) : 0.0;
    if (a.renorm) {
        const double s = wave_sum_f64(w);
        w = s > 0.0 ? w / s : 0.0;
    }
    if (live && lane < a.topk) {
        a.idx[(size_t)t * a.topk + lane] = mine;
        a.wt[(size_t)t * a.topk + lane] = (float)(w * (double)a.scale);
    }
}

template <int TYPE, int P>
void launch(const K3kRoute *a, hipStream_t st)
{
    const int waves = a->T < 1024 ? 1 : 4;
    const size_t lds = a->top_groups < a->n_groups ? (size_t)waves * a->n * 8 : 0;
    route_kernel<TYPE, P><<<(a->T + waves - 1) / waves, 64 * waves, lds, st>>>(*a);
}

template <int TYPE>
void pick(const K3kRoute *a, hipStream_t st)
{
    const int p = (a->n + 63) / 64;
    if (p <= 2) launch<TYPE, 2>(a, st);
    else if (p <= 4) launch<TYPE, 4>(a, st);
    else if (p <= 8) launch<TYPE, 8>(a, st);
    else if (p <= 16) launch<TYPE, 16>(a, st);
    else launch<TYPE, 32>(a, st);
}

}  // namespace

extern "C" int k3k_route(const K3kRoute *a, void *stream)
{
    if (a->type == K3D_F32) pick<K3D_F32>(a, (hipStream_t)stream);
    else pick<K3D_BF16>(a, (hipStream_t)stream);
    K3K_LAUNCH_CHECK("route");
    return 0;
}
