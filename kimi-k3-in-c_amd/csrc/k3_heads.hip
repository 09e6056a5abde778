/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_heads.hip -- RMSNorm of query and key heads with the position rotation (k3d_qk_norm_rope).
 *
 *   u = v / sqrt(mean(v^2) + eps) * w;  pairs of u turn by pos * freq.
 *
 * Bound by HBM: every head is read once and written once. A wave takes one token and a run of its
 * heads, 64 >> lsh of them at a time, so nothing waits for another wave. It forms the token's cosines and sines
 * once, in its part of LDS, and keeps, per element of its lane, the two factors that all heads share: an output is
 *   r (x A + p B),   A = w cos, B = -+ w' sin (p, w': the pair's other element; A = w, B = 0 outside the rotation),
 * seven vector instructions an element where the weights, cosines and sines read per head took over twenty.
 * An element's other one (half the rotated range away) is read a second time, out of the L1, rather than
 * fetched from the lane that holds it; where lengths, strides or borders do not fit 16 bytes, it comes through LDS
 * (heads_any_kernel). The next heads' rows are requested before these are worked on; the
 * reads of a head all come before its writes, so a head may be written over itself. 4096 tokens of 72 heads of 128 in bf16: 36.6 us
 * = 4.1 TB/s out of memory (two times beside each other, below, are measured alike, with heads that the last cache holds).
 */
#include "k3_common.h"
#include "k3_dev.h"
#include "k3k.h"

namespace {

constexpr int HD_WAVES = 4;              /* waves of a workgroup, each on its own */

/* cos and sin of a = pos * freq: reduced in fp64 by multiples of pi/2 (taken from it as a sum of two
 * doubles), then the Taylor polynomials to x^15 / x^14 on [-pi/4, pi/4], whose next terms are
 * under 2^-50. */
__device__ void turn(double a, float scale, float *c, float *s)
{
    const double n = rint(a * 0.63661977236758134308);
    double x = fma(-n, 1.57079632679489655800, a);
    x = fma(-n, 6.12323399573676603587e-17, x);
    const double z = x * x;
    double p = -1.0 / 1307674368000.0;
    p = fma(p, z, 1.0 / 6227020800.0);
    p = fma(p, z, -1.0 / 39916800.0);
    p = fma(p, z, 1.0 / 362880.0);
    p = fma(p, z, -1.0 / 5040.0);
    p = fma(p, z, 1.0 / 120.0);
    p = fma(p, z, -1.0 / 6.0);
    const double sn = fma(p * z, x, x);
    double q = -1.0 / 87178291200.0;
    q = fma(q, z, 1.0 / 479001600.0);
    q = fma(q, z, -1.0 / 3628800.0);
    q = fma(q, z, 1.0 / 40320.0);
    q = fma(q, z, -1.0 / 720.0);
    q = fma(q, z, 1.0 / 24.0);
    q = fma(q, z, -0.5);
    const double cs = fma(q, z, 1.0);
    const int k = (int)((long long)n & 3);
    const double co = (k & 1) ? sn : cs, si = (k & 1) ? cs : sn;
    *c = scale * (float)((k == 1 || k == 2) ? -co : co);
    *s = scale * (float)((k & 2) ? -si : si);
}

/* V elements as they lie in memory (one load), and as floats */
template <int TYPE, int V>
struct Chunk {
    static constexpr int W = TYPE == K3D_F32 ? V : (V + 1) / 2;
    uint32_t w[W];
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < W; i++) w[i] = 0;
    }
    __device__ __forceinline__ void load(const void *p, size_t i)
    {
        if constexpr (TYPE == K3D_BF16 && V == 1) w[0] = ((const uint16_t *)p)[i];
        else __builtin_memcpy(w, __builtin_assume_aligned((const char *)p + i * (TYPE == K3D_F32 ? 4 : 2), W * 4), W * 4);
    }
    /* at any alignment of an element (the hardware takes any) */
    __device__ __forceinline__ void load_any(const char *p) { __builtin_memcpy(w, __builtin_assume_aligned(p, TYPE == K3D_F32 ? 4 : 2), W * 4); }
    __device__ __forceinline__ void store_any(char *p) const { __builtin_memcpy(__builtin_assume_aligned(p, TYPE == K3D_F32 ? 4 : 2), w, W * 4); }
    __device__ __forceinline__ static Chunk pack(const float (&f)[V])
    {
        Chunk c;
        if constexpr (TYPE == K3D_F32) {
            __builtin_memcpy(c.w, f, W * 4);
        } else {
            __bf16 h[V];
#pragma unroll
            for (int j = 0; j < V; j++) h[j] = (__bf16)f[j];
            __builtin_memcpy(c.w, h, W * 4);
        }
        return c;
    }
    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (TYPE == K3D_F32) return __uint_as_float(w[i]);
        else return __uint_as_float((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
    __device__ __forceinline__ static void store(void *p, size_t i, const float (&f)[V])
    {
        if constexpr (TYPE == K3D_F32) {
            __builtin_memcpy(__builtin_assume_aligned((float *)p + i, W * 4), f, W * 4);
        } else {
            __bf16 h[V];
#pragma unroll
            for (int j = 0; j < V; j++) h[j] = (__bf16)f[j];
            __builtin_memcpy(__builtin_assume_aligned((uint16_t *)p + i, V * 2), h, V * 2);
        }
    }
};

/* 1 << lsh lanes per head, N chunks of V elements per lane; `split` waves per token */
template <int TYPE, int V, int N>
__global__ __launch_bounds__(64 * HD_WAVES) void heads_kernel(K3kHeads a, int lsh, int split)
{
    extern __shared__ float turns[];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = blockIdx.x * HD_WAVES + wv, t = wave / split, part = wave % split;
    if (t >= a.T) return;
    const double f0 = lane < a.rot / 2 ? a.freq[lane] : 0.0;
    const int pos = a.pos ? a.pos[t] : 0;
    if (pos < 0) return;
    const int h2 = a.rot / 2, L = 1 << lsh, l = lane & (L - 1), HP = 64 >> lsh;
    const int H = a.v[0].heads + a.v[1].heads, first = (int)((long)H * part / split), last = (int)((long)H * (part + 1) / split);
    float *const cs = turns + (size_t)wv * a.rot, *const sn = cs + h2;
    const float rdim = 1.0f / (float)a.dim;
    bool turned = false;

    for (int side = 0; side < 2; side++) {
        const int off = side ? a.v[0].heads : 0;
        const int hb = max(first, off) - off, he = min(last, off + a.v[side].heads) - off;
        if (hb >= he) continue;
        const void *const in = a.v[side].in;
        void *const out = a.v[side].out;
        const size_t ib = (size_t)t * a.v[side].ld, ob = (size_t)t * a.v[side].ldo;
        const float *const w = a.v[side].w;
        Chunk<TYPE, V> u[N], o[N];
        auto load = [&](int h) {
            if (h >= he) h = he - 1;        /* (lanes without a head repeat the last one's reads) */
            const size_t at = ib + (size_t)h * a.v[side].hs;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int e = (l + j * L) * V, r = e - a.rot_off;
                u[j].zero();
                o[j].zero();
                if (e >= a.dim) continue;
                u[j].load(in, at + e);
                if (r < 0 || r >= a.rot) continue;
                if (a.pairs == K3D_ROT_HALVES) o[j].load(in, at + (r < h2 ? e + h2 : e - h2));
                else if (V == 1) o[j].load(in, at + (r & 1 ? e - 1 : e + 1));
            }
        };
        load(hb + (lane >> lsh));
        if (!turned) {
            for (int i = lane; i < h2; i += 64) turn((double)pos * (i < 64 ? f0 : a.freq[i]), a.rot_scale, &cs[i], &sn[i]);
            __builtin_amdgcn_wave_barrier();
            turned = true;
        }
        float A[N][V], B[N][V];
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int e = (l + j * L) * V, r = e - a.rot_off;       /* (a chunk lies in or outside the range as a whole) */
#pragma unroll
            for (int i = 0; i < V; i++) A[j][i] = 1.0f, B[j][i] = 0.0f;
            if (e >= a.dim) continue;
            if (w) __builtin_memcpy(A[j], w + e, V * 4);
            if (r < 0 || r >= a.rot) continue;
            if (a.pairs == K3D_ROT_HALVES) {
                const bool one = r < h2;
                const int k = one ? r : r - h2;
                float c[V], d[V];
                if (w) __builtin_memcpy(B[j], w + (one ? e + h2 : e - h2), V * 4);
                __builtin_memcpy(c, __builtin_assume_aligned(cs + k, V * 4), V * 4);
                __builtin_memcpy(d, __builtin_assume_aligned(sn + k, V * 4), V * 4);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float q = w ? B[j][i] * d[i] : d[i];
                    A[j][i] *= c[i];
                    B[j][i] = one ? -q : q;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const bool one = !((r + i) & 1);
                    const float p = V > 1 ? (w ? w[e + (i ^ (V > 1))] : 1.0f) : w ? w[one ? e + 1 : e - 1] : 1.0f;
                    const float q = p * sn[(r + i) / 2];
                    A[j][i] *= cs[(r + i) / 2];
                    B[j][i] = one ? -q : q;
                }
            }
        }
        for (int h = hb + (lane >> lsh); h - (lane >> lsh) < he; h += HP) {
            float x[N][V], y[N][V], ss = 0.0f;
#pragma unroll
            for (int j = 0; j < N; j++)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    x[j][i] = u[j].get(i);
                    y[j][i] = V > 1 && a.pairs == K3D_ROT_INTERLEAVED ? u[j].get(i ^ (V > 1)) : o[j].get(i);
                    ss = fmaf(x[j][i], x[j][i], ss);
                }
            if (h - (lane >> lsh) + HP < he) load(h + HP);
            for (int q = L >> 1; q; q >>= 1) ss += __shfl_xor(ss, q);
            const float rs = 1.0f / sqrtf(fmaf(ss, rdim, a.eps));
            if (h < he) {
                const size_t at = ob + (size_t)h * a.v[side].hso;
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const int e = (l + j * L) * V, r = e - a.rot_off;
                    if (e >= a.dim) continue;
                    float f[V];
                    if (r >= 0 && r < a.rot) {
#pragma unroll
                        for (int i = 0; i < V; i++) f[i] = rs * fmaf(x[j][i], A[j][i], y[j][i] * B[j][i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < V; i++) f[i] = rs * (x[j][i] * A[j][i]);
                    }
                    Chunk<TYPE, V>::store(out, at + e, f);
                }
            }
        }
    }
}

/* Heads of any length from V, at any alignment, with the rotated range and its halves anywhere: a lane's chunk may lie on
 * both sides of a border, and the last one of a head, read where it ends with the head, holds elements of the one before it too
 * (computed twice, counted once, written twice alike). An element's other one comes out of LDS, where the wave lays its heads
 * as they are read. Out of memory 4096 tokens of 13 heads of 154 take 23 us (bytes: 6.6), bound by instructions: 1934 a wave, 341 of them for its angles,
 * most of the rest to set up two factors an element on either side. 4096 tokens of 72 heads of 128 in bf16, 74 of them rotated: 36.3 us; an element a lane and load, which such
 * borders otherwise allow, 81.7 (one token 4.8 and 3.6); 32 + 4 heads of 256 with 100 rotated 34.5, two elements a load 42.7. */
template <int TYPE, int V, int N>
__global__ __launch_bounds__(64 * HD_WAVES) void heads_any_kernel(K3kHeads a, int lsh, int split, int pitch)
{
    extern __shared__ float turns[];
    constexpr int ES = TYPE == K3D_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = blockIdx.x * HD_WAVES + wv, t = wave / split, part = wave % split;
    if (t >= a.T) return;
    const double f0 = lane < a.rot / 2 ? a.freq[lane] : 0.0;
    const int pos = a.pos ? a.pos[t] : 0;
    if (pos < 0) return;
    const int h2 = a.rot / 2, L = 1 << lsh, l = lane & (L - 1), HP = 64 >> lsh;
    const int H = a.v[0].heads + a.v[1].heads, first = (int)((long)H * part / split), last = (int)((long)H * (part + 1) / split);
    char *const mine = (char *)turns + (size_t)wv * (HP * pitch + a.rot * 4);       /* the wave's heads, then its turns */
    float *const cs = (float *)(mine + HP * pitch), *const sn = cs + h2;
    char *const row = mine + (lane >> lsh) * pitch;
    const float rdim = 1.0f / (float)a.dim;

    /* the lane's chunks: their first elements, how many of them the chunk before holds (V: no chunk), which ones turn, and where in
     * LDS their others lie */
    int e0[N], twice[N], other[N][V];
    uint32_t turns_[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int at = (l + j * L) * V;
        e0[j] = min(at, a.dim - V);
        twice[j] = min(at - e0[j], V);
        turns_[j] = 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int e = e0[j] + i, r = e - a.rot_off;
            const bool in = r >= 0 && r < a.rot;
            if (in) turns_[j] |= 1u << i;
            other[j][i] = !in ? e : a.pairs == K3D_ROT_HALVES ? (r < h2 ? e + h2 : e - h2) : r & 1 ? e - 1 : e + 1;
        }
    }
    for (int i = lane; i < h2; i += 64) turn((double)pos * (i < 64 ? f0 : a.freq[i]), a.rot_scale, &cs[i], &sn[i]);
    __builtin_amdgcn_wave_barrier();

    for (int side = 0; side < 2; side++) {
        const int off = side ? a.v[0].heads : 0;
        const int hb = max(first, off) - off, he = min(last, off + a.v[side].heads) - off;
        if (hb >= he) continue;
        const char *const in = (const char *)a.v[side].in + (size_t)t * a.v[side].ld * ES;
        char *const out = (char *)a.v[side].out + (size_t)t * a.v[side].ldo * ES;
        const float *const w = a.v[side].w;
        Chunk<TYPE, V> u[N];
        auto load = [&](int h) {
            if (h >= he) h = he - 1;        /* (lanes without a head repeat the last one's reads) */
            const char *const p = in + (size_t)h * a.v[side].hs * ES;
#pragma unroll
            for (int j = 0; j < N; j++) u[j].load_any(p + e0[j] * ES);
        };
        load(hb + (lane >> lsh));
        float A[N][V], B[N][V];
#pragma unroll
        for (int j = 0; j < N; j++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int e = e0[j] + i, r = e - a.rot_off;
                const bool halves = a.pairs == K3D_ROT_HALVES, one = halves ? r < h2 : !(r & 1);
                A[j][i] = w ? w[e] : 1.0f;
                B[j][i] = 0.0f;         /* (nothing of cs where nothing turns: rot may be 0) */
                if (turns_[j] >> i & 1) {
                    const int k = halves ? (one ? r : r - h2) : r >> 1;
                    const float q = (w ? w[other[j][i]] : 1.0f) * sn[k];
                    A[j][i] *= cs[k];
                    B[j][i] = one ? -q : q;
                }
            }
        for (int h = hb + (lane >> lsh); h - (lane >> lsh) < he; h += HP) {
            float x[N][V], ss = 0.0f;
#pragma unroll
            for (int j = 0; j < N; j++) {
                if (twice[j] < V) u[j].store_any(row + e0[j] * ES);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    x[j][i] = u[j].get(i);
                    ss = i >= twice[j] ? fmaf(x[j][i], x[j][i], ss) : ss;
                }
            }
            __builtin_amdgcn_wave_barrier();
            if (h - (lane >> lsh) + HP < he) load(h + HP);
            for (int q = L >> 1; q; q >>= 1) ss += __shfl_xor(ss, q);
            const float rs = 1.0f / sqrtf(fmaf(ss, rdim, a.eps));
            float y[N][V];
#pragma unroll
            for (int j = 0; j < N; j++)
#pragma unroll
                for (int i = 0; i < V; i++)
                    y[j][i] = TYPE == K3D_F32 ? ((const float *)row)[other[j][i]] : __uint_as_float((uint32_t)((const uint16_t *)row)[other[j][i]] << 16);
            __builtin_amdgcn_wave_barrier();
            if (h < he) {
                char *const p = out + (size_t)h * a.v[side].hso * ES;
#pragma unroll
                for (int j = 0; j < N; j++) {
                    if (twice[j] == V) continue;
                    float f[V];
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float n = x[j][i] * A[j][i];
                        f[i] = rs * (turns_[j] >> i & 1 ? fmaf(x[j][i], A[j][i], y[j][i] * B[j][i]) : n);
                    }
                    Chunk<TYPE, V>::pack(f).store_any(p + e0[j] * ES);
                }
            }
        }
    }
}

/* whether every head's rows, and the rotated range and its halves, fall on v elements */
bool fits(const K3kHeads *a, int v)
{
    const size_t bytes = (size_t)v * (a->type == K3D_F32 ? 4 : 2);
    if (a->dim % v) return false;
    for (int s = 0; s < 2; s++) {
        if (!a->v[s].heads) continue;
        if (((uintptr_t)a->v[s].in | (uintptr_t)a->v[s].out) % bytes) return false;
        if (a->T > 1 && (a->v[s].ld % v || a->v[s].ldo % v)) return false;
        if (a->v[s].heads > 1 && (a->v[s].hs % v || a->v[s].hso % v)) return false;
    }
    if (!a->rot) return true;
    return a->rot_off % v == 0 && (a->pairs == K3D_ROT_HALVES ? (a->rot / 2) % v == 0 : a->rot % v == 0);
}

/* A token's heads go over several waves while there are fewer waves than this per CU to keep the memory busy: 4 a SIMD
 * (777 tokens of 13 heads of 192 in fp32 8.1 us, 8.6 with 2 and 9.5 with 8; 4096 of 72 of 128 27.4, with 8 29.7;
 * 2000 of 72 of 256 27.3, 28.6 with 2 or 8). */
constexpr long HD_WANT = 16;

template <int TYPE, int V, int N>
void launch(const K3kHeads *a, hipStream_t st)
{
    const int chunks = (a->dim / V + N - 1) / N;
    int lsh = 0;
    while ((1 << lsh) < chunks) lsh++;
    const int HP = 64 >> lsh, H = a->v[0].heads + a->v[1].heads, passes = (H + HP - 1) / HP;
    const long want = HD_WANT * k3k_cu_count();
    int split = (int)((want + a->T - 1) / a->T);
    if (split > passes) split = passes;
    const long waves = (long)a->T * split;
    heads_kernel<TYPE, V, N><<<(unsigned)((waves + HD_WAVES - 1) / HD_WAVES), 64 * HD_WAVES, (size_t)HD_WAVES * a->rot * 4, st>>>(*a, lsh, split);
}

template <int TYPE, int V, int N>
void launch_any(const K3kHeads *a, hipStream_t st)
{
    const int chunks = ((a->dim + V - 1) / V + N - 1) / N;
    int lsh = 0;
    while ((1 << lsh) < chunks) lsh++;
    const int HP = 64 >> lsh, H = a->v[0].heads + a->v[1].heads, passes = (H + HP - 1) / HP;
    const int pitch = (a->dim * (TYPE == K3D_F32 ? 4 : 2) + 15) / 16 * 16;
    int split = (int)((HD_WANT * k3k_cu_count() + a->T - 1) / a->T);
    if (split > passes) split = passes;
    const long waves = (long)a->T * split;
    heads_any_kernel<TYPE, V, N><<<(unsigned)((waves + HD_WAVES - 1) / HD_WAVES), 64 * HD_WAVES,
                                   (size_t)HD_WAVES * (HP * pitch + a->rot * 4), st>>>(*a, lsh, split, pitch);
}

/* a head of up to 1024 elements in at most 64 lanes */
template <int TYPE>
void pick(const K3kHeads *a, hipStream_t st)
{
    constexpr int V = TYPE == K3D_F32 ? 4 : 8;
    const int c = (a->dim + V - 1) / V, n = (c + 63) / 64;
    if (a->dim < V) return launch<TYPE, 1, 1>(a, st);
    if (!fits(a, V)) {
        if (n <= 1) return launch_any<TYPE, V, 1>(a, st);
        if (n <= 2) return launch_any<TYPE, V, 2>(a, st);
        if constexpr (V <= 4) launch_any<TYPE, V, 4>(a, st);
        return;
    }
    /* Three times a power of two: three chunks a lane leave no lane idle (4096 tokens of 192 heads of 192 in bf16 164 -> 123 us),
     * where they leave waves enough (777 of 13 in fp32 8.2 us with one chunk, 9.4 with three). */
    if (c % 3 == 0 && c <= 192 && ((c / 3) & (c / 3 - 1)) == 0 &&
        (long)a->T * (a->v[0].heads + a->v[1].heads) * (c / 3) / 64 >= HD_WANT * k3k_cu_count())
        return launch<TYPE, V, 3>(a, st);
    if (n <= 1) return launch<TYPE, V, 1>(a, st);
    if (n <= 2) return launch<TYPE, V, 2>(a, st);
    if constexpr (V <= 4) launch<TYPE, V, 4>(a, st);
}

}  // namespace

extern "C" int k3k_heads(const K3kHeads *a, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    if (a->type == K3D_F32) pick<K3D_F32>(a, st);
    else pick<K3D_BF16>(a, st);
    K3K_LAUNCH_CHECK("heads");
    return 0;
}
