/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_heads.hip -- RMSNorm of query and key heads with the position rotation (k3d_qk_norm_rope).
 *
 *   u = v / sqrt(mean(v^2) + eps) * w;  pairs of u turn by pos * freq.
 *
 * Bound by HBM: every head is read once and written once. A workgroup takes some tokens and
 * some of their heads; the tokens' cosines and sines, which all heads share, are formed once per
 * workgroup in LDS (per head they would cost more vector time than the rows take to move).
 * A head lies in L lanes of one wave, V elements of 16 bytes (or fewer where a row's
 * alignment, dim or the rotated range ask for it) per load; the other element of a pair (half the
 * rotated range away) is read a second time, out of the L1, rather than fetched from the lane that
 * holds it: the reads of a head all come before its writes, so a head may be written over itself.
 */
#include "k3_common.h"
#include "k3_dev.h"
#include "k3k.h"

namespace {

constexpr int HD_THREADS = 256;
constexpr int HD_MAXANG = 2048;          /* angles that fit a workgroup's table (16 KB) */

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

template <int TYPE, int V>
struct Chunk {
    float f[V];
    __device__ __forceinline__ void load(const void *p, size_t i)
    {
        if constexpr (TYPE == K3D_F32) {
            if constexpr (V == 4) {
                const float4 v = *reinterpret_cast<const float4 *>((const float *)p + i);
                f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
            } else if constexpr (V == 2) {
                const float2 v = *reinterpret_cast<const float2 *>((const float *)p + i);
                f[0] = v.x, f[1] = v.y;
            } else {
                f[0] = ((const float *)p)[i];
            }
        } else {
            uint32_t w[(V + 1) / 2];
            if constexpr (V == 8) {
                const uint4 v = *reinterpret_cast<const uint4 *>((const uint16_t *)p + i);
                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
            } else if constexpr (V == 4) {
                const uint2 v = *reinterpret_cast<const uint2 *>((const uint16_t *)p + i);
                w[0] = v.x, w[1] = v.y;
            } else if constexpr (V == 2) {
                w[0] = *reinterpret_cast<const uint32_t *>((const uint16_t *)p + i);
            } else {
                w[0] = ((const uint16_t *)p)[i];
            }
#pragma unroll
            for (int j = 0; j < V; j++) f[j] = __uint_as_float((j & 1) ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
        }
    }
    __device__ __forceinline__ void store(void *p, size_t i) const
    {
        if constexpr (TYPE == K3D_F32) {
            if constexpr (V == 4) *reinterpret_cast<float4 *>((float *)p + i) = make_float4(f[0], f[1], f[2], f[3]);
            else if constexpr (V == 2) *reinterpret_cast<float2 *>((float *)p + i) = make_float2(f[0], f[1]);
            else ((float *)p)[i] = f[0];
        } else {
            uint32_t w[(V + 1) / 2];
#pragma unroll
            for (int j = 0; j < V; j += 2)
                w[j / 2] = (uint32_t)k3_bf16_rne(f[j]) | (j + 1 < V ? (uint32_t)k3_bf16_rne(f[j + 1 < V ? j + 1 : j]) << 16 : 0u);
            if constexpr (V == 8) *reinterpret_cast<uint4 *>((uint16_t *)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
            else if constexpr (V == 4) *reinterpret_cast<uint2 *>((uint16_t *)p + i) = make_uint2(w[0], w[1]);
            else if constexpr (V == 2) *reinterpret_cast<uint32_t *>((uint16_t *)p + i) = w[0];
            else ((uint16_t *)p)[i] = (uint16_t)w[0];
        }
    }
};

/* L = 1 << lsh lanes per head, N chunks of V elements per lane; a workgroup takes tokens
 * tpw * blockIdx.x .. and heads hpw * blockIdx.y .. of them (queries first, then keys). */
template <int TYPE, int V, int N>
__global__ __launch_bounds__(HD_THREADS) void heads_kernel(K3kHeads a, int lsh, int tpw, int hpw)
{
    __shared__ float cs[HD_MAXANG], sn[HD_MAXANG];
    const int h2 = a.rot / 2, H = a.v[0].heads + a.v[1].heads;
    const int t0 = blockIdx.x * tpw, nt = min(tpw, a.T - t0);
    const int g0 = blockIdx.y * hpw, nh = min(hpw, H - g0);
    for (int i = threadIdx.x; i < nt * h2; i += HD_THREADS)
        turn((double)a.pos[t0 + i / h2] * a.freq[i % h2], a.rot_scale, &cs[i], &sn[i]);
    __syncthreads();

    const int L = 1 << lsh, l = threadIdx.x & (L - 1);
    const float rdim = 1.0f / (float)a.dim;
    for (int it = threadIdx.x >> lsh; it < nt * nh; it += HD_THREADS >> lsh) {
        const int tt = it / nh, t = t0 + tt, gh = g0 + it % nh;
        if (a.pos && a.pos[t] < 0) continue;
        const int side = gh >= a.v[0].heads, h = side ? gh - a.v[0].heads : gh;
        const void *in = a.v[side].in;
        const size_t ib = (size_t)t * a.v[side].ld + (size_t)h * a.v[side].hs;
        const size_t ob = (size_t)t * a.v[side].ldo + (size_t)h * a.v[side].hso;
        const float *w = a.v[side].w;
        Chunk<TYPE, V> u[N], o[N];
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int e = (l + j * L) * V;
            if (e >= a.dim) continue;
            u[j].load(in, ib + e);
            const int r = e - a.rot_off;
            if (r >= 0 && r < a.rot) {
                if (a.pairs == K3D_ROT_HALVES) o[j].load(in, ib + (r < h2 ? e + h2 : e - h2));
                else if (V == 1) o[j].load(in, ib + (r & 1 ? e - 1 : e + 1));
            }
#pragma unroll
            for (int i = 0; i < V; i++) ss = fmaf(u[j].f[i], u[j].f[i], ss);
        }
        for (int x = L >> 1; x; x >>= 1) ss += __shfl_xor(ss, x);
        const float rs = 1.0f / sqrtf(fmaf(ss, rdim, a.eps));
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int e = (l + j * L) * V;
            if (e >= a.dim) continue;
            const int r = e - a.rot_off;
            if (w)
#pragma unroll
                for (int i = 0; i < V; i++) u[j].f[i] *= rs * w[e + i];
            else
#pragma unroll
                for (int i = 0; i < V; i++) u[j].f[i] *= rs;
            if (r >= 0 && r < a.rot) {
                const float *c = cs + tt * h2, *s = sn + tt * h2;
                if (a.pairs == K3D_ROT_HALVES) {
                    const bool first = r < h2;
                    const int p = first ? e + h2 : e - h2, k = first ? r : r - h2;
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float x = o[j].f[i] * (w ? rs * w[p + i] : rs);
                        u[j].f[i] = fmaf(u[j].f[i], c[k + i], first ? -x * s[k + i] : x * s[k + i]);
                    }
                } else if constexpr (V == 1) {
                    const int p = r & 1 ? e - 1 : e + 1;
                    const float x = o[j].f[0] * (w ? rs * w[p] : rs);
                    u[j].f[0] = fmaf(u[j].f[0], c[r / 2], r & 1 ? x * s[r / 2] : -x * s[r / 2]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        const float x = u[j].f[i], y = u[j].f[i + 1], cc = c[(r + i) / 2], sc = s[(r + i) / 2];
                        u[j].f[i] = fmaf(x, cc, -y * sc);
                        u[j].f[i + 1] = fmaf(y, cc, x * sc);
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int e = (l + j * L) * V;
            if (e < a.dim) u[j].store(a.v[side].out, ob + e);
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

template <int TYPE, int V, int N>
void launch(const K3kHeads *a, hipStream_t st)
{
    const int chunks = (a->dim / V + N - 1) / N;
    int lsh = 0;
    while ((1 << lsh) < chunks) lsh++;
    const int per = HD_THREADS >> lsh, H = a->v[0].heads + a->v[1].heads;   /* heads at a time */
    int tpw = H < per ? per / H : 1;
    if (tpw > a->T) tpw = a->T;
    while (tpw > 1 && tpw * (a->rot / 2) > HD_MAXANG) tpw--;
    const long cus = k3k_cu_count();
    int hpw = H;
    /* few tokens: their heads over more workgroups */
    while (hpw > per && (long)((a->T + tpw - 1) / tpw) * ((H + hpw - 1) / hpw) < 2 * cus) hpw = (hpw + 1) / 2;
    const dim3 grid((a->T + tpw - 1) / tpw, (H + hpw - 1) / hpw);
    heads_kernel<TYPE, V, N><<<grid, HD_THREADS, 0, st>>>(*a, lsh, tpw, hpw);
}

template <int TYPE, int V>
void pick(const K3kHeads *a, hipStream_t st)
{
    const int c = a->dim / V;
    if (c <= 64) launch<TYPE, V, 1>(a, st);
    else if (c <= 128) launch<TYPE, V, 2>(a, st);
    else if (c <= 256) launch<TYPE, V, 4>(a, st);
    else if constexpr (V <= 2) {
        if (c <= 512) launch<TYPE, V, 8>(a, st);
        else if constexpr (V == 1) launch<TYPE, V, 16>(a, st);
    }
}

}  // namespace

extern "C" int k3k_heads(const K3kHeads *a, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    if (a->type == K3D_F32) {
        if (fits(a, 4)) pick<K3D_F32, 4>(a, st);
        else if (fits(a, 2)) pick<K3D_F32, 2>(a, st);
        else pick<K3D_F32, 1>(a, st);
    } else {
        if (fits(a, 8)) pick<K3D_BF16, 8>(a, st);
        else if (fits(a, 4)) pick<K3D_BF16, 4>(a, st);
        else if (fits(a, 2)) pick<K3D_BF16, 2>(a, st);
        else pick<K3D_BF16, 1>(a, st);
    }
    K3K_LAUNCH_CHECK("heads");
    return 0;
}
