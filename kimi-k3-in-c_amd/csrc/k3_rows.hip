/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_rows.hip -- rows on their way to 8-bit products: the residual's addition and RMSNorm (k3d_add_norm), gated activations
 * (k3d_quant_f8), each rounded to e4m3 with a scale for each 128 columns.
 *
 *   v = x + res;  u = v / sqrt(mean(v^2) + eps) * w;   or   u = act(gate) up, or u = x
 *   s = max(max |u|, 2^-100) / 448 over 128 columns;  code = e4m3(u / s)
 *
 * Bound by memory. A lane holds eight neighbouring columns, so a block is the 16 lanes of a DPP row and its largest
 * magnitude takes four of them, without LDS; a row's elements stay in registers between the sum of squares and the rounding.
 */
#include "k3_common.h"
#include "k3_dev.h"
#include "k3_f8.h"
#include "k3k.h"

#include <math.h>

namespace {

/* (16 bytes at any alignment of their elements: as one vector, where a copy of eight elements became smaller stores, 51 against 47 us at
 * 4096 rows of 7168) */
typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

/* Elements i ..+8 of a row of n, zeros behind its end; any alignment of the elements. */
template <int TYPE>
__device__ __forceinline__ void load8(float (&f)[8], const void *row, int i, int n)
{
    if constexpr (TYPE == K3D_F32) {
        const float *p = (const float *)row + i;
        if (i + 8 <= n) __builtin_memcpy(f, p, 32);
        else
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = i + j < n ? p[j] : 0.0f;
    } else {
        const uint16_t *p = (const uint16_t *)row + i;
        uint16_t h[8];
        if (i + 8 <= n) __builtin_memcpy(h, p, 16);
        else
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] = i + j < n ? p[j] : (uint16_t)0;
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = k3_bf16_to_f32(h[j]);
    }
}

__device__ __forceinline__ void load8_of(float (&f)[8], const void *p, int type, size_t row, int i, int n)
{
    if (type == K3D_F32) load8<K3D_F32>(f, (const float *)p + row, i, n);
    else load8<K3D_BF16>(f, (const uint16_t *)p + row, i, n);
}

/* NT: not to be read again soon (rows of bf16; the sum of 4096 rows of 7168 41.0 against 46.2 us, of 1024 11.6 against 12.7, the same up to 256 and in fp32;
 * where the next call reads it at once 4096 take 39.9 against 36.9) */
template <bool NT = false>
__device__ __forceinline__ void store8_of(void *p, int type, size_t row, int i, int n, const float (&f)[8])
{
    if (type == K3D_F32) {
        float *q = (float *)p + row + i;
        if (i + 8 <= n) __builtin_memcpy(q, f, 32);
        else
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j < n) q[j] = f[j];
    } else {
        uint16_t *q = (uint16_t *)p + row + i;
        __bf16 h[8];
#pragma unroll
        for (int j = 0; j < 8; j++) h[j] = (__bf16)f[j];
        if (i + 8 <= n) {
            if (NT) __builtin_nontemporal_store(__builtin_bit_cast(u32x4a, h), (u32x4a *)q);
            else *(u32x4a *)q = __builtin_bit_cast(u32x4a, h);
        }
        else
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j < n) q[j] = __builtin_bit_cast(uint16_t, h[j]);
    }
}

/* u / s from r = 1 / s, with the remainder's share: u r alone is up to 1.5 units in the last place off, and a code is a choice that such a step
 * can turn. s of infinity gives 0 as u r does. */
__device__ __forceinline__ float quotient(float u, float s, float r)
{
    const float q = u * r;
    return fmaf(fmaf(-q, s < INFINITY ? s : 0.0f, u), r, q);
}

/* the lane's eight columns (zeros behind the row's end) as codes, the first lane of a block its scale; every lane of the block takes part.
 * EXACT: of quotients rounded once. Behind a gated activation, itself some 7 units off, they change no more than it does (32768 rows of 2048: 67.7
 * against 65.1 us). */
template <bool EXACT>
__device__ __forceinline__ void put_codes(uint8_t *q, float *qs, size_t qrow, size_t srow, int i, const float (&u)[8], bool there)
{
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, abs_bits(u[j]));
    const float s = f8_scale(row_max_bits(m)), r = 1.0f / s;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = EXACT ? quotient(u[j], s, r) : u[j] * r;
    uint2 c;
    c.x = f8_codes(v[0], v[1], v[2], v[3]);
    c.y = f8_codes(v[4], v[5], v[6], v[7]);
    if (!there) return;
    *reinterpret_cast<uint2 *>(q + qrow + i) = c;
    if ((threadIdx.x & 15) == 0) qs[srow + i / 128] = s;
}

/* A row to NW waves, P pieces of eight columns a lane. 4096 rows of 7168 in bf16 with a residual 43 us, 4.8 TB/s (a large copy 5.04); one row
 * 3.9 us, a launch. */
template <int P, int NW>
__global__ __launch_bounds__(64 * NW) void add_norm_kernel(K3kNorm a, unsigned t0)
{
    __shared__ float part[NW];
    const int tid = threadIdx.x;
    const size_t t = t0 + blockIdx.x;
    float v[P][8];
#pragma unroll
    for (int p = 0; p < P; p++) load8_of(v[p], a.x, a.x_type, t * a.ldx, (p * 64 * NW + tid) * 8, a.n);
    if (a.res) {
        float r[P][8];
#pragma unroll
        for (int p = 0; p < P; p++) load8_of(r[p], a.res, a.r_type, t * a.ldr, (p * 64 * NW + tid) * 8, a.n);
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int j = 0; j < 8; j++) v[p][j] += r[p][j];
    }
    float ss = 0.0f;
#pragma unroll
    for (int p = 0; p < P; p++) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) s = fmaf(v[p][j], v[p][j], s);
        ss += s;
    }
    ss = wave_total_f32(ss);
    if (NW > 1) {
        if ((tid & 63) == 0) part[tid >> 6] = ss;
        __syncthreads();
        ss = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) ss += part[w];
    }
    const float rms = sqrtf(ss / (float)a.n + a.eps), rstd = 1.0f / rms;
#pragma unroll
    for (int p = 0; p < P; p++) {
        const int i = (p * 64 * NW + tid) * 8;
        if (a.sum && i < a.n) store8_of<true>(a.sum, a.r_type, t * a.ldsum, i, a.n, v[p]);
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = 1.0f;
        if (a.w) load8<K3D_F32>(w, a.w, i, a.n);
#pragma unroll
        for (int j = 0; j < 8; j++) v[p][j] = i + j < a.n ? quotient(v[p][j], rms, rstd) * w[j] : 0.0f;
        if (a.y && i < a.n) store8_of(a.y, a.y_type, t * a.ldy, i, a.n, v[p]);
        if (a.q) put_codes<true>(a.q, a.qs, t * a.ldq, t * a.ldqs, i, v[p], i < (a.n + 127) / 128 * 128);
    }
}

/* 16 lanes to a block of 128 columns, 16 blocks to a workgroup. 32768 rows of 2048 in bf16 with silu 65 us, 5.1 TB/s. */
template <bool GATED>
__global__ __launch_bounds__(256) void quant_kernel(K3kQuant a, unsigned t0, int nb, int wgs)
{
    const int kb = (int)(blockIdx.x % (unsigned)wgs) * 16 + (threadIdx.x >> 4);
    const size_t t = t0 + blockIdx.x / (unsigned)wgs;
    const int i = kb * 128 + (threadIdx.x & 15) * 8;
    float u[8];
    load8_of(u, a.x, a.x_type, t * a.ldx, i, a.n);
    if (GATED) {
        float g[8];
        load8_of(g, a.x, a.x_type, t * a.ldx + a.n, i, a.n);
        const float r1 = 1.0f / a.b1, r2 = 1.0f / a.b2;
#pragma unroll
        for (int j = 0; j < 8; j++) u[j] = glu_of(u[j], g[j], a.act, a.b1, a.b2, r1, r2);
        if (i + 8 > a.n)
#pragma unroll
            for (int j = 0; j < 8; j++) u[j] = i + j < a.n ? u[j] : 0.0f;
    }
    put_codes<!GATED>(a.q, a.qs, t * a.ldq, t * a.ldqs, i, u, kb < nb);
}

/* Eight columns of one token to a thread; the slots' rows are requested four at a time. HALVES: as 16-bit floats with scales (2048
 * tokens of 8 slots of 7168 51 us, 5.4 TB/s; as fp32 113). */
template <bool HALVES>
__global__ __launch_bounds__(256) void sum_slots_kernel(K3kSum a, unsigned t0, unsigned per)
{
    const size_t t = t0 + blockIdx.x / per;
    const int i = (int)((blockIdx.x % per) * 256 + threadIdx.x) * 8;
    if (i >= a.n) return;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < a.topk; j += 4) {
        float v[4][8], w[4];
        f16x8 h[4];
        float sc[4];
        bool on[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const size_t k = t * a.topk + min(j + u, a.topk - 1);
            on[u] = j + u < a.topk && (unsigned)a.idx[k] < (unsigned)a.n_experts;
            w[u] = a.wt[k];
            if (!on[u]) continue;
            if constexpr (HALVES) {
                h[u] = *(const f16x8 *)((const _Float16 *)a.y + k * a.ldy + i);
                sc[u] = a.ys[k * (a.ldy / 64) + i / 64];
            } else load8<K3D_F32>(v[u], (const float *)a.y + k * a.ldy, i, a.n);
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (on[u])
#pragma unroll
                for (int c = 0; c < 8; c++) s[c] = fmaf(w[u], HALVES ? (float)h[u][c] * sc[u] : v[u][c], s[c]);
    }
    store8_of(a.out, a.out_type, t * a.ldo, i, a.n, s);
}

/* go(first row, rows) for as many rows at a time as a launch takes: under 2^32 work-items, `threads` a row */
template <class F>
void each_launch(int T, unsigned threads, F &&go)
{
    const unsigned most = 0xffffffffu / threads;
    for (unsigned t = 0; t < (unsigned)T; t += most) go(t, (unsigned)T - t < most ? (unsigned)T - t : most);
}

template <int P, int NW>
void norm_go(const K3kNorm *a, hipStream_t st)
{
    each_launch(a->T, 64 * NW, [&](unsigned t0, unsigned n) { add_norm_kernel<P, NW><<<n, 64 * NW, 0, st>>>(*a, t0); });
}

}  // namespace

extern "C" int k3k_add_norm(const K3kNorm *a, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    const int pieces = (a->n + 127) / 128 * 16;         /* whole blocks: their lanes all take part */
    /* (4096 rows of 7168: eight waves to a row 47 us, four 52, sixteen 47; 256 rows: 5.7, 7.7, 5.1) */
    if (pieces <= 64) norm_go<1, 1>(a, st);
    else if (pieces <= 128) norm_go<2, 1>(a, st);
    else if (a->T < 512 && pieces <= 1024) norm_go<1, 16>(a, st);
    else if (pieces <= 256) norm_go<1, 4>(a, st);
    else if (pieces <= 512) norm_go<1, 8>(a, st);
    else if (pieces <= 1024) norm_go<2, 8>(a, st);
    else if (pieces <= 2048) norm_go<2, 16>(a, st);
    else if (pieces <= 4096) norm_go<4, 16>(a, st);
    else norm_go<8, 16>(a, st);
    K3K_LAUNCH_CHECK("add_norm");
    return 0;
}

extern "C" int k3k_sum_slots(const K3kSum *a, void *stream)
{
    const unsigned per = ((unsigned)a->n + 2047) / 2048;
    each_launch(a->T, 256 * per, [&](unsigned t0, unsigned n) {
        if (a->ys) sum_slots_kernel<true><<<n * per, 256, 0, (hipStream_t)stream>>>(*a, t0, per);
        else sum_slots_kernel<false><<<n * per, 256, 0, (hipStream_t)stream>>>(*a, t0, per);
    });
    K3K_LAUNCH_CHECK("sum_slots");
    return 0;
}

extern "C" int k3k_quant_f8(const K3kQuant *a, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    const int nb = (a->n + 127) / 128, wgs = (nb + 15) / 16;
    each_launch(a->T, 256u * wgs, [&](unsigned t0, unsigned n) {
        if (a->act == K3D_GLU_NONE) quant_kernel<false><<<n * wgs, 256, 0, st>>>(*a, t0, nb, wgs);
        else quant_kernel<true><<<n * wgs, 256, 0, st>>>(*a, t0, nb, wgs);
    });
    K3K_LAUNCH_CHECK("quant_f8");
    return 0;
}
