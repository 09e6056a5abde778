/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_linear.hip -- dense products with bias, activation and residual (k3d_linear):
 *   y[t][o] = act(sum_k x[t][k] W[o][k] + bias[o]) + res[t][o],   W bf16, x bf16 or fp32.
 *
 * All products run on the matrix cores as bf16 with fp32 sums. An fp32 x is cut into three bf16 terms that hold its
 * 24 bits, so its products are as exact as fp32 ones, for three times the matrix work.
 *
 * What bounds it, and the kernel for it:
 *   - up to 64 tokens: reading W. lin_skinny_kernel, 16 to 64 rows of W to a workgroup, its waves sharing the columns, each
 *     with a ring of LDS stages of its own filled by DMA (one token of 7168 -> 12288, 176 MB, 28.6 us = 6.2 TB/s);
 *   - more: the matrix cores. lin_tile_kernel, tiles of 64 x 64 to 256 x 256, over slices of the columns where the tiles alone
 *     leave CUs idle; the slices' sums are joined in slice order by lin_join_kernel (4096 tokens of 7168 -> 12288 with
 *     silu 567 us = 1.27 PFLOP/s, the library's product alone 543);
 *   - weights that are not 16-byte aligned rows of whole 16 bytes: the same tiles, with W through registers instead of
 *     DMA (which wants 16-byte addresses); small ones for a few tokens, and rows shorter than a step, by lin_stream_kernel;
 *   - x that does not suit the DMA, and fp32 x for many tiles of outputs: lin_pack_kernel lays it out in the
 *     workspace first.
 *   - rows that end inside a step: the last step takes their last 64 columns, with zeros for those that come twice (300
 *     tokens of 4104 -> 2048 19.1 us; with x laid out first 21.9; 4096 of 4104 -> 4096, where that counts least, 136 and 130).
 * Which of them, and the tile and slices, go by the costs estimated below. Two times beside each other, here and below, are measured alike,
 * most with operands that the last cache holds from the call before; out of memory both are up to a quarter longer.
 */
#include "k3_common.h"
#include "k3_dev.h"
#include "k3k.h"

#include <math.h>
#include <type_traits>

namespace {

constexpr int LIN_KS = 64;                      /* columns of a tile kernel's step */
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));     /* (a load of uint4 loses what tells LDS arrays apart) */
constexpr uint32_t LIN_OOB = 0x80000000u;       /* a buffer offset past any descriptor used here */

/* f(0), f(1) .. f(N - 1), the numbers as constants */
template <int S, int N, class F>
__device__ __forceinline__ void each_stage(F &&f)
{
    if constexpr (S < N) {
        f(std::integral_constant<int, S>{});
        each_stage<S + 1, N>(f);
    }
}

/* ---- epilogue ------------------------------------------------------------------------ */
/* v / (1 + e^-z), z either v or of its sign. e^-z = 2^t e^c: t = -z log2 e as rounded, c = -z - t ln 2 (ln 2 as a sum of two floats) what the
 * rounding left, under 2^-16. Past t = 64, where 1 no longer counts, numerator and denominator are scaled by 2^-64, so the
 * result holds until it leaves fp32 itself (e^-z alone does so at z = -88.7). Within 7 * 2^-24 of the value (the exponential and the reciprocal two each;
 * DIV, with a corrected quotient: 6; without c, |z| more). Results of bf16 go without DIV: 8192 tokens of 512 -> 2048 with silu and a
 * residual 45.4 us, 43.5 without c and the scale too; of 4096 tokens of 1024 -> 4096 to fp32 54.6. */
template <bool DIV>
__device__ __forceinline__ float over_1p_exp(float v, float z)
{
#pragma clang fp contract(off)          /* (c belongs to t as rounded) */
    z = __builtin_amdgcn_fmed3f(z, -200.0f, 200.0f);            /* (nothing changes past these, and c stays finite) */
    const float t = -1.44269504f * z;
    const float c = fmaf(1.9046543e-9f, t, fmaf(-0.693147182f, t, -z));
    const bool far = t > 64.0f;
    const float k = far ? 0x1p-64f : 1.0f;
    const float d = fmaf(__builtin_amdgcn_exp2f(t - (far ? 64.0f : 0.0f)), 1.0f + c, k);
    const float q = __builtin_amdgcn_rcpf(d), u = v * k, w = u * q;
    if (!DIV) return w;
    const float r = fmaf(fmaf(-d, w, u), q, w);
    return r == r ? r : w;          /* (no correction where d or w is infinite) */
}

/* v (1 + erf(v / sqrt 2)) / 2 through erfc(z) = t P(t) e^-z^2, z = |v| / sqrt 2, t = 1 / (1 + 0.38 z): P of degree 8 interpolates
 * erfc(z) e^z^2 / t at the Chebyshev nodes of 0 <= z <= 10, within 2.5e-8 of itself (past it e^-z^2 is 0 in fp32).
 * By roundings: t's move erfc by up to three times as much, the square's and the exponent's by 1.5 v^2. That is
 * within 10 * 2^-24 |v| and, where v < 0, (18 + 1.5 v^2) 2^-24 of the value (6 and 13 + v^2 in emulation), which a result of bf16 rounds off. Where it is of fp32:
 * e^-z^2 = 2^s e^c with c what the square's and the exponent's rounding left, a corrected t, and up to |v| = 1 the Taylor series of
 * erf(v / sqrt 2) / 2v to v^14, whose next term is under 2^-28: within 17 * 2^-24 of the value (9 in emulation; for v > 0 6 and 2.6). 4096 tokens of
 * 1024 -> 4096 to fp32 62.3 us, 54.5 without these; to bf16 54.0. */
template <bool F32>
__device__ __forceinline__ float gelu(float v)
{
#pragma clang fp contract(off)          /* (c belongs to s and q as rounded) */
    const float a = F32 ? fminf(fabsf(v), 20.0f) : fabsf(v), q = a * a, s = -0.72134752f * q;    /* (c stays finite; erfc(14) is 0) */
    const float d = fmaf(0.26870058f, a, 1.0f);
    float t = __builtin_amdgcn_rcpf(d), e = __builtin_amdgcn_exp2f(s);
    if (F32) {
        t = fmaf(fmaf(-d, t, 1.0f), t, t);
        const float c = fmaf(1.9046543e-9f, s, fmaf(-0.693147182f, s, -0.5f * q)) - 0.5f * fmaf(a, a, -q);
        e *= 1.0f + c;
    }
    float p = 2.981513138e-02f;
    p = fmaf(p, t, -1.327961542e-01f);
    p = fmaf(p, t, 1.854386980e-01f);
    p = fmaf(p, t, -8.483748560e-02f);
    p = fmaf(p, t, 1.179101926e-01f);
    p = fmaf(p, t, 6.806875096e-02f);
    p = fmaf(p, t, 1.022790763e-01f);
    p = fmaf(p, t, 1.069136054e-01f);
    p = fmaf(p, t, 1.072081952e-01f);
    const float h = t * p * e;          /* erfc(z) / 2 */
    const float y = v > 0.0f ? 1.0f - h : h;
    if (!F32) return v * y;
    float g = -4.12266741e-08f;
    g = fmaf(g, q, 6.65969352e-07f);
    g = fmaf(g, q, -9.44465626e-06f);
    g = fmaf(g, q, 0.000115434688f);
    g = fmaf(g, q, -0.00118732822f);
    g = fmaf(g, q, 0.00997355701f);
    g = fmaf(g, q, -0.0664903801f);
    g = fmaf(g, q, 0.39894228f);
    return v * (a <= 1.0f ? fmaf(v, g, 0.5f) : y);
}

template <bool F32>
__device__ __forceinline__ float act_of(float v, int act)
{
    switch (act) {
    case K3D_ACT_RELU: return v < 0.0f ? 0.0f : v;
    case K3D_ACT_SILU: return over_1p_exp<F32>(v, v);
    case K3D_ACT_GELU: return gelu<F32>(v);
    case K3D_ACT_GELU_TANH: return over_1p_exp<F32>(v, 1.59576912f * v * fmaf(0.044715f * v, v, 1.0f));
    default: return v;
    }
}

/* the residual of outputs o ..+4 of token t as it lies in memory, requested apart from its use: an epilogue that waits for each row's
 * costs more than the bytes (8192 tokens of 512 -> 2048 with silu and a residual 54 us, four rows requested ahead 48) */
__device__ __forceinline__ uint4 res4(const K3kLinear &a, int t, int o)
{
    uint4 r = make_uint4(0, 0, 0, 0);
    if (!a.res || t >= a.T || o >= a.out) return r;
    const size_t at = (size_t)t * a.ldr + o;
    const int n = a.out - o;
    if (a.y_type == K3D_F32) {
        const uint32_t *q = (const uint32_t *)a.res + at;
        if (n >= 4) __builtin_memcpy(&r, q, 16);
        else r.x = q[0], r.y = n > 1 ? q[1] : 0u, r.z = n > 2 ? q[2] : 0u;
    } else {
        const uint16_t *q = (const uint16_t *)a.res + at;
        if (n >= 4) __builtin_memcpy(&r, q, 8);
        else r.x = q[0] | (n > 1 ? (uint32_t)q[1] << 16 : 0u), r.y = n > 2 ? q[2] : 0u;
    }
    return r;
}

/* outputs o ..+4 of token t: acc + bias b through the activation, plus the residual r (any alignment: the hardware stores 16
 * bytes to any address) */
__device__ __forceinline__ void put4(const K3kLinear &a, int t, int o, float4 acc, const float (&b)[4], uint4 r)
{
    if (t >= a.T || o >= a.out) return;
    const size_t yi = (size_t)t * a.ldy + o;
    const int n = min(4, a.out - o);
    float v[4] = {acc.x + b[0], acc.y + b[1], acc.z + b[2], acc.w + b[3]};
    if (a.y_type == K3D_F32) {
        if (a.act)
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = act_of<true>(v[i], a.act);
        float *y = (float *)a.y + yi;
        if (a.res) v[0] += __uint_as_float(r.x), v[1] += __uint_as_float(r.y), v[2] += __uint_as_float(r.z), v[3] += __uint_as_float(r.w);
        if (n == 4) {
            __builtin_memcpy(y, v, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 3; i++)
                if (i < n) y[i] = v[i];
        }
    } else {
        if (a.act)
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = act_of<false>(v[i], a.act);
        uint16_t *y = (uint16_t *)a.y + yi;
        if (a.res) {
            v[0] += __uint_as_float(r.x << 16), v[1] += __uint_as_float(r.x & 0xffff0000u);
            v[2] += __uint_as_float(r.y << 16), v[3] += __uint_as_float(r.y & 0xffff0000u);
        }
        __bf16 h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = (__bf16)v[i];
        if (n == 4) {
            __builtin_memcpy(y, h, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 3; i++)
                if (i < n) y[i] = __builtin_bit_cast(uint16_t, h[i]);
        }
    }
}

__device__ __forceinline__ void bias4(const K3kLinear &a, int o, float (&b)[4])
{
#pragma unroll
    for (int i = 0; i < 4; i++) b[i] = a.bias && o + i < a.out ? a.bias[o + i] : 0.0f;
}

/* ---- operands ------------------------------------------------------------------------ */
/* eight floats as three bf16 terms by truncation, x = h + m + l: each keeps the next 8 bits of the
 * significand, so the three hold all 24 and every product with a weight is exact. Infinities and
 * NaN are in the first term alone. */
__device__ __forceinline__ void cut3(const float (&f)[8], uint32_t (&h)[4], uint32_t (&m)[4], uint32_t (&l)[4])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t u[3][2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const float v = f[2 * i + e];
            u[0][e] = __float_as_uint(v);
            const float r1 = __builtin_amdgcn_classf(v, 0x204) ? 0.0f : v - __uint_as_float(u[0][e] & 0xffff0000u);
            u[1][e] = __float_as_uint(r1);
            u[2][e] = __float_as_uint(r1 - __uint_as_float(u[1][e] & 0xffff0000u));
        }
        /* the upper halves of a pair */
        h[i] = __builtin_amdgcn_perm(u[0][1], u[0][0], 0x07060302u);
        m[i] = __builtin_amdgcn_perm(u[1][1], u[1][0], 0x07060302u);
        l[i] = __builtin_amdgcn_perm(u[2][1], u[2][0], 0x07060302u);
    }
}

__device__ __forceinline__ k3_bf16x8 as_frag(const uint32_t (&w)[4])
{
    return k3_as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
}

/* eight bf16 from an address aligned to them only (one load: the hardware takes any alignment) */
__device__ __forceinline__ uint4 load8_any(const uint16_t *p)
{
    uint4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

/* the first n of eight bf16 (n < 1: none), zeros behind */
__device__ __forceinline__ uint4 load8_upto(const uint16_t *p, int n)
{
    uint64_t lo = 0, hi = 0;
#pragma unroll 1
    for (int i = min(n, 8) - 1; i >= 0; i--) {
        hi = (hi << 16) | (lo >> 48);
        lo = (lo << 16) | p[i];
    }
    return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

/* ---- short rows at any alignment: operands straight into registers -------------------------- */
/* A workgroup takes 16 rows of W and 16 tokens; its waves share the columns, each a run of 32-column steps, and
 * their sums meet in LDS. A lane's weights (row lane % 16, columns 8 (lane / 16) ..+8 of a step) are an MFMA operand
 * as loaded. Rows and tokens past the ends repeat the last one; only the last step can pass the end of
 * a row (guarded, zeros behind). */
template <int U, bool XF32>
__global__ __launch_bounds__(512) void lin_stream_kernel(K3kLinear a, int nw)
{
    __shared__ float4 part[8 * 64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
    const int og = (a.out + 15) / 16;
    const int o0 = (int)(blockIdx.x % og) * 16, t0 = (int)(blockIdx.x / og) * 16;
    const int steps = (a.in + 31) / 32, per = (steps + nw - 1) / nw;
    const int s0 = wv * per, n = min(per, steps - s0);          /* (n < 1: nothing for this wave) */
    constexpr int XS = XF32 ? 4 : 2;
    const uint16_t *const wp = a.W + (size_t)min(o0 + r16, a.out - 1) * a.ldw + 8 * g;
    const char *const xp = (const char *)a.x + ((size_t)min(t0 + r16, a.T - 1) * a.ldx + 8 * g) * XS;
    k3_f32x4 acc = {0.f, 0.f, 0.f, 0.f};

    struct Slot {
        uint4 w, x[XF32 ? 2 : 1];
    };
    auto load = [&](Slot &s, int step) {
        s.w = load8_any(wp + step * 32);
        const char *p = xp + (size_t)step * 32 * XS;
        s.x[0] = load8_any((const uint16_t *)p);
        if constexpr (XF32) s.x[1] = load8_any((const uint16_t *)(p + 16));
    };
    /* the step that passes the end of the rows */
    auto load_last = [&](Slot &s, int step) {
        const int k = step * 32, left = a.in - k - 8 * g;
        s.w = load8_upto(wp + k, left);
        const char *p = xp + (size_t)k * XS;
        if constexpr (XF32) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = i < left ? ((const float *)p)[i] : 0.0f;
            __builtin_memcpy(s.x, f, 32);
        } else {
            s.x[0] = load8_upto((const uint16_t *)p, left);
        }
    };
    auto use = [&](const Slot &s) {
        const k3_bf16x8 w = k3_as_bf16x8(s.w);
        if constexpr (XF32) {
            float f[8];
            uint32_t h[4], m[4], l[4];
            __builtin_memcpy(f, s.x, 32);
            cut3(f, h, m, l);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, as_frag(l), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, as_frag(m), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, as_frag(h), acc, 0, 0, 0);
        } else {
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, k3_as_bf16x8(s.x[0]), acc, 0, 0, 0);
        }
    };
    /* whole steps through a ring of U slots (past the end the last one is requested again and goes unused) */
    const int whole = min(n, a.in / 32 - s0);
    if (whole > 0) {
        Slot ring[U];
#pragma unroll
        for (int u = 0; u < U; u++) load(ring[u], s0 + min(u, whole - 1));
        int s = 0;
        for (; s + U <= whole; s += U)
#pragma unroll
            for (int u = 0; u < U; u++) {
                use(ring[u]);
                load(ring[u], s0 + min(s + u + U, whole - 1));
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (s + u < whole) use(ring[u]);
    }
    if (n > 0 && whole < n) {
        Slot s;
        load_last(s, s0 + n - 1);
        use(s);
    }
    part[wv * 64 + lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (wv == 0) {
        const int o = o0 + 4 * g;
        float b[4];
        bias4(a, o, b);
        const uint4 res = res4(a, t0 + r16, o);
        float4 s = part[lane];
        for (int w = 1; w < nw; w++) {
            const float4 v = part[w * 64 + lane];
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        put4(a, t0 + r16, o, s, b, res);
    }
}

/* ---- few tokens: a ring of LDS stages per wave ---------------------------------------------- */
/* A workgroup takes 16 RW rows of W and all tokens (8 XD of them at most); its NW waves share the columns in
 * runs of 64-column stages. Each wave fills a ring of NST stages of its own by DMA (8 lanes read a row's
 * 128 contiguous bytes; the operand layout itself, read from memory, has 16 lanes in a row on 16 rows
 * and a CU then takes in 10 bytes a cycle) and waits for its own requests alone, so there is no barrier until the
 * waves' sums meet. x takes part as bf16 or, cut into its three terms as it is read, fp32. */
template <int RW, int XR, int NW, int NST, bool XF32, int POL>
__global__ __launch_bounds__(64 * NW) void lin_skinny_kernel(K3kLinear a)
{
    constexpr int KS = LIN_KS, C = KS / 8, RD = 64 / C;         /* 16-byte columns of a row; rows of a DMA */
    constexpr int NT = (XR + 1) / 2, XB = XF32 ? 2 : 1;         /* token fragments; pieces of KS * 2 bytes of a row of x */
    constexpr int WD = 16 * RW / RD, XD = 8 * XR / RD, DN = WD + XD * XB;       /* DMAs of a stage */
    constexpr int STG = DN * 512;                               /* elements of a wave's stage */
    static_assert(RW * NT * 512 <= STG, "the sums fit the wave's part of a stage");
    __shared__ __attribute__((aligned(1024))) uint16_t S0[STG * NW], S1[STG * NW], S2[NST > 2 ? STG * NW : 8], S3[NST > 3 ? STG * NW : 8];
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int o0 = blockIdx.x * 16 * RW;
    auto swz = [](int r) { return (r >> 1) & 7; };
    const int nks = (a.in + KS - 1) / KS, k0 = (int)((long)nks * wv / NW), k1 = (int)((long)nks * (wv + 1) / NW);
    const int on = min(16 * RW, a.out - o0);

    /* 16-byte column c of an LDS row r lies in slot c ^ (r / 2 % 8): the rows of a fragment fall on all banks */
    const k3_rsrc rw = k3_make_rsrc(a.W + (size_t)o0 * a.ldw, (uint32_t)(((size_t)(on - 1) * a.ldw + a.in) * 2));
    const k3_rsrc rx = k3_make_rsrc(a.x, (uint32_t)(((size_t)(a.T - 1) * a.ldx + a.in) * (XF32 ? 4 : 2)));
    uint32_t wo[WD], xo[XD];
#pragma unroll
    for (int i = 0; i < WD; i++) {
        const int r = RD * i + lane / C;
        wo[i] = (uint32_t)min(r, on - 1) * (uint32_t)(a.ldw * 2) + ((lane & (C - 1)) ^ swz(r)) * 16;
    }
#pragma unroll
    for (int i = 0; i < XD; i++) {
        const int r = RD * i + lane / C;
        xo[i] = (uint32_t)min(r, a.T - 1) * (uint32_t)(a.ldx * (XF32 ? 4 : 2)) + ((lane & (C - 1)) ^ swz(r)) * 16;
    }
    auto buf_of = [&](auto slot) -> uint16_t * {
        constexpr int S = decltype(slot)::value;
        uint16_t *b;
        if constexpr (S == 0) b = S0;
        else if constexpr (S == 1) b = S1;
        else if constexpr (S == 2) b = S2;
        else b = S3;
        return b + wv * STG;
    };
    /* the columns of the last block that the one before it holds, per parity of a DMA (the swizzle's period) */
    const int over = nks * KS - a.in;
    uint32_t again[XF32 ? 3 : 1][2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int c = (lane & (C - 1)) ^ swz(RD * i + lane / C);
        again[0][i] = 8 * c < over ? LIN_OOB : 0u;
        if constexpr (XF32) again[1][i] = 4 * c < over ? LIN_OOB : 0u, again[2][i] = 4 * (C + c) < over ? LIN_OOB : 0u;
    }
    /* the stage of column block xk; the last block of a row ends with it, with zeros (of W and of x: either may be
     * infinite) for the columns that come twice; past the wave's run: zeros, so that every stage requests as much */
    int xk = k0;
    auto issue = [&](auto slot) {
        uint16_t *const b = buf_of(slot);
        const uint32_t none = xk < k1 ? 0u : LIN_OOB;
        const bool end = xk == nks - 1;
        const uint32_t c = end ? a.in - KS : xk * KS;
        uint32_t no[XF32 ? 3 : 1][2];
#pragma unroll
        for (int q = 0; q < (XF32 ? 3 : 1); q++)
#pragma unroll
            for (int i = 0; i < 2; i++) no[q][i] = none | (end ? again[q][i] : 0u);
#pragma unroll
        for (int i = 0; i < WD; i++) k3_dma16<POL>(rw, b + i * 512, wo[i] | no[0][i & 1], c * 2);
#pragma unroll
        for (int h = 0; h < XB; h++)
#pragma unroll
            for (int i = 0; i < XD; i++)
                k3_dma16(rx, b + (WD + h * XD + i) * 512, xo[i] | no[XF32 ? 1 + h : 0][i & 1], c * (XF32 ? 4 : 2) + h * KS * 2);
        xk++;
    };
    k3_f32x4 acc[RW][NT];
#pragma unroll
    for (int i = 0; i < RW; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = k3_f32x4{0.f, 0.f, 0.f, 0.f};
    const int sw = swz(r16);
    constexpr int WAITN = DN * (NST - 1);
    constexpr int WAIT_STAGE = (WAITN & 15) | (7 << 4) | (15 << 8) | ((WAITN >> 4) << 14);
    constexpr int WAIT_LGKM0 = 15 | (7 << 4) | (0 << 8) | (3 << 14);
    static_assert(WAITN < 64, "requests in flight");
    auto step = [&](auto slot) {
        const uint16_t *const b = buf_of(slot);
        __builtin_amdgcn_s_waitcnt(WAIT_STAGE);
        __builtin_amdgcn_sched_barrier(0);
        u32x4 wf[KS / 32][RW], xf[KS / 32][NT][XB];
#pragma unroll
        for (int h = 0; h < KS / 32; h++) {
#pragma unroll
            for (int i = 0; i < RW; i++) wf[h][i] = *reinterpret_cast<const u32x4 *>(b + (16 * i + r16) * KS + ((4 * h + g) ^ sw) * 8);
            /* (a last fragment of 8 tokens: its upper lanes repeat the lower ones') */
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const int r = 16 * j + (XR % 2 && j == NT - 1 ? r16 & 7 : r16), s = swz(r), f = 8 * h + 2 * g;
                const uint16_t *q = b + (WD * RD + r) * KS;
                if constexpr (XF32) {      /* two 16-byte columns */
                    xf[h][j][0] = *reinterpret_cast<const u32x4 *>(q + f / C * XD * 512 + ((f % C) ^ s) * 8);
                    xf[h][j][1] = *reinterpret_cast<const u32x4 *>(q + f / C * XD * 512 + ((f % C + 1) ^ s) * 8);
                } else {
                    xf[h][j][0] = *reinterpret_cast<const u32x4 *>(q + ((4 * h + g) ^ s) * 8);
                }
            }
        }
        __builtin_amdgcn_s_waitcnt(WAIT_LGKM0);
        __builtin_amdgcn_sched_barrier(0);
        issue(slot);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int h = 0; h < KS / 32; h++)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                if constexpr (XF32) {
                    float f[8];
                    uint32_t t[3][4];
#pragma unroll
                    for (int e = 0; e < 8; e++) f[e] = __uint_as_float(xf[h][j][e / 4][e % 4]);
                    cut3(f, t[2], t[1], t[0]);
#pragma unroll
                    for (int q = 0; q < 3; q++)
#pragma unroll
                        for (int i = 0; i < RW; i++)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(k3_bf16x8, wf[h][i]), as_frag(t[q]), acc[i][j], 0, 0, 0);
                } else {
                    const u32x4 v = xf[h][j][0];
#pragma unroll
                    for (int i = 0; i < RW; i++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(k3_bf16x8, wf[h][i]), __builtin_bit_cast(k3_bf16x8, v), acc[i][j], 0, 0, 0);
                }
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    each_stage<0, NST>(issue);
    int left = k1 - k0;
    for (; left >= NST; left -= NST) each_stage<0, NST>(step);
    each_stage<0, NST - 1>([&](auto slot) {
        if (decltype(slot)::value < left) step(slot);
    });
    __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));      /* the last requests land before LDS is used again */

    float4 *const mine = reinterpret_cast<float4 *>(S0 + wv * STG);
#pragma unroll
    for (int i = 0; i < RW; i++)
#pragma unroll
        for (int j = 0; j < NT; j++)
            mine[(i * NT + j) * 64 + lane] = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
    __syncthreads();
    for (int q = wv; q < RW * NT; q += NW) {
        const int o = o0 + 16 * (q / NT) + 4 * g, t = 16 * (q % NT) + r16;
        float b[4];
        bias4(a, o, b);
        const uint4 res = res4(a, t, o);
        const float4 *p = reinterpret_cast<const float4 *>(S0) + q * 64 + lane;
        float4 s = p[0];
#pragma unroll
        for (int w = 1; w < NW; w++) {
            const float4 v = p[w * (STG / 8)];
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        put4(a, t, o, s, b, res);
    }
}

/* ---- x for the tile kernel: terms and padding ------------------------------------------- */
/* xs[t][terms][kp] bf16, kp a multiple of 64: fp32 x as l, m, h; bf16 x as it is. Where the rows' length is
 * no multiple of 64, the last block of 64 columns holds the rest with zeros behind it (over 0), or columns
 * in - 64 .. in with zeros in place of those that the block before it holds (over 64 - in % 64). Under 2^31 pieces of eight
 * columns in a launch (a 64-bit division takes 0.2 us). */
template <bool XF32>
__global__ __launch_bounds__(256) void lin_pack_kernel(uint16_t *xs, const void *x, long ldx, int T, int in, int kp, int over)
{
    const int per = kp / 8;
    const unsigned i = blockIdx.x * 256 + threadIdx.x;
    const int t = (int)(i / (unsigned)per), kb = (int)(i - (unsigned)t * per) * 8;
    if (t >= T) return;
    const int last = kp - LIN_KS, k = kb >= last ? kb - over : kb;      /* the first of the eight columns */
    const bool whole = k >= (kb >= last ? last : 0) && k + 8 <= in;
    if (XF32) {
        const float *p = (const float *)x + (size_t)t * ldx;
        float f[8];
        if (whole && ((uintptr_t)(p + k) & 15) == 0) {
            __builtin_memcpy(f, __builtin_assume_aligned(p + k, 16), 32);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = k + j < in && (kb < last || k + j >= last) ? p[k + j] : 0.0f;
        }
        uint32_t h[4], m[4], l[4];
        cut3(f, h, m, l);
        uint16_t *q = xs + (size_t)t * 3 * kp + kb;
        *reinterpret_cast<uint4 *>(q) = make_uint4(l[0], l[1], l[2], l[3]);
        *reinterpret_cast<uint4 *>(q + kp) = make_uint4(m[0], m[1], m[2], m[3]);
        *reinterpret_cast<uint4 *>(q + 2 * (size_t)kp) = make_uint4(h[0], h[1], h[2], h[3]);
    } else {
        const uint16_t *p = (const uint16_t *)x + (size_t)t * ldx;
        uint4 v;
        if (whole) {
            v = load8_any(p + k);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (k + j < in && (kb < last || k + j >= last)) w[j / 2] |= (uint32_t)p[k + j] << (16 * (j & 1));
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *reinterpret_cast<uint4 *>(xs + (size_t)t * kp + kb) = v;
    }
}

/* ---- many tokens: tiles through LDS -------------------------------------------------------- */
typedef struct {
    K3kLinear a;
    const void *x;          /* bf16 rows (or fp32 ones, to be cut as they are read), 16-byte aligned with their stride */
    long ldx;
    int xcols;              /* columns of x: in, or all terms' padded ones */
    int nks, steps;         /* steps of one term, of all */
    int xend;               /* the step that reads x's last 64 columns where they end (its first ones again as zeros), or -1 */
    int nt, no;             /* tiles over tokens and outputs */
    int nsl, per;           /* slices of the steps, steps of one */
    float *part;            /* [nsl][T][out] sums of the slices (nsl > 1) */
} LinTile;

/* Which token and output tile workgroup b takes. The dispatcher deals workgroups to the XCDs in turn; each XCD
 * gets a run of tiles of its own, slice by slice, down 8 token tiles before the next outputs: what a run reads of W it reads
 * once from its L2, and its x stays there. */
__device__ __forceinline__ void tile_of(const LinTile &p, int b, int &tt, int &to, int &sl)
{
    const int tiles = p.nt * p.no, all = tiles * p.nsl;
    const int full = all / K3_NXCD * K3_NXCD;
    int i = b;
    if (b < full) i = (b % K3_NXCD) * (all / K3_NXCD) + b / K3_NXCD;
    sl = i / tiles;
    i -= sl * tiles;
    constexpr int GT = 8;
    const int blk = GT * p.no, q = i / blk, h = min(GT, p.nt - q * GT), r = i - q * blk;
    to = r / h;
    tt = q * GT + r % h;
}

/* TAIL: rows that end inside a step (without what that takes in each step 4096 tokens of 7168 -> 12288 562 us, with it 586) */
template <int BT, int BO, int WT, int WO, int NST, bool WREG, int POL, bool XF32, bool TAIL>
__global__ __launch_bounds__(64 * WT * WO) void lin_tile_kernel(LinTile p)
{
    constexpr int NW = WT * WO, FT = BT / WT / 16, FO = BO / WO / 16;
    constexpr int XE = XF32 ? 2 * LIN_KS : LIN_KS, XR = 512 / XE;                     /* a row of x in 2-byte units; rows of a DMA */
    constexpr int XD = BT / XR / NW, WD = WREG ? 0 : BO / 8 / NW, DN = XD + WD;      /* DMAs of a wave per step */
    constexpr int WR = WREG ? BO * 8 / (64 * NW) : 1;                                /* 16-byte pieces of W per thread */
    constexpr int FG = FO % 4 == 0 ? 4 : FO % 2 == 0 ? 2 : 1;       /* fragments that share a run of outputs */
    static_assert(XD >= 1 && (WREG || WD >= 1) && NST >= 2 && NST <= 4, "tile");
    constexpr int SZ = BT * XE + BO * LIN_KS;
    __shared__ __attribute__((aligned(1024))) uint16_t S0[SZ], S1[SZ], S2[NST > 2 ? SZ : 8], S3[NST > 3 ? SZ : 8];

    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wt = wv % WT, wo = wv / WT;
    int tt, to, sl;
    tile_of(p, blockIdx.x, tt, to, sl);
    const int t0 = tt * BT, o0 = to * BO;
    const int k0 = sl * p.per, n = min(p.per, p.steps - k0);

    /* Row swizzle of the LDS tiles: the 16-byte column c of row r lies in slot c ^ sw(r), so that the 16 rows of a
     * fragment read (one column) fall on all 64 banks. x: fragment rows are consecutive. W: the
     * rows of fragment q of FG are 4 FG j + 4 q + e (j: lane group, e: register of the result), so that a
     * lane's results of FG fragments are 4 FG consecutive outputs. */
    auto swx = [](int r) { return XF32 ? r & 15 : (r >> 1) & 7; };
    auto sww = [](int r) { return FG == 1 ? (r >> 1) & 7 : (((r / (4 * FG)) & 3) << 1) | ((r >> 1) & 1); };

    const int tn = min(BT, p.a.T - t0), on = min(BO, p.a.out - o0);
    constexpr int XS = XF32 ? 4 : 2;
    const k3_rsrc rx = k3_make_rsrc((const char *)p.x + (size_t)t0 * p.ldx * XS, (uint32_t)(((size_t)(tn - 1) * p.ldx + p.xcols) * XS));
    const k3_rsrc rw = k3_make_rsrc(p.a.W + (size_t)o0 * p.a.ldw, (uint32_t)(((size_t)(on - 1) * p.a.ldw + p.a.in) * 2));
    /* DMA i of wave wv fills LDS rows 8 (NW i + wv) ..+8, a lane a 16-byte slot. Rows past the last one repeat
     * it (their sums go unused), so every read lies in its matrix. */
    uint32_t xo[XD], wo_[WD > 0 ? WD : 1];
#pragma unroll
    for (int i = 0; i < XD; i++) {
        const int r = (i * NW + wv) * XR + lane / (64 / XR);
        xo[i] = (uint32_t)min(r, tn - 1) * (uint32_t)(p.ldx * XS) + ((lane & (64 / XR - 1)) ^ swx(r)) * 16;
    }
#pragma unroll
    for (int i = 0; i < WD; i++) {
        const int r = (i * NW + wv) * 8 + lane / 8;
        wo_[i] = (uint32_t)min(r, on - 1) * (uint32_t)(p.a.ldw * 2) + ((lane & 7) ^ sww(r)) * 16;
    }
    /* The last block of a row: zeros, of x (step xend) and of W (either may be infinite), for the 16-byte columns that the block before it
     * holds. A lane's column of x is the same in each of its DMAs, of W in every second one. */
    static_assert(NW * XR % 16 == 0 && NW * 16 % 64 == 0, "swizzles repeat from DMA to DMA");
    /* (one register: bit 2 - i W's DMAs of parity i, bit 0 x's) */
    const int over = p.nks * LIN_KS - p.a.in;
    auto twice = [&](int ln) -> uint32_t {
        auto w = [&](int i) { return 8 * ((ln & 7) ^ sww((i * NW + wv) * 8 + ln / 8)) < over; };
        return (16 * ((ln & (64 / XR - 1)) ^ swx(wv * XR + ln / (64 / XR))) < over * XS) | w(0) << 2 | w(1) << 1;
    };
    constexpr bool FULL = BT * BO >= 256 * 256;     /* (no register left: formed again in each step) */
    const uint32_t twice0 = FULL || !TAIL ? 0u : twice(lane);
    constexpr bool WSAME = NW * 8 % (FG == 4 ? 64 : FG == 2 ? 32 : 16) == 0;        /* one column in all of them */
    auto buf_of = [&](auto slot) -> uint16_t * {
        constexpr int S = decltype(slot)::value;
        if constexpr (S == 0) return S0;
        else if constexpr (S == 1) return S1;
        else if constexpr (S == 2) return S2;
        else return S3;
    };
    /* Stages are requested in order: step `xk` of x, which is column block `wk` of W (of a term), the last one
     * of a row from where its 64 columns end with the row (x: zeros in the columns that come twice). Past the slice: zeros, so that every step requests
     * as much and none is under a branch. */
    int xk = k0, wk = k0 % p.nks;
    const int kend = k0 + n;
    auto issue = [&](auto slot) {
        uint16_t *const b = buf_of(slot);
        const uint32_t none = xk < kend ? 0u : LIN_OOB;
        const bool end = TAIL && xk == p.xend, wend = TAIL && wk == p.nks - 1;
        const uint32_t xs = (uint32_t)(end ? p.a.in - LIN_KS : xk * LIN_KS) * XS, ws = (uint32_t)(wend ? p.a.in - LIN_KS : wk * LIN_KS) * 2;
        uint32_t again = twice0;
        if (FULL && TAIL) {
            uint32_t all = 0xffffffffu;
            asm volatile("" : "+s"(all));
            again = twice(__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0)));
        }
        const uint32_t nx = none | (end ? again << 31 : 0u), w0 = none | (wend ? again << 29 & LIN_OOB : 0u);
        const uint32_t w1 = WSAME ? w0 : none | (wend ? again << 30 & LIN_OOB : 0u);
#pragma unroll
        for (int i = 0; i < XD; i++) k3_dma16(rx, b + (i * NW + wv) * 512, xo[i] | nx, xs);
#pragma unroll
        for (int i = 0; i < WD; i++) k3_dma16<POL>(rw, b + BT * XE + (i * NW + wv) * 512, wo_[i] | (i & 1 ? w1 : w0), ws);
        xk++;
        if (++wk == p.nks) wk = 0;
    };
    /* Weights at any alignment: through registers, requested NST steps before they are stored (the hardware loads 16
     * bytes from any address). A piece that passes the end of its row is read from 8 elements before it and
     * shifted when it is stored; past the slice the last block comes again. */
    uint4 wr[WREG ? NST : 1][WR];
    const uint16_t *wb[WR];
    int gk = k0 % p.nks, gn = n, sk = gk;
    if (WREG)
#pragma unroll
        for (int i = 0; i < WR; i++) wb[i] = p.a.W + (size_t)(o0 + min((tid + 64 * NW * i) >> 3, on - 1)) * p.a.ldw;
    auto wload = [&](auto slot) {
        constexpr int S = WREG ? decltype(slot)::value : 0;
        const int k = min(gk * LIN_KS + (tid & 7) * 8, p.a.in - 8);
#pragma unroll
        for (int i = 0; i < WR; i++) wr[S][i] = load8_any(wb[i] + k);
        if (--gn > 0 && ++gk == p.nks) gk = 0;
    };
    auto wstore = [&](auto slot) {
        constexpr int S = WREG ? decltype(slot)::value : 0;
        uint16_t *const b = buf_of(slot);
        if (sk == p.nks - 1 && p.a.in % LIN_KS) {
            const int k = sk * LIN_KS + (tid & 7) * 8, over = k - min(k, p.a.in - 8), sh = 16 * (over & 3);
#pragma unroll
            for (int i = 0; i < WR; i++) {
                uint64_t lo = (uint64_t)wr[S][i].y << 32 | wr[S][i].x, hi = (uint64_t)wr[S][i].w << 32 | wr[S][i].z;
                if (over & 4) lo = hi, hi = 0;
                lo = sh ? lo >> sh | hi << (64 - sh) : lo;
                hi >>= sh;
                if (over >= 8) lo = hi = 0;
                wr[S][i] = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
            }
        }
#pragma unroll
        for (int i = 0; i < WR; i++) {
            const int c = tid + 64 * NW * i, r = c >> 3;
            *reinterpret_cast<uint4 *>(b + BT * XE + r * LIN_KS + ((c & 7) ^ sww(r)) * 8) = wr[S][i];
        }
        if (++sk == p.nks) sk = 0;
    };

    /* where the lane's fragments lie: x row 16 j + r16 of the wave's tokens, W row as above (their swizzles are
     * the same for every fragment); column 8 g of a half step */
    const int xr = wt * (BT / WT) + r16, wr0 = wo * (BO / WO) + (r16 >> 2) * 4 * FG + (r16 & 3);
    int xa[2], xb[2], wa[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int c = XF32 ? 8 * h + 2 * g : 4 * h + g;         /* (8 floats: two 16-byte columns) */
        xa[h] = xr * XE + ((c ^ swx(xr)) * 8);
        xb[h] = xr * XE + (((c + 1) ^ swx(xr)) * 8);
        wa[h] = BT * XE + wr0 * LIN_KS + (((4 * h + g) ^ sww(wr0)) * 8);
    }
    struct XFrag {
        u32x4 v[XF32 ? 2 : 1];
    };
    auto read = [&](const uint16_t *b, int half, XFrag (&xf)[FT], k3_bf16x8 (&wf)[FO]) {
#pragma unroll
        for (int i = 0; i < FO; i++)
            wf[i] = k3_as_bf16x8(*reinterpret_cast<const uint4 *>(b + wa[half] + ((i / FG) * 16 * FG + (i % FG) * 4) * LIN_KS));
#pragma unroll
        for (int j = 0; j < FT; j++) {
            xf[j].v[0] = *reinterpret_cast<const u32x4 *>(b + xa[half] + 16 * j * XE);
            if constexpr (XF32) xf[j].v[1] = *reinterpret_cast<const u32x4 *>(b + xb[half] + 16 * j * XE);
        }
    };
    k3_f32x4 acc[FO][FT];
#pragma unroll
    for (int i = 0; i < FO; i++)
#pragma unroll
        for (int j = 0; j < FT; j++) acc[i][j] = k3_f32x4{0.f, 0.f, 0.f, 0.f};
    auto mma = [&](const XFrag (&xf)[FT], const k3_bf16x8 (&wf)[FO]) {
        if constexpr (XF32) {
#pragma unroll
            for (int j = 0; j < FT; j++) {
                float f[8];
                uint32_t c[3][4];
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = __uint_as_float(xf[j].v[e / 4][e % 4]);
                cut3(f, c[2], c[1], c[0]);
#pragma unroll
                for (int q = 0; q < 3; q++)
#pragma unroll
                    for (int i = 0; i < FO; i++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[i], as_frag(c[q]), acc[i][j], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < FO; i++)
#pragma unroll
                for (int j = 0; j < FT; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[i], __builtin_bit_cast(k3_bf16x8, xf[j].v[0]), acc[i][j], 0, 0, 0);
        }
    };
    /* issue order of a half: a fragment read of the other half behind each of the first MFMAs, and, behind the
     * barrier, the next stage's requests between them too (in a burst they keep the SIMD from its MFMAs for
     * some hundred cycles) */
    constexpr int NRD = FO + FT * (XF32 ? 2 : 1), NMF = FO * FT * (XF32 ? 3 : 1), GAP = NMF / NRD > 0 ? NMF / NRD : 1;
    auto pin = [&](auto dma) {
        each_stage<0, NRD>([&](auto at) {
            constexpr int I = decltype(at)::value, ND = decltype(dma)::value, Q = (I + 1) * ND / NRD - I * ND / NRD;
            __builtin_amdgcn_sched_group_barrier(0x008, GAP, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            if constexpr (Q > 0) __builtin_amdgcn_sched_group_barrier(0x010, Q, 0);
        });
        __builtin_amdgcn_sched_group_barrier(0x008, NMF, 0);
    };
    /* all but the last NST - 2 stages' requests (with weights through registers, whose loads follow a stage's
     * requests: and those of the stage before). A count holds only where each counted load is there: the weights' are while a later step
     * stores them, which those of the last steps are not (the compiler drops them), so these request nothing and wait for all. */
    constexpr int WAITN = WREG ? WR + (XD + WR) * (NST - 2) : DN * (NST - 2);
    constexpr int WAIT_STAGE = (WAITN & 15) | (7 << 4) | (0 << 8) | ((WAITN >> 4) << 14);       /* and LDS: none */
    static_assert(WAITN < 64, "requests in flight");
    constexpr int WAIT_VM0 = (7 << 4) | (15 << 8), WAIT_ALL = 7 << 4;
    XFrag fx0[FT], fx1[FT];
    k3_bf16x8 fw0[FO], fw1[FO];

    /* Step k: its second half is read while the first is multiplied; then every wave is past its reads of
     * buffer k % NST and stage k + 1 has landed (one barrier), so stage k + NST goes into that buffer and the
     * next step's first half is read while the second is multiplied. `last`: of the steps behind the loop, past which
     * no stage is wanted. */
    auto step = [&](auto slot, auto last) {
        constexpr int S = decltype(slot)::value;
        constexpr bool DRAIN = WREG && decltype(last)::value;
        uint16_t *const b = buf_of(slot);
        uint16_t *const nb = buf_of(std::integral_constant<int, (S + 1) % NST>{});
        read(b, 1, fx1, fw1);
        mma(fx0, fw0);
        pin(std::integral_constant<int, 0>{});
        __builtin_amdgcn_sched_barrier(0);
        /* (__syncthreads would wait for every request) */
        __builtin_amdgcn_s_waitcnt(DRAIN ? WAIT_ALL : WAIT_STAGE);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (!DRAIN) {
            if (WREG) wstore(slot);
            issue(slot);
            if (WREG) {
                __builtin_amdgcn_sched_barrier(0);      /* (in this order: WAITN) */
                wload(slot);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        read(nb, 0, fx0, fw0);          /* (past the last step: what lies there, unused) */
        mma(fx1, fw1);
        pin(std::integral_constant<int, WREG ? 0 : DN>{});
        __builtin_amdgcn_sched_barrier(0);
    };
    if (WREG) each_stage<0, NST>(wload);
    each_stage<0, NST>([&](auto slot) {
        if (WREG) wstore(slot);
        issue(slot);
    });
    if (WREG) each_stage<0, NST>(wload);
    __builtin_amdgcn_s_waitcnt(WAIT_VM0);
    __syncthreads();
    read(S0, 0, fx0, fw0);
    /* (whole rounds in the loop: a way out of its middle costs copies of the accumulators) */
    int left = n;
    for (; left >= NST; left -= NST) each_stage<0, NST>([&](auto slot) { step(slot, std::false_type{}); });
    each_stage<0, NST - 1>([&](auto slot) {
        if (decltype(slot)::value < left) step(slot, std::true_type{});
    });

    /* A lane holds token r16 of each token fragment and 4 FG consecutive outputs of FG fragments. The sums go
     * through LDS (the stage buffers, a region per wave, JR token fragments at a time; 16-byte column c of row r
     * in c ^ (r % 16)), so that a wave writes whole rows of its outputs, and the epilogue's code is there once. */
    constexpr int WOUT = BO / WO, C = WOUT / 4;
    constexpr int JR = SZ * 2 / (FT * 64 * WOUT) * 2 >= NW ? FT : SZ * 2 / (FT * 32 * WOUT) * 2 >= NW ? FT / 2 : FT / 4;
    constexpr int RB = JR * 64 * WOUT, PER = SZ * 2 / RB;       /* bytes of a region; regions per stage buffer */
    static_assert(JR >= 1 && FT % JR == 0 && PER >= 1 && PER * 2 >= NW && 64 % C == 0, "epilogue regions");
    uint16_t *stage = S0;
    if (PER < NW) stage = wv / PER == 0 ? S0 : S1;
    float4 *const reg = reinterpret_cast<float4 *>(stage + (wv % PER) * (RB / 2));
    const int c = lane % C, o = o0 + wo * WOUT + 4 * c;
    /* the residuals of the first PF iterations; each, once used, makes room for the one PF further */
    constexpr int RI = 64 / C, IT = 16 * JR / RI, NIT = 16 * FT / RI, PF = IT < 4 ? IT : 4;
    static_assert(IT % PF == 0, "residuals");
    const int row0 = t0 + wt * (BT / WT) + lane / C;
    uint4 res[PF];
    if (p.nsl == 1)
#pragma unroll
        for (int k = 0; k < PF; k++) res[k] = res4(p.a, row0 + k * RI, o);
    float b[4];
    bias4(p.a, p.nsl > 1 ? p.a.out : o, b);
    __builtin_amdgcn_s_waitcnt(WAIT_VM0);      /* the last requests land before LDS is used again */
    __syncthreads();
#pragma unroll
    for (int j0 = 0; j0 < FT; j0 += JR) {
#pragma unroll
        for (int j = 0; j < JR; j++)
#pragma unroll
            for (int i = 0; i < FO; i++) {
                const int oc = (i / FG) * 4 * FG + g * FG + i % FG, r = 16 * j + r16;
                reg[r * C + (oc ^ (r16 & (C - 1)))] = make_float4(acc[i][j0 + j][0], acc[i][j0 + j][1], acc[i][j0 + j][2], acc[i][j0 + j][3]);
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int i = 0; i < IT; i += PF)
#pragma unroll
            for (int k = 0; k < PF; k++) {
                const int r = lane / C + (i + k) * RI, t = row0 + 16 * j0 + (i + k) * RI;
                const float4 v = reg[r * C + (c ^ (r & 15 & (C - 1)))];
                if (p.nsl == 1) {
                    const uint4 q = res[k];
                    if (j0 * 16 / RI + i + k + PF < NIT) res[k] = res4(p.a, t + PF * RI, o);
                    put4(p.a, t, o, v, b, q);
                } else if (t < p.a.T && o < p.a.out) {
                    float *q = p.part + ((size_t)sl * p.a.T + t) * p.a.out + o;
                    if (o + 4 <= p.a.out) {
                        __builtin_memcpy(q, &v, 16);
                    } else {
                        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int n = 0; n < 3; n++)
                            if (o + n < p.a.out) q[n] = e[n];
                    }
                }
            }
        __builtin_amdgcn_wave_barrier();
    }
}

/* the slices' sums, in slice order, and the epilogue; four slices requested at once (300 tokens of 384 outputs in 8 slices
 * 4.6 us one after another, 4.1 so). At most LIN_PART_CAP bytes of sums: their indexes fit 32 bits. */
__global__ __launch_bounds__(64) void lin_join_kernel(K3kLinear a, const float *part, int nsl)
{
    const unsigned per = (a.out + 3) / 4, i = blockIdx.x * 64 + threadIdx.x;
    const int t = (int)(i / per), o = (int)(i - (unsigned)t * per) * 4;
    if (t >= a.T) return;
    float b[4];
    bias4(a, o, b);
    const uint4 res = res4(a, t, o);
    const float *const q = part + (size_t)t * a.out + o;
    const size_t one = (size_t)a.T * a.out;
    const int n = min(4, a.out - o);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < nsl; s += 4) {
        float4 f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float *p = q + one * min(s + j, nsl - 1);
            if (n == 4) __builtin_memcpy(&f[j], p, 16);
            else f[j] = make_float4(p[0], n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, 0.f);
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (s + j < nsl) v.x += f[j].x, v.y += f[j].y, v.z += f[j].z, v.w += f[j].w;
    }
    put4(a, t, o, v, b, res);
}

/* ---- launches -------------------------------------------------------------------------------- */
/* A launch takes under 2^32 work-items: no kernel is chosen where its grid holds more. */
bool fits_launch(long workgroups, int threads) { return workgroups * threads < 1L << 32; }

constexpr int LIN_MAX_SLICES = 16;
constexpr size_t LIN_PART_CAP = (size_t)64 << 20;
/* weights that no cache keeps from one call to the next, from here on read past the caches (102 MB times 64
 * tokens 30.6 -> 29.5 us, 176 MB times one 30.2 -> 26.8; but 51 MB times 16 12.4 -> 12.8, 29 MB times 32 10.2 -> 14.5) */
constexpr size_t LIN_NT_BYTES = (size_t)96 << 20;

int kpad(int in) { return (in + LIN_KS - 1) / LIN_KS * LIN_KS; }

size_t pack_bytes(int T, int in, int x_type)
{
    return ((size_t)T * kpad(in) * (x_type == K3D_F32 ? 3 : 1) * 2 + 255) / 256 * 256;
}

/* the slices' sums of any batch up to T: a call takes slices only as far as they fit this */
size_t part_bytes(int T, int out)
{
    const size_t most = (size_t)LIN_MAX_SLICES * T * out * 4;
    return most < LIN_PART_CAP ? most : LIN_PART_CAP;
}

/* ---- short rows at any alignment ---- */
void short_rows(const K3kLinear *a, hipStream_t st)
{
    const unsigned grid = (unsigned)((a->out + 15) / 16) * (unsigned)((a->T + 15) / 16);
    /* waves that share a workgroup's columns: enough for the chip, each with a few steps */
    int nw = grid < 2 * k3k_cu_count() ? 8 : 4;
    while (nw > 1 && (a->in + 31) / 32 < 2 * nw) nw /= 2;
    if (a->x_type == K3D_F32) lin_stream_kernel<4, true><<<grid, 64 * nw, 0, st>>>(*a, nw);
    else lin_stream_kernel<8, false><<<grid, 64 * nw, 0, st>>>(*a, nw);
}

/* ---- few tokens ---- */
constexpr int SK_NW = 4;
constexpr int sk_kb(int rw, int xr, bool f32) { return 2 * rw + xr * (f32 ? 2 : 1); }      /* KB of a wave's stage */
constexpr int sk_nst(int rw, int xr, bool f32)
{
    return 4 * SK_NW * sk_kb(rw, xr, f32) <= 160 ? 4 : 3 * SK_NW * sk_kb(rw, xr, f32) <= 160 ? 3 : 2 * SK_NW * sk_kb(rw, xr, f32) <= 160 ? 2 : 0;
}
/* tokens go in groups of 8, 16, 32, 48 and 64 (and no group past the last that fits the LDS) */
constexpr int sk_group(int T) { return T <= 8 ? 1 : T <= 16 ? 2 : T <= 32 ? 4 : T <= 48 ? 6 : 8; }

template <int RW, int XR, bool XF32>
void skinny_go(const K3kLinear *a, hipStream_t st)
{
    constexpr int NST = sk_nst(RW, XR, XF32);
    if constexpr (NST > 0) {
        const unsigned grid = (a->out + 16 * RW - 1) / (16 * RW);
        if ((size_t)a->in * a->out * 2 >= LIN_NT_BYTES)
            lin_skinny_kernel<RW, XR, SK_NW, NST, XF32, K3_LD_NT><<<grid, 64 * SK_NW, 0, st>>>(*a);
        else
            lin_skinny_kernel<RW, XR, SK_NW, NST, XF32, K3_LD_DEFAULT><<<grid, 64 * SK_NW, 0, st>>>(*a);
    }
}

template <int RW, bool XF32>
void skinny_rows(const K3kLinear *a, hipStream_t st)
{
    switch (sk_group(a->T)) {
    case 1: return skinny_go<RW, 1, XF32>(a, st);
    case 2: return skinny_go<RW, 2, XF32>(a, st);
    case 4: return skinny_go<RW, 4, XF32>(a, st);
    case 6: return skinny_go<RW, 6, XF32>(a, st);
    default: return skinny_go<RW, 8, XF32>(a, st);
    }
}

template <bool XF32>
void skinny(const K3kLinear *a, int rw, hipStream_t st)
{
    if (rw == 1) skinny_rows<1, XF32>(a, st);
    else if (rw == 2) skinny_rows<2, XF32>(a, st);
    else skinny_rows<4, XF32>(a, st);
}

/* Two limits of one time: neither hides all of the other. */
float both(float a, float b) { return sqrtf(a * a + b * b); }

/* Microseconds of lin_skinny_kernel: a CU takes in 82 KB/us while the chip's 17.8 GB/ms allow it (a workgroup's
 * rows of W and all of x for them), the weights come at 5.9 GB/ms, fp32 x costs a wave 0.26 us to cut 8 tokens of a
 * stage. The constants of this and of tile_cost are fitted to 40 shapes of 1 to 4096 tokens, each on every kernel: they are off by
 * 10 % on average, and what they choose is 2.5 % slower than the best of them (16 % at 64 tokens of 7168 -> 576, 23 %
 * at 1024 of 7168 -> 384 at the worst). 0: does not fit the LDS, or a launch. */
float skinny_cost(int T, int in, int out, bool f32, int rw, long cus)
{
    const int xr = sk_group(T);
    const long wgs = (out + 16 * rw - 1) / (16 * rw), rounds = (wgs + cus - 1) / cus;
    if (sk_nst(rw, xr, f32) == 0 || !fits_launch(wgs, 64 * SK_NW)) return 0.0f;
    const float kb = (float)in * 2.0f / 1024.0f * (16 * rw + 8 * xr * (f32 ? 2 : 1));
    const float rate = fminf(82.0f, 17800.0f / (float)(wgs < cus ? wgs : cus));
    const float cut = f32 ? (float)((in + LIN_KS - 1) / LIN_KS) / SK_NW * xr * 0.26f : 0.0f;
    return 2.9f + both(rounds * fmaxf(kb / rate, cut), (float)in * out * 2.0f / 5.9e6f);
}

/* ---- many tokens ---- */
template <int BT, int BO, int WT, int WO, int NST, bool WREG, int POL = K3_LD_DEFAULT, bool XF32 = false>
void tile_go(const LinTile *p, hipStream_t st)
{
    const int grid = p->nt * p->no * p->nsl;
    if (WREG || p->a.in % LIN_KS) lin_tile_kernel<BT, BO, WT, WO, NST, WREG, POL, XF32, true><<<grid, 64 * WT * WO, 0, st>>>(*p);
    else if constexpr (!WREG) lin_tile_kernel<BT, BO, WT, WO, NST, WREG, POL, XF32, false><<<grid, 64 * WT * WO, 0, st>>>(*p);
}

/* Microseconds of a launch of lin_tile_kernel and, with slices, the join: rounds of as many workgroups as fit the chip, each
 * of `per` steps; a step takes what a CU takes in at 74 KB/us and the chip at 35 GB/ms, or the matrix cores at
 * 1.66 PFLOP/s of the chip; W and x come at 6.7 GB/ms. 0: does not fit a launch. */
struct Shape {
    int bt, bo, per_cu, threads;
};
constexpr Shape SHAPES[] = {{256, 256, 1, 512}, {256, 128, 1, 512}, {128, 128, 1, 256}, {128, 64, 2, 256}, {64, 128, 2, 256}, {64, 64, 2, 256}};
constexpr int N_SHAPES = sizeof SHAPES / sizeof SHAPES[0];

float tile_cost(const Shape &s, int T, int in, int out, int steps, int nsl, long cus)
{
    const long wgs = (long)((T + s.bt - 1) / s.bt) * ((out + s.bo - 1) / s.bo) * nsl, slots = cus * s.per_cu;
    if (!fits_launch(wgs, s.threads)) return 0.0f;
    const int per = (steps + nsl - 1) / nsl;
    const float kb = (s.bt + s.bo) * LIN_KS * 2.0f / 1024.0f, mfma = 2.0f * s.bt * s.bo * LIN_KS / 6.5e6f;
    auto round = [&](long n) {
        const float on = (float)((n + cus - 1) / cus);          /* workgroups of a CU */
        return per * both(on * fmaxf(kb / 74.0f, mfma), kb * n / 35000.0f) + 1.1f + 0.08f * kb;
    };
    float t = (float)(wgs / slots) * round(slots) + (wgs % slots ? round(wgs % slots) : 0.0f);
    t = 2.6f + both(t, ((float)out + T) * in * 2.0f / 6.7e6f);
    if (nsl > 1) t += 2.1f + (nsl + 1.0f) * T * out * 4.0f / 4.7e6f;
    return t;
}

/* Microseconds with fp32 rows cut in the kernel, 64 tokens by 64 or 128 outputs, two workgroups to a CU: a step takes one
 * 0.50 or 0.74 us alone and 0.72 or 1.01 beside another. (Cutting them once, in a launch before, costs a write and a read of
 * three terms and a longer product: 300 tokens of 7168 -> 384 26.1 us that way, 18.5 this way; 4000 tokens 135 and 74; but
 * 1024 of 7168 -> 7168 294 and 353, as each tile of outputs cuts its tokens again.) 0: does not fit a launch. */
float cut_cost(int bo, int T, int in, int out, int nsl, long cus)
{
    const int nks = (in + LIN_KS - 1) / LIN_KS, per = (nks + nsl - 1) / nsl;
    const long wgs = (long)((T + 63) / 64) * ((out + bo - 1) / bo) * nsl, slots = 2 * cus;
    if (!fits_launch(wgs, 256)) return 0.0f;
    const float one = bo == 64 ? 0.49f : 0.73f, two = bo == 64 ? 0.70f : 1.00f, kb = bo / 8.0f + 16.0f;
    auto round = [&](long n) { return both(per * (n <= cus ? one : two), per * kb * n / 25000.0f); };
    float t = (float)(wgs / slots) * round(slots) + (wgs % slots ? round(wgs % slots) : 0.0f);
    t = 4.5f + both(t, ((float)out + 2.0f * T) * in * 2.0f / 5.3e6f);
    t += nsl > 1 ? 1.3f + 0.38f * nsl + (nsl + 1.0f) * T * out * 4.0f / 3.2e6f : (float)T * out * 4.0f / 4.7e6f;
    return t;
}

}  // namespace

extern "C" size_t k3k_linear_ws(int T, int in, int out, int x_type)
{
    return pack_bytes(T, in, x_type) + part_bytes(T, out);
}

extern "C" int k3k_linear(const K3kLinear *a, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    const long cus = k3k_cu_count();
    const bool f32 = a->x_type == K3D_F32;
    const bool w16 = ((uintptr_t)a->W & 15) == 0 && a->ldw % 8 == 0;
    const bool x16 = ((uintptr_t)a->x & 15) == 0 && a->ldx % (f32 ? 4 : 8) == 0;
    /* weights by DMA, or, at other alignments and in rows shorter than a stage, through registers */
    const bool dma = w16 && a->in % 8 == 0 && a->in >= LIN_KS;
    const int nks = (a->in + LIN_KS - 1) / LIN_KS;
    int steps = nks * (f32 ? 3 : 1);
    const bool pack = f32 || !x16 || !dma;

    /* the cheapest tile shape and number of slices */
    float best = 0.0f;
    int shape = 0, nsl = 1;
    const size_t one = (size_t)a->T * a->out * 4, room = part_bytes(a->T, a->out);
    for (int i = 0; i < N_SHAPES; i++) {
        if (!dma && !(SHAPES[i].bt == SHAPES[i].bo && SHAPES[i].bt < 256)) continue;
        for (int n : {1, 2, 3, 4, 6, 8, 12, LIN_MAX_SLICES}) {
            if (n > 1 && (n * one > room || steps < 4 * n)) break;
            const float t = tile_cost(SHAPES[i], a->T, a->in, a->out, steps, n, cus);
            if (t > 0.0f && (best == 0.0f || t < best)) best = t, shape = i, nsl = n;
        }
    }
    if (pack) best += 2.5f + (float)a->T * kpad(a->in) * (f32 ? 10 : 4) / 4e6f;
    /* or fp32 rows as they are */
    int cut = 0;
    if (f32 && dma && x16)
        for (int bo : {64, 128})
            for (int n : {1, 2, 3, 4, 6, 8, 12, LIN_MAX_SLICES}) {
                if (n > 1 && (n * one > room || nks < 4 * n)) break;
                const float t = cut_cost(bo, a->T, a->in, a->out, n, cus);
                if (t > 0.0f && t < best) best = t, cut = bo, nsl = n;
            }
    if (a->T <= 64) {
        int rw = 0;
        if (dma && x16)
            for (int r = 1; r <= 4; r *= 2) {
                const float t = skinny_cost(a->T, a->in, a->out, f32, r, cus);
                if (t > 0.0f && t < best) best = t, rw = r;
            }
        if (rw) {
            if (f32) skinny<true>(a, rw, st);
            else skinny<false>(a, rw, st);
            K3K_LAUNCH_CHECK("linear: few tokens");
            return 0;
        }
    }
    /* (16 tokens of 777 -> 999 9.6 us, as tiles 10.7, one 6.8 and 9.9; but 16 of 5001 -> 4097 47 us, as tiles 21) */
    if (!dma && (a->in < LIN_KS || (a->T <= 16 && (long)a->in * a->out <= 1L << 21))) {
        short_rows(a, st);
        K3K_LAUNCH_CHECK("linear: short rows");
        return 0;
    }

    LinTile p;
    p.a = *a;
    p.nks = nks;
    if (cut) steps = nks;
    p.steps = steps;
    if (pack && !cut) {
        const int kp = kpad(a->in), over = dma ? kp - a->in : 0;
        const int most = (int)((1u << 31) / (unsigned)(kp / 8)), terms = f32 ? 3 : 1;       /* tokens of a launch */
        for (int t = 0; t < a->T; t += most) {
            const int n = a->T - t < most ? a->T - t : most;
            uint16_t *const xs = (uint16_t *)a->ws + (size_t)t * terms * kp;
            const char *const x = (const char *)a->x + (size_t)t * a->ldx * (f32 ? 4 : 2);
            const unsigned grid = (unsigned)(((size_t)n * (kp / 8) + 255) / 256);
            if (f32) lin_pack_kernel<true><<<grid, 256, 0, st>>>(xs, x, a->ldx, n, a->in, kp, over);
            else lin_pack_kernel<false><<<grid, 256, 0, st>>>(xs, x, a->ldx, n, a->in, kp, over);
            K3K_LAUNCH_CHECK("linear: pack");
        }
        p.x = a->ws;
        p.ldx = p.xcols = p.steps * LIN_KS;
        p.xend = -1;
    } else {
        p.x = a->x;
        p.ldx = a->ldx;
        p.xcols = a->in;
        p.xend = nks - 1;
    }
    p.part = (float *)((char *)a->ws + pack_bytes(a->T, a->in, a->x_type));
    const int bt = cut ? 64 : SHAPES[shape].bt, bo = cut ? cut : SHAPES[shape].bo;
    p.nt = (a->T + bt - 1) / bt;
    p.no = (a->out + bo - 1) / bo;
    p.per = (steps + nsl - 1) / nsl;
    p.nsl = (steps + p.per - 1) / p.per;
    if (cut == 64) {
        tile_go<64, 64, 4, 1, 3, false, K3_LD_DEFAULT, true>(&p, st);
    } else if (cut) {
        tile_go<64, 128, 4, 1, 2, false, K3_LD_DEFAULT, true>(&p, st);
    } else if (dma) {
        switch (shape) {
        case 0: tile_go<256, 256, 2, 4, 2, false>(&p, st); break;
        case 1: tile_go<256, 128, 4, 2, 3, false>(&p, st); break;
        case 2: tile_go<128, 128, 2, 2, 4, false>(&p, st); break;
        case 3: tile_go<128, 64, 2, 2, 3, false>(&p, st); break;
        case 4:
            /* (one tile of tokens: W is read once) */
            if (p.nt == 1 && (size_t)a->in * a->out * 2 >= LIN_NT_BYTES) tile_go<64, 128, 1, 4, 3, false, K3_LD_NT>(&p, st);
            else tile_go<64, 128, 1, 4, 3, false>(&p, st);
            break;
        default: tile_go<64, 64, 2, 2, 4, false>(&p, st); break;
        }
    } else if (shape == 2) {
        tile_go<128, 128, 2, 2, 3, true>(&p, st);
    } else {
        tile_go<64, 64, 2, 2, 4, true>(&p, st);
    }
    K3K_LAUNCH_CHECK("linear: tiles");
    if (p.nsl > 1) {
        const size_t n = (size_t)a->T * ((a->out + 3) / 4);
        lin_join_kernel<<<(unsigned)((n + 63) / 64), 64, 0, st>>>(*a, p.part, p.nsl);
        K3K_LAUNCH_CHECK("linear: join");
    }
    return 0;
}
