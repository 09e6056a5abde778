/* SPDX-License-Identifier: Apache-2.0 */
/* k3_epilogue.h -- what the dense products do with their sums: bias, activation, residual, one rounding. A: the arguments of
 * a product (y, ldy, y_type, bias, act, res, ldr, T, out). */
#ifndef K3_EPILOGUE_H
#define K3_EPILOGUE_H

#include "k3_common.h"
#include "k3_dev.h"

namespace {

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
template <class A>
__device__ __forceinline__ uint4 res4(const A &a, int t, int o)
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
template <class A>
__device__ __forceinline__ void put4(const A &a, int t, int o, float4 acc, const float (&b)[4], uint4 r)
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

template <class A>
__device__ __forceinline__ void bias4(const A &a, int o, float (&b)[4])
{
#pragma unroll
    for (int i = 0; i < 4; i++) b[i] = a.bias && o + i < a.out ? a.bias[o + i] : 0.0f;
}

}  // namespace

#endif
