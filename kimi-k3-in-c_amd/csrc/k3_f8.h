/* SPDX-License-Identifier: Apache-2.0 */
/* k3_f8.h -- e4m3 codes with a scale for each 128 columns: rounding to them, and the gated activations in front of it. */
#ifndef K3_F8_H
#define K3_F8_H

#include "k3_common.h"
#include "k3_dev.h"
#include "k3_epilogue.h"
#include "k3_wave.h"

namespace {

/* The largest magnitude among 16 neighbouring lanes (a block of 128 columns, eight a lane) from each lane's, as bits: NaN is
 * above infinity, so a block that holds one has it. */
__device__ __forceinline__ uint32_t row_max_bits(uint32_t v)
{
    v = max(v, dpp_u32<0xB1, 0xf, 0u>(v));      /* quad_perm [1,0,3,2] */
    v = max(v, dpp_u32<0x4E, 0xf, 0u>(v));      /* quad_perm [2,3,0,1] */
    v = max(v, dpp_u32<0x141, 0xf, 0u>(v));     /* row_half_mirror */
    return max(v, dpp_u32<0x140, 0xf, 0u>(v));  /* row_mirror */
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

/* A block's scale from its largest magnitude: max(amax, 2^-100) / 448, NaN where amax is. (Below 2^-100 the quotient, and
 * its reciprocal, would leave fp32; the codes of such a block still stand for its values within 2^-119.) */
__device__ __forceinline__ float f8_scale(uint32_t amax)
{
    return __uint_as_float(max(amax, __float_as_uint(0x1p-100f))) / 448.0f;
}

/* Four codes, a byte each, of four values already divided by their scale: to nearest, ties to even. Magnitudes reach 448 and a few
 * units in the last place, which round to it; NaN becomes the code of NaN. */
__device__ __forceinline__ uint32_t f8_codes(float a, float b, float c, float d)
{
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}

/* tanh within a few units of 2^-24 of its value: the Taylor series to y^9 up to |y| = 1/4, whose next term is under 2^-24 of
 * it, where 1 - 2 / (e^2y + 1) would lose what it subtracts. */
__device__ __forceinline__ float tanh_of(float y)
{
    const float q = y * y;
    float p = fmaf(q, 62.0f / 2835.0f, -17.0f / 315.0f);
    p = fmaf(q, p, 2.0f / 15.0f);
    p = fmaf(q, p, -1.0f / 3.0f);
    const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(2.88539008f * y));
    return fabsf(y) <= 0.25f ? fmaf(y * q, p, y) : far;
}

/* act(gate) * up as k3_act_pair has it, in forms that hold their precision for small and far arguments */
__device__ __forceinline__ float glu_of(float g, float u, int act, float b1, float b2, float r1, float r2)
{
    if (act == K3D_GLU_SILU) return over_1p_exp<false>(g, g) * u;
    return over_1p_exp<false>(b1 * tanh_of(g * r1), g) * (b2 * tanh_of(u * r2));
}

}  // namespace

#endif
