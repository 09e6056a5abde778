/* SPDX-License-Identifier: Apache-2.0 */
/* k3_wave.h -- reductions over a wave shared by the selection kernels. */
#ifndef K3_WAVE_H
#define K3_WAVE_H

#include "k3_common.h"

namespace {

/* 32-bit max / min of the wave by DPP, the same in every lane: pairs, quads (quad_perm),
 * 8 (row half mirror), 16 (row mirror), then rows 0-1 and 2-3 (row_bcast15 into rows 1,
 * 3) and rows 0-3 (row_bcast31 into rows 2, 3), so lane 63 holds the result. */
/* (rows outside RM read the identity of the operation, so each step is one DPP max/min) */
template <int CTRL, int RM, uint32_t ID>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp((int)ID, (int)v, CTRL, RM, 0xf, false);
}

template <bool MAX>
__device__ __forceinline__ uint32_t wave_reduce_u32(uint32_t v)
{
    constexpr uint32_t ID = MAX ? 0u : 0xffffffffu;
    auto op = [](uint32_t a, uint32_t b) { return MAX ? (a > b ? a : b) : (a < b ? a : b); };
    v = op(v, dpp_u32<0xB1, 0xf, ID>(v));      /* quad_perm [1,0,3,2] */
    v = op(v, dpp_u32<0x4E, 0xf, ID>(v));      /* quad_perm [2,3,0,1] */
    v = op(v, dpp_u32<0x141, 0xf, ID>(v));     /* row_half_mirror */
    v = op(v, dpp_u32<0x140, 0xf, ID>(v));     /* row_mirror */
    v = op(v, dpp_u32<0x142, 0xa, ID>(v));     /* row_bcast15 */
    v = op(v, dpp_u32<0x143, 0xc, ID>(v));     /* row_bcast31 */
    return __builtin_amdgcn_readlane(v, 63);
}

/* Sum of the wave's doubles, the same in every lane, in a fixed order (the steps of wave_reduce_u32; 18 instructions, where
 * shuffles through the LDS take 12 round trips). */
template <int CTRL, int RM>
__device__ __forceinline__ double dpp_f64(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint64_t r = (uint64_t)dpp_u32<CTRL, RM, 0u>((uint32_t)(b >> 32)) << 32 | dpp_u32<CTRL, RM, 0u>((uint32_t)b);
    return __longlong_as_double((long long)r);
}

__device__ __forceinline__ double wave_total_f64(double v)
{
    v += dpp_f64<0xB1, 0xf>(v);
    v += dpp_f64<0x4E, 0xf>(v);
    v += dpp_f64<0x141, 0xf>(v);
    v += dpp_f64<0x140, 0xf>(v);
    v += dpp_f64<0x142, 0xa>(v);
    v += dpp_f64<0x143, 0xc>(v);
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint64_t r = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), 63) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)b, 63);
    return __longlong_as_double((long long)r);
}

}  // namespace

#endif
