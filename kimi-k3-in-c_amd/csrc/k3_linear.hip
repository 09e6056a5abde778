/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_linear.hip -- dense products with bias, activation and residual (k3d_linear):
 *   y[t][o] = act(sum_k x[t][k] W[o][k] + bias[o]) + res[t][o],   W bf16, x bf16 or fp32.
 */
#include "k3_common.h"
#include "k3_dev.h"
#include "k3k.h"

namespace {

__device__ __forceinline__ float act_of(float v, int act)
{
    switch (act) {
    case K3D_ACT_RELU: return v < 0.0f ? 0.0f : v;
    case K3D_ACT_SILU: return v / (1.0f + expf(-v));
    case K3D_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678f));
    case K3D_ACT_GELU_TANH: return v / (1.0f + expf(-1.5957691f * (v + 0.044715f * v * v * v)));
    default: return v;
    }
}

__device__ __forceinline__ void put(const K3kLinear &a, int t, int o, float v)
{
    if (a.bias) v += a.bias[o];
    v = act_of(v, a.act);
    const size_t i = (size_t)t * a.ldy + o, r = (size_t)t * a.ldr + o;
    if (a.y_type == K3D_F32) {
        if (a.res) v += ((const float *)a.res)[r];
        ((float *)a.y)[i] = v;
    } else {
        if (a.res) v += k3_bf16_to_f32(((const uint16_t *)a.res)[r]);
        ((uint16_t *)a.y)[i] = k3_bf16_rne(v);
    }
}

/* A wave per 16 rows of W and 16 tokens, operands element by element from memory. */
__global__ __launch_bounds__(256) void linear_kernel(K3kLinear a)
{
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
    const int o0 = (blockIdx.x * 4 + wv) * 16, t0 = blockIdx.y * 16;
    const int o = o0 + r16, t = t0 + r16;
    k3_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < a.in; k0 += 32) {
        k3_bf16x8 w, x[3];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int k = k0 + 8 * g + i;
            const bool in = k < a.in;
            const uint16_t wb = in && o < a.out ? a.W[(size_t)o * a.ldw + k] : (uint16_t)0;
            float v = 0.0f;
            if (in && t < a.T)
                v = a.x_type == K3D_F32 ? ((const float *)a.x)[(size_t)t * a.ldx + k]
                                        : k3_bf16_to_f32(((const uint16_t *)a.x)[(size_t)t * a.ldx + k]);
            w[i] = __builtin_bit_cast(__bf16, wb);
            const bool fin = (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
            float r = v;
#pragma unroll
            for (int s = 0; s < 3; s++) {
                uint32_t u = __float_as_uint(r) & 0xffff0000u;
                if (r != r) u |= 0x00400000u;
                x[s][i] = __builtin_bit_cast(__bf16, (uint16_t)(u >> 16));
                r = fin ? r - __uint_as_float(u) : 0.0f;
            }
        }
#pragma unroll
        for (int s = 2; s >= 0; s--) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x[s], acc, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (t < a.T && o0 + 4 * g + i < a.out) put(a, t, o0 + 4 * g + i, acc[i]);
}

}  // namespace

extern "C" size_t k3k_linear_ws(int T, int in, int out, int x_type) { return 0; }

extern "C" int k3k_linear(const K3kLinear *a, void *stream)
{
    const dim3 grid((a->out + 63) / 64, (a->T + 15) / 16);
    linear_kernel<<<grid, 256, 0, (hipStream_t)stream>>>(*a);
    K3K_LAUNCH_CHECK("linear");
    return 0;
}
