/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_f8.hip -- products of e4m3 codes with a scale for each 128 columns of a row of x and for each 128 x 128 block of W
 * (k3d_linear_f8, k3d_grouped_f8 and the products of k3d_moe_f8):
 *   y[t][o] = act(sum_b xs[t][b] ws[o / 128][b] (sum over block b of x[t][k] W[o][k]) + bias[o]) + res[t][o]
 *
 * A block's 128 columns are one 8-bit matrix instruction (16 x 16 x 128), so each instruction starts from zero and its sums enter the
 * fp32 accumulators through one multiplication by the two scales' product: four vector FMAs to 32 cycles of the matrix cores. The
 * 8-bit instructions (all shapes of them alike, as measured) add each 8 neighbouring products after aligning them to the largest's exponent, and what is more
 * than 13 bits below that is cut off: 1.5 * 2^-16 of a sum of random products. That is far under the rounding of a bf16 result, but not of an fp32 one,
 * nor harmless in front of 8-bit codes, which it turns (k3k_gateup_f8); those products (WIDE) are formed by the bf16 instruction out of the codes
 * widened to bf16 (exactly), at half the rate.
 *
 * W is laid out once, by k3d_f8_tile: tiles of 16 rows x 128 columns in the operand's own order, 2 KB, F8_G row tiles side by side,
 * column block after column block, zeros where rows or columns end. So every load of W is contiguous at any size.
 */
#include "k3_common.h"
#include "k3_dev.h"
#include "k3_f8.h"
#include "k3k.h"

#include <math.h>
#include <type_traits>

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));     /* (a load of uint4 loses what tells LDS arrays apart) */
constexpr uint32_t F8_OOB = 0x80000000u;        /* a buffer offset past any descriptor used here */

/* f(0), f(1) .. f(N - 1), the numbers as constants */
template <int S, int N, class F>
__device__ __forceinline__ void each_of(F &&f)
{
    if constexpr (S < N) {
        f(std::integral_constant<int, S>{});
        each_of<S + 1, N>(f);
    }
}

/* sum over a block's 128 columns: a lane holds 32 bytes of row lane % 16 of either operand, 16-byte pieces g and 4 + g of the
 * block (g = lane / 16); it gets token lane % 16, outputs 4 g ..+4 */
__device__ __forceinline__ k3_f32x4 f8_mfma(u32x4 w0, u32x4 w1, u32x4 x0, u32x4 x1)
{
    const i32x8 w = {(int)w0.x, (int)w0.y, (int)w0.z, (int)w0.w, (int)w1.x, (int)w1.y, (int)w1.z, (int)w1.w};
    const i32x8 x = {(int)x0.x, (int)x0.y, (int)x0.z, (int)x0.w, (int)x1.x, (int)x1.y, (int)x1.z, (int)x1.w};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, k3_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

/* 32 codes as bf16: exact */
struct Wide {
    k3_bf16x8 v[4];
};
__device__ __forceinline__ k3_bf16x8 widen8(uint32_t a, uint32_t b)
{
    const k3_bf16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false), p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
    const k3_bf16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false), p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
    return k3_bf16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}
__device__ __forceinline__ Wide widen(u32x4 a, u32x4 b)
{
    return Wide{{widen8(a.x, a.y), widen8(a.z, a.w), widen8(b.x, b.y), widen8(b.z, b.w)}};
}

/* f8_mfma's sum with products and additions in fp32 */
__device__ __forceinline__ k3_f32x4 wide_mfma(const Wide &w, const Wide &x)
{
    k3_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; q++) v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[q], x.v[q], v, 0, 0, 0);
    return v;
}

/* Requests from a buffer straight into LDS, 4 or 16 bytes a lane: lane L writes lds + 4 L or 16 L. As instructions of their own that the compiler does
 * not count: it would have reads of the same array wait for all of them, also where they read what arrived long before. The caller
 * waits, by count, before a barrier. (Raw buffer: what lies past `bytes` comes as zeros.) */
__device__ __forceinline__ i32x4 f8_rsrc(const void *base, uint32_t bytes)
{
    const uint64_t b = (uint64_t)(uintptr_t)base;
    return i32x4{__builtin_amdgcn_readfirstlane((int)b), __builtin_amdgcn_readfirstlane((int)(b >> 32)), __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}

/* where an array lies in LDS (of the array itself: an address computed from it would be checked for null) */
__device__ __forceinline__ uint32_t lds_at(uint32_t *lds) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint32_t *)lds; }

template <int BYTES>
__device__ __forceinline__ void f8_dma(i32x4 r, uint32_t at, uint32_t voff, uint32_t soff)
{
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (BYTES == 16) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(at), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
    else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(at), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
#else
    (void)r; (void)at; (void)voff; (void)soff;
#endif
}

template <int POL>
__device__ __forceinline__ u32x4 bload16(k3_rsrc r, uint32_t off)
{
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, POL));
}

/* ---- layout ---------------------------------------------------------------------------- */
constexpr int F8_TILE = 2048;                   /* bytes of 16 rows x 128 columns */
constexpr int F8_G = 8;                         /* row tiles side by side: the 128 rows of a scale */
constexpr uint32_t F8_KSTEP = F8_G * F8_TILE;   /* from one column block to the next */

__host__ __device__ __forceinline__ int blocks(int n) { return (n + 127) / 128; }
__host__ __device__ __forceinline__ size_t tiled_bytes(int rows, int in) { return (size_t)blocks(rows) * blocks(in) * F8_KSTEP; }

/* 16 bytes of tile (128-row block, column block, row tile) to a thread; loads by the row's alignment */
__global__ __launch_bounds__(128) void tile_kernel(uint8_t *t, const uint8_t *W, size_t ldw, int rows, int in, int nkb, unsigned first)
{
    /* a workgroup: 2 KB, one row tile of one column block of one matrix */
    const size_t i = (size_t)first + blockIdx.x;
    const size_t per = (size_t)blocks(rows) * nkb * F8_G, m = i / per;
    const unsigned j = (unsigned)(i - m * per), rt = j % F8_G, kb = j / F8_G % nkb, rb = j / F8_G / nkb;
    const int h = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int row = (int)(rb * F8_G + rt) * 16 + (lane & 15), col = (int)kb * 128 + (4 * h + (lane >> 4)) * 16;
    uint32_t v[4] = {0, 0, 0, 0};
    if (row < rows && col < in) {
        const uint8_t *p = W + m * rows * ldw + (size_t)row * ldw + col;
        if (col + 16 <= in) __builtin_memcpy(v, p, 16);
        else
            for (int b = 0; b < in - col; b++) v[b / 4] |= (uint32_t)p[b] << (8 * (b % 4));
    }
    *reinterpret_cast<uint4 *>(t + i * F8_TILE + threadIdx.x * 16) = make_uint4(v[0], v[1], v[2], v[3]);
}

/* ---- which rows ------------------------------------------------------------------------ */
struct Job {
    int e, r0, n;       /* expert, its first row here, rows (0: nothing to do) */
};

/* Of the experts' rows, cut into passes of `most`: how many passes there are, and (find_job) the j-th. Each lane holds a run of
 * experts. Offsets out of order or range count as no rows. */
struct Jobs {
    int total, before, mine, per;       /* passes; of the lanes before; of this lane; experts a lane */
    int n, r0;                          /* (one expert a lane) its rows, the first */
};

__device__ __forceinline__ int rows_of(const K3kF8 &a, int e, int &r0)
{
    if (e >= a.n_experts) return 0;
    const int p = a.offsets[e], q = min(a.offsets[e + 1], a.rows);
    r0 = p;
    return p < 0 || q <= p ? 0 : q - p;
}

__device__ __forceinline__ Jobs count_jobs(const K3kF8 &a, int most)
{
    const int lane = threadIdx.x & 63;
    Jobs s;
    s.per = (a.n_experts + 63) / 64;
    s.mine = 0;
    for (int i = 0; i < s.per; i += 4) {
        int n[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            int r0 = 0;
            n[u] = i + u < s.per ? rows_of(a, lane * s.per + i + u, r0) : 0;
            if (u == 0) s.n = n[0], s.r0 = r0;
        }
#pragma unroll
        for (int u = 0; u < 4; u++) s.mine += (n[u] + most - 1) / most;
    }
    int sum = s.mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(sum, d);
        sum += lane >= d ? o : 0;
    }
    s.before = sum - s.mine;
    s.total = __builtin_amdgcn_readlane(sum, 63);
    return s;
}

__device__ __forceinline__ Job find_job(const K3kF8 &a, const Jobs &s, int j, int most)
{
    const int lane = threadIdx.x & 63;
    Job job = {0, 0, 0};
    const uint64_t who = __ballot(j >= s.before && j < s.before + s.mine);
    if (!who) return job;
    const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)who) - 1);
    int left = j - __builtin_amdgcn_readlane(s.before, l);
    if (s.per == 1) {           /* (no second look at the offsets: 2048 tokens on 64 experts 1229 -> 1214 us) */
        const int n = __builtin_amdgcn_readlane(s.n, l);
        return Job{l, __builtin_amdgcn_readlane(s.r0, l) + left * most, min(most, n - left * most)};
    }
    /* the lane's experts, one to a lane now */
    int r0 = 0, n = lane < s.per ? rows_of(a, l * s.per + lane, r0) : 0;
    const int p = (n + most - 1) / most;
    int sum = p;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(sum, d);
        sum += lane >= d ? o : 0;
    }
    const int f = __builtin_amdgcn_readfirstlane(__ffsll(__ballot(left >= sum - p && left < sum)) - 1);
    left -= __builtin_amdgcn_readlane(sum - p, f);
    job.e = l * s.per + f;
    job.r0 = __builtin_amdgcn_readlane(r0, f) + left * most;
    job.n = min(most, __builtin_amdgcn_readlane(n, f) - left * most);
    return job;
}

/* the row of x of a job's i-th row, -1 for none */
__device__ __forceinline__ int x_row(const K3kF8 &a, int r)
{
    if (a.slot_e) return r / a.x_div;
    if (!a.offsets) return r;
    int t = r;
    if (a.x_rows) {
        t = a.x_rows[r];
        t = t < 0 ? -1 : t / a.x_div;
    }
    return t < a.x_cap ? t : -1;
}

/* the row of y, past every row for one that is left as it was */
__device__ __forceinline__ int y_row(const K3kF8 &a, int r)
{
    if (!a.offsets) return r;
    int t = a.y_rows ? a.y_rows[r] : r;
    if (x_row(a, r) < 0) t = -1;
    return (unsigned)t < (unsigned)a.T ? t : a.T;
}

/* ---- up to 64 rows: W straight into operands ---------------------------------------------- */
constexpr int SK_NW = 4;                        /* waves */

/* a stage, an array of its own: that tells the accesses of one from those of another */
template <int S, int SZ>
__device__ __forceinline__ uint32_t *stage_of()
{
    __shared__ __attribute__((aligned(1024))) uint32_t b[SZ];
    return b;
}

/* A workgroup takes 16 RW rows of W and up to 8 NP rows of x; its four waves share the column blocks, each with a ring of R blocks: W's tiles
 * are operands as loaded, 1 KB a load, into registers; rows of x come by DMA, 8 lanes to a row's 128 bytes, into LDS of the wave's own
 * (16-byte column c of row r in slot c ^ (r / 2 % 8): the 16 rows of a fragment fall on all banks). So there is no barrier until the waves'
 * sums meet. Past the wave's run and behind the last row requests return zeros without reading.
 * Bound by reading W (one token of 7168 -> 12288, 88 MB, 16.3 us; 64 tokens on 384 experts of 7168 -> 2048, 4.1 GB, 603 us = 6.8 TB/s) and, for many
 * rows, by what a CU takes in: x comes again for each 16 RW rows of W (64 tokens of 7168 -> 12288 24.5 us). Deeper rings change nothing. */
template <int RW, int NP, int R, int POL, bool WIDE>
__global__ __launch_bounds__(64 * SK_NW) void f8_skinny_kernel(K3kF8 a, int o0, int og)
{
    constexpr int NW = SK_NW;
    constexpr int NT = (NP + 1) / 2, XW = NP * 256;              /* a wave's stage of x, in 4-byte units */
    static_assert(NP % 2 == 0, "whole fragments");
    __shared__ uint32_t SC[NW * NT * 256];
    Job job = {0, 0, a.T};
    int o = blockIdx.x;
    if (a.offsets || a.slot_e) {
        const int j = blockIdx.x / (unsigned)og;
        o -= j * og;
        if (a.W2 && 2 * o >= og) {              /* the second matrix, its outputs behind the first's */
            o -= og / 2;
            a.W = a.W2;
            a.Ws = a.Ws2;
            a.y = (float *)a.y + a.out;
        }
        if (a.slot_e) {
            const int e = a.slot_e[j];
            job = Job{e, j, (unsigned)e < (unsigned)a.n_experts ? 1 : 0};
        } else job = find_job(a, count_jobs(a, 8 * NP), j, 8 * NP);
        if (job.n == 0) return;
    }
    const int rt0 = (o0 + o) * RW;
    const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nkb = blocks(a.in), k0 = nkb * wv / NW, k1 = nkb * (wv + 1) / NW, n = k1 - k0;

    /* (three tiles can lie in two groups, with scales of their own) */
    constexpr bool TWO = F8_G % RW != 0;
    const int rb = rt0 / F8_G, left_rb = blocks(a.out) - rb;
    const k3_rsrc rw = k3_make_rsrc(a.W + (size_t)job.e * a.w_step + (size_t)rb * nkb * F8_KSTEP, (uint32_t)min(left_rb, TWO ? 2 : 1) * (uint32_t)nkb * F8_KSTEP);
    auto w_at = [&](int q) -> uint32_t {
        const int rt = rt0 + q;
        return (uint32_t)(rt / F8_G - rb) * (uint32_t)nkb * F8_KSTEP + (uint32_t)(rt % F8_G) * F8_TILE;
    };
    const k3_rsrc rx = k3_make_rsrc(a.x, F8_OOB), rs = k3_make_rsrc(a.xs, F8_OOB);
    auto sw = [](int r) { return (r >> 1) & 7; };
    uint32_t xo[NP], so[NT];
#pragma unroll
    for (int p = 0; p < NP; p++) {
        const int r = 8 * p + lane / 8, t = r < job.n ? x_row(a, job.r0 + r) : -1;
        xo[p] = t < 0 ? F8_OOB : (uint32_t)t * (uint32_t)a.ldx + ((lane & 7) ^ sw(r)) * 16;
    }
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int r = 16 * j + r16, t = r < job.n ? x_row(a, job.r0 + r) : -1;
        so[j] = t < 0 ? F8_OOB : (uint32_t)t * (uint32_t)a.ldxs * 4;
    }
    const float *const Ws = a.Ws + (size_t)job.e * a.ws_step;
    auto scales = [&](int b, int i) {
        float v = Ws[(size_t)min(b, blocks(a.out) - 1) * a.ldws + min(k0 + i + lane, nkb - 1)];
        asm volatile("" : "+v"(v));
        return v;
    };
    float wsc = scales(rb, 0), wsc2 = TWO ? scales(rb + 1, 0) : 0.0f;
    /* scales of x: 16 blocks at a time through LDS, [block][row] (one block's alone would be a line of memory for each row and block) */
    uint32_t *const sc = SC + wv * NT * 256;
    auto x_scales = [&](int c) {                /* of blocks k0 + c ..+16 */
        float v[NT][4];
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int kb = k0 + c + 4 * g + e;
                v[j][e] = __uint_as_float(k3_bload4(rs, (so[j] + kb * 4) | (kb < nkb ? 0u : F8_OOB)));
            }
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) sc[(4 * g + e) * NT * 16 + 16 * j + r16] = __float_as_uint(v[j][e]);
        __builtin_amdgcn_wave_barrier();
    };
    x_scales(0);
    auto buf_of = [&](auto slot) -> uint32_t * { return stage_of<decltype(slot)::value, NW * XW>() + wv * XW; };
    u32x4 wr[R][RW][2];
    int at = 0;                                 /* the block requested next */
    /* (inlined in any case: a call would put what the bodies share in memory, 64 tokens of 7168 -> 12288 to fp32 in 360 us) */
    auto load = [&](auto slot) __attribute__((always_inline)) {
        constexpr int S = decltype(slot)::value;
        const uint32_t none = at < n ? 0u : F8_OOB, kb = k0 + at;
#pragma unroll
        for (int p = 0; p < NP; p++) k3_dma16(rx, buf_of(slot) + p * 256, xo[p] | none, kb * 128);
#pragma unroll
        for (int q = 0; q < RW; q++)
#pragma unroll
            for (int h = 0; h < 2; h++) wr[S][q][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rw, (w_at(q) + lane * 16 + h * 1024) | none, kb * F8_KSTEP, POL));
        at++;
    };
    k3_f32x4 acc[RW][NT];
#pragma unroll
    for (int q = 0; q < RW; q++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[q][j] = k3_f32x4{0.f, 0.f, 0.f, 0.f};
    int i = 0;
    auto use = [&](auto slot) __attribute__((always_inline)) {
        constexpr int S = decltype(slot)::value;
        const uint32_t *const b = buf_of(slot);
        const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wsc), i & 63));
        const float w2 = TWO ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wsc2), i & 63)) : w;
        /* W's last request of this block is younger than its rows of x: with it all have arrived */
#pragma unroll
        for (int q = 0; q < RW; q++) asm volatile("" : "+v"(wr[S][q][0]), "+v"(wr[S][q][1]));
        __builtin_amdgcn_sched_barrier(0);
        u32x4 xf[NT][2];
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) xf[j][h] = *reinterpret_cast<const u32x4 *>(b + (16 * j + r16) * 32 + (((4 * h + g) ^ sw(r16)) & 7) * 4);
        Wide ww[WIDE ? RW : 1];
        if constexpr (WIDE) each_of<0, RW>([&](auto q) { ww[decltype(q)::value] = widen(wr[S][decltype(q)::value][0], wr[S][decltype(q)::value][1]); });
        each_of<0, NT>([&](auto jj) __attribute__((always_inline)) {
            constexpr int j = decltype(jj)::value;
            const float xs = __uint_as_float(sc[(i & 15) * NT * 16 + 16 * j + r16]);
            Wide xw;
            if constexpr (WIDE) xw = widen(xf[j][0], xf[j][1]);
            each_of<0, RW>([&](auto qq) __attribute__((always_inline)) {
                constexpr int q = decltype(qq)::value;
                const float f = xs * (TWO && (rt0 + q) / F8_G != rb ? w2 : w);
                k3_f32x4 v;
                if constexpr (WIDE) v = wide_mfma(ww[q], xw);
                else v = f8_mfma(wr[S][q][0], wr[S][q][1], xf[j][0], xf[j][1]);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[q][j][e] = fmaf(f, v[e], acc[q][j][e]);
                asm volatile("" : "+v"(acc[q][j]));
            });
        });
        __builtin_amdgcn_sched_barrier(0);
        if ((++i & 15) == 0 && i < n) {
            x_scales(i);
            if ((i & 63) == 0) {
                wsc = scales(rb, i);
                if (TWO) wsc2 = scales(rb + 1, i);
            }
        }
    };
    each_of<0, R - 1>(load);
    int left = n;
    /* block k is used while block k + R - 1 is requested, into the stage that block k - 1 left */
    for (; left >= R; left -= R)
        each_of<0, R>([&](auto slot) __attribute__((always_inline)) {
            load(std::integral_constant<int, (decltype(slot)::value + R - 1) % R>{});
            use(slot);
        });
    each_of<0, R - 1>([&](auto slot) __attribute__((always_inline)) {
        if (decltype(slot)::value < left) use(slot);
    });

    /* the waves' sums, in their order, 16 rows of W at a time, where the last requests (of zeros) have landed */
    __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));
    float4 *const part = reinterpret_cast<float4 *>(buf_of(std::integral_constant<int, 0>{}));
    each_of<0, RW>([&](auto qq) __attribute__((always_inline)) {
        constexpr int q = decltype(qq)::value;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; j++) part[j * 64 + lane] = make_float4(acc[q][j][0], acc[q][j][1], acc[q][j][2], acc[q][j][3]);
        __syncthreads();
        for (int j = wv; j < NT; j += NW) {
            const int out = (rt0 + q) * 16 + 4 * g, r = 16 * j + r16;
            const int t = r < job.n ? y_row(a, job.r0 + r) : a.T;
            float b[4];
            bias4(a, out, b);
            const uint4 res = res4(a, t, out);
            const float4 *p = reinterpret_cast<const float4 *>(stage_of<0, NW * XW>()) + j * 64 + lane;
            float4 s = p[0];
#pragma unroll
            for (int w = 1; w < NW; w++) {
                const float4 v = p[w * (XW / 4)];
                s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
            }
            put4(a, t, out, s, b, res);
        }
    });
}

/* ---- many rows: LDS tiles ---------------------------------------------------------------- */
typedef struct {
    K3kF8 a;
    int nt, no;             /* tiles over rows (dense) and outputs */
    int nsl, per;           /* slices of the column blocks, blocks of one */
    float *part;            /* [nsl][T][out] sums of the slices (nsl > 1) */
} F8Tile;

/* Which row and output tile workgroup b of nt * no * nsl takes: each XCD gets a run of tiles of its own, slice by
 * slice, down 8 row tiles before the next outputs (what a run reads of W it reads once from its L2, and its x stays there). */
__device__ __forceinline__ bool tile_of(int nt, int no, int nsl, int b, int &tt, int &to, int &sl)
{
    const int tiles = nt * no, all = tiles * nsl;
    if (b >= all) return false;
    const int full = all / K3_NXCD * K3_NXCD;
    int i = b;
    if (b < full) i = (b % K3_NXCD) * (all / K3_NXCD) + b / K3_NXCD;
    sl = i / tiles;
    i -= sl * tiles;
    constexpr int GT = 8;
    const int blk = GT * no, q = i / blk, h = min(GT, nt - q * GT), r = i - q * blk;
    to = r / h;
    tt = q * GT + r % h;
    return true;
}

/* up to n of eight sums of a slice */
__device__ __forceinline__ void part8(float *q, const float (&v)[8], int n)
{
    if (n >= 8) {
        __builtin_memcpy(q, v, 32);
    } else {
#pragma unroll
        for (int m = 0; m < 7; m++)
            if (m < n) q[m] = v[m];
    }
}

/* (one choice for the eight: the activation is the same for all) */
template <bool F32>
__device__ __forceinline__ void act8(float (&v)[8], int act)
{
    each_of<K3D_ACT_RELU, K3D_ACT_GELU_TANH + 1>([&](auto which) {
        if (act == decltype(which)::value)
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = act_of<F32>(v[i], decltype(which)::value);
    });
}

/* the residual of outputs o ..+8 of row t as it lies in memory */
struct Res8 {
    uint4 a, b;
};
__device__ __forceinline__ Res8 res8(const K3kF8 &a, int t, int o)
{
    Res8 r = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (!a.res || t >= a.T || o + 8 > a.out) return r;
    const bool bf = a.y_type == K3D_BF16;
    const char *q = (const char *)a.res + ((size_t)t * a.ldr + o) * (bf ? 2 : 4);
    __builtin_memcpy(&r.a, q, 16);
    if (!bf) __builtin_memcpy(&r.b, q + 16, 16);
    return r;
}

/* outputs o ..+8 of row t: v + bias b through the activation, plus the residual */
__device__ __forceinline__ void put8(const K3kF8 &a, int t, int o, float (&v)[8], const float (&b)[8], const Res8 &r)
{
    if (t >= a.T || o >= a.out) return;
    if (o + 8 > a.out) {                /* (the end of a row) */
        put4(a, t, o, make_float4(v[0], v[1], v[2], v[3]), *(const float(*)[4])b, res4(a, t, o));
        put4(a, t, o + 4, make_float4(v[4], v[5], v[6], v[7]), *(const float(*)[4])(b + 4), res4(a, t, o + 4));
        return;
    }
    const bool bf = a.y_type == K3D_BF16;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += b[i];
    if (bf) act8<false>(v, a.act);
    else act8<true>(v, a.act);
    const size_t at = (size_t)t * a.ldy + o;
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (bf) {
        if (a.res)
#pragma unroll
            for (int i = 0; i < 4; i++) v[2 * i] += __uint_as_float(w[i] << 16), v[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
        __bf16 h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = (__bf16)v[i];
        __builtin_memcpy((uint16_t *)a.y + at, h, 16);
    } else {
        if (a.res)
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] += __uint_as_float(w[i]);
        __builtin_memcpy((float *)a.y + at, v, 32);
    }
}

/* The largest magnitude among 8 neighbouring lanes. */
__device__ __forceinline__ uint32_t max8_bits(uint32_t v)
{
    v = max(v, dpp_u32<0xB1, 0xf, 0u>(v));      /* quad_perm [1,0,3,2] */
    v = max(v, dpp_u32<0x4E, 0xf, 0u>(v));      /* quad_perm [2,3,0,1] */
    return max(v, dpp_u32<0x141, 0xf, 0u>(v));  /* row_half_mirror */
}

/* outputs o ..+8 of row t as 16-bit floats, 8 lanes to a group of 64 columns and its scale, the power of two that brings the largest finite magnitude
 * (2^-100 at least) to 2^14 ..+2^14; every lane of the 8 takes part. Within 2^-11 of the value, down to 2^-28 of the group's largest; half the bytes of fp32
 * (16-bit integers, as exact beside the largest, left an output 2^11 below it four bits). What is no number stays alone. */
__device__ __forceinline__ void put8_halves(const K3kF8 &a, int t, int o, const float (&v)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, abs_bits(v[i]) < 0x7f800000u ? abs_bits(v[i]) : 0u);
    const uint32_t e = max(max8_bits(m) >> 23, 27u);            /* (biased) */
    const float r = __uint_as_float((268 - e) << 23);
    if (t >= a.T || o >= a.ldy) return;
    f16x8 h;
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = (_Float16)(v[i] * r);
    *reinterpret_cast<f16x8 *>((_Float16 *)a.y + (size_t)t * a.ldy + o) = h;
    if (o % 64 == 0) a.ys[(size_t)t * (a.ldy / 64) + o / 64] = __uint_as_float((e - 14) << 23);
}

/* bytes of LDS: the stages, the scales of x for 16 column blocks, and where each row's lie */
constexpr int tile_lds(int bt, int bo, int nw, int nst) { return nst * (bt + bo) * 128 + 3 * ((bt / 8 + nw - 1) / nw * nw) * 256; }

/* PAIR: the tile is 128 rows of W (gate) and the same of W2 (up), a wave has 32 of both, and what leaves is act(gate) up in 8 bits: a
 * row's 128 columns are one block of it, so its scale is the workgroup's own business. HALVES: a.ys may ask for 16-bit floats. */
template <int BT, int BO, int WT, int WO, int NST, bool WIDE, bool PAIR, bool HALVES>
__device__ __forceinline__ void tile_run(const F8Tile &p, const Job &job, int to, int sl, uint32_t *lds)
{
    constexpr int NW = WT * WO, FT = BT / WT / 16, FO = BO / WO / 16;
    constexpr int XD = BT / 8 / NW, WD = BO / 8 / NW, SD = (BT / 8 + NW - 1) / NW, DN = XD + WD;       /* requests of a wave: a step's, scales' */
    constexpr int SZ = (BT + BO) * 32, SC = SD * NW * 64;       /* a stage, the scales of 8 column blocks, in 4-byte units */
    /* two barriers a step, which release half a stage each: where a DMA of the workgroup fills half of a wave's rows */
    constexpr bool EARLY = NST == 2 && BT / WT == 2 * NW * 8 && FT == 8;
    static_assert(!PAIR || (BO == 256 && WO == 4 && WD % 2 == 0 && !WIDE), "a block of gate and one of up");
    static_assert(XD >= 1 && WD >= 1 && NST >= 2 && NST <= 4 && BO / WO <= 128 && (BO <= 128 || BO % 128 == 0), "tile");
    static_assert((NST * SZ + 3 * SC) * 4 <= tile_lds(BT, BO, NW, NST), "LDS");
    uint32_t *const SX = lds + NST * SZ, *const SO = SX + 2 * SC;

    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wt = wv % WT, wo = wv / WT;
    const K3kF8 &a = p.a;
    const int o0 = to * (PAIR ? BO / 2 : BO), nkb = blocks(a.in);
    const int k0 = sl * p.per, n = min(p.per, nkb - k0);

    /* Row r's 16-byte column c lies in slot c ^ (r / 2 % 8): the 16 rows of a fragment read fall on all 64 banks. */
    auto sw = [](int r) { return (r >> 1) & 7; };
    const size_t xbase = a.offsets ? 0 : (size_t)job.r0;        /* (dense: offsets from the tile's own rows) */
    const i32x4 rx = f8_rsrc(a.x + xbase * a.ldx, F8_OOB), rs = f8_rsrc(a.xs + xbase * a.ldxs, F8_OOB);
    const int rb = o0 / 128;
    const uint32_t wbytes = (uint32_t)min(blocks(a.out) - rb, PAIR ? 1 : (BO + 127) / 128) * (uint32_t)nkb * F8_KSTEP;     /* of the tile's row blocks */
    const size_t wfrom = (size_t)job.e * a.w_step + (size_t)rb * nkb * F8_KSTEP;
    const i32x4 rw = f8_rsrc(a.W + wfrom, wbytes), rw2 = PAIR ? f8_rsrc(a.W2 + wfrom, wbytes) : rw;
    /* DMA i of wave wv fills rows 8 (NW i + wv) ..+8 of x, a lane a 16-byte slot; rows past the job's come as zeros */
    uint32_t xo[XD];
    auto row_at = [&](int r) -> int { return r < job.n ? (a.offsets ? x_row(a, job.r0 + r) : r) : -1; };
#pragma unroll
    for (int i = 0; i < XD; i++) {
        const int r = (i * NW + wv) * 8 + lane / 8, t = row_at(r);
        xo[i] = t < 0 ? F8_OOB : (uint32_t)t * (uint32_t)a.ldx + ((lane & 7) ^ sw(r)) * 16;
    }
    /* Scales of x: 8 column blocks at a time, 8 lanes to a row's 32 bytes (a step's alone would be a line of memory for each row and
     * step); block c of row r in slot c ^ (r / 8 % 2 * 4), so that 16 rows' fall on 64 banks */
#pragma unroll
    for (int i = 0; i < SD; i++) {
        const int r = (i * NW + wv) * 8 + lane / 8, t = r < BT ? row_at(r) : -1;
        SO[i * NW * 64 + tid] = t < 0 ? F8_OOB : (uint32_t)t * (uint32_t)a.ldxs * 4;     /* (read by the thread that wrote it) */
    }
    /* W: the stage holds row tiles in their order, DMA i half tile NW i + wv: where it lies, from the first tile's row block */
    auto w_at = [&](int i) -> uint32_t {
        const int h = i * NW + wv, rt = o0 / 16 + (PAIR ? h / 2 % F8_G : h / 2);
        return (uint32_t)(rt / F8_G - rb) * (uint32_t)nkb * F8_KSTEP + (uint32_t)(rt % F8_G) * F8_TILE + (h & 1) * 1024;
    };
    auto buf_of = [&](auto slot) -> uint32_t * { return lds + decltype(slot)::value * SZ; };
    const uint32_t base = lds_at(lds);
    const int kend = k0 + n;
    auto issue_x = [&](auto slot, int i, int k) {
        f8_dma<16>(rx, base + decltype(slot)::value * SZ * 4 + (i * NW + wv) * 1024, xo[i] | (k < kend ? 0u : F8_OOB), k * 128);
    };
    auto issue_w = [&](auto slot, int i, int k) {
        const uint32_t at = w_at(i), none = k < kend && at < wbytes ? 0u : F8_OOB;
        f8_dma<16>(PAIR && i >= WD / 2 ? rw2 : rw, base + decltype(slot)::value * SZ * 4 + BT * 128 + (i * NW + wv) * 1024, (lane * 16) | none, none ? 0 : at + k * F8_KSTEP);
    };
    auto issue_scales = [&](int c) {            /* of blocks k0 + 8 c ..+8 */
        const int kb = k0 + 8 * c + ((lane & 7) ^ (wv & 1) * 4);
        static_assert(NW % 2 == 0, "a request's rows are 8 i + wv, their parity the wave's");
#pragma unroll
        for (int i = 0; i < SD; i++) f8_dma<4>(rs, base + (NST * SZ + (c & 1) * SC + (i * NW + wv) * 64) * 4, (SO[i * NW * 64 + tid] + kb * 4) | (kb < nkb ? 0u : F8_OOB), 0);
    };
    /* W's scales of the wave's outputs: a lane each, 64 column blocks at a time */
    const size_t sfrom = (size_t)job.e * a.ws_step + (size_t)(PAIR ? rb : min((o0 + wo * (BO / WO)) / 128, blocks(a.out) - 1)) * a.ldws;
    /* (arrived when it returns: a wait at its use would be one for every request since) */
    auto scales = [&](const float *Ws, int i) {
        float v = Ws[sfrom + min(k0 + i + lane, nkb - 1)];
        asm volatile("" : "+v"(v));
        return v;
    };
    float wsc = scales(a.Ws, 0), wsc2 = PAIR ? scales(a.Ws2, 0) : 0.0f;

    k3_f32x4 acc[FO][FT];
#pragma unroll
    for (int i = 0; i < FO; i++)
#pragma unroll
        for (int j = 0; j < FT; j++) acc[i][j] = k3_f32x4{0.f, 0.f, 0.f, 0.f};
    const int xr = wt * (BT / WT) + r16;
    const int xa0 = xr * 32 + ((g ^ sw(xr)) & 7) * 4, xa1 = xr * 32 + (((4 + g) ^ sw(xr)) & 7) * 4;
    const int wa = BT * 32 + wo * (BO / WO) * (PAIR ? 16 : 32) + lane * 4, sa = xr * 8 + ((r16 >> 3 & 1) * 4);
    /* all but the youngest N requests, and LDS: none */
    constexpr int WAITN = EARLY ? XD + WD : DN * (NST - 2);
    constexpr int WAIT_STAGE = (WAITN & 15) | (7 << 4) | (0 << 8) | ((WAITN >> 4) << 14);
    constexpr int WAIT_VM0 = (7 << 4) | (15 << 8);
    static_assert(WAITN < 64, "requests in flight");
    /* Step k: fragments of rows one after another, read three ahead. Three fragments before the end the last one's read has returned: behind
     * a barrier every wave is past its reads of buffer k % NST, and stage k + 1 has landed. So stage k + NST goes into that
     * buffer, and the next step's first rows and, behind their last use, fragments of W are read under the last rows' products. With two stages a
     * request would have a step's time to arrive (256 x 256: 550 of its 3110 cycles were waits for them); so there (EARLY) W's part and half the rows', which are in registers
     * by fragment 1, go behind a barrier of their own then, and what the last fragments read is waited for at the next step's. The scaled sums join the accumulators
     * three products later: behind their own they would wait for it. */
    constexpr int XR = 4, LA = 3, VR = 4, LAG = 3, NM = FT * FO, FR = 2;
    static_assert(FO > LAG, "scales of two fragments");
    static_assert(FT % XR == 0 && NM % VR == 0, "fragment rings");
    u32x4 wf[FO][2], xf[XR][2];
    Wide ww[WIDE ? FO : 1], xw;
    float sf[XR], f[FR], f2[FR];
    k3_f32x4 v[VR];
    auto read_w = [&](const uint32_t *b, int i) {
#pragma unroll
        for (int h = 0; h < 2; h++) wf[i][h] = *reinterpret_cast<const u32x4 *>(b + wa + (PAIR ? i / 2 * F8_G * 512 + i % 2 * 512 : i * 512) + h * 256);
    };
    auto read_x = [&](const uint32_t *b, int j, int k) {        /* of the k-th block */
        xf[j % XR][0] = *reinterpret_cast<const u32x4 *>(b + xa0 + j * 512);
        xf[j % XR][1] = *reinterpret_cast<const u32x4 *>(b + xa1 + j * 512);
        sf[j % XR] = __uint_as_float(SX[(k >> 3 & 1) * SC + (sa ^ (k & 7)) + 128 * j]);
    };
    auto add = [&](int m) {
        const int i = m % FO, j = m / FO;
#pragma unroll
        for (int e = 0; e < 4; e++) acc[i][j][e] = fmaf(PAIR && i >= FO / 2 ? f2[j % FR] : f[j % FR], v[m % VR][e], acc[i][j][e]);
        /* (formed here: the compiler would put all of them off, and hold the products) */
        asm volatile("" : "+v"(acc[i][j]));
    };
    int at = 0;
    auto step = [&](auto slot) {
        constexpr int S = decltype(slot)::value;
        const uint32_t *const b = buf_of(slot);
        const uint32_t *const nb = buf_of(std::integral_constant<int, (S + 1) % NST>{});
        const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wsc), at & 63));
        const float w2 = PAIR ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wsc2), at & 63)) : 0.0f;
        each_of<0, FT>([&](auto jj) {
            constexpr int j = decltype(jj)::value, past = j - (FT - LA);        /* fragments past the barrier (from 0 on) */
            if constexpr (past == 0 || (EARLY && j == 1)) {
                /* (__syncthreads would wait for every request) */
                __builtin_amdgcn_s_waitcnt(WAIT_STAGE);
                asm volatile("s_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (past == 2)
                if ((at & 7) == 0) issue_scales(at / 8 + 1);
            if constexpr (past < 0) {
                read_x(b, j + LA, at);
            } else {                            /* (past the last step: what lies there, unused) */
                read_x(nb, past, at + 1);
            }
            if constexpr (WIDE) {
                if constexpr (j == 0)
#pragma unroll
                    for (int i = 0; i < FO; i++) ww[i] = widen(wf[i][0], wf[i][1]);
                xw = widen(xf[j % XR][0], xf[j % XR][1]);
            }
            f[j % FR] = sf[j % XR] * w;
            if (PAIR) f2[j % FR] = sf[j % XR] * w2;
            each_of<0, FO>([&](auto ii) {
                constexpr int i = decltype(ii)::value, m = j * FO + i;
                if constexpr (WIDE) v[m % VR] = wide_mfma(ww[i], xw);
                else v[m % VR] = f8_mfma(wf[i][0], wf[i][1], xf[j % XR][0], xf[j % XR][1]);
                add((m + NM - LAG) % NM);
                if constexpr (j == FT - 1) read_w(nb, i);
                /* a request behind each product */
                constexpr int q = EARLY ? (past >= 0 ? past * FO + i : (j - 1) * FO + i) : past * FO + i;
                if constexpr (EARLY && past < 0 && q >= 0) {
                    if constexpr (q < WD) issue_w(slot, q, k0 + at + NST);
                    else if constexpr (q - WD < XD / 2) issue_x(slot, 2 * (q - WD), k0 + at + NST);
                }
                if constexpr (EARLY && past >= 0 && q < XD / 2) issue_x(slot, 2 * q + 1, k0 + at + NST);
                if constexpr (!EARLY && q >= 0 && q < XD) issue_x(slot, q, k0 + at + NST);
                if constexpr (!EARLY && q >= XD && q - XD < WD) issue_w(slot, q - XD, k0 + at + NST);
                __builtin_amdgcn_sched_barrier(0);
            });
            static_assert(XD + WD <= LA * FO, "requests behind the products");
            __builtin_amdgcn_sched_barrier(0);
        });
        if ((++at & 63) == 0) {
            wsc = scales(a.Ws, at);
            if (PAIR) wsc2 = scales(a.Ws2, at);
        }
    };
#pragma unroll
    for (int m = 0; m < VR; m++) v[m] = k3_f32x4{0.f, 0.f, 0.f, 0.f}, f[m % FR] = f2[m % FR] = 0.0f;
    issue_scales(0);
    each_of<0, NST>([&](auto slot) {
        constexpr int S = decltype(slot)::value;
#pragma unroll
        for (int i = 0; i < XD; i++) issue_x(slot, i, k0 + S);
#pragma unroll
        for (int i = 0; i < WD; i++) issue_w(slot, i, k0 + S);
    });
    __builtin_amdgcn_s_waitcnt(WAIT_VM0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FO; i++) read_w(lds, i);
#pragma unroll
    for (int j = 0; j < LA; j++) read_x(lds, j, 0);
    int left = n;
    for (; left >= NST; left -= NST) each_of<0, NST>(step);
    each_of<0, NST - 1>([&](auto slot) {
        if (decltype(slot)::value < left) step(slot);
    });
    each_of<NM - LAG, NM>([&](auto m) { add(decltype(m)::value); });

    if constexpr (PAIR) {
        const float r1 = 1.0f / a.b1, r2 = 1.0f / a.b2;
        auto glu = [&](auto act) {              /* in the gate's place */
#pragma unroll
            for (int j = 0; j < FT; j++)
#pragma unroll
                for (int i = 0; i < FO / 2; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][j][e] = glu_of(acc[i][j][e], acc[i + FO / 2][j][e], decltype(act)::value, a.b1, a.b2, r1, r2);
        };
        if (a.glu == K3D_GLU_SILU) glu(std::integral_constant<int, K3D_GLU_SILU>{});
        else glu(std::integral_constant<int, K3D_GLU_SITU>{});
        __builtin_amdgcn_s_waitcnt(WAIT_VM0);  /* the last requests land before LDS is used again */
        __syncthreads();
        /* a row's largest magnitude: of the lane's eight columns, the wave's 32, the four waves' */
        static_assert(2 * SC >= 4 * BT, "largest magnitudes");
#pragma unroll
        for (int j = 0; j < FT; j++) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < FO / 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) m = max(m, abs_bits(acc[i][j][e]));
            m = max(m, (uint32_t)__shfl_xor((int)m, 16));
            m = max(m, (uint32_t)__shfl_xor((int)m, 32));
            if (g == 0) SX[(xr + 16 * j) * 4 + wo] = m;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < FT; j++) {
            const int r = xr + 16 * j;
            const uint4 m = *reinterpret_cast<const uint4 *>(SX + r * 4);
            const float sc = f8_scale(max(max(m.x, m.y), max(m.z, m.w))), inv = 1.0f / sc;
            if (wo == 0 && g == 0 && r < job.n) a.hs[(size_t)(job.r0 + r) * blocks(a.out) + to] = sc;
            /* codes 32 wo + 16 i + 4 g ..+4: 16-byte column 2 wo + i of the row, swizzled as x's */
#pragma unroll
            for (int i = 0; i < FO / 2; i++)
                lds[r * 32 + ((2 * wo + i) ^ sw(r)) * 4 + g] = f8_codes(acc[i][j][0] * inv, acc[i][j][1] * inv, acc[i][j][2] * inv, acc[i][j][3] * inv);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < BT / 8 / NW; i++) {
            const int r = (i * NW + wv) * 8 + lane / 8, c = lane & 7;
            if (r < job.n) *reinterpret_cast<u32x4 *>(a.hq + (size_t)(job.r0 + r) * blocks(a.out) * 128 + to * 128 + c * 16) = *reinterpret_cast<const u32x4 *>(lds + r * 32 + (c ^ sw(r)) * 4);
        }
        return;
    }
    /* The sums go through LDS (the stage buffers, a region per wave, JR fragments of rows at a time; 16-byte column c of row r in
     * c ^ (r % 16)), so that a wave writes whole rows of its outputs, eight to a lane, and the epilogue's code is there once. */
    constexpr int WOUT = BO / WO, C = WOUT / 4;
    constexpr int RB1 = 16 * WOUT;              /* 4-byte units of one fragment of rows */
    constexpr int LR = NST * SZ / NW;           /* of a wave's region */
    constexpr int JR = LR >= FT * RB1 ? FT : LR >= FT / 2 * RB1 ? FT / 2 : FT / 4, RB = JR * RB1;
    static_assert(!HALVES || WOUT == 64, "a group of 64 columns");
    static_assert(JR >= 1 && FT % JR == 0 && RB <= LR && 128 % C == 0, "epilogue regions");
    float4 *const reg = reinterpret_cast<float4 *>(lds + wv * RB);
    constexpr int RI = 128 / C, IT = 16 * JR / RI;              /* rows of a round of the wave, rounds */
    const int c = lane % (C / 2), o = o0 + wo * WOUT + 8 * c, row0 = wt * (BT / WT) + lane / (C / 2);
    float bs[8];
    bias4(a, p.nsl > 1 ? a.out : o, *(float(*)[4])bs);
    bias4(a, p.nsl > 1 ? a.out : o + 4, *(float(*)[4])(bs + 4));
    __builtin_amdgcn_s_waitcnt(WAIT_VM0);      /* the last requests land before LDS is used again */
    __syncthreads();
    each_of<0, FT / JR>([&](auto part) {
        constexpr int j0 = decltype(part)::value * JR;
#pragma unroll
        for (int j = 0; j < JR; j++)
#pragma unroll
            for (int i = 0; i < FO; i++) {
                const int r = 16 * j + r16, oc = 4 * i + g;
                reg[r * C + (oc ^ (r16 & (C - 1)))] = make_float4(acc[i][j0 + j][0], acc[i][j0 + j][1], acc[i][j0 + j][2], acc[i][j0 + j][3]);
            }
        __builtin_amdgcn_wave_barrier();
        /* (residuals of four rounds requested ahead: one after another each round would wait for its own) */
        constexpr int PF = IT < 4 ? IT : 4;
        static_assert(IT % PF == 0, "rounds");
#pragma unroll 1
        for (int i0 = 0; i0 < IT; i0 += PF) {
            int t[PF];
            Res8 res[PF];
#pragma unroll
            for (int i = 0; i < PF; i++) {
                const int at = row0 + 16 * j0 + (i0 + i) * RI;
                t[i] = at < job.n ? y_row(a, job.r0 + at) : a.T;
                if (p.nsl == 1) res[i] = res8(a, t[i], o);
            }
#pragma unroll
            for (int i = 0; i < PF; i++) {
                const int r = lane / (C / 2) + (i0 + i) * RI, x = r & 15 & (C - 1);
                const float4 v0 = reg[r * C + (2 * c ^ x)], v1 = reg[r * C + ((2 * c + 1) ^ x)];
                float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
                if (HALVES && a.ys) put8_halves(a, t[i], o, v);
                else if (p.nsl == 1) put8(a, t[i], o, v, bs, res[i]);
                else if (t[i] < a.T && o < a.out) part8(p.part + ((size_t)sl * a.T + t[i]) * a.out + o, v, a.out - o);
            }
        }
        __builtin_amdgcn_wave_barrier();
    });
}

/* Bound by the matrix cores and the clock under their power where rows are many (4096 tokens of 7168 -> 12288 with silu 316 to 328 us, 2.2 PFLOP/s at some
 * 1.95 GHz; without the scales a library's product takes 263), 13 us of a tile's first requests and epilogue with nothing beside them among it. Experts of about a
 * tile's rows ask for W, 8 MB a step of all workgroups, as fast as memory gives it, and wait: gate and up of 64 experts of 256 rows 606 us, the same
 * rows on 32 experts 447. Tiles of 128 rows there, with three stages, took 10 % more at 256 rows and 4 % less at 264. */
/* DUAL: passes of at most half the rows by a kernel of half the rows and three stages, which takes little over half the time (2048 tokens, eight of 64
 * experts each: half of the experts have a pass of some 16 rows behind one of 256) */
template <int BT, int BO, int WT, int WO, int NST, bool WIDE, bool PAIR, bool DUAL>
__global__ __launch_bounds__(64 * WT * WO) void f8_tile_kernel(F8Tile p)
{
    constexpr int NW = WT * WO, A = tile_lds(BT, BO, NW, NST), B = DUAL ? tile_lds(BT / 2, BO, NW, 3) : 0;
    __shared__ __attribute__((aligned(1024))) uint32_t lds[(A > B ? A : B) / 4];
    const K3kF8 &a = p.a;
    int tt, to, sl;
    Job job;
    if (a.offsets) {
        const Jobs s = count_jobs(a, BT);
        if (!tile_of(s.total, p.no, 1, blockIdx.x, tt, to, sl)) return;
        job = find_job(a, s, tt, BT);
    } else {
        if (!tile_of(p.nt, p.no, p.nsl, blockIdx.x, tt, to, sl)) return;
        job = Job{0, tt * BT, min(BT, a.T - tt * BT)};
    }
    if constexpr (DUAL)
        if (job.n <= BT / 2) return tile_run<BT / 2, BO, WT, WO, 3, WIDE, PAIR, !PAIR>(p, job, to, sl, lds);
    tile_run<BT, BO, WT, WO, NST, WIDE, PAIR, DUAL && !PAIR>(p, job, to, sl, lds);
}

/* the slices' sums, in slice order, and the epilogue; four slices requested at once */
__global__ __launch_bounds__(64) void f8_join_kernel(K3kF8 a, const float *part, int nsl)
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
constexpr int F8_FEW = 64;              /* rows of a dense product that f8_skinny_kernel takes, without slices */
constexpr int F8_MAX_SLICES = 16;
constexpr size_t F8_PART_CAP = (size_t)64 << 20;

/* the slices' sums of any batch up to T: a call takes slices only as far as they fit this */
size_t part_bytes(int T, int out)
{
    const size_t most = (size_t)F8_MAX_SLICES * T * out * 4;
    return most < F8_PART_CAP ? most : F8_PART_CAP;
}

/* passes of up to `most` rows that the experts can need */
long most_jobs(const K3kF8 *a, int most)
{
    return (long)a->rows / most + (a->rows < a->n_experts ? a->rows : a->n_experts);
}

/* weights that no cache keeps from one call to the next, from here on read past the caches (88 MB times one token 16.3 us, 18.2 otherwise; but
 * 15 MB 6.1 and 5.9) */
constexpr size_t F8_NT_BYTES = (size_t)48 << 20;

template <int RW, int NP, int R>
void skinny_go(const K3kF8 *a, long jobs, hipStream_t st)
{
    /* (a launch takes under 2^32 work-items) */
    const long og = ((a->out + 15) / 16 + RW - 1) / RW, mats = a->W2 ? 2 : 1, most = ((1L << 32) - 1) / (64 * SK_NW) / (jobs * mats);
    const bool nt = tiled_bytes(a->out, a->in) * (a->offsets || a->slot_e ? a->n_experts * mats : 1) >= F8_NT_BYTES;
    for (long o = 0; o < og; o += most) {
        const int n = (int)(og - o < most ? og - o : most) * mats;
        const unsigned grid = (unsigned)(jobs * n);
        if (a->wide && nt) f8_skinny_kernel<RW, NP, R, K3_LD_NT, true><<<grid, 64 * SK_NW, 0, st>>>(*a, (int)o, n);
        else if (a->wide) f8_skinny_kernel<RW, NP, R, K3_LD_DEFAULT, true><<<grid, 64 * SK_NW, 0, st>>>(*a, (int)o, n);
        else if (nt) f8_skinny_kernel<RW, NP, R, K3_LD_NT, false><<<grid, 64 * SK_NW, 0, st>>>(*a, (int)o, n);
        else f8_skinny_kernel<RW, NP, R, K3_LD_DEFAULT, false><<<grid, 64 * SK_NW, 0, st>>>(*a, (int)o, n);
    }
}

template <int NP>
void skinny_rows(const K3kF8 *a, hipStream_t st)
{
    /* The rows of W of a workgroup: a CU takes in 46 KB/us, W and x for each of its workgroups (64 tokens of 7168 -> 12288: 256 workgroups of 48 rows
     * 24.5 us, 384 of 32 33, 192 of 64 26.7). By expert: as if each expert had one pass. */
    const bool by = a->offsets || a->slot_e;
    const long jobs = a->slot_e ? a->rows : a->offsets ? most_jobs(a, 8 * NP) : 1, about = by ? (a->rows < a->n_experts ? a->rows : a->n_experts) * (a->W2 ? 2 : 1) : 1;
    const long tiles = (a->out + 15) / 16, cus = k3k_cu_count();
    int rw = 1;
    long best = 0;
    for (int r = 1; r <= 3; r++) {
        const long cost = ((about * ((tiles + r - 1) / r) + cus - 1) / cus) * (2 * r + NP);
        if (r == 1 || cost < best) best = cost, rw = r;
    }
    if (rw == 1) skinny_go<1, NP, NP < 8 ? 4 : 3>(a, jobs, st);
    else if (rw == 2) skinny_go<2, NP, NP < 8 ? 4 : 2>(a, jobs, st);
    else skinny_go<3, NP, NP < 8 ? 4 : 3>(a, jobs, st);
}

void skinny(const K3kF8 *a, int rows, hipStream_t st)
{
    if (rows <= 16) skinny_rows<2>(a, st);
    else if (rows <= 32) skinny_rows<4>(a, st);
    else if (rows <= 48) skinny_rows<6>(a, st);
    else skinny_rows<8>(a, st);
}

template <int BT, int BO, int WT, int WO, int NST, bool WIDE = false, bool PAIR = false, bool DUAL = false>
void tile_go(F8Tile *p, int nsl, hipStream_t st)
{
    const int nkb = blocks(p->a.in);
    p->nt = (p->a.T + BT - 1) / BT;
    p->no = PAIR ? blocks(p->a.out) : (p->a.out + BO - 1) / BO;
    p->per = (nkb + nsl - 1) / nsl;
    p->nsl = (nkb + p->per - 1) / p->per;
    const long grid = (p->a.offsets ? most_jobs(&p->a, BT) : (long)p->nt) * p->no * p->nsl;
    f8_tile_kernel<BT, BO, WT, WO, NST, WIDE, PAIR, DUAL><<<(unsigned)grid, 64 * WT * WO, 0, st>>>(*p);
}

/* Microseconds of a launch of f8_tile_kernel and, with slices, the join: rounds of as many workgroups as fit the chip, each of `per` steps, its first
 * requests and its epilogue (activations and residuals cost a tile more than the join); W comes at 5 GB/ms at the most. What it chooses is within 8 % of the best of all shapes and slices for 12 shapes of 100 to 4096
 * tokens (1000 tokens of 2048 -> 12288 39 us as 256 x 256, 49 as 128 x 256, 57 as 128 x 128; 2048 of 7168 -> 4096 89, 60 and 77). */
struct Shape {
    int bt, bo, per_cu, wide;
    float alone, full, over;    /* of a step, on a CU alone or with as many as fit; of the rest */
};
constexpr Shape SHAPES[] = {{256, 256, 1, 0, 1.62f, 1.62f, 13.0f}, {128, 256, 1, 0, 0.91f, 0.91f, 9.0f}, {128, 128, 1, 0, 0.64f, 0.64f, 7.0f}, {128, 128, 2, 1, 1.0f, 1.65f, 8.0f}};
constexpr int N_SHAPES = sizeof SHAPES / sizeof SHAPES[0];

float tile_cost(const Shape &s, int T, int in, int out, int nsl, float epilogue, long cus)
{
    const long wgs = (long)((T + s.bt - 1) / s.bt) * ((out + s.bo - 1) / s.bo) * nsl, slots = cus * s.per_cu;
    const int per = (blocks(in) + nsl - 1) / nsl;
    const float t = 3.0f + (float)((wgs + slots - 1) / slots) * (per * (wgs <= cus ? s.alone : s.full) + s.over + (nsl > 1 ? 0.0f : epilogue));
    return fmaxf(t, 5.0f + (float)in * out / 5e6f) + (nsl > 1 ? 2.5f + (nsl + 1.0f) * T * out * 4.0f / 4.7e6f : 0.0f);
}

}  // namespace

extern "C" size_t k3k_f8_tiled_bytes(int rows, int in) { return tiled_bytes(rows, in); }

extern "C" int k3k_f8_tile(uint8_t *t, const uint8_t *W, long ldw, int rows, int in, int mats, void *stream)
{
    const int nkb = blocks(in);
    const size_t all = (size_t)mats * blocks(rows) * nkb * F8_G, most = (size_t)1 << 24;
    for (size_t i = 0; i < all; i += most) {
        /* (a launch counts its workgroups from the first one's number, which fits 32 bits: see k3d_f8_tile) */
        tile_kernel<<<(unsigned)(all - i < most ? all - i : most), 128, 0, (hipStream_t)stream>>>(t, W, (size_t)ldw, rows, in, nkb, (unsigned)i);
        K3K_LAUNCH_CHECK("f8_tile");
    }
    return 0;
}

extern "C" size_t k3k_linear_f8_ws(int T, int in, int out)
{
    (void)in;
    return T <= F8_FEW ? 0 : part_bytes(T, out);
}

extern "C" int k3k_linear_f8(const K3kF8 *a, void *stream_)
{
    hipStream_t st = (hipStream_t)stream_;
    if (a->T <= F8_FEW) {
        skinny(a, a->T, st);
        K3K_LAUNCH_CHECK("linear_f8: few rows");
        return 0;
    }
    F8Tile p;
    p.a = *a;
    p.part = (float *)a->ws;
    /* the cheapest tile shape and number of slices */
    float best = 0.0f;
    int shape = 0, nsl = 1;
    const size_t one = (size_t)a->T * a->out * 4, room = part_bytes(a->T, a->out);
    for (int i = 0; i < N_SHAPES; i++) {
        if (SHAPES[i].wide != a->wide) continue;
        for (int n = 1; n <= F8_MAX_SLICES; n *= 2) {
            if (n > 1 && (n * one > room || blocks(a->in) < 2 * n)) break;
            const float t = tile_cost(SHAPES[i], a->T, a->in, a->out, n, (a->act ? 5.0f : 0.0f) + (a->res ? 4.0f : 0.0f), k3k_cu_count());
            if (best == 0.0f || t < best) best = t, shape = i, nsl = n;
        }
    }
    switch (shape) {
    case 0: tile_go<256, 256, 2, 4, 2>(&p, nsl, st); break;
    case 1: tile_go<128, 256, 2, 4, 3>(&p, nsl, st); break;
    case 2: tile_go<128, 128, 2, 2, 4>(&p, nsl, st); break;
    default: tile_go<128, 128, 2, 2, 2, true>(&p, nsl, st); break;
    }
    K3K_LAUNCH_CHECK("linear_f8: tiles");
    if (p.nsl > 1) {
        const size_t n = (size_t)a->T * ((a->out + 3) / 4);
        f8_join_kernel<<<(unsigned)((n + 63) / 64), 64, 0, st>>>(*a, p.part, p.nsl);
        K3K_LAUNCH_CHECK("linear_f8: join");
    }
    return 0;
}

/* Experts' rows without tiles: up to 10 on average in passes of 16 (64 experts of 7168 -> 2048: 8 each 145 us, as tiles 167), up to 16 of long rows
 * in passes of 32 (162 us, as tiles 170; but of 2048 -> 7168 236 and 199). */
static bool few_rows(const K3kF8 *a)
{
    const int each = (a->rows + a->n_experts - 1) / a->n_experts;
    return each <= 10 || (each <= 16 && a->in >= 4096);
}

extern "C" int k3k_grouped_f8(const K3kF8 *a, void *stream_)
{
    hipStream_t st = (hipStream_t)stream_;
    const int each = (a->rows + a->n_experts - 1) / a->n_experts;       /* rows of an expert, on average */
    if (few_rows(a)) {
        skinny(a, each <= 10 ? 16 : 32, st);
        K3K_LAUNCH_CHECK("grouped_f8: few rows");
        return 0;
    }
    F8Tile p;
    p.a = *a;
    p.part = NULL;
    if (a->wide) tile_go<128, 128, 2, 2, 2, true>(&p, 1, st);
    else tile_go<256, 256, 2, 4, 2, false, false, true>(&p, 1, st);
    K3K_LAUNCH_CHECK("grouped_f8: tiles");
    return 0;
}

extern "C" int k3k_slots_f8(const K3kF8 *a, float **ys, void *stream)
{
    K3kF8 s = *a;
    s.y_type = K3D_F32;
    *ys = s.ys = a->wide || few_rows(a) ? NULL : (float *)((_Float16 *)a->y + (size_t)a->T * a->ldy);
    return k3k_grouped_f8(&s, stream);
}

/* Gate and up: W, W2 [experts], into hq / hs; gu: room for their sums where they are formed as fp32 first. A code is a choice: what a sum's cut turns
 * is a whole step of it. So the 8-bit instructions' cut (2e-5 of a sum) shows as 1.1e-3 of the layer's result, and they are for many rows alone, where they
 * halve the time, and for a result that is rounded to bf16 (1.7e-3) anyway. Few rows wait for W: exact products cost
 * them nothing (one token on 8 of 64 experts 69.7 us, 70.1 cut; its error 1.66e-3 as bf16's own, 2.12e-3 cut). An fp32 result of 2048 tokens takes 2003 us, 1497 cut. */
extern "C" int k3k_gateup_f8(const K3kF8 *a, float *gu, void *stream_)
{
    hipStream_t st = (hipStream_t)stream_;
    const bool few = few_rows(a);
    if (!few && !a->wide) {
        F8Tile p;
        p.a = *a;
        p.part = NULL;
        tile_go<256, 256, 2, 4, 2, false, true, true>(&p, 1, st);
        K3K_LAUNCH_CHECK("gateup_f8");
        return 0;
    }
    K3kF8 s = *a;
    s.y = gu;
    s.ldy = 2L * a->out;
    s.T = a->rows;
    s.wide = 1;
    if (!few) s.W2 = NULL;              /* (tiles have one matrix to a launch) */
    if (k3k_grouped_f8(&s, stream_)) return -1;
    if (!few) {
        s.W = a->W2;
        s.Ws = a->Ws2;
        s.y = gu + a->out;
        if (k3k_grouped_f8(&s, stream_)) return -1;
    }
    K3kQuant q = {a->hq, a->hs, gu, blocks(a->out) * 128L, blocks(a->out), 2L * a->out, K3D_F32, a->rows, a->out, a->glu, a->b1, a->b2};
    return k3k_quant_f8(&q, stream_);
}
