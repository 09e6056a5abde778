/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_group.hip -- a routing's slots by expert (k3d_group): offsets[e] .. offsets[e + 1] of perm are the slots t * topk + j
 * whose expert is e, ascending; slots without an expert are in none.
 *
 * A counting sort, the same order every time: a wave ranks its slots among equal experts by ballots, each expert's counts are summed over
 * the workgroup's waves in their order. Up to 4096 slots in one workgroup; more in chunks of 1024, whose
 * counts are summed by chunk before the slots take their places, by one workgroup: beyond 10^5 slots that walk is the time (2^20 slots of 384 experts 125 us, of
 * 2048 413). Bound by latency: barriers and launches (one token of 8 3.3 us, 64 3.9, 512
 * 8.0, 2048 in three launches 8.4; 20000 23.4).
 */
#include "k3_common.h"
#include "k3k.h"

namespace {

constexpr int GR_C = 1024, GR_ONE = 4, GR_MAXE = 2048;

/* This slot's place among the wave's slots of its expert, their number, and whether it is the first of them: the lanes whose expert agrees in
 * each bit (a ballot a bit; one for each expert that the wave holds would be up to 64). */
__device__ __forceinline__ void rank_wave(int e, bool valid, int bits, int &rank, int &count, bool &first)
{
    const uint64_t below = (1ull << (threadIdx.x & 63)) - 1;
    uint64_t same = __ballot(valid);
    for (int b = 0; b < bits; b++) {
        const bool on = e >> b & 1;
        const uint64_t m = __ballot(on);
        same &= on ? m : ~m;
    }
    rank = __popcll(same & below);
    count = __popcll(same);
    first = valid && rank == 0;
}

__device__ __forceinline__ int bits_of(int E) { return E < 2 ? 0 : 32 - __clz(E - 1); }

/* The slot's place among its expert's slots up to here: cnt counts them, over the chunk's n slots; by: counts of each wave, [waves][E up to a
 * pair]. (Waves that add to cnt one after another, with a barrier each, took twice as long: 4096 slots 13.4 us.) */
__device__ __forceinline__ int rank_chunk(int *cnt, uint16_t *by, int e, bool valid, int E, int n)
{
    int rank, count;
    bool first;
    const int waves = min(GR_C / 64, (n + 63) / 64), S = (E + 1) / 2 * 2;
    for (int k = threadIdx.x; k < waves * S / 2; k += GR_C) reinterpret_cast<uint32_t *>(by)[k] = 0;
    rank_wave(e, valid, bits_of(E), rank, count, first);
    uint16_t *const mine = by + (threadIdx.x >> 6) * S;
    __syncthreads();
    if (first) mine[e] = (uint16_t)count;
    __syncthreads();
    for (int k = threadIdx.x; k < E; k += GR_C) {
        int s = cnt[k];
        for (int w = 0; w < waves; w++) {
            const int c = by[w * S + k];
            by[w * S + k] = (uint16_t)s;
            s += c;
        }
        cnt[k] = s;
    }
    __syncthreads();
    const int at = valid ? mine[e] + rank : 0;
    __syncthreads();            /* (the next chunk's counts take the same place) */
    return at;
}

/* off[e]: the sum of n[0 .. e) of GR_MAXE entries, two a thread; the whole sum returned */
__device__ __forceinline__ int scan_experts(const int *n, int *off, int *waves)
{
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int a = n[2 * tid], b = n[2 * tid + 1];
    int sum = a + b;
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(sum, d);
        sum += lane >= d ? o : 0;
    }
    if (lane == 63) waves[wv] = sum;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < GR_C / 64; w++) {
        if (w < wv) before += waves[w];
        total += waves[w];
    }
    off[2 * tid] = before + sum - a - b;
    off[2 * tid + 1] = before + sum - b;
    __syncthreads();
    return total;
}

__global__ __launch_bounds__(GR_C) void group_one_kernel(int *offsets, int *perm, const int *idx, int N, int E)
{
    __shared__ int cnt[GR_MAXE], off[GR_MAXE], waves[GR_C / 64];
    __shared__ uint32_t by[GR_C / 64 * GR_MAXE / 2];
    const int tid = threadIdx.x;
    int e[GR_ONE], rank[GR_ONE];
    for (int u = 0; u < GR_ONE; u++) e[u] = u * GR_C + tid < N ? idx[u * GR_C + tid] : -1;
    cnt[tid] = cnt[GR_C + tid] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < GR_ONE; u++)
        if (u * GR_C < N) rank[u] = rank_chunk(cnt, (uint16_t *)by, e[u], (unsigned)e[u] < (unsigned)E, E, N - u * GR_C);
    const int total = scan_experts(cnt, off, waves);
    for (int i = tid; i <= E; i += GR_C) offsets[i] = i < E ? off[i] : total;
#pragma unroll
    for (int u = 0; u < GR_ONE; u++)
        if ((unsigned)e[u] < (unsigned)E) perm[off[e[u]] + rank[u]] = u * GR_C + tid;
}

/* hist[c][e]: slots of expert e in chunk c */
__global__ __launch_bounds__(GR_C) void group_count_kernel(int *hist, const int *idx, int N, int E)
{
    __shared__ int cnt[GR_MAXE];
    const int tid = threadIdx.x, i = blockIdx.x * GR_C + tid;
    const int e = i < N ? idx[i] : -1;
    cnt[tid] = cnt[GR_C + tid] = 0;
    __syncthreads();
    if ((unsigned)e < (unsigned)E) atomicAdd(&cnt[e], 1);
    __syncthreads();
    for (int k = tid; k < E; k += GR_C) hist[(size_t)blockIdx.x * E + k] = cnt[k];
}

/* hist[c][e] becomes the place of the chunk's first slot of expert e */
__global__ __launch_bounds__(GR_C) void group_scan_kernel(int *offsets, int *hist, int E, int chunks)
{
    __shared__ int cnt[GR_MAXE], off[GR_MAXE], waves[GR_C / 64];
    const int tid = threadIdx.x;
    cnt[tid] = cnt[GR_C + tid] = 0;
    for (int e = tid; e < E; e += GR_C) {
        int s = 0;
#pragma unroll 8
        for (int c = 0; c < chunks; c++) s += hist[(size_t)c * E + e];
        cnt[e] = s;
    }
    __syncthreads();
    const int total = scan_experts(cnt, off, waves);
    for (int e = tid; e <= E; e += GR_C) offsets[e] = e < E ? off[e] : total;
    for (int e = tid; e < E; e += GR_C) {
        int s = off[e];
#pragma unroll 8
        for (int c = 0; c < chunks; c++) {
            int *const h = hist + (size_t)c * E + e;
            const int v = *h;
            *h = s;
            s += v;
        }
    }
}

__global__ __launch_bounds__(GR_C) void group_place_kernel(int *perm, const int *hist, const int *idx, int N, int E)
{
    __shared__ int cnt[GR_MAXE];
    __shared__ uint32_t by[GR_C / 64 * GR_MAXE / 2];
    const int tid = threadIdx.x, i = blockIdx.x * GR_C + tid;
    const int e = i < N ? idx[i] : -1;
    const bool valid = (unsigned)e < (unsigned)E;
    const int from = valid ? hist[(size_t)blockIdx.x * E + e] : 0;
    for (int k = tid; k < E; k += GR_C) cnt[k] = 0;
    __syncthreads();
    const int at = rank_chunk(cnt, (uint16_t *)by, e, valid, E, N - (int)blockIdx.x * GR_C);
    if (valid) perm[from + at] = i;
}

}  // namespace

extern "C" size_t k3k_group_ws(int N, int n_experts)
{
    return N <= GR_ONE * GR_C ? 0 : (size_t)((N + GR_C - 1) / GR_C) * n_experts * 4;
}

extern "C" int k3k_group(int *offsets, int *perm, const int *idx, int N, int n_experts, int *hist, void *stream)
{
    hipStream_t st = (hipStream_t)stream;
    if (N <= GR_ONE * GR_C) {
        group_one_kernel<<<1, GR_C, 0, st>>>(offsets, perm, idx, N, n_experts);
    } else {
        const int chunks = (N + GR_C - 1) / GR_C;
        group_count_kernel<<<chunks, GR_C, 0, st>>>(hist, idx, N, n_experts);
        K3K_LAUNCH_CHECK("group: count");
        group_scan_kernel<<<1, GR_C, 0, st>>>(offsets, hist, n_experts, chunks);
        K3K_LAUNCH_CHECK("group: scan");
        group_place_kernel<<<chunks, GR_C, 0, st>>>(perm, hist, idx, N, n_experts);
    }
    K3K_LAUNCH_CHECK("group");
    return 0;
}
