/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_layer8.c -- the device entry points of a layer's 8-bit path (include/k3_dev.h): the checks of their arguments,
 * in C99 over the kernel ABI (k3k.h). A call is refused here, before any device call, or its kernels stay within what it
 * describes.
 */
#include "k3_dev.h"
#include "k3.h"
#include "k3k.h"

#include <stdio.h>
#include <string.h>

static int refuse(const char *fn, const char *why)
{
    char m[512];
    snprintf(m, sizeof m, "%s: %s", fn, why);
    k3dx_bad(m);
    return -1;
}

static int fail(const char *fn) { return refuse(fn, k3k_error()); }

static int type_ok(int t) { return t == K3D_F32 || t == K3D_BF16; }
static size_t type_size(int t) { return t == K3D_F32 ? 4 : 2; }
static int aligned(const void *p, size_t n) { return ((uintptr_t)p % n) == 0; }
static int blocks(int n) { return (n + 127) / 128; }

/* p is one of the n places at q (none is no place) */
static int among(const void *p, const void *const *q, size_t n)
{
    for (size_t i = 0; p && i < n; i++)
        if (p == q[i]) return 1;
    return 0;
}
#define AMONG(p, ...) among(p, (const void *const[]){__VA_ARGS__}, sizeof((const void *const[]){__VA_ARGS__}) / sizeof(void *))

/* 8-bit rows of n columns and their scales: NULL, or what is wrong with them */
static const char *rows_bad(const void *q, long ldq, const void *s, long lds, int n)
{
    if (!q || !s) return "codes and their scales must be given";
    if (!aligned(q, 16) || ldq % 16) return "codes must be 16-byte aligned, and so their rows";
    if (!aligned(s, 4)) return "a pointer is not aligned to its elements";
    if (ldq < (long)blocks(n) * 128) return "a row of codes holds whole blocks of 128 columns: the stride is shorter";
    if (lds < blocks(n)) return "the scales' stride is shorter than a row of them";
    return NULL;
}

static const char *act_bad(int act, float b1, float b2)
{
    if (act != K3D_GLU_SITU && act != K3D_GLU_SILU) return "unknown activation";
    /* (within these a limit's reciprocal, and what the kernels multiply with them, stay in fp32) */
    if (act == K3D_GLU_SITU && !(b1 >= 0x1p-64f && b1 <= 0x1p64f && b2 >= 0x1p-64f && b2 <= 0x1p64f)) return "situ needs limits from 2^-64 to 2^64";
    return NULL;
}

/* ---- residual, norm, 8 bits ------------------------------------------------------------ */
int k3d_add_norm(void *y, int y_type, long ldy, uint8_t *q, long ldq, float *qs, long ldqs, void *sum, long ldsum,
                 const void *x, int x_type, long ldx, const void *res, int r_type, long ldr, int T, int n, const float *w,
                 float eps, void *stream)
{
    static const char fn[] = "k3d_add_norm";
    if (!type_ok(x_type) || !type_ok(y_type) || !type_ok(r_type)) return refuse(fn, "x_type, y_type and r_type are K3D_F32 or K3D_BF16");
    if (T < 0 || n < 1 || n > K3D_NORM_MAX_N) return refuse(fn, "need T >= 0 and 1 <= n <= K3D_NORM_MAX_N");
    if (!(eps >= 0.0f)) return refuse(fn, "eps >= 0");
    if (T == 0) return 0;
    if (T > K3D_MAX_TOKENS) return refuse(fn, "up to K3D_MAX_TOKENS tokens");
    if (!x || (!y && !q && !sum)) return refuse(fn, "x and an output must be given");
    if (ldx < n || (y && ldy < n) || (sum && ldsum < n) || (res && ldr < n)) return refuse(fn, "a stride is shorter than its row");
    if (!aligned(x, type_size(x_type)) || !aligned(y, type_size(y_type)) || !aligned(res, type_size(r_type)) ||
        !aligned(sum, type_size(r_type)) || !aligned(w, 4))
        return refuse(fn, "a pointer is not aligned to its elements");
    if (q) {
        const char *bad = rows_bad(q, ldq, qs, ldqs, n);
        if (bad) return refuse(fn, bad);
    }
    if (sum && sum == res && ldsum != ldr) return refuse(fn, "sum in res's place needs its stride");
    if (sum && sum == x && (ldsum != ldx || r_type != x_type)) return refuse(fn, "sum in x's place needs its stride and type");
    if (y && y == x && (ldy != ldx || y_type != x_type)) return refuse(fn, "y in x's place needs its stride and type");
    if (y && y == res && (ldy != ldr || y_type != r_type)) return refuse(fn, "y in res's place needs its stride and type");
    if (AMONG(y, sum, q) || AMONG(sum, q) || (q && AMONG(qs, y, sum, q))) return refuse(fn, "two outputs are one place");
    if (AMONG(q, x, res, w) || (q && AMONG(qs, x, res, w)) || AMONG(w, y, sum)) return refuse(fn, "an output lies in an operand's place");
    K3kNorm a;
    a.y = y;
    a.sum = sum;
    a.q = q;
    a.qs = qs;
    a.x = x;
    a.res = res;
    a.w = w;
    a.ldy = ldy;
    a.ldsum = ldsum;
    a.ldq = ldq;
    a.ldqs = ldqs;
    a.ldx = ldx;
    a.ldr = ldr;
    a.y_type = y_type;
    a.x_type = x_type;
    a.r_type = r_type;
    a.T = T;
    a.n = n;
    a.eps = eps;
    if (k3k_add_norm(&a, stream)) return fail(fn);
    return 0;
}

/* ---- gated activation, 8 bits ---------------------------------------------------------- */
int k3d_quant_f8(uint8_t *q, long ldq, float *qs, long ldqs, const void *x, int x_type, long ldx, int T, int n, int act,
                 float b1, float b2, void *stream)
{
    static const char fn[] = "k3d_quant_f8";
    if (!type_ok(x_type)) return refuse(fn, "x_type is K3D_F32 or K3D_BF16");
    if (act != K3D_GLU_NONE) {
        const char *bad = act_bad(act, b1, b2);
        if (bad) return refuse(fn, bad);
    }
    if (T < 0 || n < 1 || n > K3D_NORM_MAX_N) return refuse(fn, "need T >= 0 and 1 <= n <= K3D_NORM_MAX_N");
    if (T == 0) return 0;
    if (T > K3D_MAX_TOKENS) return refuse(fn, "up to K3D_MAX_TOKENS tokens");
    if (!x) return refuse(fn, "x must be given");
    if (ldx < (act == K3D_GLU_NONE ? n : 2L * n)) return refuse(fn, "a stride is shorter than its row");
    if (!aligned(x, type_size(x_type))) return refuse(fn, "a pointer is not aligned to its elements");
    const char *bad = rows_bad(q, ldq, qs, ldqs, n);
    if (bad) return refuse(fn, bad);
    if ((const void *)q == qs) return refuse(fn, "two outputs are one place");
    if (AMONG(x, q, qs)) return refuse(fn, "an output lies in an operand's place");
    K3kQuant a;
    a.q = q;
    a.qs = qs;
    a.x = x;
    a.ldq = ldq;
    a.ldqs = ldqs;
    a.ldx = ldx;
    a.x_type = x_type;
    a.T = T;
    a.n = n;
    a.act = act;
    a.b1 = b1;
    a.b2 = b2;
    if (k3k_quant_f8(&a, stream)) return fail(fn);
    return 0;
}

/* ---- weights ----------------------------------------------------------------------------- */
size_t k3d_f8_tiled_bytes(int rows, int in)
{
    if (rows <= 0 || in <= 0) return 0;
    return k3k_f8_tiled_bytes(rows, in);
}

int k3d_f8_tile(uint8_t *t, const uint8_t *W, long ldw, int rows, int in, int mats, void *stream)
{
    static const char fn[] = "k3d_f8_tile";
    if (rows < 1 || in < 1 || mats < 0) return refuse(fn, "need rows >= 1, in >= 1, mats >= 0");
    if (in > K3D_F8_MAX_IN || rows > K3D_F8_MAX_OUT) return refuse(fn, "in up to K3D_F8_MAX_IN, rows up to K3D_F8_MAX_OUT");
    if (mats == 0) return 0;
    if (ldw < in) return refuse(fn, "a stride is shorter than its row");
    if ((double)mats * (double)k3k_f8_tiled_bytes(rows, in) >= 0x1p43) return refuse(fn, "up to 2^43 bytes");
    if (!t || !W) return refuse(fn, "t and W must be given");
    if (!aligned(t, 16)) return refuse(fn, "t must be 16-byte aligned");
    if (t == W) return refuse(fn, "t lies in W's place");
    if (k3k_f8_tile(t, W, ldw, rows, in, mats, stream)) return fail(fn);
    return 0;
}

/* ---- dense product ----------------------------------------------------------------------- */
size_t k3d_linear_f8_ws(int T, int in, int out)
{
    if (T <= 0 || in <= 0 || out <= 0) return 0;
    return k3k_linear_f8_ws(T, in, out);
}

static const char *sizes_bad(int in, int out)
{
    if (in < 1 || out < 0) return "need in >= 1 and out >= 0";
    if (in > K3D_F8_MAX_IN || out > K3D_F8_MAX_OUT) return "in up to K3D_F8_MAX_IN, out up to K3D_F8_MAX_OUT";
    return NULL;
}

int k3d_linear_f8(void *y, int y_type, long ldy, const uint8_t *x, long ldx, const float *xs, long ldxs, int T,
                  const uint8_t *W, const float *Ws, long ldws, int in, int out, const float *bias, int act,
                  const void *res, long ldr, void *ws, size_t ws_bytes, void *stream)
{
    static const char fn[] = "k3d_linear_f8";
    const char *bad = sizes_bad(in, out);
    if (bad) return refuse(fn, bad);
    if (!type_ok(y_type)) return refuse(fn, "y_type is K3D_F32 or K3D_BF16");
    if (act < K3D_ACT_NONE || act > K3D_ACT_GELU_TANH) return refuse(fn, "unknown activation");
    if (T < 0) return refuse(fn, "need T >= 0");
    if (T == 0 || out == 0) return 0;
    if (T > K3D_MAX_TOKENS) return refuse(fn, "up to K3D_MAX_TOKENS tokens");
    if ((long)T * out > K3D_F8_MAX_RESULTS) return refuse(fn, "T * out up to K3D_F8_MAX_RESULTS");
    if ((bad = rows_bad(x, ldx, xs, ldxs, in))) return refuse(fn, bad);
    if (ldx > K3D_F8_MAX_LD || ldxs > K3D_F8_MAX_LD / 4) return refuse(fn, "ldx up to K3D_F8_MAX_LD, ldxs up to a quarter of it");
    if (!y || !W || !Ws) return refuse(fn, "y, W and Ws must be given");
    if (ldy < out || (res && ldr < out) || ldws < blocks(in)) return refuse(fn, "a stride is shorter than its row");
    if (!aligned(y, type_size(y_type)) || !aligned(res, type_size(y_type)) || !aligned(Ws, 4) || !aligned(bias, 4))
        return refuse(fn, "a pointer is not aligned to its elements");
    if (!aligned(W, 16)) return refuse(fn, "W must be 16-byte aligned");
    if (res == y && ldr != ldy) return refuse(fn, "res in y's place needs y's stride");
    const size_t need = k3k_linear_f8_ws(T, in, out);
    if (need && (!ws || ws_bytes < need)) return refuse(fn, "workspace too small");
    if (need && !aligned(ws, 16)) return refuse(fn, "the workspace must be 16-byte aligned");
    if (AMONG(y, x, xs, W, Ws, ws, bias)) return refuse(fn, "y lies in an operand's place");
    if (need && AMONG(ws, x, xs, W, Ws, bias, res)) return refuse(fn, "the workspace lies in an operand's place");
    K3kF8 a;
    memset(&a, 0, sizeof a);
    a.y = y;
    a.x = x;
    a.W = W;
    a.xs = xs;
    a.Ws = Ws;
    a.bias = bias;
    a.res = res;
    a.ldy = ldy;
    a.ldx = ldx;
    a.ldxs = ldxs;
    a.ldws = ldws;
    a.ldr = ldr;
    a.y_type = y_type;
    a.T = T;
    a.in = in;
    a.out = out;
    a.act = act;
    a.ws = ws;
    a.wide = y_type == K3D_F32;
    k3k_prof_mark(stream, K3D_STAGE_BEGIN);
    if (k3k_linear_f8(&a, stream)) return fail(fn);
    k3k_prof_mark(stream, K3D_STAGE_GEMV);
    return 0;
}

/* ---- slots by expert --------------------------------------------------------------------- */
static const char *slots_bad(int T, int topk, int n_experts)
{
    if (T < 0 || topk < 1 || topk > K3_MAX_TOPK) return "need T >= 0 and 1 <= topk <= 64";
    if (n_experts < 1 || n_experts > 2048) return "1 to 2048 experts";
    if ((long)T * topk > K3D_F8_MAX_SLOTS) return "T * topk up to K3D_F8_MAX_SLOTS";
    return NULL;
}

size_t k3d_group_ws(int T, int topk, int n_experts)
{
    if (T <= 0 || slots_bad(T, topk, n_experts)) return 0;
    return k3k_group_ws(T * topk, n_experts);
}

int k3d_group(int *offsets, int *perm, const int *idx, int T, int topk, int n_experts, void *ws, size_t ws_bytes, void *stream)
{
    static const char fn[] = "k3d_group";
    const char *bad = slots_bad(T, topk, n_experts);
    if (bad) return refuse(fn, bad);
    if (!offsets || (T && (!perm || !idx))) return refuse(fn, "offsets, perm and idx must be given");
    if (!aligned(offsets, 4) || !aligned(perm, 4) || !aligned(idx, 4)) return refuse(fn, "a pointer is not aligned to its elements");
    if (offsets == perm || offsets == idx || (T && perm == idx)) return refuse(fn, "an output lies in another argument's place");
    const size_t need = k3k_group_ws(T * topk, n_experts);
    if (need && (!ws || ws_bytes < need)) return refuse(fn, "workspace too small");
    if (need && !aligned(ws, 4)) return refuse(fn, "a pointer is not aligned to its elements");
    if (need && AMONG(ws, offsets, perm, idx)) return refuse(fn, "the workspace lies in another argument's place");
    if (k3k_group(offsets, perm, idx, T * topk, n_experts, (int *)ws, stream)) return fail(fn);
    return 0;
}

/* ---- products by expert ------------------------------------------------------------------ */
int k3d_grouped_f8(void *y, int y_type, long ldy, const int *y_rows, int y_cap, const uint8_t *x, long ldx, const float *xs,
                   long ldxs, const int *x_rows, int x_div, int x_cap, const int *offsets, int rows, int n_experts,
                   const uint8_t *W, const float *Ws, int in, int out, void *stream)
{
    static const char fn[] = "k3d_grouped_f8";
    const char *bad = sizes_bad(in, out);
    if (bad) return refuse(fn, bad);
    if (!type_ok(y_type)) return refuse(fn, "y_type is K3D_F32 or K3D_BF16");
    if (n_experts < 1 || n_experts > 2048) return refuse(fn, "1 to 2048 experts");
    if (rows < 0 || x_cap < 0 || y_cap < 0 || x_div < 1) return refuse(fn, "need rows, x_cap, y_cap >= 0 and x_div >= 1");
    if (rows == 0 || x_cap == 0 || y_cap == 0 || out == 0) return 0;
    if (rows > K3D_F8_MAX_SLOTS || y_cap > K3D_MAX_TOKENS || x_cap > K3D_MAX_TOKENS)
        return refuse(fn, "rows up to K3D_F8_MAX_SLOTS, x_cap and y_cap up to K3D_MAX_TOKENS");
    if ((long)rows * out > K3D_F8_MAX_RESULTS) return refuse(fn, "rows * out up to K3D_F8_MAX_RESULTS");
    if ((bad = rows_bad(x, ldx, xs, ldxs, in))) return refuse(fn, bad);
    if (ldx > K3D_F8_MAX_LD || ldxs > K3D_F8_MAX_LD / 4) return refuse(fn, "ldx up to K3D_F8_MAX_LD, ldxs up to a quarter of it");
    if ((long)x_cap * ldx > K3D_F8_MAX_X || (long)x_cap * ldxs * 4 > K3D_F8_MAX_X) return refuse(fn, "x and its scales up to K3D_F8_MAX_X bytes");
    if (!y || !W || !Ws || !offsets) return refuse(fn, "y, offsets, W and Ws must be given");
    if (ldy < out) return refuse(fn, "a stride is shorter than its row");
    if (!aligned(y, type_size(y_type)) || !aligned(Ws, 4) || !aligned(offsets, 4) || !aligned(x_rows, 4) || !aligned(y_rows, 4))
        return refuse(fn, "a pointer is not aligned to its elements");
    if (!aligned(W, 16)) return refuse(fn, "W must be 16-byte aligned");
    if (AMONG(y, x, xs, W, Ws, offsets, x_rows, y_rows)) return refuse(fn, "y lies in an operand's place");
    K3kF8 a;
    memset(&a, 0, sizeof a);
    a.y = y;
    a.x = x;
    a.W = W;
    a.xs = xs;
    a.Ws = Ws;
    a.offsets = offsets;
    a.x_rows = x_rows;
    a.y_rows = y_rows;
    a.ldy = ldy;
    a.ldx = ldx;
    a.ldxs = ldxs;
    a.ldws = blocks(in);
    a.w_step = k3k_f8_tiled_bytes(out, in);
    a.ws_step = (size_t)blocks(out) * blocks(in);
    a.y_type = y_type;
    a.T = y_cap;
    a.in = in;
    a.out = out;
    a.rows = rows;
    a.x_div = x_div;
    a.x_cap = x_cap;
    a.n_experts = n_experts;
    a.wide = y_type == K3D_F32;
    k3k_prof_mark(stream, K3D_STAGE_BEGIN);
    if (k3k_grouped_f8(&a, stream)) return fail(fn);
    k3k_prof_mark(stream, K3D_STAGE_GATEUP);
    return 0;
}

/* ---- the experts' layer ------------------------------------------------------------------ */
typedef struct {
    int *offsets, *perm, *hist;
    uint8_t *hq;
    float *hs, *gu;
    void *y;
} MoeF8Ws;

/* where each part lies in ws; the bytes of all (256-byte aligned parts). gu (gate and up as fp32, where they do not become codes at once) is done with
 * before y (the slots' rows) begins: one place. */
static size_t moe_layout(MoeF8Ws *w, void *ws, int T, int hidden, int inter, int n_experts, int topk)
{
    const size_t N = (size_t)T * topk, nb = blocks(inter), wide = ((size_t)hidden + 63) / 64 * 64;
    const size_t gu = N * 2 * inter * 4, y = N * wide * 4;
    const size_t sizes[6] = {((size_t)n_experts + 1) * 4, N * 4, k3k_group_ws((int)N, n_experts), N * nb * 128, N * nb * 4, gu > y ? gu : y};
    size_t off = 0, at[6];
    for (int i = 0; i < 6; i++) {
        at[i] = off;
        off += (sizes[i] + 255) / 256 * 256;
    }
    if (w) {
        char *const b = (char *)ws;
        w->offsets = (int *)(b + at[0]);
        w->perm = (int *)(b + at[1]);
        w->hist = (int *)(b + at[2]);
        w->hq = (uint8_t *)(b + at[3]);
        w->hs = (float *)(b + at[4]);
        w->gu = (float *)(b + at[5]);
        w->y = w->gu;
    }
    return off;
}

size_t k3d_moe_f8_ws(int T, int hidden, int inter, int n_experts, int topk)
{
    if (T <= 0 || hidden <= 0 || inter <= 0 || slots_bad(T, topk, n_experts)) return 0;
    return moe_layout(NULL, NULL, T, hidden, inter, n_experts, topk);
}

int k3d_moe_f8(void *out, int out_type, long ldo, const int *idx, const float *wt, const uint8_t *x, long ldx, const float *xs,
               long ldxs, int T, const uint8_t *w1, const float *s1, const uint8_t *w3, const float *s3, const uint8_t *w2,
               const float *s2, int hidden, int inter, int n_experts, int topk, int act, float b1, float b2, void *ws,
               size_t ws_bytes, void *stream)
{
    static const char fn[] = "k3d_moe_f8";
    const char *bad = slots_bad(T, topk, n_experts);
    if (bad) return refuse(fn, bad);
    if (!type_ok(out_type)) return refuse(fn, "out_type is K3D_F32 or K3D_BF16");
    if ((bad = act_bad(act, b1, b2))) return refuse(fn, bad);
    if (hidden < 1 || inter < 1 || hidden > K3D_NORM_MAX_N || inter > K3D_NORM_MAX_N) return refuse(fn, "hidden and inter are 1 to K3D_NORM_MAX_N");
    if (T == 0) return 0;
    if ((bad = rows_bad(x, ldx, xs, ldxs, hidden))) return refuse(fn, bad);
    if (ldx > K3D_F8_MAX_LD || ldxs > K3D_F8_MAX_LD / 4) return refuse(fn, "ldx up to K3D_F8_MAX_LD, ldxs up to a quarter of it");
    if ((long)T * ldx > K3D_F8_MAX_X || (long)T * ldxs * 4 > K3D_F8_MAX_X || (long)T * topk * blocks(inter) * 128 > K3D_F8_MAX_X)
        return refuse(fn, "x, its scales and the gated activations' codes up to K3D_F8_MAX_X bytes");
    if (!out || !idx || !wt || !w1 || !s1 || !w3 || !s3 || !w2 || !s2) return refuse(fn, "out, idx, wt, weights and scales must be given");
    if (ldo < hidden) return refuse(fn, "a stride is shorter than its row");
    if (!aligned(out, type_size(out_type)) || !aligned(idx, 4) || !aligned(wt, 4) || !aligned(s1, 4) || !aligned(s3, 4) || !aligned(s2, 4))
        return refuse(fn, "a pointer is not aligned to its elements");
    if (!aligned(w1, 16) || !aligned(w3, 16) || !aligned(w2, 16)) return refuse(fn, "weights must be 16-byte aligned");
    MoeF8Ws w;
    if (!ws || ws_bytes < moe_layout(&w, ws, T, hidden, inter, n_experts, topk)) return refuse(fn, "workspace too small");
    if (!aligned(ws, 16)) return refuse(fn, "the workspace must be 16-byte aligned");
    if (AMONG(out, x, xs, wt, idx, w1, s1, w3, s3, w2, s2, ws)) return refuse(fn, "out lies in an operand's place");
    if (AMONG(ws, x, xs, wt, idx, w1, s1, w3, s3, w2, s2)) return refuse(fn, "the workspace lies in an operand's place");
    const int N = T * topk, one = T == 1 && topk <= n_experts;
    k3k_prof_mark(stream, K3D_STAGE_BEGIN);
    /* (one token's slots are rows of experts of their own: no launch to sort them, and no offsets to search) */
    if (!one && k3k_group(w.offsets, w.perm, idx, N, n_experts, w.hist, stream)) return fail(fn);
    k3k_prof_mark(stream, K3D_STAGE_GATHER);
    K3kF8 a;
    memset(&a, 0, sizeof a);
    a.x = x;
    a.W = w1;
    a.W2 = w3;
    a.xs = xs;
    a.Ws = s1;
    a.Ws2 = s3;
    a.offsets = one ? NULL : w.offsets;
    a.slot_e = one ? idx : NULL;
    a.x_rows = one ? NULL : w.perm;
    a.ldx = ldx;
    a.ldxs = ldxs;
    a.ldws = blocks(hidden);
    a.w_step = k3k_f8_tiled_bytes(inter, hidden);
    a.ws_step = (size_t)blocks(inter) * blocks(hidden);
    a.y_type = K3D_F32;
    a.T = N;
    a.in = hidden;
    a.out = inter;
    a.rows = N;
    a.x_div = topk;
    a.x_cap = T;
    a.n_experts = n_experts;
    a.hq = w.hq;
    a.hs = w.hs;
    a.glu = act;
    a.b1 = b1;
    a.b2 = b2;
    a.wide = out_type == K3D_F32;
    if (k3k_gateup_f8(&a, w.gu, stream)) return fail(fn);
    k3k_prof_mark(stream, K3D_STAGE_GATEUP);
    a.y = w.y;
    a.x = w.hq;
    a.W = w2;
    a.W2 = NULL;
    a.xs = w.hs;
    a.Ws = s2;
    a.x_rows = NULL;
    a.y_rows = one ? NULL : w.perm;
    a.ldy = (hidden + 63L) / 64 * 64;
    a.ldx = blocks(inter) * 128L;
    a.ldxs = blocks(inter);
    a.ldws = blocks(inter);
    a.w_step = k3k_f8_tiled_bytes(hidden, inter);
    a.ws_step = (size_t)blocks(hidden) * blocks(inter);
    a.in = inter;
    a.out = hidden;
    a.x_div = 1;
    a.x_cap = N;
    float *ys;
    if (k3k_slots_f8(&a, &ys, stream)) return fail(fn);
    k3k_prof_mark(stream, K3D_STAGE_DOWN);
    K3kSum s;
    s.out = out;
    s.y = w.y;
    s.ys = ys;
    s.ldy = a.ldy;
    s.wt = wt;
    s.idx = idx;
    s.ldo = ldo;
    s.out_type = out_type;
    s.T = T;
    s.topk = topk;
    s.n = hidden;
    s.n_experts = n_experts;
    if (k3k_sum_slots(&s, stream)) return fail(fn);
    k3k_prof_mark(stream, K3D_STAGE_COMBINE);
    return 0;
}
