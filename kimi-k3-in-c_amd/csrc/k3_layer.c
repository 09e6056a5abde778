/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_layer.c -- the device entry points of the operators around the routed experts
 * (include/k3_dev.h): the checks of their arguments, in C99 over the kernel ABI (k3k.h). A call
 * is refused here, before any device call, or its kernels stay within what it describes.
 */
#include "k3_dev.h"
#include "k3.h"
#include "k3k.h"

#include <stdio.h>

static int fail(const char *what)
{
    char m[512];
    snprintf(m, sizeof m, "%s: %s", what, k3k_error());
    k3dx_bad(m);
    return -1;
}

static int type_ok(int t) { return t == K3D_F32 || t == K3D_BF16; }
static size_t type_size(int t) { return t == K3D_F32 ? 4 : 2; }
static int aligned(const void *p, size_t n) { return ((uintptr_t)p % n) == 0; }

/* ---- dense product with an epilogue ---------------------------------------------------- */
size_t k3d_linear_ws(int T, int in, int out, int x_type)
{
    if (T <= 0 || in <= 0 || out <= 0) return 0;
    return k3k_linear_ws(T, in, out, x_type);
}

int k3d_linear(void *y, int y_type, long ldy, const void *x, int x_type, long ldx, int T, const uint16_t *W,
               long ldw, int in, int out, const float *bias, int act, const void *res, long ldr, void *ws,
               size_t ws_bytes, void *stream)
{
    if (!type_ok(x_type) || !type_ok(y_type)) return k3dx_bad("k3d_linear: x_type and y_type are K3D_F32 or K3D_BF16");
    if (act < K3D_ACT_NONE || act > K3D_ACT_GELU_TANH) return k3dx_bad("k3d_linear: unknown activation");
    if (T < 0 || out < 0 || in < 1) return k3dx_bad("k3d_linear: need T >= 0, out >= 0, in >= 1");
    if (T == 0 || out == 0) return 0;
    if (T > K3D_MAX_TOKENS) return k3dx_bad("k3d_linear: up to K3D_MAX_TOKENS tokens");
    if (ldx < in || ldw < in || ldy < out || (res && ldr < out)) return k3dx_bad("k3d_linear: a stride is shorter than its row");
    if (ldx > K3D_LINEAR_MAX_LD || ldw > K3D_LINEAR_MAX_LD || in > K3D_LINEAR_MAX_IN)
        return k3dx_bad("k3d_linear: ldx and ldw up to K3D_LINEAR_MAX_LD, in up to K3D_LINEAR_MAX_IN");
    if (out > K3D_LINEAR_MAX_OUT) return k3dx_bad("k3d_linear: out up to K3D_LINEAR_MAX_OUT");
    if ((long)T * out > K3D_LINEAR_MAX_RESULTS) return k3dx_bad("k3d_linear: T * out up to K3D_LINEAR_MAX_RESULTS");
    if (in < 64 && (long)T * out > 1L << 33) return k3dx_bad("k3d_linear: up to 2^33 results of rows under 64 columns");
    if (!y || !x || !W) return k3dx_bad("k3d_linear: y, x and W must be given");
    if (res == y && ldr != ldy) return k3dx_bad("k3d_linear: res in y's place needs y's stride");
    if (!aligned(y, type_size(y_type)) || !aligned(res, type_size(y_type)) || !aligned(x, type_size(x_type)) ||
        !aligned(W, 2) || !aligned(bias, 4))
        return k3dx_bad("k3d_linear: a pointer is not aligned to its elements");
    const size_t need = k3k_linear_ws(T, in, out, x_type);
    if (need && (!ws || ws_bytes < need)) return k3dx_bad("k3d_linear: workspace too small");
    if (need && !aligned(ws, 16)) return k3dx_bad("k3d_linear: the workspace must be 16-byte aligned");
    if (y == x || y == W || y == ws || (const void *)y == bias) return k3dx_bad("k3d_linear: y lies in an operand's place");
    K3kLinear a;
    a.y = y;
    a.x = x;
    a.res = res;
    a.W = W;
    a.bias = bias;
    a.ldy = ldy;
    a.ldx = ldx;
    a.ldw = ldw;
    a.ldr = ldr;
    a.y_type = y_type;
    a.x_type = x_type;
    a.T = T;
    a.in = in;
    a.out = out;
    a.act = act;
    a.ws = ws;
    a.ws_bytes = ws_bytes;
    k3k_prof_mark(stream, K3D_STAGE_BEGIN);
    if (k3k_linear(&a, stream)) return fail("k3d_linear");
    k3k_prof_mark(stream, K3D_STAGE_GEMV);
    return 0;
}

/* ---- routing from logits ----------------------------------------------------------------- */
int k3d_route(int *idx, float *wt, const void *logits, int type, long ld, int T, int n_experts, const float *bias,
              int score, int n_groups, int top_groups, int group_top, int topk, int renorm, float routed_scale,
              void *stream)
{
    if (!type_ok(type)) return k3dx_bad("k3d_route: type is K3D_F32 or K3D_BF16");
    if (score != K3D_SCORE_SIGMOID && score != K3D_SCORE_SOFTMAX) return k3dx_bad("k3d_route: unknown score");
    if (T < 0) return k3dx_bad("k3d_route: need T >= 0");
    if (n_experts < 1 || n_experts > 2048) return k3dx_bad("k3d_route: 1 to 2048 experts");
    if (n_groups < 1 || n_groups > 64 || n_experts % n_groups) return k3dx_bad("k3d_route: n_groups is 1 to 64 and divides n_experts");
    if (top_groups < 1 || top_groups > n_groups) return k3dx_bad("k3d_route: top_groups is 1 to n_groups");
    if (group_top != 1 && group_top != 2) return k3dx_bad("k3d_route: group_top is 1 or 2");
    if (topk < 1 || topk > K3_MAX_TOPK || topk > n_experts / n_groups * top_groups)
        return k3dx_bad("k3d_route: topk is 1 to 64 and at most the experts of top_groups groups");
    if (ld < n_experts) return k3dx_bad("k3d_route: ld is shorter than a row");
    if (T == 0) return 0;
    if (T > K3D_MAX_TOKENS) return k3dx_bad("k3d_route: up to K3D_MAX_TOKENS tokens");
    if (!idx || !wt || !logits) return k3dx_bad("k3d_route: idx, wt and logits must be given");
    if (!aligned(idx, 4) || !aligned(wt, 4) || !aligned(bias, 4) || !aligned(logits, type_size(type)))
        return k3dx_bad("k3d_route: a pointer is not aligned to its elements");
    K3kRoute a;
    a.idx = idx;
    a.wt = wt;
    a.logits = logits;
    a.bias = bias;
    a.ld = ld;
    a.type = type;
    a.T = T;
    a.n = n_experts;
    a.score = score;
    a.n_groups = n_groups;
    a.top_groups = top_groups;
    a.group_top = group_top;
    a.topk = topk;
    a.renorm = renorm && topk > 1;
    a.scale = routed_scale;
    k3k_prof_mark(stream, K3D_STAGE_BEGIN);
    if (k3k_route(&a, stream)) return fail("k3d_route");
    k3k_prof_mark(stream, K3D_STAGE_ROUTER);
    return 0;
}

/* ---- head norms and rotation --------------------------------------------------------------- */
int k3d_qk_norm_rope(void *qo, long ldqo, long hsqo, void *ko, long ldko, long hsko, const void *q, long ldq, long hsq,
                     const void *k, long ldk, long hsk, int type, int T, int hq, int hk, int dim, const float *qw,
                     const float *kw, float eps, const int *pos, const double *inv_freq, int rot, int rot_off,
                     int pairs, float rot_scale, void *stream)
{
    if (!type_ok(type)) return k3dx_bad("k3d_qk_norm_rope: type is K3D_F32 or K3D_BF16");
    if (pairs != K3D_ROT_HALVES && pairs != K3D_ROT_INTERLEAVED) return k3dx_bad("k3d_qk_norm_rope: unknown pairs");
    if (T < 0 || hq < 0 || hk < 0 || hq > 65536 || hk > 65536) return k3dx_bad("k3d_qk_norm_rope: need T >= 0 and 0 to 65536 heads");
    if (dim < 1 || dim > 1024) return k3dx_bad("k3d_qk_norm_rope: dim is 1 to 1024");
    if (rot < 0 || rot % 2 || rot_off < 0 || rot > dim || rot_off > dim - rot)
        return k3dx_bad("k3d_qk_norm_rope: rot is even and lies within the head");
    if (!(eps >= 0.0f)) return k3dx_bad("k3d_qk_norm_rope: eps >= 0");
    if (T == 0 || hq + hk == 0) return 0;
    if (T > K3D_MAX_TOKENS) return k3dx_bad("k3d_qk_norm_rope: up to K3D_MAX_TOKENS tokens");
    if (rot && (!pos || !inv_freq)) return k3dx_bad("k3d_qk_norm_rope: a rotation needs pos and inv_freq");
    if ((hq && (!q || !qo)) || (hk && (!k || !ko))) return k3dx_bad("k3d_qk_norm_rope: heads without their tensors");
    if (!aligned(pos, 4) || !aligned(inv_freq, 8) || !aligned(qw, 4) || !aligned(kw, 4)) return k3dx_bad("k3d_qk_norm_rope: a pointer is not aligned to its elements");
    K3kHeads a;
    a.v[0].out = qo;
    a.v[0].in = q;
    a.v[0].w = qw;
    a.v[0].ldo = ldqo;
    a.v[0].hso = hsqo;
    a.v[0].ld = ldq;
    a.v[0].hs = hsq;
    a.v[0].heads = hq;
    a.v[1].out = ko;
    a.v[1].in = k;
    a.v[1].w = kw;
    a.v[1].ldo = ldko;
    a.v[1].hso = hsko;
    a.v[1].ld = ldk;
    a.v[1].hs = hsk;
    a.v[1].heads = hk;
    for (int i = 0; i < 2; i++) {
        if (!a.v[i].heads) continue;
        if (!aligned(a.v[i].in, type_size(type)) || !aligned(a.v[i].out, type_size(type)))
            return k3dx_bad("k3d_qk_norm_rope: a pointer is not aligned to its elements");
        /* (heads of one token may lie at any distance from each other, but not in each other; token-major or head-major) */
        if (a.v[i].heads > 1 && (a.v[i].hs < dim || a.v[i].hso < dim)) return k3dx_bad("k3d_qk_norm_rope: heads overlap");
        if (T > 1 && (a.v[i].ld < dim || a.v[i].ldo < dim)) return k3dx_bad("k3d_qk_norm_rope: tokens overlap");
        if (a.v[i].in == a.v[i].out && ((T > 1 && a.v[i].ld != a.v[i].ldo) || (a.v[i].heads > 1 && a.v[i].hs != a.v[i].hso)))
            return k3dx_bad("k3d_qk_norm_rope: in place needs the same strides");
        if (a.v[i].heads > 1 && T > 1) {                       /* of two writes to one place either could come last */
            const unsigned __int128 ld = a.v[i].ldo, hs = a.v[i].hso;
            if (ld < hs * (unsigned)(a.v[i].heads - 1) + (unsigned)dim && hs < ld * (unsigned)(T - 1) + (unsigned)dim)
                return k3dx_bad("k3d_qk_norm_rope: the outputs of a token and of a head overlap");
        }
    }
    if (hq && hk && qo == ko) return k3dx_bad("k3d_qk_norm_rope: qo and ko are one place");
    a.type = type;
    a.T = T;
    a.dim = dim;
    a.rot = rot;
    a.rot_off = rot_off;
    a.pairs = pairs;
    a.eps = eps;
    a.rot_scale = rot_scale;
    a.pos = pos;
    a.freq = inv_freq;
    if (k3k_heads(&a, stream)) return fail("k3d_qk_norm_rope");
    return 0;
}
