/* SPDX-License-Identifier: Apache-2.0 */
/*
 * k3_dev.h -- device-pointer entry points of libk3amd.so.
 *
 * The reference has no device: its kernels take host buffers (include/k3/k3.h). These
 * entry points are the same operations for callers whose activations and weights are
 * already resident in HBM (a serving loop, the benchmark): every pointer is a DEVICE
 * pointer, work is enqueued on the caller's HIP stream (NULL = the null stream) and the
 * call returns without synchronising. None of them allocates: scratch comes from a
 * caller-provided workspace of the size the matching *_ws() function reports, which also
 * serves any smaller batch of the same widths. They
 * return 0, or a negative value with a message available from k3d_error() (kept per host
 * thread).
 *
 * Work that runs beside the caller's (the activation split beside the router, the hot
 * experts' passes of a skewed prefill batch) goes to a side stream that belongs to the
 * caller's stream, forked from it and joined back into it by events of its own; so calls
 * from several host threads on different streams, at once, never share a stream or an
 * event, and each gives the result it gives alone. A stream's side stream is made by
 * k3d_stream_create (the null stream's by k3d_init), or by the first call on a stream made
 * elsewhere; at most 256 caller streams at once have one (k3d_stream_create then fails, and on
 * a stream made elsewhere everything runs on the stream itself). Calls that overlap on one
 * stream, or share a workspace, race.
 *
 * Each names the reference function whose arithmetic it performs.
 */
#ifndef K3_DEV_H
#define K3_DEV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Selects the device and uploads the router's tables once; after it, no entry point below
 * allocates or synchronises (except k3d_malloc/free/sync and the copies). */
int k3d_init(void);
const char *k3d_error(void);
void *k3d_malloc(size_t bytes);
int k3d_free(void *p);
int k3d_h2d(void *dst, const void *src, size_t bytes, void *stream);
int k3d_d2h(void *dst, const void *src, size_t bytes, void *stream);
int k3d_sync(void *stream);

/* Streams (default priority) and HIP graphs: k3d_graph_begin/end capture everything the
 * k3d_* calls enqueue on a created stream between them (no allocation or synchronisation
 * happens inside those calls); k3d_graph_launch replays it with one launch. The captured
 * pointers are baked in: replay with the same buffers, new contents. */
void *k3d_stream_create(void);
int k3d_stream_destroy(void *stream);
int k3d_graph_begin(void *stream);
int k3d_graph_end(void *stream, void **exec);
int k3d_graph_launch(void *exec, void *stream);
int k3d_graph_destroy(void *exec);

/* Stage profiler (HIP events). Between k3d_prof_begin and k3d_prof_end, the MoE and GEMV
 * entry points record an event at each stage boundary; k3d_prof_end synchronises and
 * returns, per stage, the summed milliseconds and the number of samples. Stage ids: */
enum { K3D_STAGE_BEGIN = 0, K3D_STAGE_ROUTER = 1, K3D_STAGE_GATHER = 2, K3D_STAGE_GATEUP = 3,
       K3D_STAGE_DOWN = 4, K3D_STAGE_COMBINE = 5, K3D_STAGE_GEMV = 6, K3D_STAGE_SHARED = 7,
       K3D_STAGE_COUNT = 8 };
/* Per-workgroup stamps of the batched expert kernels (mx_moe_kernel, mx_prefill_kernel), a
 * profiling aid beside the stage profiler: between k3d_stamps_begin and k3d_stamps_end, each
 * launch of those kernels writes, for each of its workgroups, three u64 into the device
 * buffer dbuf, launch after launch: the workgroup's start and end on the 100 MHz clock and
 * the hardware id it ran on (XCC id << 32 | the HW_ID register: CU in bits 8-11, shader
 * array 12, shader engine 13-15). Launches that no longer fit are not stamped. k3d_stamps_end
 * gives the kinds (K3D_STAMP_*) and grids of the stamped launches in order (up to max; *n =
 * their number) and stops stamping. Not for graph capture: the buffer region is chosen when a
 * call enqueues its work. */
enum { K3D_STAMP_MOE_GATEUP = 1, K3D_STAMP_MOE_DOWN = 2, K3D_STAMP_PREFILL_GATEUP = 3,
       K3D_STAMP_PREFILL_DOWN = 4 };
int k3d_stamps_begin(void *dbuf, size_t bytes);
int k3d_stamps_end(int *kinds, int *grids, int max, int *n);
int k3d_prof_begin(int max_marks);
int k3d_prof_mark(void *stream, int stage);
int k3d_prof_end(double *ms, int *count, int n_stages);

/* Y[ntok][rows] = X[ntok][in] . W^T, W packed MXFP4 with group 32, in % 32 == 0.
 * prec 0: fp32-accurate (activations split into two bf16 terms), prec 1: activations
 * rounded to bf16. Arithmetic of k3_matmul_mxfp4 (reference k3_ops.c:1380-1785). */
size_t k3d_matmul_mxfp4_ws(int ntok, int in);
int k3d_matmul_mxfp4(float *y, const float *x, int ntok, const uint8_t *packed,
                     const uint8_t *scales, int in, int rows, int prec, void *ws,
                     size_t ws_bytes, void *stream);

/* Y[ntok][out] = X[ntok][in] . W^T for fp32 / bf16 weights (reference k3_ops.c:265-291,
 * 1108-1213), fp32-accurate. One token: bf16 weights give the bits of fp32 weights of the same
 * values. Two and more run on the matrix cores: there the two agree within rounding, and a token's
 * result depends in its last bits on the number of tokens. */
int k3d_matmul_f32(float *y, const float *x, int ntok, const float *W, int in, int out,
                   void *stream);
int k3d_matmul_bf16(float *y, const float *x, int ntok, const uint16_t *W, int in, int out,
                    void *stream);

/* Router over T tokens: idx/wt [T][topk] (reference k3_ops.c:419-478, per token).
 * n_experts 1..2048 (the selection holds every expert's record in one workgroup's LDS);
 * more returns an error. */
size_t k3d_router_ws(int T, int hidden, int n_experts);
int k3d_router(int *idx, float *wt, const float *x, int T, const float *W, const float *bias,
               int hidden, int n_experts, int topk, int renorm, float routed_scale, void *ws,
               size_t ws_bytes, void *stream);

/* Device layouts of an expert bank's MXFP4 matrices.
 *   K3D_LAYOUT_ROWS:  the reference's, packed [rows][in/2] + scales [rows][in/32] bytes.
 *   K3D_LAYOUT_TILED: the same bytes regrouped per tile of 16 rows x 512 columns in the
 *     order the expert kernel reads them (k3d_mxfp4_tile), the four tiles of each group of
 *     64 rows side by side chunk after chunk; rows are padded to a multiple of 64, in must
 *     be a multiple of 512. A block with scale byte 255 (NaN; zero in the reference) is
 *     stored as zero codes with scale byte 127. Same arithmetic, results bit-identical to
 *     ROWS; the expert kernel streams it at a higher fraction of HBM bandwidth. */
enum { K3D_LAYOUT_ROWS = 0, K3D_LAYOUT_TILED = 1 };
int k3d_mxfp4_tiled_size(int rows, int in, size_t *packed_bytes, size_t *scales_bytes);
int k3d_mxfp4_tile(uint8_t *tpacked, uint8_t *tscales, const uint8_t *packed,
                   const uint8_t *scales, int rows, int in, void *stream);

/* Diagnostics of the last k3d_router call that used workspace `ws` (after the device has
 * finished it; synchronises): h_counts[t] = number of token t's logits whose fp32 rounding
 * the split fp64 sum could not certify and that were recomputed with the reference's
 * sequential chain. */
int k3d_router_recomputed(int *h_counts, const void *ws, int T, int hidden, int n_experts);
/* The chunk partials of the same call (more than four tokens; synchronises): *h_chunk = the
 * chunk width, h_part / h_rbound [ks][T][n_experts] (ks = ceil(hidden / chunk), at most
 * `cap` entries each) the chunk sums P_k and the bounds R_k, |P_k - exact| <= 2^-53 R_k and
 * R_k >= the sum of |the chunk's exact prefix sums|, that the certification uses. Returns
 * ks, or -1. */
int k3d_router_partials(double *h_part, float *h_rbound, int *h_chunk, size_t cap, const void *ws, int T,
                        int hidden, int n_experts);

/* The routed MoE layer (k3_moe's routed loop, reference k3_ops.c:576-643, with z := x),
 * expert-major. bank is a DEVICE array of n_experts K3ExpertQ (k3.h) whose pointers are
 * device pointers, in the given layout; an entry with a NULL pointer is a dropped expert.
 * hidden and inter: multiples of 32 (ROWS) or of 512 (TILED). perm_out (T*topk) and
 * offsets_out (n_experts+1), when not NULL, receive the gather permutation. *drops_out,
 * when not NULL, receives (after the stream reaches it) the number of dropped
 * assignments; it must be a device int. */
size_t k3d_moe_ws(int T, int hidden, int inter, int n_experts, int topk, int prec);
int k3d_moe_routed(float *out, int *idx, float *wt, const float *x, int T,
                   const float *router_w, const float *bias, const void *bank, int layout,
                   int hidden, int inter, int n_experts, int topk, int renorm, float routed_scale,
                   int act, float b1, float b2, int prec, void *ws, size_t ws_bytes,
                   int *perm_out, int *offsets_out, int *drops_out, void *stream);

/* k3d_moe_routed with no workspace argument and no allocation, for callers that cannot
 * allocate (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc). No counterpart in the reference. The scratch lives in a static device array
 * of K3D_STATIC_WS_BYTES (40 MiB) that each GPU holds until the process ends: enough for
 * decode batches of up to 64 tokens at hidden 7168 / inter 2048 / 384 experts / top-8 or
 * at 3584 / 3072 / 896 / top-16 (what the call itself takes must not exceed it, which can be less
 * than k3d_moe_ws, sized for any smaller batch too; larger calls return an error). k3d_init must have run on the device first (it looks the array up and
 * makes the one-time uploads). All calls on one GPU share the array: calls that overlap
 * on one GPU race. Otherwise identical to k3d_moe_routed, results bit for bit. */
#define K3D_STATIC_WS_BYTES ((size_t)40 << 20)
size_t k3d_static_ws_bytes(void);
int k3d_moe_routed_static(float *out, int *idx, float *wt, const float *x, int T,
                          const float *router_w, const float *bias, const void *bank, int layout,
                          int hidden, int inter, int n_experts, int topk, int renorm,
                          float routed_scale, int act, float b1, float b2, int prec, int *perm_out,
                          int *offsets_out, int *drops_out, void *stream);

/* The always-on dense shared expert with bf16 weights, on the matrix cores:
 *   s[t] = W2 . act(W1 x[t], W3 x[t]),  W1, W3 [inter][hidden], W2 [hidden][inter] bf16,
 * y = s (accumulate 0) or y += s (accumulate 1, after the routed sum: the order of the
 * reference's shared tail, k3_ops.c:650-654). The reference computes each product with
 * k3_matmul_bf16 (fp64 accumulation); here fp32 MFMA accumulation in the library's own
 * bf16 GEMM kernels (gate and up in one pass with the activation in the epilogue, then
 * down) with the activations as two bf16 terms (prec 0, max|err| <= 1e-4 ||ref||inf) or
 * one (prec 1, 2e-2 relative). hidden and inter must be multiples of 64. Nothing is
 * allocated and no library is initialised, so the call can be captured in a HIP graph. */
size_t k3d_shared_ws(int T, int hidden, int inter, int prec);
int k3d_shared_expert(float *y, int accumulate, const float *x, int T, const uint16_t *w1,
                      const uint16_t *w3, const uint16_t *w2, int hidden, int inter, int act,
                      float b1, float b2, int prec, void *ws, size_t ws_bytes, void *stream);

/* The expert half of the layer for a routing already in idx/wt (device). Slots whose
 * expert index lies outside [0, n_experts), or whose bank entry has a NULL pointer,
 * contribute nothing; drops_out counts the latter. */
int k3d_moe_experts(float *out, const int *idx, const float *wt, const float *x, int T,
                    const void *bank, int layout, int hidden, int inter, int n_experts, int topk,
                    int act, float b1, float b2, int prec, void *ws, size_t ws_bytes,
                    int *perm_out, int *offsets_out, int *drops_out, void *stream);

/* ---- the operators of the layer around the routed experts -------------------------------
 * No counterpart in the reference as single calls. Strides are in elements; nothing is allocated,
 * nothing synchronises, and the calls can be captured in a HIP graph. The stream and the tensors
 * belong to the current device. Up to K3D_MAX_TOKENS tokens in a call. */
#define K3D_MAX_TOKENS (1 << 24)

/* Element types of the tensors below. */
enum { K3D_F32 = 0, K3D_BF16 = 1 };

/* Dense product with bias, activation and residual:
 *   y[t][o] = act(sum_k x[t][k] W[o][k] + bias[o]) + res[t][o],   t < T, o < out, k < in.
 * W bf16 [out][ldw], x [T][ldx] of x_type, bias fp32 [out] or NULL, res [T][ldr] of y_type or NULL
 * (it may be y itself, with its stride), y [T][ldy] of y_type; rows and pointers at any alignment of
 * their elements. fp32 x counts in full: cut into three bf16 terms that hold all 24 bits of it,
 * down to bf16's least step of 2^-133 (an infinite weight then gives NaN where it meets a finite x). Sums, bias, activation and
 * residual are formed in fp32 and rounded once to y_type; silu is within 8 * 2^-24 of its value under either type, gelu_tanh
 * within 6 |z| 2^-24 more, z = 1.6 v (1 + .045 v^2), which z's own roundings cost; gelu within 18 * 2^-24 of its value
 * (for bf16 10 * 2^-24 |v|, and where v < 0 (18 + 1.5 v^2) 2^-24 of its value, before that rounding). Which kernel runs, and with it the order
 * of a sum, goes by the shape, the types and the alignment; a call's bits repeat. ldx and ldw up to
 * K3D_LINEAR_MAX_LD, in up to K3D_LINEAR_MAX_IN, out up to K3D_LINEAR_MAX_OUT, T * out up to
 * K3D_LINEAR_MAX_RESULTS, 2^33 where in is under 64. y must not overlap x, W, bias or ws, nor res unless it is y itself. ws
 * (k3d_linear_ws bytes, which hold any fewer tokens too; 16-byte aligned) is scratch of one call: calls
 * and graphs that may run at the same time need one each. */
enum { K3D_ACT_NONE = 0, K3D_ACT_RELU = 1, K3D_ACT_SILU = 2, K3D_ACT_GELU = 3 /* erf */, K3D_ACT_GELU_TANH = 4 };
#define K3D_LINEAR_MAX_LD (1 << 22)
#define K3D_LINEAR_MAX_IN (1 << 20)
#define K3D_LINEAR_MAX_OUT (1 << 28)
#define K3D_LINEAR_MAX_RESULTS (1L << 37)
size_t k3d_linear_ws(int T, int in, int out, int x_type);
int k3d_linear(void *y, int y_type, long ldy, const void *x, int x_type, long ldx, int T, const uint16_t *W,
               long ldw, int in, int out, const float *bias, int act, const void *res, long ldr, void *ws,
               size_t ws_bytes, void *stream);

/* Routing from logits [T][ld] (of `type`; k3d_linear's, say): idx/wt [T][topk], the form that
 * k3d_moe_experts takes. Per token:
 *   score[e]  = sigmoid(logit) (K3D_SCORE_SIGMOID) or softmax over the token's experts (K3D_SCORE_SOFTMAX);
 *   choice[e] = score[e] + bias[e] (bias fp32 [n_experts] or NULL);
 *   groups    : n_groups runs of n_experts / n_groups experts; a group's value is the sum of its
 *               group_top (1 or 2) largest choices; the top_groups groups of largest value stay;
 *   idx       : the topk largest choices among them, descending; wt their scores, divided by their
 *               sum if renorm and topk > 1 (as k3_router does), times routed_scale.
 * Equal values go to the lower index, of groups and of experts. Scores, choices, sums and
 * comparisons are formed in 64 bits, wt is rounded once. A logit of -inf or NaN, or a choice of -inf or
 * NaN, is an expert that cannot be taken (a masked one; a NaN logit is left out of the softmax too); a
 * group has the value of those it can give, and one without any is never taken; where fewer than topk
 * are left, the last slots get idx -1 and wt 0 (k3d_moe_experts skips them), and weights
 * that sum to 0 are 0. (-inf masks an expert at no cost; a large finite bias is as right, but every choice of a token that has one is
 * formed in 64 bits, which takes three times as long.) Logits of +inf share a softmax among themselves.
 * 1 <= n_experts <= 2048, n_groups <= 64 and a divisor of it, topk <= 64 and at most the experts of
 * top_groups groups. */
enum { K3D_SCORE_SIGMOID = 0, K3D_SCORE_SOFTMAX = 1 };
int k3d_route(int *idx, float *wt, const void *logits, int type, long ld, int T, int n_experts, const float *bias,
              int score, int n_groups, int top_groups, int group_top, int topk, int renorm, float routed_scale,
              void *stream);

/* RMSNorm of every query and key head, and the position rotation behind it. Head h of token t
 * is the `dim` elements at q + t * ldq + h * hsq (k likewise); it goes to qo / ko in the same form,
 * which may be the input itself (same pointer and strides), else must overlap neither q nor k; qo and
 * ko are apart. Outputs lie token by token (ldqo >= (hq - 1) * hsqo + dim) or head by head (hsqo >= (T - 1) * ldqo + dim).
 *   u = v / sqrt(mean(v^2) + eps) * w     (w: qw or kw, fp32 [dim], or NULL for ones)
 *   rotated over u[rot_off .. rot_off + rot): the pairs (i, i + rot/2) (K3D_ROT_HALVES) or
 *   (2i, 2i + 1) (K3D_ROT_INTERLEAVED) turn by the angle pos[t] * inv_freq[i], i < rot/2, and are
 *   multiplied by rot_scale; the rest of u stays as it is.
 * Angles are formed and reduced in 64 bits (inv_freq fp64), so far positions lose nothing; the rest is fp32,
 * rounded once (the squares too: a head whose sum of them passes fp32's range, values of 10^18 and more, becomes 0). A token of negative position is padding: its rows of qo and ko are left as they were.
 * hq or hk may be 0. 1 <= dim <= 1024; rot even (0: no rotation, pos may then be NULL: no padding);
 * eps >= 0. */
enum { K3D_ROT_HALVES = 0, K3D_ROT_INTERLEAVED = 1 };
int k3d_qk_norm_rope(void *qo, long ldqo, long hsqo, void *ko, long ldko, long hsko, const void *q, long ldq, long hsq,
                     const void *k, long ldk, long hsk, int type, int T, int hq, int hk, int dim, const float *qw,
                     const float *kw, float eps, const int *pos, const double *inv_freq, int rot, int rot_off,
                     int pairs, float rot_scale, void *stream);

/* ---- a layer's path in 8 bits -------------------------------------------------------------
 * No counterpart in the reference. Activations: rows of OCP e4m3 codes, one fp32 scale for each 128 columns of a row; a
 * value is code * scale. A row holds whole blocks: ceil(n / 128) * 128 codes, those behind column n the code of 0 (the entry
 * points that write rows write them so); rows and pointers of codes 16-byte aligned. Weights: e4m3 codes laid out once by k3d_f8_tile, one fp32
 * scale for each block of 128 rows x 128 columns. Strides are in elements; nothing is allocated, nothing synchronises, the calls can be captured
 * in a HIP graph. The stream and the tensors belong to the current device. Outputs and workspaces overlap no operand and no other output, but where it is said. */
#define K3D_NORM_MAX_N (1 << 16)
#define K3D_F8_MAX_IN (1 << 20)
#define K3D_F8_MAX_OUT (1 << 18)
#define K3D_F8_MAX_LD (1 << 22)
#define K3D_F8_MAX_RESULTS (1L << 37)
#define K3D_F8_MAX_SLOTS (1 << 24)
#define K3D_F8_MAX_X (1L << 31)

/* The gated activations act(gate) * up: K3D_GLU_SILU silu(gate) * up; K3D_GLU_SITU b1 tanh(gate / b1) sigmoid(gate) * b2 tanh(up / b2), as
 * K3_ACT_SITU of k3.h. */
enum { K3D_GLU_NONE = -1, K3D_GLU_SITU = 0, K3D_GLU_SILU = 1 };

/* Residual and RMSNorm, into 8 bits and / or y, t < T, i < n <= K3D_NORM_MAX_N:
 *   v = x[t][i] + res[t][i] (res may be NULL);  sum = v, rounded to r_type (sum may be NULL);
 *   u = v / sqrt(mean_i(v^2) + eps) * w[i]  (w fp32 or NULL for ones);  y = u, rounded to y_type (y may be NULL);
 *   q, qs (may be NULL): scale = max(max |u| over 128 columns, 2^-100) / 448, code = u / scale to nearest, ties to even.
 * All in fp32, v unrounded (the squares too: a row whose sum of them passes fp32's range becomes 0, and squares under 2^-126 lose bits, which an eps of 1e-37 or less
 * does not hide: such a row's u is inexact, and NaN where all of them vanish beside an eps of 0, as of a row of zeros). x is of x_type, res and sum of r_type; res, sum and y at any alignment of
 * their elements. sum may be res or x itself, y too (same type and stride). A NaN in a block of u makes its scale and codes NaN; an infinity the scale infinite. */
int k3d_add_norm(void *y, int y_type, long ldy, uint8_t *q, long ldq, float *qs, long ldqs, void *sum, long ldsum,
                 const void *x, int x_type, long ldx, const void *res, int r_type, long ldr, int T, int n, const float *w,
                 float eps, void *stream);

/* The rows of x in 8 bits (act K3D_GLU_NONE), or of act(gate) * up: row t of x is gate [n], then up [n]. Scales and codes as above;
 * the activation in fp32; behind one a code is the nearest to u times the scale's rounded reciprocal, within 2^-23 of u / scale. b1, b2 from 2^-64 to 2^64 for K3D_GLU_SITU. */
int k3d_quant_f8(uint8_t *q, long ldq, float *qs, long ldqs, const void *x, int x_type, long ldx, int T, int n, int act,
                 float b1, float b2, void *stream);

/* The layout of weights: mats matrices of e4m3 codes [rows][ldw] one after another (rows * ldw apart) into k3d_f8_tiled_bytes(rows, in) bytes
 * each, one after another; t 16-byte aligned, W at any alignment. Tiles of 16 rows x 128 columns in the order the
 * kernels read them; rows up to a multiple of 128 and columns up to whole blocks are there as zeros. */
size_t k3d_f8_tiled_bytes(int rows, int in);
int k3d_f8_tile(uint8_t *t, const uint8_t *W, long ldw, int rows, int in, int mats, void *stream);

/* Dense product, t < T, o < out:
 *   y[t][o] = act(sum_b xs[t][b] Ws[o / 128][b] p[t][o][b] + bias[o]) + res[t][o],
 * p the sum over block b's 128 columns of the codes' products. x [T][ldx] codes with scales xs [T][ldxs];
 * W from k3d_f8_tile, Ws [ceil(out / 128)][ldws]; bias, act, res and y as k3d_linear has them. For y of K3D_F32 p is formed with fp32 products and
 * sums; for K3D_BF16 by 8-bit matrix instructions, which align each 8 neighbouring products to the largest of them and cut 13 bits below it (1.5 * 2^-16 of a
 * sum of random products, a 70th of what y's own rounding adds) and take half the time. The two scales' product is formed
 * in fp32, as are the sum over blocks, bias, activation and residual; one rounding to y_type. Which kernel runs, and with it the order of the
 * sum over blocks, goes by the shape; a call's bits repeat. ws (k3d_linear_f8_ws bytes, which hold any fewer tokens too, none up to 64; 16-byte aligned) is
 * scratch of one call: calls and graphs that may run at the same time need one each. y must not overlap an operand, nor res unless
 * it is y itself. */
size_t k3d_linear_f8_ws(int T, int in, int out);
int k3d_linear_f8(void *y, int y_type, long ldy, const uint8_t *x, long ldx, const float *xs, long ldxs, int T,
                  const uint8_t *W, const float *Ws, long ldws, int in, int out, const float *bias, int act,
                  const void *res, long ldr, void *ws, size_t ws_bytes, void *stream);

/* A routing's slots by expert: offsets [n_experts + 1], perm [T * topk]: perm[offsets[e] .. offsets[e + 1]) are the slots t * topk + j with
 * idx[t][j] == e, ascending. Slots whose idx lies outside [0, n_experts) are in none, and perm behind offsets[n_experts] is left
 * as it was. n_experts up to 2048, topk up to 64, T * topk up to K3D_F8_MAX_SLOTS. ws (k3d_group_ws bytes, none up to 4096 slots) is scratch of one call. */
size_t k3d_group_ws(int T, int topk, int n_experts);
int k3d_group(int *offsets, int *perm, const int *idx, int T, int topk, int n_experts, void *ws, size_t ws_bytes, void *stream);

/* Products by expert: rows offsets[e] <= r < offsets[e + 1] (device; `rows` is what offsets[n_experts] is at most) with expert e's weights,
 *   y[Y(r)][o] = sum_b xs[X(r)][b] Ws[e][o / 128][b] p[..],  X(r) = x_rows ? x_rows[r] / x_div : r,  Y(r) = y_rows ? y_rows[r] : r.
 * with p as in k3d_linear_f8, by y_type too. W: n_experts matrices [out][in] from k3d_f8_tile, Ws [n_experts][ceil(out / 128)][ceil(in / 128)]. With k3d_group's perm as x_rows and x_div = topk a
 * row takes its token of x; as y_rows it returns to its slot. x has x_cap rows, y y_cap; a row with X(r) or Y(r) outside them is left as it was,
 * and so is every row of y that no r has. No Y(r) may come twice. Experts without rows cost nothing; an expert's end past `rows` counts as `rows`, and one whose offsets fall,
 * or begin below 0, has none. */
int k3d_grouped_f8(void *y, int y_type, long ldy, const int *y_rows, int y_cap, const uint8_t *x, long ldx, const float *xs,
                   long ldxs, const int *x_rows, int x_div, int x_cap, const int *offsets, int rows, int n_experts,
                   const uint8_t *W, const float *Ws, int in, int out, void *stream);

/* The experts' layer for a routing in idx/wt [T][topk] (k3d_route's), weights in 8 bits: out[t] = sum_j wt[t][j] W2_e (act(W1_e x[t]) * (W3_e x[t])),
 * e = idx[t][j], act and b1, b2 as in k3d_quant_f8. The gated activation goes through 8 bits as k3d_quant_f8 rounds it. With out_type K3D_F32 every product is
 * formed as k3d_linear_f8's of fp32 are. With K3D_BF16 the down products are formed by 8-bit instructions, as k3d_linear_f8's of bf16 are, and so are gate and up where the experts have more than
 * about 10 rows each (16 of hidden >= 4096): some of their codes fall a step aside there, 1.1e-3 of the result beside the 1.7e-3 of its rounding; and many tokens' down products
 * wait for their sum as 16-bit floats with a power of two for each 64 columns (within 2^-11 of the value, or 2^-39 of the largest of them). The weighted sum
 * is fp32, rounded once to out_type. Slots whose idx lies outside [0, n_experts) contribute nothing; a token without any becomes 0. w1, w3 [n_experts] matrices [inter][hidden], w2
 * [hidden][inter] from k3d_f8_tile, s1, s3, s2 their scales as in k3d_grouped_f8. ws (k3d_moe_f8_ws bytes; 16-byte aligned) is scratch of one call. */
size_t k3d_moe_f8_ws(int T, int hidden, int inter, int n_experts, int topk);
int k3d_moe_f8(void *out, int out_type, long ldo, const int *idx, const float *wt, const uint8_t *x, long ldx, const float *xs,
               long ldxs, int T, const uint8_t *w1, const float *s1, const uint8_t *w3, const float *s3, const uint8_t *w2,
               const float *s2, int hidden, int inter, int n_experts, int topk, int act, float b1, float b2, void *ws,
               size_t ws_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
