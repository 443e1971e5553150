/*
 * hoard_ops.h -- C ABI of the operators around the MI355X expert stage.
 *
 * What a layer runs next to the stage of hoard_moe.h: the norms before and
 * after its block with the block's gate and the residual, the (token, slot)
 * pairs sorted by expert and back (with gradients), and products with 4-bit
 * weights and group scales (projections, and experts that come as such codes
 * rather than as GGUF K-quants).
 *
 * As in hoard_moe.h every call is extern "C", returns 0 or a negative
 * HOARD_ERR_* code (hoard_last_error() then describes it), throws nothing and
 * takes the hipStream_t to run on as a void*.  There is no handle: a call keeps
 * nothing from one call to the next, allocates nothing and only launches
 * kernels, so it can be captured into a graph, and calls on different streams
 * are independent as long as their outputs and workspaces are.  The current
 * device must be the stream's, and every pointer without "host" in its
 * description is device memory of it.
 *
 * Arrays are dense, rows one after the other.  An activation type is
 * HOARD_TYPE_F32, _F16 or _BF16; sums are formed in 32 bits and rounded once
 * when stored.  A row count of zero is valid: there is nothing to write but sums
 * over the rows, which are 0.  Outputs must not overlap inputs or each other
 * except where said.
 */
#ifndef HOARD_OPS_H
#define HOARD_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "hoard_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* further ggml type ids (ggml.h enum ggml_type), for activations and scales */
#define HOARD_TYPE_F16 1
#define HOARD_TYPE_BF16 30

/* ---- products with 4-bit weights ------------------------------------------ */

/* n_mat matrices of rows x cols weights, row r of matrix e at index e*rows + r:
   weight k = scale[k / group] * (code[k] - zero[k / group]), zero 8 without
   zeros.  rows is at most 2^22, n_mat 2^30; cols is a multiple of group, at most 2^20. */
typedef struct hoard_q4_matrix {
    const void *codes;    /* [n_mat*rows][cols/2] bytes, 16-byte aligned: byte j holds code 2j in
                             its low half and code 2j+1 in its high half */
    const void *scales;   /* [n_mat*rows][cols/group] of scale_type */
    const uint8_t *zeros; /* [n_mat*rows][cols/group] zero points, any byte; or NULL */
    int32_t rows, cols;
    int32_t group;        /* 32, 64 or 128 */
    int32_t n_mat;
    int32_t scale_type;   /* HOARD_TYPE_F32, _F16 or _BF16 */
} hoard_q4_matrix;

/* y[r] = W x[r] for n_rows rows: x [n_rows][cols] and y [n_rows][rows] of `type`,
   x 16-byte aligned.  With `up` (same rows, cols, group and n_mat; its zeros and
   scale type may differ) y[r] = silu(W x[r]) * (W_up x[r]).  W has n_mat 1.  The
   products are formed with the activations as given, not quantised; fp32 ones are
   held, for more than one row and by offsets, to 2^-23 of a value or to 2^-39 of its
   group's largest.  A group's sum is formed before its scale, in 16 bits also of codes
   with an offset of up to 16 that is then corrected, so it overflows where the sum of
   |x| over the group reaches 2^119.  A row of x that holds an infinity or a NaN gives a
   row of y without a defined value (infinities and NaN); other rows are not touched by
   it. */
int hoard_q4_matmul(const hoard_q4_matrix *w, const hoard_q4_matrix *up, int type, int n_rows, const void *x,
                    void *y, void *stream);

/* Every row by the matrix its id names: y[r] = W[ids[r]] x[r / x_share], x
   [n_rows / x_share][cols] (x_share divides n_rows): a token's row shared by its
   x_share chosen experts, or 1.  ids[n_rows] int32; a row whose id lies outside
   [0, n_mat) is NaN.  The form for one token or a few: every row reads its
   matrix. */
int hoard_q4_matmul_ids(const hoard_q4_matrix *w, const hoard_q4_matrix *up, int type, int n_rows, const void *x,
                        int x_share, const int32_t *ids, void *y, void *stream);

/* Rows sorted by matrix: rows offsets[e] .. offsets[e+1]-1 take matrix e, as
   hoard_sort_pairs writes offsets[n_mat + 1] (ascending; read as if clamped to
   [0, n_rows]).  Rows of y outside every range are left as they are. */
int hoard_q4_matmul_sorted(const hoard_q4_matrix *w, const hoard_q4_matrix *up, int type, int n_rows, const void *x,
                           const int32_t *offsets, void *y, void *stream);

/* ---- pairs sorted by expert, and back -------------------------------------- */

/* The n_tokens * k pairs (t, j), numbered p = t*k + j, sorted by their expert
   ids[p], pairs of one expert in the order of p.  place[p]: the sorted row of
   pair p; order[row]: the pair at it; offsets[e] .. offsets[e+1]-1: the rows of
   expert e.  A pair whose id lies outside [0, n_expert) is dropped: its place is
   -1, and order is -1 in the rows from offsets[n_expert] on.  An id may repeat
   within a token.  1 <= k <= 64, 1 <= n_expert <= 1024, n_tokens * k < 2^31.
   workspace: hoard_sort_workspace's bytes (possibly 0), 4-byte aligned, used by
   the call alone while it runs. */
int hoard_sort_pairs(int n_tokens, int k, int n_expert, const int32_t *ids, int32_t *place, int32_t *order,
                     int32_t *offsets, void *workspace, size_t workspace_bytes, void *stream);
int hoard_sort_workspace(int n_tokens, int k, int n_expert, size_t *bytes);

/* xs[place[t][j]] = w[t][j] * x[t] (w NULL: 1): the tokens' rows [n_tokens][n]
   laid out by sorted row, xs [n_tokens*k][n], 1 <= n <= 2^30.  In these calls a place outside
   [0, n_tokens*k) drops its pair, and the places that are not dropped must be
   distinct; rows of xs that no pair names are left as they are. */
int hoard_sort_gather(int type, int n_tokens, int k, int n, const void *x, const int32_t *place, const float *w,
                      void *xs, void *stream);

/* out[t] = res[t] + sum_j w[t][j] * y[place[t][j]], j ascending (w NULL: 1, the
   gradient of hoard_sort_gather without weights; res NULL: 0).  y [n_tokens*k][n],
   res and out [n_tokens][n] of `type`, w [n_tokens][k] f32.  A dropped pair adds
   nothing.  out may be res. */
int hoard_sort_combine(int type, int n_tokens, int k, int n, const void *y, const int32_t *place, const float *w,
                       const void *res, void *out, void *stream);

/* Gradients of hoard_sort_combine given dout [n_tokens][n] (that of res is dout
   itself): dy[place[t][j]] = w[t][j] * dout[t] and dw[t][j] = <dout[t],
   y[place[t][j]]>; dw is 0 for a dropped pair, and rows of dy that no pair names
   are left as they are.  dy may be NULL (not wanted), or y. */
int hoard_sort_combine_grad(int type, int n_tokens, int k, int n, const void *dout, const void *y,
                            const int32_t *place, const float *w, void *dy, float *dw, void *stream);

/* ---- norms around a block --------------------------------------------------- */

#define HOARD_GATE_NONE 0
#define HOARD_GATE_CHANNEL 1 /* gate f32 [n] */
#define HOARD_GATE_TOKEN 2   /* gate f32 [n_rows] */
#define HOARD_GATE_FULL 3    /* gate of `type`, [n_rows][n] */

/* Between two blocks, for every row of n values:

     c     = b * rho_b * (w_offset + w_post)        (w_post NULL: c = b)
     v     = r + scale * gate * c                   (b NULL: v = r, nothing is written to r_out)
     r_out = v                                      rounded to res_type
     h     = v * rho_v * (w_offset + w_pre)         of v as stored; h NULL: not wanted

   rho_x = 1 / sqrt(mean(x^2) + eps).  r is the residual stream, b the output of
   the block before, h the input of the block after (hoard_moe_layer's fx).  The
   gate multiplies as it is, or as sigmoid(gate) with gate_sigmoid.  w_offset is 1
   for models that store their norm weights less one.  r_out may be r.
   1 <= n <= 16384. */
typedef struct hoard_norm_args {
    int32_t type;     /* of b, h and a full gate: HOARD_TYPE_F32, _F16 or _BF16 */
    int32_t res_type; /* of r and r_out: HOARD_TYPE_F32 or `type` */
    int32_t gate_kind, gate_sigmoid;
    int32_t n_rows, n;
    float eps;        /* > 0 */
    float scale, w_offset;
    const void *r;       /* [n_rows][n] */
    const void *b;       /* [n_rows][n], or NULL */
    const void *gate;    /* as gate_kind says; NULL with HOARD_GATE_NONE */
    const float *w_post; /* [n], or NULL; needs b */
    const float *w_pre;  /* [n]; needed with h */
    void *r_out;         /* [n_rows][n]; needed with b */
    void *h;             /* [n_rows][n], or NULL */
    float *stats;        /* [n_rows][2]: rho_b and rho_v for the gradient (1 for a norm that is not
                            taken), or NULL */
} hoard_norm_args;

int hoard_norm_forward(const hoard_norm_args *a, void *stream);

/* Gradients of hoard_norm_forward.  `a` is the forward call's (r and h are not
   read, r_out and stats are: with b NULL r_out is the r that was normed).  dr_out
   and dh are the gradients of r_out and h (NULL: zero; dh needs w_pre, and at
   least one is given); the outputs are NULL where not wanted, and need what they
   are the gradient of.  Those of w_post, w_pre and a channel gate are sums over
   the rows in a fixed order.  dr may be dr_out.  workspace: hoard_norm_workspace's
   bytes (possibly 0), 4-byte aligned, used by the call alone while it runs. */
typedef struct hoard_norm_grads {
    const void *dr_out; /* [n_rows][n] of res_type, or NULL */
    const void *dh;     /* [n_rows][n] of type, or NULL */
    void *dr;           /* [n_rows][n] of res_type */
    void *db;           /* [n_rows][n] of type */
    void *dgate;        /* as gate */
    float *dw_post;     /* [n] */
    float *dw_pre;      /* [n] */
} hoard_norm_grads;

int hoard_norm_backward(const hoard_norm_args *a, const hoard_norm_grads *g, void *workspace, size_t workspace_bytes,
                        void *stream);
int hoard_norm_workspace(const hoard_norm_args *a, size_t *bytes);

#ifdef __cplusplus
}
#endif
#endif
