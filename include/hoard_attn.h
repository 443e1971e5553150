/*
 * hoard_attn.h -- C ABI of the operators of a layer's attention half on MI355X.
 *
 * What a layer runs between the projection to queries, keys and values and the
 * output projection (both hoard_q4_matmul of hoard_ops.h, or the caller's): the
 * norms of each query and key head with the rotation by its position (with
 * gradients), keys and values written to a paged cache of 16 or 8 bits and read
 * back, and the attention of one new token a sequence, or the few of a verify
 * step, over that cache.
 *
 * The manner is that of hoard_ops.h: extern "C", 0 or a negative HOARD_ERR_* code
 * (hoard_last_error() then describes it), no handle, nothing kept, nothing
 * allocated and only kernels launched, on the stream given; the current device
 * must be the stream's, pointers are device memory of it unless "host" is said.
 * An activation type is HOARD_TYPE_F32, _F16 or _BF16; sums, norms and softmax
 * statistics are formed in 32 bits and rounded once when stored.  Counts of tokens
 * and sequences may be zero.  Outputs must not overlap inputs or each other except
 * where said.
 */
#ifndef HOARD_ATTN_H
#define HOARD_ATTN_H

#include <stddef.h>
#include <stdint.h>

#include "hoard_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HOARD_TYPE_I8 24 /* 8-bit codes (ggml.h GGML_TYPE_I8), for caches */

/* ---- a paged cache ------------------------------------------------------------ */

/* Pages of `page` tokens each.  A slot names a token's place: slot / page is the
   page's number, slot % page the place in it.  head_dim is a multiple of 16 up to
   256, page 16, 32, 64, 128 or 256, n_pages * page < 2^31.

   With HOARD_TYPE_I8 a row of head_dim values is held as codes and one scale
   s = max |x| / 127: code = x / s rounded to nearest, ties to even, value = s * code.
   A row of zeros has the scale 0; one that holds an infinity or a NaN is NaN
   throughout, and a value's scale that is infinite makes as much of it. */
typedef struct hoard_kv_cache {
    void *k, *v;              /* [n_pages][n_kv_heads][page][head_dim] of `type`, 16-byte aligned */
    float *k_scale, *v_scale; /* [n_pages][n_kv_heads][page] with HOARD_TYPE_I8, 16-byte aligned; else NULL */
    int32_t type;             /* HOARD_TYPE_F16, _BF16 or _I8 */
    int32_t n_pages, page, n_kv_heads, head_dim;
} hoard_kv_cache;

/* Rows of keys and values to their slots, and back: k and v [n_tokens][n_kv_heads]
   [head_dim] of `type`, a token's row k_stride (v_stride) elements behind the one
   before; k or v may be NULL (left out).  slots[n_tokens]: one outside
   [0, n_pages * page) drops its token (a read leaves its rows as they are); the
   others of a write must be distinct.  `cache` is host memory. */
int hoard_kv_write(const hoard_kv_cache *cache, int type, int n_tokens, const int32_t *slots, const void *k,
                   int64_t k_stride, const void *v, int64_t v_stride, void *stream);
int hoard_kv_read(const hoard_kv_cache *cache, int type, int n_tokens, const int32_t *slots, void *k,
                  int64_t k_stride, void *v, int64_t v_stride, void *stream);

/* ---- heads normed and rotated --------------------------------------------------- */

#define HOARD_ROPE_HALVES 0 /* value i turns with value i + rot_dim / 2 */
#define HOARD_ROPE_PAIRS 1  /* value 2i turns with value 2i + 1 */

/* For every token and every head x of head_dim values, those of q by w_q and of k by w_k:

     y = x * rho * (w_offset + w),  rho = 1 / sqrt(mean(x^2) + eps)     (w NULL: y = x)
     z = y with pair i of its first rot_dim values turned by the angle
         pos[axis[i]][token] * freq[i], formed in 64 bits               (rot_dim 0: z = y)

   q_out and k_out receive z.  With a cache, z of k and v as it is go to slots[token]
   as by hoard_kv_write, from 32 bits, and k_out may be NULL.  q, k and v are each
   optional; v needs a cache.  The rows of a token are n heads one after the other, a
   token's row a stride (in elements) behind the one before, so that q, k and v may be
   columns of one projection's rows.  q_out may be q and k_out may be k, at their
   strides.  head_dim is a multiple of 8 up to 256 (with a cache as its head_dim), a
   stride at least a row and below 2^31. */
typedef struct hoard_heads_args {
    int32_t type;     /* of q, k, v, q_out and k_out */
    int32_t n_tokens, n_q_heads, n_kv_heads, head_dim;
    int32_t rot_dim;  /* multiple of 8 up to head_dim */
    int32_t rope;     /* HOARD_ROPE_* */
    int32_t n_axes;   /* rows of pos, 1..255 */
    float eps;        /* > 0 */
    float w_offset;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    const void *q, *k, *v;
    const float *w_q, *w_k; /* [head_dim], or NULL */
    const int32_t *pos;     /* [n_axes][n_tokens]; NULL with rot_dim 0 */
    const double *freq;     /* [rot_dim / 2], radians a position; NULL with rot_dim 0 */
    const uint8_t *axis;    /* [rot_dim / 2], one past the last axis counts as the last; NULL: 0 */
    void *q_out, *k_out;
    float *stats;           /* [n_tokens][n_q_heads + n_kv_heads]: rho for the gradient, or NULL; written
                               for the heads that are given, 1 for those without a norm */
    const hoard_kv_cache *cache; /* host memory, or NULL */
    const int32_t *slots;   /* [n_tokens], with a cache */
} hoard_heads_args;

int hoard_heads_forward(const hoard_heads_args *a, void *stream);

/* Gradients of hoard_heads_forward given those of q_out and k_out (dq_out at
   q_out_stride, dk_out at k_out_stride).  `a` is the forward call's; v, q_out, k_out,
   cache and slots are not used, q (k) and stats only with w_q (w_k).  dq may be dq_out
   and dk may be dk_out, at equal strides.
   dw_q and dw_k are sums over tokens and heads in a fixed order.  Outputs are NULL
   where not wanted.  workspace: hoard_heads_workspace's bytes (possibly 0), 4-byte
   aligned, used by the call alone while it runs. */
typedef struct hoard_heads_grads {
    const void *dq_out, *dk_out; /* of type, or NULL */
    void *dq, *dk;               /* of type, or NULL */
    float *dw_q, *dw_k;          /* [head_dim], or NULL */
    int64_t dq_stride, dk_stride; /* 0: q_stride and k_stride */
} hoard_heads_grads;

int hoard_heads_backward(const hoard_heads_args *a, const hoard_heads_grads *g, void *workspace,
                         size_t workspace_bytes, void *stream);
int hoard_heads_workspace(const hoard_heads_args *a, size_t *bytes);

/* ---- attention over the cache ---------------------------------------------------- */

/* For every sequence s, new token t and query head h, with the key head h / (n_q_heads
   / n_kv_heads) and n = lens[s][t]:

     S_j = scale * <q[s][t][h], k_j>,  0 <= j < n
     out[s][t][h] = sum_j softmax(S)_j v_j,  lse[s][t][h] = log sum_j exp(S_j)

   where key j of the sequence is place j % page of page pages[s][j / page].  A row that
   sees no key (n <= 0) has out 0 and lse -infinity.  n beyond max_pages * page counts as
   that; a page number outside [0, n_pages) hides the keys of its page.  Keys and values
   that a row does not see may hold anything, and so may a page table's entries behind
   the last key.  Keys and values are used as the cache holds them.  q and the weights are
   held to 2^-16 of each (2^-22 for fp32 activations) or, over f16 and I8 caches, to 2^-37
   of the row's largest, whichever is more; with I8 a weight's product with its value's
   scale is held so, by the keys that the row sees.  A weight below 2^-126 may count as
   none.
   What a row sees that is not finite counts as in the formula, wherever it lies: a score
   of -infinity weighs nothing (where all are, the row is as one that sees no key), one
   of +infinity or NaN makes the row NaN, as a query does that is not finite; an infinity
   among the values makes its column infinite, NaN beside one of the other sign, and
   either of these where its weight is too small for 32 bits.  1 <= n_new <= 64,
   n_q_heads a multiple of the cache's n_kv_heads up to 1024, n_seq * n_new < 2^24,
   max_pages * page <= 2^30.
   workspace: hoard_attn_workspace's bytes (possibly 0), 16-byte aligned, used by the
   call alone while it runs.  `cache` and `a` are host memory. */
typedef struct hoard_attn_args {
    int32_t type; /* of q and out */
    int32_t n_seq, n_new, n_q_heads;
    int32_t max_pages;    /* columns of pages */
    float scale;
    int64_t q_stride;     /* elements from a new token's row of q to the next */
    const void *q;        /* [n_seq][n_new] rows of [n_q_heads][head_dim] */
    const int32_t *pages; /* [n_seq][max_pages] */
    const int32_t *lens;  /* [n_seq][n_new] */
    void *out;            /* [n_seq][n_new][n_q_heads][head_dim] */
    float *lse;           /* [n_seq][n_new][n_q_heads], or NULL */
} hoard_attn_args;

int hoard_attn_decode(const hoard_kv_cache *cache, const hoard_attn_args *a, void *workspace, size_t workspace_bytes,
                      void *stream);
int hoard_attn_workspace(const hoard_kv_cache *cache, const hoard_attn_args *a, size_t *bytes);

#ifdef __cplusplus
}
#endif
#endif
