/*
 * The decoder's sublayers around the AttnRes reads: the heads of a fused query /
 * key / value projection (per-head rms-norm and rotary positions in one pass) and
 * the gated feed-forward block's two projections with their activation and
 * product.  Additions to attnres_hip.h; its conventions hold.
 */
#ifndef ATTNRES_SUBLAYERS_H
#define ATTNRES_SUBLAYERS_H

#include "attnres_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ATTNRES_QKV_ROTARY_MAX_HEAD_DIM 1024

/*
 * The heads of one projection [batch, tokens, (q_heads + 2 kv_heads) head_dim]:
 * queries, keys, values (model.py:430-569).  With qk_norm each query and key head
 * is rms-normed (model.py:28-31); then each is rotated, interleaved pairs, by row
 * p of sin and cos (model.py:291-313): out[2i] = cos x[2i] - sin x[2i+1], out[2i+1]
 * = sin x[2i] + cos x[2i+1].  fp32 throughout, one rounding to the dtype.  Token
 * (b, t) takes table row start + t, or positions[b * positions_batch_stride + t *
 * positions_token_stride]; a position outside the table gives NaN in that token's
 * queries and keys (and in their gradients) and reads nothing.
 */
typedef struct attnres_qkv_rotary_desc {
  int32_t dtype;          /* ATTNRES_DTYPE_* */
  int32_t table_dtype;    /* of sin and cos: ATTNRES_DTYPE_F32 or dtype */
  int64_t batch;          /* batch * tokens 0 is allowed: nothing is launched */
  int64_t tokens;
  int32_t q_heads;
  int32_t kv_heads;
  int32_t head_dim;       /* even, at most ATTNRES_QKV_ROTARY_MAX_HEAD_DIM */
  int32_t qk_norm;
  float norm_eps;
  const void* qkv;        /* a token's heads are contiguous */
  int64_t batch_stride;   /* elements */
  int64_t token_stride;   /* elements */
  const void* sin;        /* [table_rows, head_dim / 2] */
  const void* cos;
  int64_t table_rows;
  int64_t table_row_stride; /* elements, both tables */
  const int64_t* positions; /* device, or NULL */
  int64_t positions_batch_stride;
  int64_t positions_token_stride;
  int64_t start;          /* without positions: start >= 0, start + tokens <= table_rows */
} attnres_qkv_rotary_desc;

/* q [batch, q_heads, tokens, head_dim] and k [batch, kv_heads, tokens, head_dim],
 * dense in dtype.  The values are read where they are. */
int attnres_qkv_rotary_forward(const attnres_qkv_rotary_desc* desc, void* q, void* k, void* stream);

/* grads: dq, dk, dv as [batch, heads, tokens, head_dim] in dtype with any strides
 * (elements, over batch, heads and tokens: strides[3 * i + 0..2] of gradient i) and
 * a contiguous last dimension; NULL = zero.  dqkv [batch, tokens, (q_heads + 2
 * kv_heads) head_dim], dense. */
int attnres_qkv_rotary_backward(const attnres_qkv_rotary_desc* desc, const void* const* grads, const int64_t* strides,
                                void* dqkv, void* stream);

/*
 * Gated feed-forward projections (model.py:572-589): with weight [2 hidden, dim],
 * rows [0, hidden) up and [hidden, 2 hidden) gate, u = x up^T, z = x gate^T and
 *   h = u silu(z),  silu(z) = z / (1 + exp(-z)).
 * Products and activation in fp32.  h is rounded to the dtype once.  The backward
 * forms the projections' gradient from u and z as the forward kept them (20 bits in
 * bf16, 24 in fp16, all in fp32) and rounds it to the dtype, as the matrix cores take
 * it, before the products that give dx and dweight, which are rounded once more.
 */
typedef struct attnres_swiglu_desc {
  int32_t dtype;          /* ATTNRES_DTYPE_* */
  int64_t n_tok;          /* at most 2^22; 0 is allowed: the forward launches nothing, the backward clears dweight */
  int32_t dim;
  int32_t hidden;
  const void* x;          /* [n_tok, dim], contiguous last dimension */
  int64_t x_row_stride;   /* elements */
  const void* weight;     /* [2 hidden, dim], contiguous last dimension */
  int64_t weight_row_stride;
} attnres_swiglu_desc;

/* Bytes of what the forward keeps of u and z for the backward (its own layout; more
 * bits than the 16-bit dtypes hold).  Host computation. */
size_t attnres_swiglu_saved_size(const attnres_swiglu_desc* desc);

/* Workspace bytes of the forward / of the backward (host computation). */
size_t attnres_swiglu_forward_workspace_size(const attnres_swiglu_desc* desc);
size_t attnres_swiglu_backward_workspace_size(const attnres_swiglu_desc* desc, int32_t want_dx, int32_t want_dweight);

/* h [n_tok, hidden] dense.  saved: NULL, or attnres_swiglu_saved_size bytes aligned to
 * 16, for the backward.  workspace aligned to 256 bytes. */
int attnres_swiglu_forward(const attnres_swiglu_desc* desc, void* h, void* saved, void* workspace,
                           size_t workspace_bytes, void* stream);

/* grad_h [n_tok, hidden], rows of grad_row_stride elements; saved: the forward's.
 * dx [n_tok, dim] and dweight [2 hidden, dim], dense in dtype; either may be NULL. */
int attnres_swiglu_backward(const attnres_swiglu_desc* desc, const void* grad_h, int64_t grad_row_stride,
                            const void* saved, void* dx, void* dweight, void* workspace, size_t workspace_bytes,
                            void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ATTNRES_SUBLAYERS_H */
