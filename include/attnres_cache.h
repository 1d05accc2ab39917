/*
 * A decoder layer's key-value cache in pages, and what generation does with it: the
 * heads of new tokens written into it, attention of the newest tokens over it, and
 * its reduction to the tokens that attention used most.  The reference's attention
 * keeps its cache as one tensor that grows by concatenation (model.py:430-569).
 * Additions to attnres_hip.h; its conventions hold.
 */
#ifndef ATTNRES_CACHE_H
#define ATTNRES_CACHE_H

#include "attnres_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ATTNRES_CACHE_MAX_HEAD_DIM 256
#define ATTNRES_CACHE_MAX_TOKENS (1 << 30) /* of one sequence */
#define ATTNRES_CACHE_MAX_SCALE 1e38f      /* (base-2 logarithms: log2(e) times it is finite) */
/*
 * Of one call (what the kernels count in 32 bits; more is ATTNRES_EUNSUPPORTED, but for the first ATTNRES_EINVAL):
 */
#define ATTNRES_CACHE_MAX_HEADS (1 << 20)       /* sequences; query heads; key / value heads */
#define ATTNRES_CACHE_MAX_APPENDED INT32_MAX    /* batch * tokens * (q_heads + 2 kv_heads) */
#define ATTNRES_CACHE_MAX_QUERIES (1 << 23)     /* batch * tokens * q_heads of attention */
#define ATTNRES_CACHE_MAX_PIECES (INT32_MAX / 2) /* batch * kv_heads * blocks of 16 or 32 query rows * 128-token units of the table */
#define ATTNRES_CACHE_MAX_EVICTED (1 << 21)     /* batch * kv_heads, times 8192-token slices of the table */
#define ATTNRES_CACHE_MAX_KEPT INT32_MAX        /* batch * kv_heads * budget */

/*
 * One layer's pages.  Token j of sequence b, head h lies at
 *   page block_table[b * table_stride + j / page_size], slot j % page_size,
 * its key at k + page * page_stride + h * head_stride + slot * slot_stride, its value
 * likewise at v, and, where they are kept, the attention it received at
 * weights[page * weight_page_stride + h * weight_head_stride + slot].
 * The values of the device tables are not known to the host: an entry of the block
 * table outside [0, pages), a negative count or more tokens than the table has room
 * for is never read or written through (each call says what becomes of it).
 */
typedef struct attnres_cache_desc {
  int32_t dtype;          /* ATTNRES_DTYPE_* of keys, values and queries */
  int32_t kv_heads;
  int32_t head_dim;       /* at most ATTNRES_CACHE_MAX_HEAD_DIM */
  int32_t page_size;      /* tokens of a page */
  int64_t pages;
  void* k;
  void* v;
  int64_t page_stride;    /* elements, of both k and v; the last dimension is contiguous */
  int64_t head_stride;
  int64_t slot_stride;
  float* weights;         /* or NULL */
  int64_t weight_page_stride;
  int64_t weight_head_stride;
  int64_t batch;          /* 0 is allowed: nothing is launched */
  const int32_t* block_table; /* device [batch, table_pages] */
  int64_t table_stride;
  int64_t table_pages;    /* table_pages * page_size at most ATTNRES_CACHE_MAX_TOKENS */
  const int32_t* cached;  /* device [batch]: tokens that each sequence has, without the call's new ones */
  const int32_t* fresh;   /* device [batch]: how many of the call's new tokens are the sequence's, the first ones; NULL: all */
} attnres_cache_desc;

/*
 * Heads of the new tokens from one projection [batch, tokens, (q_heads + 2 kv_heads)
 * head_dim], as attnres_qkv_rotary_forward computes them (per-head rms-norm, rotation
 * of interleaved pairs, fp32, one rounding), with keys and values written to slots
 * cached[b] + t of the cache, and 0 to their weights.  Token t of sequence b takes
 * table row positions[b] + t, or cached[b] + t without positions; a row outside the
 * tables gives NaN in its query and key.  A token that its sequence does not have (t >=
 * fresh[b]) is not written and has zeros for its query and key; one that has no slot is
 * not written either.
 */
typedef struct attnres_cache_append_desc {
  int64_t tokens;         /* 0 is allowed */
  int32_t q_heads;
  int32_t qk_norm;
  float norm_eps;
  int32_t table_dtype;    /* of sin and cos: ATTNRES_DTYPE_F32 or the cache's dtype */
  const void* qkv;        /* a token's heads are contiguous */
  int64_t batch_stride;   /* elements */
  int64_t token_stride;
  const void* sin;        /* [table_rows, head_dim / 2] */
  const void* cos;
  int64_t table_rows;
  int64_t table_row_stride; /* elements, both tables */
  const int32_t* positions; /* device [batch], or NULL */
} attnres_cache_append_desc;

/* q [batch, q_heads, tokens, head_dim], dense; k [batch, kv_heads, tokens, head_dim],
 * dense, or NULL: the rotated keys go to the cache alone. */
int attnres_cache_append(const attnres_cache_desc* cache, const attnres_cache_append_desc* desc, void* q, void* k,
                         void* stream);

/*
 * Attention of the newest tokens over the cache (their own keys and values in it
 * already): query row (b, h, t) reads tokens j < cached[b] + t + 1 through key / value
 * head h / (q_heads / kv_heads),
 *   p_j = softmax_j(scale <q, k_j>),   out = sum_j p_j v_j,
 * in fp32 (the products' operands in the dtype, p in two terms of it), one rounding to
 * the dtype.  With weights (tokens 1): each cached token's weight becomes decay * weight +
 * the sum of p_j over the key / value head's queries; with decay 0 the old one is not read.
 * Pages may be shared between sequences, but not with weights.
 * A query that its sequence does not have (t >= fresh[b]) gives zeros; a page outside the
 * cache gives NaN in that sequence, in every row that reads it, and a count that is
 * negative or beyond the table's room gives NaN in all its rows.
 */
typedef struct attnres_cache_attend_desc {
  int64_t tokens;         /* 0 is allowed */
  int32_t q_heads;        /* a multiple of kv_heads */
  float scale;            /* at most ATTNRES_CACHE_MAX_SCALE either way */
  const void* q;          /* [batch, q_heads, tokens, head_dim], last dimension contiguous */
  int64_t q_batch_stride; /* elements */
  int64_t q_head_stride;
  int64_t q_token_stride;
  float decay;            /* with weights */
} attnres_cache_attend_desc;

/* Workspace bytes (host computation; aligned to 256): pieces of at most 256 workgroups' rows
 * and, with weights, 4 bytes for each query head and token that the table has room for (a
 * table of the pages in use keeps it small). */
size_t attnres_cache_attend_workspace_size(const attnres_cache_desc* cache, const attnres_cache_attend_desc* desc);

/* out [batch, tokens, q_heads, head_dim], dense */
int attnres_cache_attend(const attnres_cache_desc* cache, const attnres_cache_attend_desc* desc, void* out,
                         void* workspace, size_t workspace_bytes, void* stream);

/*
 * Each key / value head of a sequence keeps at most `budget` of its cached[b] tokens:
 * the last `recent` and, of the others, those of the largest weights (a NaN is below
 * every number; equal ones: the earlier token).  What is kept is copied in its order,
 * keys, values and weights, to the first slots of the pages new_table[b * new_stride +
 * ...], which are all different and hold no token that the call reads; only a sequence
 * within its budget may keep its own pages, in the same order, and is then left as it is.  `fresh` is not used.
 * kept [batch, kv_heads, budget]: the tokens kept, ascending, -1 behind them; left
 * [batch]: their number.  Counts beyond the table's room are taken as 0.  A token whose
 * page lies outside the cache has the lowest weight and is not copied.
 */
int attnres_cache_evict(const attnres_cache_desc* cache, const int32_t* new_table, int64_t new_stride, int64_t budget,
                        int64_t recent, int32_t* kept, int32_t* left, void* workspace, size_t workspace_bytes,
                        void* stream);

/* Workspace bytes (host computation; aligned to 256); 0 for tables of few tokens. */
size_t attnres_cache_evict_workspace_size(const attnres_cache_desc* cache, int64_t budget, int64_t recent);

#ifdef __cplusplus
}
#endif

#endif /* ATTNRES_CACHE_H */
