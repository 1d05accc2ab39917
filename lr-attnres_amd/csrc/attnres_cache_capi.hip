// C ABI of the paged cache's kernels: argument checks and kernel selection.
// Declared in include/attnres_cache.h.
#include <float.h>
#include <math.h>
#include <string.h>

#include "../../include/attnres_cache.h"
#include "attnres_cache.h"

using namespace attnres;

namespace {

constexpr int kCus = 256;

int es_of(int dtype) { return dtype == ATTNRES_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

// the cache itself; what the calls write and read through it is checked by each
int check_cache(const attnres_cache_desc* c) {
  if (!c) return api_fail(ATTNRES_EINVAL, "cache is NULL");
  if (c->dtype != ATTNRES_DTYPE_F32 && c->dtype != ATTNRES_DTYPE_BF16 && c->dtype != ATTNRES_DTYPE_F16)
    return api_fail(ATTNRES_EINVAL, "unknown dtype %d", c->dtype);
  if (c->kv_heads < 1 || c->kv_heads > ATTNRES_CACHE_MAX_HEADS)
    return api_fail(ATTNRES_EINVAL, "kv_heads=%d must be 1 .. %d", c->kv_heads, ATTNRES_CACHE_MAX_HEADS);
  if (c->head_dim < 1) return api_fail(ATTNRES_EINVAL, "head_dim=%d must be >= 1", c->head_dim);
  if (c->head_dim > ATTNRES_CACHE_MAX_HEAD_DIM)
    return api_fail(ATTNRES_EUNSUPPORTED, "head_dim=%d above %d", c->head_dim, ATTNRES_CACHE_MAX_HEAD_DIM);
  if (c->page_size < 1) return api_fail(ATTNRES_EINVAL, "page_size=%d must be >= 1", c->page_size);
  if (c->batch < 0 || c->batch > ATTNRES_CACHE_MAX_HEADS)
    return api_fail(ATTNRES_EINVAL, "batch=%lld must be 0 .. %d", (long long)c->batch, ATTNRES_CACHE_MAX_HEADS);
  if (c->pages < 0 || c->pages > INT32_MAX) return api_fail(ATTNRES_EINVAL, "pages=%lld", (long long)c->pages);
  if (c->table_pages < 0) return api_fail(ATTNRES_EINVAL, "table_pages=%lld < 0", (long long)c->table_pages);
  if (c->table_pages > ATTNRES_CACHE_MAX_TOKENS / c->page_size)
    return api_fail(ATTNRES_EUNSUPPORTED, "table_pages=%lld of %d tokens: above %d tokens a sequence",
                    (long long)c->table_pages, c->page_size, ATTNRES_CACHE_MAX_TOKENS);
  if (c->batch == 0) return ATTNRES_OK;
  if (!c->cached || (c->table_pages > 0 && !c->block_table)) return api_fail(ATTNRES_EINVAL, "block_table / cached is NULL");
  if (c->table_stride < 0) return api_fail(ATTNRES_EINVAL, "table_stride < 0");
  if (c->pages > 0 && (!c->k || !c->v)) return api_fail(ATTNRES_EINVAL, "k / v is NULL");
  if (c->page_stride < 0 || c->head_stride < 0 || c->slot_stride < 0)
    return api_fail(ATTNRES_EINVAL, "page, head and slot strides must be >= 0");
  if (c->weights && (c->weight_page_stride < 0 || c->weight_head_stride < 0))
    return api_fail(ATTNRES_EINVAL, "weight strides must be >= 0");
  return ATTNRES_OK;
}

CachePages pages_of(const attnres_cache_desc* c) {
  CachePages p{};
  p.k = c->k;
  p.v = c->v;
  p.page_stride = c->page_stride;
  p.head_stride = c->head_stride;
  p.slot_stride = c->slot_stride;
  p.w = c->weights;
  p.w_page_stride = c->weight_page_stride;
  p.w_head_stride = c->weight_head_stride;
  p.table = c->block_table;
  p.table_stride = c->table_stride;
  p.cached = c->cached;
  p.fresh = c->fresh;
  p.batch = (int32_t)c->batch;
  p.kv_heads = c->kv_heads;
  p.head_dim = c->head_dim;
  p.page_size = c->page_size;
  p.pages = (int32_t)c->pages;
  p.room = (int32_t)(c->table_pages * c->page_size);
  p.by_page = fast_div(c->page_size);
  p.page_bytes = (uint32_t)(c->page_stride * es_of(c->dtype));
  p.slot_bytes = (uint32_t)(c->slot_stride * es_of(c->dtype));
  return p;
}

// whether every row of the pages starts at a multiple of `per` values
bool rows_at(const attnres_cache_desc* c, int per) {
  const int bytes = per * es_of(c->dtype);
  return c->head_dim % per == 0 && aligned(c->k, bytes) && aligned(c->v, bytes) && c->page_stride % per == 0 &&
         c->head_stride % per == 0 && c->slot_stride % per == 0;
}

// the widest of 16, 8, 4 bytes that every row of the pages starts and ends at a multiple of, or a value's
int row_bytes(const attnres_cache_desc* c) {
  const int es = es_of(c->dtype);
  for (int b = 16; b > es; b /= 2)
    if (rows_at(c, b / es)) return b;
  return es;
}

int check_append(const attnres_cache_desc* c, const attnres_cache_append_desc* d) {
  if (int rc = check_cache(c)) return rc;
  if (!d) return api_fail(ATTNRES_EINVAL, "desc is NULL");
  if (d->table_dtype != ATTNRES_DTYPE_F32 && d->table_dtype != c->dtype)
    return api_fail(ATTNRES_EINVAL, "table dtype %d is neither fp32 nor the cache's %d", d->table_dtype, c->dtype);
  if (d->tokens < 0 || d->tokens > (int64_t)1 << 30)
    return api_fail(ATTNRES_EINVAL, "tokens=%lld must be 0 .. 2^30", (long long)d->tokens);
  if (d->q_heads < 1 || d->q_heads > ATTNRES_CACHE_MAX_HEADS)
    return api_fail(ATTNRES_EINVAL, "q_heads=%d must be 1 .. %d", d->q_heads, ATTNRES_CACHE_MAX_HEADS);
  if (c->head_dim % 2) return api_fail(ATTNRES_EINVAL, "head_dim=%d must be even", c->head_dim);
  if (c->batch == 0 || d->tokens == 0) return ATTNRES_OK;
  if (c->batch * d->tokens > ATTNRES_CACHE_MAX_APPENDED / ((int64_t)d->q_heads + 2 * c->kv_heads))
    return api_fail(ATTNRES_EUNSUPPORTED, "batch=%lld, tokens=%lld, %d + 2 * %d heads: too many", (long long)c->batch,
                    (long long)d->tokens, d->q_heads, c->kv_heads);
  if (!d->qkv || !d->sin || !d->cos) return api_fail(ATTNRES_EINVAL, "qkv / sin / cos is NULL");
  if (d->batch_stride < 0 || d->token_stride < 0)
    return api_fail(ATTNRES_EINVAL, "batch_stride and token_stride must be >= 0");
  if (d->table_rows < 1) return api_fail(ATTNRES_EINVAL, "table_rows=%lld < 1", (long long)d->table_rows);
  if (d->table_row_stride < c->head_dim / 2)
    return api_fail(ATTNRES_EINVAL, "table_row_stride=%lld below head_dim / 2 = %d", (long long)d->table_row_stride,
                    c->head_dim / 2);
  return ATTNRES_OK;
}

int check_attend(const attnres_cache_desc* c, const attnres_cache_attend_desc* d) {
  if (int rc = check_cache(c)) return rc;
  if (!d) return api_fail(ATTNRES_EINVAL, "desc is NULL");
  if (d->tokens < 0 || d->tokens > ATTNRES_CACHE_MAX_TOKENS)
    return api_fail(ATTNRES_EINVAL, "tokens=%lld must be 0 .. 2^30", (long long)d->tokens);
  if (d->q_heads < 1 || d->q_heads > ATTNRES_CACHE_MAX_HEADS || d->q_heads % c->kv_heads)
    return api_fail(ATTNRES_EINVAL, "q_heads=%d must be a multiple of kv_heads=%d, at most %d", d->q_heads, c->kv_heads,
                    ATTNRES_CACHE_MAX_HEADS);
  if (!(fabsf(d->scale) <= ATTNRES_CACHE_MAX_SCALE))
    return api_fail(ATTNRES_EINVAL, "scale must be finite, of at most %g", (double)ATTNRES_CACHE_MAX_SCALE);
  if (c->weights && d->tokens > 1) return api_fail(ATTNRES_EINVAL, "weights need a single new token, got %lld", (long long)d->tokens);
  if (c->weights && !(d->decay >= 0.f && d->decay <= 1.f)) return api_fail(ATTNRES_EINVAL, "decay must be 0 .. 1");
  if (c->batch == 0 || d->tokens == 0) return ATTNRES_OK;
  if (c->batch * d->tokens > ATTNRES_CACHE_MAX_QUERIES / d->q_heads)
    return api_fail(ATTNRES_EUNSUPPORTED, "batch=%lld, tokens=%lld, q_heads=%d: too many queries, above %d", (long long)c->batch,
                    (long long)d->tokens, d->q_heads, ATTNRES_CACHE_MAX_QUERIES);
  if (!d->q) return api_fail(ATTNRES_EINVAL, "q is NULL");
  if (d->q_batch_stride < 0 || d->q_head_stride < 0 || d->q_token_stride < 0)
    return api_fail(ATTNRES_EINVAL, "q strides must be >= 0");
  return ATTNRES_OK;
}

}  // namespace

extern "C" int attnres_cache_append(const attnres_cache_desc* c, const attnres_cache_append_desc* d, void* q, void* k,
                                    void* stream) {
  if (int rc = check_append(c, d)) return rc;
  if (c->batch == 0 || d->tokens == 0) return ATTNRES_OK;
  if (!q) return api_fail(ATTNRES_EINVAL, "q is NULL");
  CacheAppendParams p{};
  p.c = pages_of(c);
  p.qkv = d->qkv;
  p.b_stride = d->batch_stride;
  p.t_stride = d->token_stride;
  p.n_tok = (int32_t)(c->batch * d->tokens);
  p.tokens = (int32_t)d->tokens;
  p.by_tokens = fast_div(p.tokens);
  p.q_heads = d->q_heads;
  p.qk_norm = d->qk_norm != 0;
  p.eps = d->norm_eps;
  p.sin = d->sin;
  p.cos = d->cos;
  p.table_rows = d->table_rows;
  p.table_stride = d->table_row_stride;
  p.pos = d->positions;
  p.q = q;
  p.k = k;
  // the widest vector that every row starts at a multiple of, and the lanes that cover a
  // head with one each; vec 1 is the general kernel
  const int es = es_of(c->dtype), ts = es_of(d->table_dtype);
  int vec = 1, lanes = 1;
  for (int v = 16 / es; v >= 2 && vec == 1; v /= 2) {
    if (!rows_at(c, v) || !aligned(d->qkv, v * es) || d->batch_stride % v || d->token_stride % v || !aligned(q, v * es) ||
        !aligned(k, v * es) || !aligned(d->sin, v / 2 * ts) || !aligned(d->cos, v / 2 * ts) || d->table_row_stride % (v / 2))
      continue;
    for (int n = v == 8 ? 4 : v == 4 ? 8 : 32; n <= (v == 8 ? 32 : v == 4 ? 64 : 128); n *= 2)
      if (vec == 1 && n * v >= c->head_dim) vec = v, lanes = n;
  }
  const hipError_t err = launch_cache_append(c->dtype, d->table_dtype == ATTNRES_DTYPE_F32, p, vec, lanes, (hipStream_t)stream);
  if (err != hipSuccess) return api_fail(ATTNRES_ELAUNCH, "cache append launch failed: %s", hipGetErrorString(err));
  return ATTNRES_OK;
}

namespace {

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

struct AttendPlan {
  int tile, rows, blocks, row_bits, wgs, direct, page16;
  int64_t logit_stride;
  size_t part, part_ml, row_ml, logits, need;  // offsets in the workspace, and its size
};

int plan_attend(const attnres_cache_desc* c, const attnres_cache_attend_desc* d, AttendPlan* a) {
  const int es = es_of(c->dtype);
  const int64_t rows = d->q_heads / c->kv_heads * d->tokens, heads = c->batch * c->kv_heads;
  const int64_t room = c->table_pages * c->page_size, units = (room + kAttUnit - 1) / kAttUnit;
  const double room_bytes = 2.0 * room * c->head_dim * es;
  // (pages, and tokens inside one, within 32-bit offsets of each other)
  constexpr int64_t kFar = (int64_t)1 << 32;
  a->page16 = row_bytes(c) == 16 && c->page_size % 16 == 0 && c->page_stride < kFar / es && c->slot_stride < kFar / es / c->page_size;
  // Each block of rows reads its head's tokens, from L2 after the first.  Blocks of 32 halve that and take longer to
  // start, so they are for many bytes (us, 16 rows / 32: 16 x 2 heads of up to 8192 x 64 bf16, 128 rows 53 / 40, 32 rows 21.7 / 20.4;
  // x 128 92 / 67; 28 x 14 heads of up to 1337 x 64, 56 rows 39.6 / 27.7; 4 x 4 heads of up to 4096 x 64, 2048 rows 237 / 170.  Of fewer:
  // 4 x 2 heads of up to 4096 x 128, 128 rows 22.3 / 25.3; 8 x 2 of 400, 9.6 / 13.6.  In pages of 11 tokens 47.6 / 46.1 and 72 / 95.)
  const int64_t blocks16 = (rows + 15) / 16;
  a->row_bits = a->page16 && blocks16 > 1 && heads * blocks16 * room_bytes >= 256 << 20 ? 5 : 4;
  const int64_t blocks = (rows + (1 << a->row_bits) - 1) >> a->row_bits, segs = heads * blocks;
  // (rows, and segs with them, are at most the queries)
  if (segs * (units > 0 ? units : 1) > ATTNRES_CACHE_MAX_PIECES)
    return api_fail(ATTNRES_EUNSUPPORTED, "batch=%lld, tokens=%lld, q_heads=%d, %lld cached: too many tokens", (long long)c->batch,
                    (long long)d->tokens, d->q_heads, (long long)room);
  a->tile = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  a->rows = (int)rows;
  a->blocks = (int)blocks;
  // One workgroup a CU takes all that a CU can have in flight (2, 3 or 4, or twice the waves: the same to 3%).
  const int64_t all = segs * units;
  a->wgs = (int)(all < kCus ? (all > 0 ? all : 1) : kCus);
  // A CU reads at most 48 bytes a ns, and a round of its waves' tiles takes 650 ns (1100 with tokens looked up one by
  // one); all CUs read 5500; joining takes 6 us.  A segment that is read in one piece, if it fills its table, ends the
  // call at best after its rounds, all of them (half full) after segs * room_bytes / 2 / 5500.  Where that is later by
  // less than the join, a workgroup takes a whole segment and writes its rows.  (us, whole / split: 16 x 12 heads of up to 2048 x
  // 64 bf16 15.4 / 14 + 4; 12 heads of 300 5.6 / 6.8 + 4; 32 segments of up to 4096 25 / 9.4 + 4; 64 of up to 8192 x 128 fp16 100 / 48
  // + 5; 15 heads of up to 700 x 40 fp32 15.5 / 10.3 + 4.)  Lengths are on the device alone, so longer tables are split though they
  // may be nearly empty, and one long sequence among short ones is shared.
  const double rounds = (double)room / (es == 4 || a->tile == 256 ? 64 : 128);
  const double round_ns = a->page16 ? 650 : 1100;
  const double piece_ns = rounds * round_ns > room_bytes / 48 ? rounds * round_ns : room_bytes / 48;
  a->direct = c->pages > 0 && room_bytes <= 1 << 20 && piece_ns - segs * room_bytes / 11000.0 <= 6000;
  if (a->direct) a->wgs = 0;
  a->logit_stride = (room + 31) / 32 * 32;
  size_t at = 0;
  a->part = at;
  at += up256(((size_t)2 * a->wgs << a->row_bits) * a->tile * 4);
  a->part_ml = at;
  at += up256(((size_t)2 * a->wgs << a->row_bits) * 2 * 4);
  a->row_ml = at;
  if (c->weights) at += up256((size_t)c->batch * d->q_heads * 2 * 4);
  a->logits = at;
  if (c->weights) at += up256((size_t)c->batch * d->q_heads * a->logit_stride * 4);
  a->need = at;
  return ATTNRES_OK;
}

}  // namespace

extern "C" size_t attnres_cache_attend_workspace_size(const attnres_cache_desc* c, const attnres_cache_attend_desc* d) {
  AttendPlan a;
  if (check_attend(c, d) || c->batch == 0 || d->tokens == 0 || plan_attend(c, d, &a)) return 0;
  return a.need;
}

extern "C" int attnres_cache_attend(const attnres_cache_desc* c, const attnres_cache_attend_desc* d, void* out,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_attend(c, d)) return rc;
  if (c->batch == 0 || d->tokens == 0) return ATTNRES_OK;
  AttendPlan a;
  if (int rc = plan_attend(c, d, &a)) return rc;
  if (!out) return api_fail(ATTNRES_EINVAL, "out is NULL");
  if (a.need && (!workspace || workspace_bytes < a.need || !aligned(workspace, 256)))
    return api_fail(ATTNRES_EWORKSPACE, "workspace of %zu bytes needed, got %zu", a.need, workspace ? workspace_bytes : (size_t)0);
  const int es = es_of(c->dtype), per = 16 / es;
  CacheAttendParams p{};
  p.c = pages_of(c);
  p.q = d->q;
  p.q_b_stride = d->q_batch_stride;
  p.q_h_stride = d->q_head_stride;
  p.q_t_stride = d->q_token_stride;
  p.tokens = (int32_t)d->tokens;
  p.q_heads = d->q_heads;
  p.group = d->q_heads / c->kv_heads;
  p.rows = a.rows;
  p.blocks = a.blocks;
  p.wgs = a.wgs;
  p.direct = a.direct;
  p.by_group = fast_div(p.group);
  p.by_blocks = fast_div(a.blocks);
  p.by_segs = fast_div(c->kv_heads * a.blocks);
  p.by_wgs = fast_div(a.wgs);
  p.own_weights = c->weights && a.direct && a.blocks == 1;
  if (c->weights && !p.own_weights) {
    const int64_t units = c->batch * c->kv_heads * ((p.c.room + kAttUnit - 1) / kAttUnit);
    const int64_t wgs = (units + 3) / 4;
    p.weight_waves = (int32_t)(wgs < 8 * kCus ? wgs : 8 * kCus) * 4;
    p.by_weight_waves = fast_div(p.weight_waves);
  }
  p.tile = a.tile;
  p.row_bits = a.row_bits;
  p.vb = row_bytes(c);
  p.page16 = a.page16;
  p.whole = c->head_dim == a.tile;
  p.q_vec = aligned(d->q, 16) && d->q_batch_stride % per == 0 && d->q_head_stride % per == 0 && d->q_token_stride % per == 0;
  // (the kernels take the maximum before they scale: a negative scale goes into the queries' sign, and 0 is as good as
  // the smallest number, which masked scores of -inf times it stay -inf with)
  p.negate = d->scale < 0;
  p.scale = (float)(fabs((double)d->scale) * 1.4426950408889634);
  if (!(p.scale >= FLT_MIN)) p.scale = FLT_MIN;
  p.decay = d->decay;
  p.out = out;
  char* ws = (char*)workspace;
  p.part = (float*)(ws + a.part);
  p.part_ml = (float*)(ws + a.part_ml);
  if (c->weights) {
    p.row_ml = (float*)(ws + a.row_ml);
    p.logits = (float*)(ws + a.logits);
    p.logit_stride = a.logit_stride;
  }
  hipStream_t st = (hipStream_t)stream;
  hipError_t err = c->dtype == ATTNRES_DTYPE_F32    ? launch_cache_attend_f32(p, st)
                   : c->dtype == ATTNRES_DTYPE_BF16 ? launch_cache_attend_bf16(p, st)
                                                    : launch_cache_attend_f16(p, st);
  if (err != hipSuccess) return api_fail(ATTNRES_ELAUNCH, "cache attend launch failed: %s", hipGetErrorString(err));
  return ATTNRES_OK;
}

namespace {

int check_evict(const attnres_cache_desc* c, int64_t budget, int64_t recent) {
  if (int rc = check_cache(c)) return rc;
  if (budget < 1 || budget > ATTNRES_CACHE_MAX_TOKENS) return api_fail(ATTNRES_EINVAL, "budget=%lld must be 1 .. 2^30", (long long)budget);
  if (recent < 0 || recent > budget)
    return api_fail(ATTNRES_EINVAL, "recent=%lld must be 0 .. budget=%lld", (long long)recent, (long long)budget);
  const int64_t heads = c->batch * c->kv_heads, slices = (c->table_pages * c->page_size + kEvictSlice - 1) / kEvictSlice;
  if (heads > ATTNRES_CACHE_MAX_EVICTED || heads * budget > ATTNRES_CACHE_MAX_KEPT || heads * slices > ATTNRES_CACHE_MAX_EVICTED)
    return api_fail(ATTNRES_EUNSUPPORTED, "batch=%lld, kv_heads=%d, budget=%lld, %lld pages of %d: too many tokens",
                    (long long)c->batch, c->kv_heads, (long long)budget, (long long)c->table_pages, c->page_size);
  return ATTNRES_OK;
}

// workgroups that choose a head's tokens: one, where it can hold all keys or there is nothing to choose
int64_t evict_slices(const attnres_cache_desc* c, int64_t budget, int64_t recent) {
  const int64_t room = c->table_pages * c->page_size;
  return room <= 2 * kEvictSlice || budget == recent ? 1 : (room + kEvictSlice - 1) / kEvictSlice;
}

}  // namespace

extern "C" size_t attnres_cache_evict_workspace_size(const attnres_cache_desc* c, int64_t budget, int64_t recent) {
  if (check_evict(c, budget, recent) || c->batch == 0) return 0;
  const int64_t slices = evict_slices(c, budget, recent);
  return slices > 1 ? (size_t)c->batch * c->kv_heads * slices * kEvictSlots * 4 : 0;
}

extern "C" int attnres_cache_evict(const attnres_cache_desc* c, const int32_t* new_table, int64_t new_stride,
                                   int64_t budget, int64_t recent, int32_t* kept, int32_t* left, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (int rc = check_evict(c, budget, recent)) return rc;
  if (c->batch == 0) return ATTNRES_OK;
  if (!new_table || !kept || !left) return api_fail(ATTNRES_EINVAL, "new_table / kept / left is NULL");
  if (c->pages > 0 && !c->weights) return api_fail(ATTNRES_EINVAL, "weights is NULL");
  if (new_stride < (budget + c->page_size - 1) / c->page_size && c->batch > 1)
    return api_fail(ATTNRES_EINVAL, "new_stride=%lld below the pages of %lld tokens", (long long)new_stride, (long long)budget);
  const size_t need = attnres_cache_evict_workspace_size(c, budget, recent);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 256)))
    return api_fail(ATTNRES_EWORKSPACE, "workspace of %zu bytes needed, got %zu", need, workspace ? workspace_bytes : (size_t)0);
  CacheEvictParams p{};
  p.c = pages_of(c);
  p.new_table = new_table;
  p.new_stride = new_stride;
  p.budget = (int32_t)budget;
  p.recent = (int32_t)recent;
  p.kept = kept;
  p.left = left;
  p.es = es_of(c->dtype);
  p.slices = (int32_t)evict_slices(c, budget, recent);
  p.hist = (int32_t*)workspace;
  p.vb = row_bytes(c);
  const hipError_t err = launch_cache_evict(p, (hipStream_t)stream);
  if (err != hipSuccess) return api_fail(ATTNRES_ELAUNCH, "cache evict launch failed: %s", hipGetErrorString(err));
  return ATTNRES_OK;
}
