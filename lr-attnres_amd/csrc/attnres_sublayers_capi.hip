// C ABI of the sublayer kernels: argument checks, kernel selection and launch
// geometry.  Declared in include/attnres_sublayers.h.
#include <string.h>

#include "../../include/attnres_sublayers.h"
#include "attnres_sublayers.h"
#include "attnres_swiglu.h"

using namespace attnres;

namespace {

int es_of(int dtype) { return dtype == ATTNRES_DTYPE_F32 ? 4 : 2; }
bool known(int dtype) {
  return dtype == ATTNRES_DTYPE_F32 || dtype == ATTNRES_DTYPE_BF16 || dtype == ATTNRES_DTYPE_F16;
}
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

int check_rotary(const attnres_qkv_rotary_desc* d) {
  if (!d) return api_fail(ATTNRES_EINVAL, "desc is NULL");
  if (!known(d->dtype)) return api_fail(ATTNRES_EINVAL, "unknown dtype %d", d->dtype);
  if (d->table_dtype != ATTNRES_DTYPE_F32 && d->table_dtype != d->dtype)
    return api_fail(ATTNRES_EINVAL, "table dtype %d is neither fp32 nor the values' %d", d->table_dtype, d->dtype);
  if (d->batch < 0 || d->tokens < 0)
    return api_fail(ATTNRES_EINVAL, "batch=%lld, tokens=%lld must be >= 0", (long long)d->batch, (long long)d->tokens);
  if (d->q_heads < 1 || d->kv_heads < 1 || d->q_heads > (1 << 20) || d->kv_heads > (1 << 20))
    return api_fail(ATTNRES_EINVAL, "q_heads=%d, kv_heads=%d must be >= 1", d->q_heads, d->kv_heads);
  if (d->head_dim < 2 || d->head_dim % 2)
    return api_fail(ATTNRES_EINVAL, "head_dim=%d must be even and >= 2", d->head_dim);
  if (d->head_dim > ATTNRES_QKV_ROTARY_MAX_HEAD_DIM)
    return api_fail(ATTNRES_EUNSUPPORTED, "head_dim=%d above %d", d->head_dim, ATTNRES_QKV_ROTARY_MAX_HEAD_DIM);
  if (d->batch == 0 || d->tokens == 0) return ATTNRES_OK;
  if (d->batch > INT64_MAX / d->tokens || d->batch * d->tokens > (int64_t)1 << 40)
    return api_fail(ATTNRES_EUNSUPPORTED, "too many tokens");
  if (!d->qkv || !d->sin || !d->cos) return api_fail(ATTNRES_EINVAL, "qkv / sin / cos is NULL");
  if (d->batch_stride < 0 || d->token_stride < 0)
    return api_fail(ATTNRES_EINVAL, "batch_stride and token_stride must be >= 0");
  if (d->table_rows < 1) return api_fail(ATTNRES_EINVAL, "table_rows=%lld < 1", (long long)d->table_rows);
  if (d->table_row_stride < d->head_dim / 2)
    return api_fail(ATTNRES_EINVAL, "table_row_stride=%lld below head_dim / 2 = %d", (long long)d->table_row_stride,
                    d->head_dim / 2);
  if (!d->positions && (d->start < 0 || d->start > d->table_rows - d->tokens))
    return api_fail(ATTNRES_EINVAL, "rows %lld .. %lld are outside the tables' %lld", (long long)d->start,
                    (long long)(d->start + d->tokens - 1), (long long)d->table_rows);
  return ATTNRES_OK;
}

void fill_rotary(const attnres_qkv_rotary_desc* d, QkvRotaryParams* p) {
  memset(p, 0, sizeof(*p));
  p->qkv = d->qkv;
  p->b_stride = d->batch_stride;
  p->t_stride = d->token_stride;
  p->n_tok = d->batch * d->tokens;
  p->tokens = d->tokens;
  p->q_heads = d->q_heads;
  p->kv_heads = d->kv_heads;
  p->head_dim = d->head_dim;
  p->qk_norm = d->qk_norm != 0;
  p->eps = d->norm_eps;
  p->sin = d->sin;
  p->cos = d->cos;
  p->table_rows = d->table_rows;
  p->table_stride = d->table_row_stride;
  p->pos = d->positions;
  p->pos_b_stride = d->positions_batch_stride;
  p->pos_t_stride = d->positions_token_stride;
  p->start = d->start;
}

// The widest vector that every row starts at a multiple of, and the lanes that
// cover a head with it; vec 1 is the general kernel (any alignment).
void rotary_layout(const attnres_qkv_rotary_desc* d, const QkvRotaryParams& p, int* vec, int* lanes, int* chunks) {
  const int es = es_of(d->dtype), ts = es_of(d->table_dtype), Dh = d->head_dim;
  for (int v = es == 4 ? 4 : 8; v >= 2; v /= 2) {
    bool ok = Dh % v == 0 && aligned(p.qkv, (int64_t)v * es) && p.b_stride % v == 0 && p.t_stride % v == 0 &&
              aligned(p.sin, (int64_t)v / 2 * ts) && aligned(p.cos, (int64_t)v / 2 * ts) &&
              p.table_stride % (v / 2) == 0 && aligned(p.q, (int64_t)v * es) && aligned(p.k, (int64_t)v * es) &&
              aligned(p.dqkv, (int64_t)v * es);
    for (int i = 0; i < 3 && ok; ++i) {
      if (!p.grad[i]) continue;
      ok = aligned(p.grad[i], (int64_t)v * es);
      for (int j = 0; j < 3; ++j) ok = ok && p.grad_stride[i][j] % v == 0;
    }
    if (!ok) continue;
    *chunks = 1;
    for (*lanes = v == 8 ? 4 : v == 4 ? 8 : 32; *lanes <= (v == 8 ? 32 : 64); *lanes *= 2)
      if (*lanes * v >= Dh) {
        *vec = v;
        return;
      }
    if (v == 2 && Dh <= 256) {
      *vec = 2;
      *lanes = 64;
      *chunks = 2;
      return;
    }
  }
  *vec = *lanes = *chunks = 1;
}

}  // namespace

extern "C" int attnres_qkv_rotary_forward(const attnres_qkv_rotary_desc* d, void* q, void* k, void* stream) {
  if (int rc = check_rotary(d)) return rc;
  if (d->batch == 0 || d->tokens == 0) return ATTNRES_OK;
  if (!q || !k) return api_fail(ATTNRES_EINVAL, "q / k is NULL");
  QkvRotaryParams p;
  fill_rotary(d, &p);
  p.q = q;
  p.k = k;
  int vec, lanes, chunks;
  rotary_layout(d, p, &vec, &lanes, &chunks);
  const hipError_t err = launch_qkv_rotary(d->dtype, d->table_dtype == ATTNRES_DTYPE_F32, false, p, vec, lanes, chunks,
                                           (hipStream_t)stream);
  if (err != hipSuccess) return api_fail(ATTNRES_ELAUNCH, "qkv rotary forward launch failed: %s", hipGetErrorString(err));
  return ATTNRES_OK;
}

extern "C" int attnres_qkv_rotary_backward(const attnres_qkv_rotary_desc* d, const void* const* grads,
                                           const int64_t* strides, void* dqkv, void* stream) {
  if (int rc = check_rotary(d)) return rc;
  if (d->batch == 0 || d->tokens == 0) return ATTNRES_OK;
  if (!grads || !strides || !dqkv) return api_fail(ATTNRES_EINVAL, "grads / strides / dqkv is NULL");
  QkvRotaryParams p;
  fill_rotary(d, &p);
  for (int i = 0; i < 3; ++i) {
    p.grad[i] = grads[i];
    for (int j = 0; j < 3; ++j) {
      p.grad_stride[i][j] = grads[i] ? strides[3 * i + j] : 0;
      if (p.grad_stride[i][j] < 0) return api_fail(ATTNRES_EINVAL, "negative gradient stride");
    }
  }
  p.dqkv = dqkv;
  int vec, lanes, chunks;
  rotary_layout(d, p, &vec, &lanes, &chunks);
  const hipError_t err = launch_qkv_rotary(d->dtype, d->table_dtype == ATTNRES_DTYPE_F32, true, p, vec, lanes, chunks,
                                           (hipStream_t)stream);
  if (err != hipSuccess) return api_fail(ATTNRES_ELAUNCH, "qkv rotary backward launch failed: %s", hipGetErrorString(err));
  return ATTNRES_OK;
}

// ---------------------------------------------------------------- gated feed-forward

namespace {

constexpr int kCus = 256;

struct SwLayout {
  int es, per, step;   // bytes of a value, values of a chunk and of a k step
  int Fp;              // hidden, in whole steps
  int Dp;              // dim, in whole chunks
  bool x_ok, w_ok;     // the products can read the operand as it is
  bool w_ok_dx;        // and dx the weight: its halves fill k steps
};

int round_up(int v, int to) { return (v + to - 1) / to * to; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

SwLayout sw_layout(const attnres_swiglu_desc* d) {
  SwLayout l;
  l.es = es_of(d->dtype);
  l.per = 16 / l.es;
  l.step = kSwStepBytes / l.es;
  l.Fp = round_up(d->hidden, l.step);
  l.Dp = round_up(d->dim, l.per);
  // direct loads of 16 bytes; a tile's rows within 32-bit offsets of its first one
  const int64_t far = ((int64_t)1 << 32) / (256 * l.es) - d->dim;
  l.x_ok = d->dim % l.per == 0 && aligned(d->x, 16) && d->x_row_stride % l.per == 0 && d->x_row_stride < far;
  l.w_ok = d->dim % l.per == 0 && aligned(d->weight, 16) && d->weight_row_stride % l.per == 0 &&
           d->weight_row_stride < far &&
           (int64_t)2 * d->hidden * d->weight_row_stride * l.es < (int64_t)1 << 32;
  l.w_ok_dx = l.w_ok && d->hidden == l.Fp;
  return l;
}

// Tile and splits of a product with `steps` k steps: the least cost in a model of a
// launch.  The CUs take workgroups in rounds, as many together as LDS holds;
// together they share the matrix cores.  A split product's sums are written and read
// once more, by a second launch.  The constants were fitted, in us, to 1900 launches of these
// products before their last speed-up (24 shapes of 60 to 16384 tokens, every tile, 1 to 64
// splits, fp32 and bf16).  They rank choices and are no times: the model has no term for what a
// tile stores (16384 tokens, dim 1024, hidden 4096, bf16: 215 for a forward of 304 us) nor for the
// single-value stores of odd widths.  Its choices, measured again since: 1422 launches of 63 products (100 to 16384
// tokens; dx and dw with the activation's gradient before them): the model's choice is 1.3%
// slower than the best one in the mean, 17% at most (dx of 100 tokens, dim 512, hidden 1024:
// 13.3 us, 11.4 with 8 splits) and 8% otherwise.
// The large tile moves the least data a product, the small one fills the CUs: forward of
// 2000 tokens, dim 1024, hidden 4096, bf16, with what the backward needs: 38 us with 256 x
// 256, 39 with 128 x 128, 45 with 64 x 128; of 512 tokens, dim 1024, hidden 1024: 8.9 with
// 64 x 128, 11.8 with 128 x 128.
struct SwShape {
  int tile, tiles_m, tiles_n, splits, steps;
};

struct SwCosts {
  double step[kSwTiles];      // a k step of one workgroup
  double together[kSwTiles];  // of g workgroups on a CU: g * together times that, if more
  double fixed[kSwTiles];     // a workgroup's begin and end
  double launch, bytes_us;    // a split's second launch, and its traffic
};
constexpr SwCosts kCost16 = {{0.638, 0.394, 0.239, 0.181}, {1.0, 0.961, 0.899, 0.778}, {6.45, 3.35, 2.63, 1.82}, 4.17, 9.5e6};
constexpr SwCosts kCost32 = {{3.955, 2.036, 1.024, 0.557}, {1.0, 0.934, 0.971, 0.912}, {4.25, 0.92, 0.88, 0.2}, 5.31, 7.9e6};

SwShape sw_shape(int form, int dtype, int64_t M, int N, int steps) {  // (forward: of two k steps each)
  const SwCosts& k = dtype == ATTNRES_DTYPE_F32 ? kCost32 : kCost16;
  SwShape best{};
  double least = 1e300;
  for (int t = 0; t < kSwTiles; ++t) {
    if (!sw_has_tile(form, dtype, t)) continue;
    const int cols = form == kFwd ? kSwTileN[t] / 2 : kSwTileN[t];
    const int64_t tm = (M + kSwTileM[t] - 1) / kSwTileM[t], tn = (N + cols - 1) / cols;
    const int together = sw_per_cu(kSwTileM[t], kSwTileN[t]);
    for (int splits = 1; splits <= 64 && splits <= steps; ++splits) {
      const int per = (steps + splits - 1) / splits;
      if ((steps + per - 1) / per != splits) continue;
      const int64_t wgs = tm * tn * splits;
      if (wgs >= (1 << 24)) break;  // fewer than 2^32 threads
      const int64_t rounds = (wgs + kCus - 1) / kCus;  // workgroups that one CU works on
      auto group = [&](int g) { return (form == kFwd ? 2 : 1) * per * k.step[t] * (g * k.together[t] > 1.0 ? g * k.together[t] : 1.0) + k.fixed[t]; };
      double cost = (double)(rounds / together) * group(together);
      if (rounds % together) cost += group((int)(rounds % together));
      if (splits > 1) cost += k.launch + (double)wgs * kSwTileM[t] * kSwTileN[t] * 8 / k.bytes_us;
      if (cost < least) {
        least = cost;
        best = SwShape{t, (int)tm, (int)tn, splits, per};
      }
    }
  }
  return best;
}

size_t sw_partials(const SwShape& s) {
  return s.splits > 1 ? up256((size_t)s.splits * s.tiles_m * s.tiles_n * kSwTileM[s.tile] * kSwTileN[s.tile] * 4) : 0;
}

int check_swiglu(const attnres_swiglu_desc* d) {
  if (!d) return api_fail(ATTNRES_EINVAL, "desc is NULL");
  if (!known(d->dtype)) return api_fail(ATTNRES_EINVAL, "unknown dtype %d", d->dtype);
  if (d->n_tok < 0) return api_fail(ATTNRES_EINVAL, "n_tok=%lld < 0", (long long)d->n_tok);
  if (d->dim < 1 || d->hidden < 1) return api_fail(ATTNRES_EINVAL, "dim=%d, hidden=%d must be >= 1", d->dim, d->hidden);
  if (d->n_tok > (1 << 22) || d->dim > (1 << 20) || d->hidden > (1 << 20) ||
      (int64_t)2 * round_up(d->hidden, 32) * round_up(d->dim, 8) * es_of(d->dtype) >= (int64_t)1 << 32)
    return api_fail(ATTNRES_EUNSUPPORTED, "n_tok=%lld, dim=%d, hidden=%d: outside the kernels' 32-bit offsets",
                    (long long)d->n_tok, d->dim, d->hidden);
  if (d->n_tok == 0) return ATTNRES_OK;
  if (!d->x || !d->weight) return api_fail(ATTNRES_EINVAL, "x / weight is NULL");
  if (d->n_tok > 1 && d->x_row_stride < 0) return api_fail(ATTNRES_EINVAL, "x_row_stride < 0");
  if (d->weight_row_stride < d->dim)
    return api_fail(ATTNRES_EINVAL, "weight_row_stride=%lld < dim=%d", (long long)d->weight_row_stride, d->dim);
  return ATTNRES_OK;
}

SwShape fwd_shape(const attnres_swiglu_desc* d, const SwLayout& l) {
  return sw_shape(kFwd, d->dtype, d->n_tok, d->hidden, (d->dim + 2 * l.step - 1) / (2 * l.step));
}
SwShape dx_shape(const attnres_swiglu_desc* d, const SwLayout& l) {
  return sw_shape(kDx, d->dtype, d->n_tok, d->dim, 2 * l.Fp / l.step);
}
SwShape dw_shape(const attnres_swiglu_desc* d, const SwLayout& l) {
  return sw_shape(kDw, d->dtype, 2 * l.Fp, d->dim, (int)((d->n_tok + l.step - 1) / l.step));
}

size_t packed_x(const attnres_swiglu_desc* d, const SwLayout& l) {
  return l.x_ok ? 0 : up256((size_t)d->n_tok * l.Dp * l.es);
}
size_t packed_w(const attnres_swiglu_desc* d, const SwLayout& l, bool dx) {
  return (dx ? l.w_ok_dx : l.w_ok) ? 0 : up256((size_t)2 * (dx ? l.Fp : d->hidden) * l.Dp * l.es);
}

// the operands as the products read them: where they are, or (one launch) copied
struct SwOperands {
  const void *x, *w;
  int64_t x_stride, w_stride;
};
hipError_t sw_operands(const attnres_swiglu_desc* d, const SwLayout& l, bool dx, char* x_to, char* w_to, hipStream_t st,
                       SwOperands* o) {
  *o = SwOperands{d->x, d->weight, d->x_row_stride, d->weight_row_stride};
  SwPackParams k{};
  k.cols = d->dim;
  k.to_stride = l.Dp;
  if (x_to) {
    k.part[k.parts++] = SwPack{d->x, x_to, d->n_tok, d->n_tok, d->x_row_stride, 1};
    o->x = x_to;
    o->x_stride = l.Dp;
  }
  if (w_to) {
    k.part[k.parts++] = SwPack{d->weight, w_to, d->hidden, dx ? l.Fp : d->hidden, d->weight_row_stride, 2};
    o->w = w_to;
    o->w_stride = l.Dp;
  }
  return k.parts ? launch_swiglu_pack(d->dtype, k, st) : hipSuccess;
}

void set_shape(const SwShape& s, SwGemmParams* g) {
  g->tiles_m = s.tiles_m;
  g->tiles_n = s.tiles_n;
  g->splits = s.splits;
  g->steps = s.steps;
}

}  // namespace

extern "C" size_t attnres_swiglu_saved_size(const attnres_swiglu_desc* d) {
  if (check_swiglu(d) || d->n_tok == 0) return 0;
  const SwLayout l = sw_layout(d);
  const size_t low = d->dtype == ATTNRES_DTYPE_F32 ? 0 : 2 * (d->dtype == ATTNRES_DTYPE_BF16 ? 4 : 8);  // bits a pair
  return (size_t)d->n_tok * l.Fp * 2 * l.es + (size_t)d->n_tok * l.Fp * low / 8;
}

extern "C" size_t attnres_swiglu_forward_workspace_size(const attnres_swiglu_desc* d) {
  if (check_swiglu(d) || d->n_tok == 0) return 0;
  const SwLayout l = sw_layout(d);
  return packed_x(d, l) + packed_w(d, l, false) + (d->n_tok <= kSwFew ? 0 : sw_partials(fwd_shape(d, l)));
}

namespace {

// The backward's products (only those that are wanted: the search for one takes a microsecond, and a product that
// nobody asked for refuses no call) and its workspace: [du dz], copied operands, one product's partial sums at a time.
struct SwBackward {
  SwShape dx, dw;
  size_t d, x, w, need;
};
SwBackward sw_backward(const attnres_swiglu_desc* d, const SwLayout& l, bool want_dx, bool want_dw) {
  SwBackward b{};
  if (want_dx) b.dx = dx_shape(d, l);
  if (want_dw) b.dw = dw_shape(d, l);
  b.d = up256((size_t)d->n_tok * 2 * l.Fp * l.es);
  b.x = want_dw ? packed_x(d, l) : 0;
  b.w = want_dx ? packed_w(d, l, true) : 0;
  const size_t dx = want_dx ? sw_partials(b.dx) : 0, dw = want_dw ? sw_partials(b.dw) : 0;
  b.need = b.d + b.x + b.w + (dx > dw ? dx : dw);
  return b;
}

}  // namespace

extern "C" size_t attnres_swiglu_backward_workspace_size(const attnres_swiglu_desc* d, int32_t want_dx, int32_t want_dw) {
  if (check_swiglu(d) || d->n_tok == 0) return 0;
  return sw_backward(d, sw_layout(d), want_dx != 0, want_dw != 0).need;
}

extern "C" int attnres_swiglu_forward(const attnres_swiglu_desc* d, void* h, void* saved, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  if (int rc = check_swiglu(d)) return rc;
  if (d->n_tok == 0) return ATTNRES_OK;
  if (!h) return api_fail(ATTNRES_EINVAL, "h is NULL");
  if (saved && !aligned(saved, 16)) return api_fail(ATTNRES_EINVAL, "saved is not aligned to 16 bytes");
  const SwLayout l = sw_layout(d);
  const bool few = d->n_tok <= kSwFew;
  const SwShape s = few ? SwShape{0, 0, 0, 1, 1} : fwd_shape(d, l);
  const size_t px = packed_x(d, l), pw = packed_w(d, l, false), need = px + pw + sw_partials(s);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 256)))
    return api_fail(ATTNRES_EWORKSPACE, "workspace of %zu bytes needed, got %zu", need, workspace ? workspace_bytes : (size_t)0);
  if (!s.steps) return api_fail(ATTNRES_EUNSUPPORTED, "too many tiles");
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace;
  SwGemmParams g{};
  SwOperands o;
  hipError_t err = sw_operands(d, l, false, px ? ws : nullptr, pw ? ws + px : nullptr, st, &o);
  g.q = o.x;
  g.q_stride = o.x_stride;
  g.p = o.w;
  g.p_stride = o.w_stride;
  g.M = (int)d->n_tok;
  g.N = g.F = g.n_out = d->hidden;
  g.Fp = l.Fp;
  g.K = l.Dp;
  g.n_tok = d->n_tok;
  set_shape(s, &g);
  g.out = h;
  g.out_stride = d->hidden;
  g.out_vec = d->hidden % l.per == 0 && aligned(h, 16);
  g.saved = saved;
  g.partials = (float*)(ws + px + pw);
  if (err == hipSuccess) err = few ? launch_swiglu_few(d->dtype, g, st) : launch_swiglu_gemm(d->dtype, kFwd, s.tile, g, st);
  if (err != hipSuccess) return api_fail(ATTNRES_ELAUNCH, "swiglu forward launch failed: %s", hipGetErrorString(err));
  return ATTNRES_OK;
}

extern "C" int attnres_swiglu_backward(const attnres_swiglu_desc* d, const void* grad_h, int64_t grad_row_stride,
                                       const void* saved, void* dx, void* dweight, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  if (int rc = check_swiglu(d)) return rc;
  hipStream_t st = (hipStream_t)stream;
  hipError_t err = hipSuccess;
  if (d->n_tok == 0) {
    if (dweight) err = launch_swiglu_clear(d->dtype, dweight, (int64_t)2 * d->hidden * d->dim, st);
    if (err != hipSuccess) return api_fail(ATTNRES_ELAUNCH, "swiglu backward launch failed: %s", hipGetErrorString(err));
    return ATTNRES_OK;
  }
  if (!dx && !dweight) return ATTNRES_OK;
  if (!grad_h || !saved) return api_fail(ATTNRES_EINVAL, "grad_h / saved is NULL");
  if (!aligned(saved, 16)) return api_fail(ATTNRES_EINVAL, "saved is not aligned to 16 bytes");
  if (grad_row_stride < 0) return api_fail(ATTNRES_EINVAL, "grad_row_stride < 0");
  const SwLayout l = sw_layout(d);
  const SwBackward b = sw_backward(d, l, dx != nullptr, dweight != nullptr);
  if ((dx && !b.dx.steps) || (dweight && !b.dw.steps)) return api_fail(ATTNRES_EUNSUPPORTED, "too many tiles");
  if (!workspace || workspace_bytes < b.need || !aligned(workspace, 256))
    return api_fail(ATTNRES_EWORKSPACE, "workspace of %zu bytes needed, got %zu", b.need, workspace ? workspace_bytes : (size_t)0);
  char* ws = (char*)workspace;
  float* const partials = (float*)(ws + b.d + b.x + b.w);
  SwGradParams e{};
  e.dh = grad_h;
  e.dh_stride = grad_row_stride;
  e.saved = saved;
  e.d = ws;
  e.n = d->n_tok;
  e.F = d->hidden;
  e.Fp = l.Fp;
  e.vec = aligned(grad_h, 16) && grad_row_stride % l.per == 0;
  SwOperands o;
  err = sw_operands(d, l, true, b.x ? ws + b.d : nullptr, b.w ? ws + b.d + b.x : nullptr, st, &o);
  if (err == hipSuccess) err = launch_swiglu_grad(d->dtype, e, st);
  if (dx && err == hipSuccess) {
    SwGemmParams g{};
    g.p = o.w;
    g.p_stride = o.w_stride;
    g.q = ws;
    g.n_tok = d->n_tok;
    g.M = (int)d->n_tok;
    g.N = l.Dp;
    g.K = 2 * l.Fp;
    g.F = d->hidden;
    g.Fp = l.Fp;
    set_shape(b.dx, &g);
    g.out = dx;
    g.out_stride = d->dim;
    g.n_out = d->dim;
    g.out_vec = d->dim % l.per == 0 && aligned(dx, 16);
    g.partials = partials;
    err = launch_swiglu_gemm(d->dtype, kDx, b.dx.tile, g, st);
  }
  if (dweight && err == hipSuccess) {
    SwGemmParams g{};
    g.p = o.x;
    g.p_stride = o.x_stride;
    g.q = ws;
    g.n_tok = d->n_tok;
    g.M = 2 * l.Fp;
    g.N = l.Dp;
    g.K = (int)d->n_tok;
    g.F = d->hidden;
    g.Fp = l.Fp;
    set_shape(b.dw, &g);
    g.out = dweight;
    g.out_stride = d->dim;
    g.n_out = d->dim;
    g.out_vec = d->dim % l.per == 0 && aligned(dweight, 16);
    g.partials = partials;
    err = launch_swiglu_gemm(d->dtype, kDw, b.dw.tile, g, st);
  }
  if (err != hipSuccess) return api_fail(ATTNRES_ELAUNCH, "swiglu backward launch failed: %s", hipGetErrorString(err));
  return ATTNRES_OK;
}
