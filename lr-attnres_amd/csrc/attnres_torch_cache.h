// Host side of the paged cache's calls (qkv_norm_rotary_cached, cached_attention,
// evict_cached_tokens): part of attnres_torch.cpp, inside its namespace, with its rules
// -- plain eager calls only, None for everything else.

bool ints(const py::object& o, const Tensor& like, Tensor* out) {
  return unpack(o.ptr(), out) && out->scalar_type() == at::kInt && out->device() == like.device();
}

bool counts(const py::object& o, const Tensor& like, int64_t B, Tensor* out) {
  return ints(o, like, out) && out->dim() == 1 && out->size(0) == B && (B <= 1 || out->stride(0) == 1);
}

bool overlaps(const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return true;
  return false;
}

struct Cache {
  Tensor k, v, w, table, cached, fresh;
  attnres_cache_desc d = {};
};

// the cache of `batch` sequences (-1: as many as the table has rows)
bool cache_of(const py::object& k_, const py::object& v_, const py::object& w_, const py::object& table_,
              const py::object& cached_, const py::object& fresh_, int64_t batch, bool writes, Cache* c) {
  if (!unpack(k_.ptr(), &c->k) || !unpack(v_.ptr(), &c->v) || !unpack_opt(w_, &c->w)) return false;
  const Tensor &k = c->k, &v = c->v, &w = c->w;
  if (k.dim() != 4 || dtype_code(k.scalar_type()) < 0 || k.numel() < 1 || k.size(3) > ATTNRES_CACHE_MAX_HEAD_DIM) return false;
  if (v.scalar_type() != k.scalar_type() || v.device() != k.device() || v.sizes() != k.sizes() || v.strides() != k.strides() ||
      !last_dense(k))
    return false;
  if (w.defined() && (w.dim() != 3 || w.sizes() != k.sizes().slice(0, 3) || w.scalar_type() != at::kFloat ||
                      w.device() != k.device() || !last_dense(w) || overlaps(w)))
    return false;
  if (writes && (overlaps(k) || overlaps(v))) return false;
  if (!ints(table_, k, &c->table) || c->table.dim() != 2 || c->table.numel() < 1 || !last_dense(c->table)) return false;
  if (batch < 0) batch = c->table.size(0);
  if (c->table.size(0) != batch || c->table.size(1) > ATTNRES_CACHE_MAX_TOKENS / k.size(2)) return false;
  if (!counts(cached_, k, batch, &c->cached)) return false;
  if (!fresh_.is_none() && !counts(fresh_, k, batch, &c->fresh)) return false;
  if (any_grad({k, v, w})) return false;
  attnres_cache_desc& d = c->d;
  d.dtype = dtype_code(k.scalar_type());
  d.pages = k.size(0);
  d.kv_heads = (int)k.size(1);
  d.page_size = (int)k.size(2);
  d.head_dim = (int)k.size(3);
  d.k = k.data_ptr();
  d.v = v.data_ptr();
  d.page_stride = k.size(0) > 1 ? k.stride(0) : 0;
  d.head_stride = k.size(1) > 1 ? k.stride(1) : 0;
  d.slot_stride = k.size(2) > 1 ? k.stride(2) : 0;
  if (w.defined()) {
    d.weights = w.data_ptr<float>();
    d.weight_page_stride = w.size(0) > 1 ? w.stride(0) : 0;
    d.weight_head_stride = w.size(1) > 1 ? w.stride(1) : 0;
  }
  d.batch = batch;
  d.block_table = c->table.data_ptr<int32_t>();
  d.table_stride = batch > 1 ? c->table.stride(0) : 0;
  d.table_pages = c->table.size(1);
  d.cached = c->cached.data_ptr<int32_t>();
  d.fresh = c->fresh.defined() ? c->fresh.data_ptr<int32_t>() : nullptr;
  return true;
}

// a tensor that a kernel wrote in place, as autograd sees it
void written(const Tensor& t) {
  if (t.defined()) t.unsafeGetTensorImpl()->bump_version();
}

py::object cache_append(const py::object& projected, int64_t H, const py::object& sin_, const py::object& cos_,
                        const py::object& k_, const py::object& v_, const py::object& table_, const py::object& cached_,
                        const py::object& fresh_, const py::object& positions_, bool qk_norm, const py::object& w_,
                        bool heads) {
  Tensor qkv, sin, cos, at;
  Cache c;
  if (!plain_mode() || !unpack(projected.ptr(), &qkv) || !unpack(sin_.ptr(), &sin) || !unpack(cos_.ptr(), &cos))
    return py::none();
  if (qkv.dim() != 3 || qkv.numel() < 1 || !last_dense(qkv) || any_grad({qkv, sin, cos})) return py::none();
  const int64_t B = qkv.size(0), T = qkv.size(1);
  if (!cache_of(k_, v_, w_, table_, cached_, fresh_, B, true, &c)) return py::none();
  const int64_t K = c.d.kv_heads, Dh = c.d.head_dim;
  if (qkv.scalar_type() != c.k.scalar_type() || qkv.device() != c.k.device() || Dh % 2) return py::none();
  if (H < 1 || H > (1 << 20) || qkv.size(2) != (H + 2 * K) * Dh) return py::none();
  if (!rotary_table(sin, qkv, Dh / 2) || !rotary_table(cos, qkv, Dh / 2) || sin.sizes() != cos.sizes() ||
      sin.scalar_type() != cos.scalar_type())
    return py::none();
  if (!positions_.is_none() && !counts(positions_, qkv, B, &at)) return py::none();
  attnres_cache_append_desc d = {};
  d.tokens = T;
  d.q_heads = (int)H;
  d.qk_norm = qk_norm;
  d.norm_eps = kEps;
  d.table_dtype = dtype_code(sin.scalar_type());
  d.qkv = qkv.data_ptr();
  d.batch_stride = B > 1 ? qkv.stride(0) : 0;
  d.token_stride = T > 1 ? qkv.stride(1) : 0;
  d.sin = sin.data_ptr();
  d.cos = cos.data_ptr();
  d.table_row_stride = Dh / 2;
  d.table_rows = sin.numel() / d.table_row_stride;
  d.positions = at.defined() ? at.data_ptr<int32_t>() : nullptr;
  c10::DeviceGuard guard(qkv.device());
  const auto opt = qkv.options().requires_grad(false);
  Tensor q = at::empty({B, H, T, Dh}, opt), k;
  if (heads) k = at::empty({B, K, T, Dh}, opt);
  check(lib.attnres_cache_append(&c.d, &d, q.data_ptr(), ptr(k), stream_of(qkv.device())), "cache append");
  written(c.k);
  written(c.v);
  written(c.w);
  if (!heads) return py::cast(q);
  Tensor v = qkv.as_strided({B, K, T, Dh}, {qkv.stride(0), Dh, qkv.stride(1), 1}, qkv.storage_offset() + (H + K) * Dh);
  return py::make_tuple(q, k, v);
}

py::object cache_attend(const py::object& q_, const py::object& k_, const py::object& v_, const py::object& table_,
                        const py::object& cached_, const py::object& fresh_, const py::object& scale_, const py::object& w_,
                        const py::object& decay_) {
  Tensor q;
  Cache c;
  if (!plain_mode() || !unpack(q_.ptr(), &q) || q.dim() != 4 || q.numel() < 1 || !last_dense(q) || any_grad({q}))
    return py::none();
  if (!cache_of(k_, v_, w_, table_, cached_, fresh_, q.size(0), false, &c)) return py::none();
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), Dh = q.size(3);
  if (q.scalar_type() != c.k.scalar_type() || q.device() != c.k.device() || Dh != c.d.head_dim || H % c.d.kv_heads ||
      H > (1 << 20) || (c.w.defined() && T > 1))
    return py::none();
  attnres_cache_attend_desc d = {};
  if (!PyFloat_CheckExact(decay_.ptr())) return py::none();
  const double decay = PyFloat_AS_DOUBLE(decay_.ptr());
  if (!(decay >= 0.0 && decay <= 1.0)) return py::none();
  d.decay = (float)decay;
  if (scale_.is_none()) {
    d.scale = (float)(1.0 / std::sqrt((double)Dh));
  } else {
    if (!PyFloat_CheckExact(scale_.ptr())) return py::none();
    d.scale = (float)PyFloat_AS_DOUBLE(scale_.ptr());
    if (!(std::fabs(d.scale) <= ATTNRES_CACHE_MAX_SCALE)) return py::none();
  }
  d.tokens = T;
  d.q_heads = (int)H;
  d.q = q.data_ptr();
  d.q_batch_stride = B > 1 ? q.stride(0) : 0;
  d.q_head_stride = H > 1 ? q.stride(1) : 0;
  d.q_token_stride = T > 1 ? q.stride(2) : 0;
  c10::DeviceGuard guard(q.device());
  Tensor out = at::empty({B, T, H, Dh}, q.options().requires_grad(false)), ws;
  const size_t n = lib.attnres_cache_attend_workspace_size(&c.d, &d);
  if (n) ws = bytes(n, q.device());
  check(lib.attnres_cache_attend(&c.d, &d, out.data_ptr(), ptr(ws), n, stream_of(q.device())), "cache attend");
  written(c.w);
  return py::cast(out.transpose(1, 2));
}

py::object cache_evict(const py::object& k_, const py::object& v_, const py::object& w_, const py::object& table_,
                       const py::object& cached_, const py::object& new_, int64_t budget, int64_t recent) {
  Cache c;
  Tensor to;
  if (!plain_mode() || w_.is_none() || !cache_of(k_, v_, w_, table_, cached_, py::none(), -1, true, &c)) return py::none();
  const int64_t B = c.d.batch;
  if (budget < 1 || recent < 0 || recent > budget || budget > ATTNRES_CACHE_MAX_TOKENS) return py::none();
  if (!ints(new_, c.k, &to) || to.dim() != 2 || to.size(0) != B || !last_dense(to) || (B > 1 && to.stride(0) < to.size(1)) ||
      to.size(1) * c.d.page_size < budget)
    return py::none();
  c10::DeviceGuard guard(c.k.device());
  const auto opt = c.table.options();
  Tensor kept = at::empty({B, c.d.kv_heads, budget}, opt), left = at::empty({B}, opt);
  const size_t bytes_needed = lib.attnres_cache_evict_workspace_size(&c.d, budget, recent);
  Tensor ws;
  if (bytes_needed) ws = bytes(bytes_needed, c.k.device());
  check(lib.attnres_cache_evict(&c.d, to.data_ptr<int32_t>(), B > 1 ? to.stride(0) : to.size(1), budget, recent,
                                kept.data_ptr<int32_t>(), left.data_ptr<int32_t>(), ptr(ws), bytes_needed,
                                stream_of(c.k.device())),
        "cache evict");
  written(c.k);
  written(c.v);
  written(c.w);
  return py::make_tuple(kept, left);
}
