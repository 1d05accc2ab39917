// Host side of the sublayer calls (qkv_norm_rotary, swiglu_projection): part of
// attnres_torch.cpp, inside its namespace, with its rules -- plain eager calls only,
// None for everything else.

// ------------------------------------------------------------------ the heads of a projection

struct RotaryMeta : torch::CustomClassHolder {
  int64_t H = 0, K = 0, start = 0;
  bool qk_norm = true;
};

int64_t last_dense(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

// qkv [B, T, C], sin / cos [rows, Dh / 2] dense, positions [T] or [B, T] int64 or undefined
void fill_rotary(const RotaryMeta& m, const Tensor& qkv, const Tensor& sin, const Tensor& cos, const Tensor& at,
                 attnres_qkv_rotary_desc* d) {
  *d = {};
  d->dtype = dtype_code(qkv.scalar_type());
  d->table_dtype = dtype_code(sin.scalar_type());
  d->batch = qkv.size(0);
  d->tokens = qkv.size(1);
  d->q_heads = (int)m.H;
  d->kv_heads = (int)m.K;
  d->head_dim = (int)(qkv.size(2) / (m.H + 2 * m.K));
  d->qk_norm = m.qk_norm;
  d->norm_eps = kEps;
  d->qkv = qkv.data_ptr();
  d->batch_stride = d->batch > 1 ? qkv.stride(0) : 0;
  d->token_stride = d->tokens > 1 ? qkv.stride(1) : 0;
  d->sin = sin.data_ptr();
  d->cos = cos.data_ptr();
  d->table_row_stride = sin.size(-1);
  d->table_rows = sin.numel() / sin.size(-1);
  if (at.defined()) {
    d->positions = at.data_ptr<int64_t>();
    d->positions_batch_stride = at.dim() == 2 ? at.stride(0) : 0;
    d->positions_token_stride = at.stride(-1);
  }
  d->start = m.start;
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  // in: qkv, sin, cos, positions where given; out: q, k, v (a view of qkv)
  static variable_list run(const RotaryMeta& m, const variable_list& in) {
    const Tensor& qkv = in[0];
    c10::DeviceGuard guard(qkv.device());
    attnres_qkv_rotary_desc d;
    fill_rotary(m, qkv, in[1], in[2], in.size() > 3 ? in[3] : Tensor(), &d);
    const auto opt = qkv.options().requires_grad(false);
    const int64_t B = d.batch, T = d.tokens, Dh = d.head_dim;
    Tensor q = at::empty({B, m.H, T, Dh}, opt), k = at::empty({B, m.K, T, Dh}, opt);
    check(lib.attnres_qkv_rotary_forward(&d, q.data_ptr(), k.data_ptr(), stream_of(qkv.device())), "qkv rotary forward");
    Tensor v = qkv.as_strided({B, m.K, T, Dh}, {qkv.stride(0), Dh, qkv.stride(1), 1},
                              qkv.storage_offset() + (m.H + m.K) * Dh);
    return {q, k, v};
  }

  static variable_list forward(AutogradContext* ctx, c10::intrusive_ptr<RotaryMeta> m, at::TensorList list) {
    variable_list in = list.vec();
    variable_list res = run(*m, in);
    ctx->saved_data["m"] = c10::IValue::make_capsule(m);
    ctx->save_for_backward(std::move(in));
    ctx->set_materialize_grads(false);
    return res;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    auto m = meta_of<RotaryMeta>(ctx);
    variable_list s = ctx->get_saved_variables();
    variable_list res(1 + s.size());
    if (!grads[0].defined() && !grads[1].defined() && !grads[2].defined()) return res;
    {
      at::NoGradGuard no_grad;
      // (a saved-tensor hook may give a tensor back in another layout)
      if (!last_dense(s[0])) s[0] = s[0].contiguous();
      for (int i = 1; i < 3; ++i) s[i] = s[i].contiguous();
      const Tensor& qkv = s[0];
      c10::DeviceGuard guard(qkv.device());
      attnres_qkv_rotary_desc d;
      fill_rotary(*m, qkv, s[1], s[2], s.size() > 3 ? s[3] : Tensor(), &d);
      Tensor g[3];
      const void* p[3];
      int64_t st[9] = {};
      for (int i = 0; i < 3; ++i) {
        if (grads[i].defined()) g[i] = last_dense(grads[i]) ? grads[i] : grads[i].contiguous();
        p[i] = ptr(g[i]);
        for (int j = 0; j < 3; ++j)
          if (g[i].defined() && g[i].size(j) > 1) st[3 * i + j] = g[i].stride(j);
      }
      Tensor out = at::empty(qkv.sizes(), qkv.options().requires_grad(false));
      check(lib.attnres_qkv_rotary_backward(&d, p, st, out.data_ptr(), stream_of(qkv.device())), "qkv rotary backward");
      res[1] = out;
    }
    return once(std::move(res), grads);
  }
};

bool rotary_table(const Tensor& t, const Tensor& qkv, int64_t half) {
  return t.dim() >= 2 && t.size(-1) == half && t.numel() > 0 && t.numel() == t.size(-2) * half && t.is_contiguous() && !t.requires_grad() &&
         t.device() == qkv.device() && (t.scalar_type() == at::kFloat || t.scalar_type() == qkv.scalar_type());
}

py::object qkv_rotary(const py::object& projected, int64_t H, int64_t K, const py::object& sin_, const py::object& cos_,
                      const py::object& positions, bool qk_norm) {
  Tensor qkv, sin, cos, at;
  if (!plain_mode() || !unpack(projected.ptr(), &qkv) || !unpack(sin_.ptr(), &sin) || !unpack(cos_.ptr(), &cos))
    return py::none();
  if (qkv.dim() != 3 || dtype_code(qkv.scalar_type()) < 0 || qkv.numel() < 1 || !last_dense(qkv)) return py::none();
  if (H < 1 || K < 1 || H > (1 << 20) || K > (1 << 20) || qkv.size(2) % (H + 2 * K)) return py::none();
  const int64_t T = qkv.size(1), Dh = qkv.size(2) / (H + 2 * K);
  if (Dh % 2 || Dh > ATTNRES_QKV_ROTARY_MAX_HEAD_DIM) return py::none();
  if (!rotary_table(sin, qkv, Dh / 2) || !rotary_table(cos, qkv, Dh / 2) || sin.sizes() != cos.sizes() ||
      sin.scalar_type() != cos.scalar_type())
    return py::none();
  auto m = c10::make_intrusive<RotaryMeta>();
  m->H = H;
  m->K = K;
  m->qk_norm = qk_norm;
  variable_list in = {qkv, sin, cos};
  if (PyLong_CheckExact(positions.ptr())) {
    int overflow = 0;
    m->start = PyLong_AsLongLongAndOverflow(positions.ptr(), &overflow);
    if (overflow) return py::none();
  } else if (!positions.is_none()) {
    if (!unpack(positions.ptr(), &at) || at.scalar_type() != at::kLong || at.device() != qkv.device()) return py::none();
    if (!(at.dim() == 1 && at.size(0) == T) && !(at.dim() == 2 && at.size(0) == qkv.size(0) && at.size(1) == T))
      return py::none();
    in.push_back(at);
  }
  if (!at.defined() && (m->start < 0 || m->start > sin.numel() / (Dh / 2) - T)) return py::none();
  variable_list res = any_grad({qkv}) ? RotaryFn::apply(m, at::TensorList(in)) : RotaryFn::run(*m, in);
  return py::make_tuple(res[0], res[1], res[2]);
}

// ------------------------------------------------------------------ the gated feed-forward projections

// elements between the rows of x [..., D]; -1: they are not uniform
int64_t uniform_rows(const Tensor& x) {
  const int64_t D = x.size(-1);
  if (D > 1 && x.stride(-1) != 1) return -1;
  int64_t row = -1, next = 0;  // the stride of the rows, and of the next outer dimension in it
  for (int64_t i = x.dim() - 2; i >= 0; --i) {
    if (x.size(i) == 1) continue;
    if (row < 0) row = x.stride(i), next = row * x.size(i);
    else if (x.stride(i) != next) return -1;
    else next *= x.size(i);
  }
  return row < 0 ? D : row;
}

void fill_swiglu(const Tensor& x, const Tensor& w, attnres_swiglu_desc* d) {
  *d = {};
  d->dtype = dtype_code(x.scalar_type());
  d->dim = (int)x.size(-1);
  d->n_tok = x.numel() / x.size(-1);
  d->hidden = (int)(w.size(0) / 2);
  d->x = x.data_ptr();
  d->x_row_stride = uniform_rows(x);
  d->weight = w.data_ptr();
  d->weight_row_stride = w.stride(0);
}

struct SwigluFn : torch::autograd::Function<SwigluFn> {
  static Tensor run(const Tensor& x, const Tensor& w, bool save, Tensor* saved) {
    c10::DeviceGuard guard(x.device());
    attnres_swiglu_desc d;
    fill_swiglu(x, w, &d);
    const auto opt = x.options().requires_grad(false);
    auto shape = x.sizes().vec();
    shape.back() = d.hidden;
    Tensor h = at::empty(shape, opt), ws;
    if (save) *saved = bytes(lib.attnres_swiglu_saved_size(&d), x.device());
    const size_t n = lib.attnres_swiglu_forward_workspace_size(&d);
    if (n) ws = bytes(n, x.device());
    check(lib.attnres_swiglu_forward(&d, h.data_ptr(), ptr(*saved), ptr(ws), n, stream_of(x.device())), "swiglu forward");
    return h;
  }

  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w) {
    Tensor saved;
    Tensor h = run(x, w, true, &saved);
    ctx->save_for_backward({x, w, saved});
    ctx->set_materialize_grads(false);
    return h;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list res(2);
    if (!grads[0].defined()) return res;
    variable_list s = ctx->get_saved_variables();
    {
      at::NoGradGuard no_grad;
      // (a saved-tensor hook may give a tensor back in another layout)
      if (uniform_rows(s[0]) < 0) s[0] = s[0].contiguous();
      if (!last_dense(s[1]) || s[1].stride(0) < s[1].size(1)) s[1] = s[1].contiguous();
      s[2] = s[2].contiguous();
      if ((uintptr_t)s[2].data_ptr() % 16) copy_dense(&s[2]);
      const Tensor &x = s[0], &w = s[1];
      c10::DeviceGuard guard(x.device());
      attnres_swiglu_desc d;
      fill_swiglu(x, w, &d);
      const Tensor go = uniform_rows(grads[0]) < 0 ? grads[0].contiguous() : grads[0];
      const auto opt = x.options().requires_grad(false);
      if (ctx->needs_input_grad(0)) res[0] = at::empty(x.sizes(), opt);
      if (ctx->needs_input_grad(1)) res[1] = at::empty(w.sizes(), opt);
      const size_t n = lib.attnres_swiglu_backward_workspace_size(&d, res[0].defined(), res[1].defined());
      Tensor ws = bytes(n, x.device());
      check(lib.attnres_swiglu_backward(&d, go.data_ptr(), uniform_rows(go), s[2].data_ptr(), ptr(res[0]), ptr(res[1]),
                                        ws.data_ptr(), n, stream_of(x.device())), "swiglu backward");
    }
    return once(std::move(res), grads);
  }
};

// An operand as a linear layer takes it: under autocast in the autocast dtype (fp64 as it is).  The cast is
// differentiable, and a weight's is kept by the autocast context as it keeps a linear layer's.
Tensor autocast_operand(const Tensor& t) {
  if (!at::autocast::is_autocast_enabled(at::kCUDA)) return t;
  const auto to = at::autocast::get_autocast_dtype(at::kCUDA);
  Tensor c = at::autocast::cached_cast(to, t, at::kCUDA);
  // (a cast that was kept from a call without gradients has none to give)
  if (at::GradMode::is_enabled() && t.requires_grad() && !c.requires_grad()) c = t.to(to);
  return c;
}

py::object swiglu(const py::object& x_, const py::object& w_) {
  Tensor x, w;
  if (!plain_mode() || !unpack(x_.ptr(), &x) || !unpack(w_.ptr(), &w)) return py::none();
  x = autocast_operand(x);
  w = autocast_operand(w);
  if (x.dim() < 1 || x.numel() < 1 || dtype_code(x.scalar_type()) < 0 || w.scalar_type() != x.scalar_type() ||
      w.device() != x.device() || w.dim() != 2 || w.size(1) != x.size(-1) || w.size(0) < 2 || w.size(0) % 2)
    return py::none();
  if (uniform_rows(x) < 0 || !last_dense(w) || w.stride(0) < w.size(1)) return py::none();
  if (any_grad({x, w})) return py::cast(SwigluFn::apply(x, w));
  Tensor none;
  return py::cast(SwigluFn::run(x, w, false, &none));
}
