// The host side of the wide layers (norm, 8-bit rows and products, the linear layer that keeps its input in 8 bits), in the manner of
// host_native.cpp: a function for the plain case that returns None for everything else, and launch functions on checked arguments for
// the Python functions that then take over.
#include "host_common.h"

namespace {

// An eager graph of a leaf that is still alive holds the node that adds up the leaf's gradient, on the stream that it was built on.  Where that is the
// default stream, which cannot take part in a capture, a captured backward would end there: it has to wait for the captured stream, and torch ends the
// process.  Refused in the forward, while nothing has happened yet.  (Any other stream joins the capture and is joined again.)
void refuse_eager_graph(const Tensor& t) {
  if (!t.defined() || !t.is_cuda() || !t.requires_grad() || !t.is_leaf()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (node == nullptr || node->num_inputs() == 0) return;
  if (node->input_metadata(0).stream().id() != c10::hip::getDefaultHIPStream(t.device().index()).id() ||
      c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None)
    return;
  TORCH_CHECK(false, "a graph that was built outside of this capture, on the default stream, still holds one of the leaves: delete what it computed (outputs, losses) before capturing a "
                     "step that takes gradients");
}

// refuse_eager_graphs(tensors or None ...): the same for the Python functions, in front of the autograd Functions that take over from here
PyObject* refuse_eager_graphs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (at::GradMode::is_enabled())
    for (Py_ssize_t i = 0; i < n; ++i)
      if (THPVariable_Check(a[i])) refuse_eager_graph(THPVariable_Unpack(a[i]));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

bool float_type(const Tensor& t) { return code_of(t.scalar_type()) >= 0; }

// ------------------------------------------------------------------------------------------------ norm
struct Norm {
  Tensor x, w, r;  // w, r: undefined without
  float eps;
  at::ScalarType stream_type() const { return r.defined() ? r.scalar_type() : x.scalar_type(); }
};

// An element type and sizes that the kernels take (the same conditions as the Python function's checks).
bool norm_fits(const Norm& m) {
  if (m.x.dim() < 1 || m.x.size(-1) < 1 || !float_type(m.x)) return false;
  if (m.w.defined() && (!float_type(m.w) || m.w.dim() != 1 || m.w.size(0) != m.x.size(-1) || m.w.device() != m.x.device())) return false;
  if (m.r.defined() && (m.r.sizes() != m.x.sizes() || m.r.device() != m.x.device() ||
                        (m.r.scalar_type() != m.x.scalar_type() && m.r.scalar_type() != at::kFloat)))
    return false;
  return m.eps >= 0.0f;
}

struct NormOut {
  Tensor y, scale, stream, rstd;
};

NormOut norm_forward(const Norm& m, bool eight, bool keep) {
  const c10::DeviceGuard guard(m.x.device());
  const int64_t width = m.x.size(-1);
  const Rows x(m.x, width);
  NormOut o;
  o.y = at::empty(m.x.sizes(), eight ? m.x.options().dtype(at::kChar) : m.x.options());
  if (eight) o.scale = at::empty(m.x.sizes().slice(0, m.x.dim() - 1), m.x.options().dtype(at::kFloat));
  if (keep) o.rstd = at::empty({x.n}, m.x.options().dtype(at::kFloat));
  std::optional<Rows> r;
  if (m.r.defined()) {
    r.emplace(m.r, width);
    o.stream = at::empty(m.r.sizes(), m.r.options());
  }
  const Tensor w = contiguous(m.w);
  check(nf_rms_norm_fwd(x.p, x.stride, code_of(m.x.scalar_type()), r ? r->p : nullptr, r ? r->stride : width, code_of(m.stream_type()), ptr(w),
                        w.defined() ? code_of(w.scalar_type()) : NF_F32, o.y.data_ptr(), (float*)ptr(o.scale), ptr(o.stream), (float*)ptr(o.rstd), x.n,
                        width, m.eps, stream_of(m.x)),
        "nf_rms_norm_fwd");
  return o;
}

// (dx, dw, dr).  h: the kept rows; dy, ds: the gradients of the output and of the new residual, either may be undefined.  `two`: dx and dr go
// to leaves, which need a tensor each (autograd would copy a shared one).
variable_list norm_backward(const Tensor& h, const Tensor& rstd, const Tensor& weight, at::ScalarType xt, Tensor dy, Tensor ds, bool residual,
                            bool need_rows, bool need_w, bool two) {
  const c10::DeviceGuard guard(h.device());
  const int64_t width = h.size(-1);  // (h and the factors may come back from a saved-tensor hook in any layout)
  const auto ht = h.scalar_type();
  if (!dy.defined()) dy = at::zeros(h.sizes(), h.options().dtype(xt));
  if (dy.scalar_type() != xt) dy = dy.to(xt);
  if (ds.defined() && ds.scalar_type() != ht) ds = ds.to(ht);
  const Rows rh(h, width), rd(dy, width);
  std::optional<Rows> rs;
  if (ds.defined()) rs.emplace(ds, width);
  const Tensor w = contiguous(weight), factors = contiguous(rstd);
  Tensor dx, dr, dw;
  if (need_rows) {
    dx = at::empty(h.sizes(), h.options().dtype(xt));
    if (residual) dr = ht != xt || two ? at::empty(h.sizes(), h.options()) : dx;
  }
  need_w = need_w && w.defined();
  if (need_w) dw = rh.n > 0 ? at::empty(w.sizes(), w.options()) : at::zeros(w.sizes(), w.options());
  if (rh.n > 0 && (need_rows || need_w)) {
    const int64_t bytes = need_w ? nf_rms_norm_bwd_workspace_bytes(rh.n, width) : 0;
    const Tensor ws = scratch(bytes, h);
    check(nf_rms_norm_bwd(rd.p, rd.stride, code_of(xt), rs ? rs->p : nullptr, rs ? rs->stride : width, rh.p, rh.stride, code_of(ht),
                          factors.data_ptr<float>(), ptr(w), w.defined() ? code_of(w.scalar_type()) : NF_F32, ptr(dx),
                          dr.defined() && !dr.is_same(dx) ? dr.data_ptr() : nullptr, ptr(dw), rh.n, width, ptr(ws), bytes, stream_of(h)),
          "nf_rms_norm_bwd");
  }
  return {dx, dw, dr};
}

// The forward's tensors are x, the weight where there is one, the residual.
void norm_once(const variable_list& g, const Tensor& dy, const Tensor& ds, bool weight) {
  const Once once("rms_norm");
  if (!dy.defined()) {  // the new residual's gradient goes on as it is
    once.mark(g[0], {}, {ds});
    if (g[2].defined() && !g[2].is_same(g[0])) once.mark(g[2], {}, {ds});
    return;
  }
  once.mark(g[0], {0, 1, 2}, {dy, ds});
  if (weight) once.mark(g[1], {0, 2}, {dy});
  if (g[2].defined() && !g[2].is_same(g[0])) once.mark(g[2], {0, 1, 2}, {dy, ds});
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, std::optional<Tensor> w, std::optional<Tensor> r, double eps) {
    const bool two = r && x.is_leaf() && r->is_leaf() && x.requires_grad() && r->requires_grad();
    const at::AutoDispatchBelowADInplaceOrView below;
    const Norm m{x, w.value_or(Tensor()), r.value_or(Tensor()), (float)eps};
    NormOut o = norm_forward(m, false, true);
    ctx->save_for_backward({r ? o.stream : x, o.rstd, m.w});
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->saved_data["residual"] = r.has_value();
    ctx->saved_data["two"] = two;
    ctx->set_materialize_grads(false);
    return r ? variable_list{o.y, o.stream} : variable_list{o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const at::AutoDispatchBelowADInplaceOrView below;
    const bool residual = ctx->saved_data["residual"].toBool();
    // the engine counts the tensors that there are: an absent weight has no number
    const bool weight = s[2].defined(), need_w = weight && ctx->needs_input_grad(1);
    const bool need_rows = ctx->needs_input_grad(0) || (residual && ctx->needs_input_grad(weight ? 2 : 1));
    variable_list g = norm_backward(s[0], s[1], s[2], (at::ScalarType)ctx->saved_data["type"].toInt(), grads[0], residual ? grads[1] : Tensor(), residual,
                                    need_rows, need_w, ctx->saved_data["two"].toBool());
    norm_once(g, grads[0], residual ? grads[1] : Tensor(), weight);
    return {g[0], g[1], g[2], Tensor()};
  }
};

bool norm_args(PyObject* const* a, Norm* m) {
  Tensor x;
  std::optional<Tensor> w, r;
  double eps;
  if (modes_active() || !plain(a[0], &x) || !plain_or_none(a[1], &w) || !as_double(a[2], &eps) || !plain_or_none(a[3], &r)) return false;
  *m = Norm{x, w.value_or(Tensor()), r.value_or(Tensor()), (float)eps};
  return norm_fits(*m);
}

bool wants_grad(const Norm& m) {
  return at::GradMode::is_enabled() && (m.x.requires_grad() || (m.w.defined() && m.w.requires_grad()) || (m.r.defined() && m.r.requires_grad()));
}

// rms_norm(x, weight, eps, residual): y, or (y, new residual)
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(4);
  Norm m;
  if (!norm_args(a, &m)) Py_RETURN_NONE;
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    if (wants_grad(m)) {
      for (const Tensor* t : {&m.x, &m.w, &m.r}) refuse_eager_graph(*t);
      const auto opt = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
      out = RmsNorm::apply(m.x, opt(m.w), opt(m.r), (double)m.eps);
    } else {
      const at::AutoDispatchBelowADInplaceOrView below;
      NormOut o = norm_forward(m, false, false);
      out = m.r.defined() ? variable_list{o.y, o.stream} : variable_list{o.y};
    }
  }
  return out.size() == 1 ? wrap(out[0]) : wrap_list(out);
  END_HANDLE_TH_ERRORS
}

// rms_norm_int8(x, weight, eps, residual): (q, scale), or (q, scale, new residual)
PyObject* rms_norm_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(4);
  Norm m;
  if (!norm_args(a, &m) || wants_grad(m)) Py_RETURN_NONE;
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    const at::AutoDispatchBelowADInplaceOrView below;
    NormOut o = norm_forward(m, true, false);
    out = {o.y, o.scale};
    if (m.r.defined()) out.push_back(o.stream);
  }
  return wrap_list(out);
  END_HANDLE_TH_ERRORS
}

// rms_norm_launch_forward(x, weight, eps, residual, eight) on checked arguments: (y, scale or None, new residual or None, rstd or None)
PyObject* rms_norm_launch_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(5);
  double eps;
  TORCH_CHECK(as_double(a[2], &eps), "eps expected");
  const Norm m{tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[3]), (float)eps};
  const bool eight = a[4] == Py_True;
  NormOut o;
  {
    pybind11::gil_scoped_release release;
    const at::AutoDispatchBelowADInplaceOrView below;
    o = norm_forward(m, eight, !eight);
  }
  return wrap_list({o.y, o.scale, o.stream, o.rstd});
  END_HANDLE_TH_ERRORS
}

// rms_norm_launch_backward(h, rstd, weight, like, dy, d_residual, residual, need_rows, need_w): (dx, dw, dr); `like`: a tensor of x's type
PyObject* rms_norm_launch_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(9);
  const Tensor h = tensor_arg(a[0]), rstd = tensor_arg(a[1]), w = tensor_arg(a[2]), like = tensor_arg(a[3]), dy = tensor_arg(a[4]), ds = tensor_arg(a[5]);
  const bool residual = a[6] == Py_True, need_rows = a[7] == Py_True, need_w = a[8] == Py_True;
  variable_list g;
  {
    pybind11::gil_scoped_release release;
    const at::AutoDispatchBelowADInplaceOrView below;
    g = norm_backward(h, rstd, w, like.scalar_type(), dy, ds, residual, need_rows, need_w, residual);
    norm_once(g, dy, ds, w.defined());
  }
  return wrap_list(g);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ 8-bit rows and products
// (q, scale)
variable_list quantize(const Tensor& x) {
  const c10::DeviceGuard guard(x.device());
  const int64_t width = x.size(-1);
  const Rows r(x, width);
  const Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar));
  const Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  check(nf_quantize_rows(r.p, r.stride, code_of(x.scalar_type()), (int8_t*)q.data_ptr(), (float*)scale.data_ptr(), nullptr, width, NF_ACT_NONE, r.n,
                         width, stream_of(x)),
        "nf_quantize_rows");
  return {q, scale};
}

struct Int8 {
  Tensor q, scale, w, w_scale, bias;
  int act;
  at::ScalarType type;
};

bool int8_fits(const Int8& m) {
  if (m.q.dim() < 1 || m.w.dim() != 2 || m.q.size(-1) < 1 || m.q.size(-1) > 131071 || m.w.size(0) < 1 || m.w.size(1) != m.q.size(-1)) return false;
  if (m.q.scalar_type() != at::kChar || m.w.scalar_type() != at::kChar || m.scale.scalar_type() != at::kFloat || m.w_scale.scalar_type() != at::kFloat)
    return false;
  if (m.scale.sizes() != m.q.sizes().slice(0, m.q.dim() - 1) || m.w_scale.dim() != 1 || m.w_scale.size(0) != m.w.size(0)) return false;
  if (m.bias.defined() && (!float_type(m.bias) || m.bias.dim() != 1 || m.bias.size(0) != m.w.size(0))) return false;
  for (const Tensor* t : {&m.scale, &m.w, &m.w_scale, &m.bias})
    if (t->defined() && t->device() != m.q.device()) return false;
  return code_of(m.type) >= 0;
}

Tensor int8_forward(const Int8& m) {
  const c10::DeviceGuard guard(m.q.device());
  const int64_t k = m.q.size(-1), n = m.w.size(0);
  const Rows q(m.q, k), w(m.w, k);
  c10::SmallVector<int64_t, 5> shape(m.q.sizes().begin(), m.q.sizes().end());
  shape.back() = n;
  const Tensor y = at::empty(shape, m.q.options().dtype(m.type)), scale = contiguous(m.scale), w_scale = contiguous(m.w_scale), bias = contiguous(m.bias);
  const auto* qp = (const int8_t*)q.p;
  const auto* wp = (const int8_t*)w.p;
  const int64_t bytes = nf_int8_linear_workspace_bytes(qp, q.stride, wp, w.stride, q.n, n, k);
  const Tensor ws = scratch(bytes, m.q);
  check(nf_int8_linear(qp, q.stride, (const float*)scale.data_ptr(), wp, w.stride, (const float*)w_scale.data_ptr(), ptr(bias),
                       bias.defined() ? code_of(bias.scalar_type()) : NF_F32, y.data_ptr(), n, code_of(m.type), q.n, n, k, m.act, ptr(ws), bytes,
                       stream_of(m.q)),
        "nf_int8_linear");
  return y;
}

bool needs_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.defined() && t.requires_grad(); }

// quantize_rows(x): (q, scale)
PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(1);
  Tensor x;
  if (modes_active() || !plain(a[0], &x) || x.dim() < 1 || x.size(-1) < 1 || !float_type(x) || needs_grad(x)) Py_RETURN_NONE;
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    const at::AutoDispatchBelowADInplaceOrView below;
    out = quantize(x);
  }
  return wrap_list(out);
  END_HANDLE_TH_ERRORS
}

// int8_linear(q, scale, w, w_scale, bias, activation, code of the result's type)
PyObject* int8_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(7);
  Int8 m;
  std::optional<Tensor> bias;
  int64_t type;
  m.act = activation(a[5], true);
  if (modes_active() || m.act < 0 || !plain(a[0], &m.q) || !plain(a[1], &m.scale) || !plain(a[2], &m.w) || !plain(a[3], &m.w_scale) ||
      !plain_or_none(a[4], &bias) || !as_int(a[6], &type) || type < NF_F32 || type > NF_BF16)
    Py_RETURN_NONE;
  m.bias = bias.value_or(Tensor());
  m.type = type == NF_F32 ? at::kFloat : type == NF_F16 ? at::kHalf : at::kBFloat16;
  if (!int8_fits(m) || needs_grad(m.scale) || needs_grad(m.w_scale) || needs_grad(m.bias)) Py_RETURN_NONE;
  Tensor y;
  {
    pybind11::gil_scoped_release release;
    const at::AutoDispatchBelowADInplaceOrView below;
    y = int8_forward(m);
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// quantize_rows_launch(x), int8_linear_launch(q, scale, w, w_scale, bias, activation code, type code): on checked arguments
PyObject* quantize_rows_launch(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(1);
  const Tensor x = tensor_arg(a[0]);
  variable_list out;
  {
    pybind11::gil_scoped_release release;
    const at::AutoDispatchBelowADInplaceOrView below;
    out = quantize(x);
  }
  return wrap_list(out);
  END_HANDLE_TH_ERRORS
}

PyObject* int8_linear_launch(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(7);
  int64_t act, type;
  TORCH_CHECK(as_int(a[5], &act) && as_int(a[6], &type), "codes expected");
  const Int8 m{tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), tensor_arg(a[3]), tensor_arg(a[4]), (int)act,
               type == NF_F32 ? at::kFloat : type == NF_F16 ? at::kHalf : at::kBFloat16};
  Tensor y;
  {
    pybind11::gil_scoped_release release;
    const at::AutoDispatchBelowADInplaceOrView below;
    y = int8_forward(m);
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ linear layer with 8-bit checkpoints
struct Keep {
  Tensor x, w, b;  // b: undefined without
  int act;
};

bool keep_fits(const Keep& m, bool cast) {
  if (m.x.dim() < 1 || m.w.dim() != 2 || m.x.size(-1) < 1 || m.w.size(0) < 1 || m.w.size(1) != m.x.size(-1) || m.w.device() != m.x.device()) return false;
  if (m.b.defined() && (!float_type(m.b) || m.b.dim() != 1 || m.b.size(0) != m.w.size(0) || m.b.device() != m.x.device())) return false;
  const auto half = [](const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; };
  return cast ? float_type(m.x) && float_type(m.w) : half(m.x) && m.w.scalar_type() == m.x.scalar_type();
}

// (y, q, scale); the last two only where they are kept
variable_list keep_forward(const Keep& m, bool keep) {
  const c10::DeviceGuard guard(m.x.device());
  const int64_t k = m.x.size(-1), n = m.w.size(0);
  const Rows x(m.x, k), w(m.w, k);
  const Tensor b = contiguous(m.b);
  c10::SmallVector<int64_t, 5> shape(m.x.sizes().begin(), m.x.sizes().end());
  shape.back() = n;
  const Tensor y = at::empty(shape, m.x.options());
  Tensor q, scale;
  if (keep) {
    q = at::empty(m.x.sizes(), m.x.options().dtype(at::kChar));
    scale = at::empty({x.n}, m.x.options().dtype(at::kFloat));
  }
  if (x.n > 0) {
    const int64_t bytes = nf_linear_keep_fwd_workspace_bytes(x.p, x.stride, w.p, w.stride, x.n, n, k, m.act);
    const Tensor ws = scratch(bytes, m.x);
    check(nf_linear_keep_fwd(x.p, x.stride, code_of(m.x.scalar_type()), w.p, w.stride, ptr(b), b.defined() ? code_of(b.scalar_type()) : NF_F32, y.data_ptr(),
                             n, (int8_t*)ptr(q), (float*)ptr(scale), x.n, n, k, m.act, ptr(ws), bytes, stream_of(m.x)),
          "nf_linear_keep_fwd");
  }
  return {y, q, scale};
}

// (dx, dw, db); dw in float32 where `float_dw`, db of type `bt`
variable_list keep_backward(Tensor q, Tensor scale, const Tensor& weight, int act, Tensor dy, bool need_dx, bool need_dw, bool need_db,
                            bool float_dw, at::ScalarType bt) {
  const c10::DeviceGuard guard(weight.device());
  const int64_t n = weight.size(0), k = weight.size(1);
  if (dy.scalar_type() != weight.scalar_type()) dy = dy.to(weight.scalar_type());
  // (what was kept may come back from a saved-tensor hook in any layout)
  q = contiguous(q);
  scale = contiguous(scale);
  if (q.defined() && (uintptr_t)q.data_ptr() % 16 != 0) q = q.clone();
  const Rows g(dy, n), w(weight, k);
  Tensor dx, dw, db;
  c10::SmallVector<int64_t, 5> shape(dy.sizes().begin(), dy.sizes().end());
  shape.back() = k;
  if (need_dx) dx = at::empty(shape, weight.options());
  const auto made = [&](at::IntArrayRef sizes, at::ScalarType t) {
    return g.n > 0 ? at::empty(sizes, weight.options().dtype(t)) : at::zeros(sizes, weight.options().dtype(t));
  };
  if (need_dw) dw = made({n, k}, float_dw ? at::kFloat : weight.scalar_type());
  if (need_db) db = made({n}, bt);
  if (g.n > 0) {
    const int64_t bytes = nf_linear_keep_bwd_workspace_bytes(g.p, g.stride, w.p, w.stride, g.n, n, k, need_dx, need_dw, need_db);
    const Tensor ws = scratch(bytes, weight);
    check(nf_linear_keep_bwd(g.p, g.stride, code_of(weight.scalar_type()), (const int8_t*)ptr(q), (const float*)ptr(scale), w.p, w.stride, ptr(dx), ptr(dw),
                             dw.defined() ? code_of(dw.scalar_type()) : NF_F32, ptr(db), code_of(bt), g.n, n, k, act, ptr(ws), bytes, stream_of(weight)),
          "nf_linear_keep_bwd");
  }
  return {dx, dw, db};
}

// The forward's tensors are x, w, b.
void keep_once(const variable_list& g, const Tensor& dy, int act) {
  const Once once("checkpointed_linear");
  if (act == NF_ACT_NONE) once.mark(g[0], {1}, {dy});
  else once.mark(g[0], {0, 1}, {dy});
  once.mark(g[1], {0}, {dy});
  once.mark(g[2], {}, {dy});
}

struct LinearKeep : torch::autograd::Function<LinearKeep> {
  // cast: the type that autocast asks for, or the tensors' own
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, std::optional<Tensor> b, int64_t act, int64_t cast) {
    const auto type = (at::ScalarType)cast;
    const bool keep = w.requires_grad() || act != NF_ACT_NONE;
    const at::AutoDispatchBelowADInplaceOrView below;
    const Keep m{x.to(type), w.to(type), b.value_or(Tensor()), (int)act};
    const variable_list r = keep_forward(m, keep);
    ctx->save_for_backward({r[1], r[2], m.w});
    ctx->saved_data["act"] = act;
    ctx->saved_data["float_dw"] = w.scalar_type() == at::kFloat;
    ctx->saved_data["bias"] = b ? (int64_t)b->scalar_type() : (int64_t)-1;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const at::AutoDispatchBelowADInplaceOrView below;
    const int64_t bias = ctx->saved_data["bias"].toInt();
    const int act = (int)ctx->saved_data["act"].toInt();
    variable_list g = keep_backward(s[0], s[1], s[2], act, grads[0], ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                    bias >= 0 && ctx->needs_input_grad(2), ctx->saved_data["float_dw"].toBool(),
                                    bias >= 0 ? (at::ScalarType)bias : at::kFloat);
    keep_once(g, grads[0], act);
    g.resize(5);
    return g;
  }
};

// checkpointed_linear(x, w, b, activation)
PyObject* checkpointed_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(4);
  Keep m;
  std::optional<Tensor> b;
  m.act = activation(a[3], true);
  if (modes_active() || m.act < 0 || !plain(a[0], &m.x) || !plain(a[1], &m.w) || !plain_or_none(a[2], &b)) Py_RETURN_NONE;
  m.b = b.value_or(Tensor());
  const bool cast = autocast();
  if (!keep_fits(m, cast)) Py_RETURN_NONE;
  const at::ScalarType type = cast ? at::autocast::get_autocast_dtype(at::kCUDA) : m.x.scalar_type();
  if (type != at::kHalf && type != at::kBFloat16) Py_RETURN_NONE;
  Tensor y;
  {
    pybind11::gil_scoped_release release;
    if (needs_grad(m.x) || needs_grad(m.w) || needs_grad(m.b)) {
      for (const Tensor* t : {&m.x, &m.w, &m.b}) refuse_eager_graph(*t);
      y = LinearKeep::apply(m.x, m.w, b, (int64_t)m.act, (int64_t)type);
    } else {
      const at::AutoDispatchBelowADInplaceOrView below;
      y = keep_forward(Keep{m.x.to(type), m.w.to(type), m.b, m.act}, false)[0];
    }
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// checkpointed_linear_launch_forward(x, w, b, activation code) on checked arguments: (y, q, scale)
PyObject* checkpointed_linear_launch_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(4);
  int64_t act;
  TORCH_CHECK(as_int(a[3], &act), "activation code expected");
  const Keep m{tensor_arg(a[0]), tensor_arg(a[1]), tensor_arg(a[2]), (int)act};
  variable_list r;
  {
    pybind11::gil_scoped_release release;
    const at::AutoDispatchBelowADInplaceOrView below;
    r = keep_forward(m, true);
  }
  return wrap_list(r);
  END_HANDLE_TH_ERRORS
}

// checkpointed_linear_launch_backward(q, scale, w, activation code, dy, need_dx, need_dw, need_db, float_dw, code of db's type): (dx, dw, db)
PyObject* checkpointed_linear_launch_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  NARGS(10);
  int64_t act, bt;
  TORCH_CHECK(as_int(a[3], &act) && as_int(a[9], &bt), "codes expected");
  const Tensor q = tensor_arg(a[0]), scale = tensor_arg(a[1]), w = tensor_arg(a[2]), dy = tensor_arg(a[4]);
  const bool dx = a[5] == Py_True, dw = a[6] == Py_True, db = a[7] == Py_True, wide = a[8] == Py_True;
  variable_list r;
  {
    pybind11::gil_scoped_release release;
    const at::AutoDispatchBelowADInplaceOrView below;
    r = keep_backward(q, scale, w, (int)act, dy, dx, dw, db, wide, bt == NF_F32 ? at::kFloat : bt == NF_F16 ? at::kHalf : at::kBFloat16);
    keep_once(r, dy, (int)act);
  }
  return wrap_list(r);
  END_HANDLE_TH_ERRORS
}

}  // namespace

PyMethodDef wide_methods[] = {ENTRY(refuse_eager_graphs), ENTRY(rms_norm), ENTRY(rms_norm_int8), ENTRY(rms_norm_launch_forward), ENTRY(rms_norm_launch_backward),
                              ENTRY(quantize_rows), ENTRY(quantize_rows_launch), ENTRY(int8_linear), ENTRY(int8_linear_launch),
                              ENTRY(checkpointed_linear), ENTRY(checkpointed_linear_launch_forward), ENTRY(checkpointed_linear_launch_backward),
                              {nullptr, nullptr, 0, nullptr}};
