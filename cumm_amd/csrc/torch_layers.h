// The calls of cumm_amd/torch_layers.py in native code: argument checks, allocation, the C entry points, and the nodes in
// torch's autograd graph.  What is not plain here - other types or devices, shapes that do not fit, dispatch modes,
// forward-mode derivatives - is left to the Python functions, which say what is wrong or do the same; a call that this
// file makes has their results.  Part of torch_native.cpp.
#pragma once
#include <algorithm>

// tensors that these calls take as they are
bool simple(const Tensor &t, const c10::Device &device, at::ScalarType type) {
  return t.device() == device && t.scalar_type() == type && t.layout() == at::kStrided && !t.is_conj() && !t.is_neg() && t.numel() > 0 &&
         !t.key_set().has(c10::DispatchKey::Python) && !t._fw_grad(0).defined();
}

// A tensor's rows: the tensor itself, or a contiguous copy where its rows are not contiguous and evenly apart, or further apart than
// a product takes them (8 MiB)
struct Rows {
  Tensor t;
  int64_t rows = 0, cols = 0, pitch = 0;
  Rows() = default;
  explicit Rows(const Tensor &of) : t(of) {
    cols = t.size(-1);
    rows = t.numel() / cols;
    pitch = cols;
    if (t.is_contiguous()) return;
    if (t.dim() != 2) t = t.reshape({-1, cols});      // (a view where the rows are evenly apart)
    if (t.dim() == 2 && (t.stride(1) == 1 || cols == 1) && (rows == 1 || (t.stride(0) >= cols && t.stride(0) * (int64_t)t.element_size() < (int64_t)8 << 20))) {
      if (rows > 1) pitch = t.stride(0);
      return;
    }
    t = t.contiguous();
  }
  void *at() const { return t.data_ptr(); }
};

Tensor given(const std::optional<Tensor> &t) { return t.has_value() ? *t : Tensor(); }
std::optional<Tensor> maybe(const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// a call with a workspace of the size that it asks for
template <class Args, class Query, class Call>
void with_workspace(Args &a, Query query, Call call, const c10::Device &device) {
  const int64_t need = query(&a);
  Tensor ws;
  if (need > 0) {
    ws = bytes(need, device);
    a.workspace = ws.data_ptr();
    a.workspace_bytes = (size_t)need;
  }
  check(call(&a, current_stream().stream()));
}

at::TensorOptions kind_of(at::ScalarType type, const c10::Device &device) { return at::TensorOptions().dtype(type).device(device); }

std::vector<int64_t> with_last(const Tensor &x, int64_t n) {
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n;
  return shape;
}

int layer_type(at::ScalarType t) { return t == at::kChar ? CUMM_HIP_S8 : (t == at::kFloat ? CUMM_HIP_F32 : tv_type(t)); }

// out, and what the activation got (undefined unless wanted); scales: of 8-bit operands
std::pair<Tensor, Tensor> linear_result(const Tensor &x_, const Tensor &w_, const Tensor &bias, const Tensor &residual, int64_t act, double slope, at::ScalarType out_type,
                                        bool want_pre, const Tensor &x_scale, const Tensor &w_scale, const Tensor &gate = Tensor()) {
  const Rows x(x_), w(w_);
  const c10::Device device = x_.device();
  const auto options = kind_of(out_type, device);
  const Tensor out = at::empty(with_last(x_, w.rows), options), pre = want_pre ? at::empty({x.rows, w.rows}, options) : Tensor();
  CummHipLinearArgs a = {};
  a.dtype = layer_type(x.t.scalar_type());
  a.out_dtype = layer_type(out_type);
  a.m = x.rows;
  a.n = (int32_t)w.rows;
  a.k = (int32_t)x.cols;
  a.x = x.at();
  a.weight = w.at();
  a.out = out.data_ptr();
  a.ld_x = x.pitch;
  a.ld_weight = w.pitch;
  a.ld_out = a.ld_pre_act = w.rows;
  Tensor b, xs, ws;
  if (bias.defined()) a.bias = (b = bias.contiguous()).data_ptr();
  Rows r;
  if (residual.defined()) {
    r = Rows(residual);
    a.residual = r.at();
    a.ld_residual = r.pitch;
  }
  if (want_pre) a.pre_act = pre.data_ptr();
  if (gate.defined()) a.gate = gate.data_ptr();
  if (x_scale.defined()) {
    a.x_scale = (xs = x_scale.contiguous()).data_ptr<float>();
    a.weight_scale = (ws = w_scale.contiguous()).data_ptr<float>();
  }
  a.act_type = (int32_t)act;
  a.act_alpha = (float)slope;
  with_workspace(a, api.linear_workspace, api.linear, device);
  return {out, pre};
}

// A gradient of a gradient is refused where it would be asked for, as torch's once_differentiable does
torch::autograd::variable_list once(torch::autograd::variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable",
                                                               (int64_t)grads.size());
  torch::autograd::variable_list marked;
  for (const Tensor &g : grads) marked.push_back(g.defined() ? g.detach().requires_grad_() : g);
  return (*error)(std::move(marked));
}

// A tensor that was kept for the backward pass, as it comes back: an unpack hook may give another one
const Tensor &kept(const Tensor &t, const char *name, const c10::Device &device, at::ScalarType type, c10::IntArrayRef sizes) {
  TORCH_CHECK_VALUE(t.defined() && simple(t, device, type) && t.sizes() == sizes, "the tensor kept as ", name, " came back as ", t.toString(), " ", t.sizes(), " on ", t.device(),
                    ", not as ", type, " ", sizes, " on ", device);
  return t;
}

struct LinearLayer : torch::autograd::Function<LinearLayer> {
  // (a tensor that is not there has no edge in the graph: its gradient's place is counted in `edges`)
  static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &w, const std::optional<Tensor> &bias_,
                        const std::optional<Tensor> &residual_, int64_t act, double slope, bool save_x, bool save_w) {
    const Tensor bias = given(bias_), residual = given(residual_);
    // what the backward pass needs of the activation's argument.  Of few channels it is worked out again, or, where only its side of a
    // kink counts, kept as a bit; the sign of a ReLU's result is that of its argument, unless something is added to it
    const auto narrow = [](int64_t c) { return c % 8 == 0 && c <= CUMM_HIP_LINEAR_NARROW; };
    const bool again = narrow(w.size(0)) && narrow(w.size(1)), kink = again && (act == CUMM_HIP_ACT_RELU || act == CUMM_HIP_ACT_LEAKY_RELU);
    const bool whole = again && act != CUMM_HIP_ACT_NONE && !kink;
    const bool by_result = act == CUMM_HIP_ACT_RELU && !residual.defined() && !again;
    const bool keep = act != CUMM_HIP_ACT_NONE && !by_result && !again;
    const Tensor gate = kink ? bytes(x.numel() / x.size(-1) * CUMM_HIP_LINEAR_GATE_BYTES(w.size(0)), x.device()) : Tensor();
    const auto got = linear_result(x, w, bias, residual, act, slope, x.scalar_type(), keep, Tensor(), Tensor(), gate);
    ctx->save_for_backward({save_x || whole ? x : Tensor(), save_w || whole ? w : Tensor(), kink ? gate : (whole ? bias : (by_result ? got.first : got.second))});
    ctx->saved_data["again"] = again;
    ctx->saved_data["edges"] = (int64_t)(bias.defined() ? 1 : 0) | (residual.defined() ? 2 : 0);
    ctx->saved_data["act"] = act;
    ctx->saved_data["slope"] = slope;
    ctx->saved_data["shape"] = x.sizes();
    return got.first;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    const Tensor &grad = grads[0];
    torch::autograd::variable_list result(8);
    if (!grad.defined()) return result;
    const auto saved = ctx->get_saved_variables();
    const int64_t edges = ctx->saved_data["edges"].toInt();
    const bool need[4] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), (edges & 1) && ctx->needs_input_grad(2),
                          (edges & 2) && ctx->needs_input_grad(2 + (edges & 1))};
    if (need[3]) result[3] = grad;
    if (need[0] || need[1] || need[2]) {
      at::AutoGradMode no_grad(false);
      const c10::Device device = grad.device();
      const c10::DeviceGuard guard(device);
      const Rows g(grad.detach());
      const auto options = kind_of(grad.scalar_type(), device);
      Rows x, w;
      CummHipLinearGradArgs a = {};
      a.dtype = layer_type(grad.scalar_type());
      a.m = g.rows;
      a.n = (int32_t)g.cols;
      a.grad_out = g.at();
      a.ld_grad_out = g.pitch;
      const at::ScalarType type = grad.scalar_type();
      const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
      a.from_inputs = ctx->saved_data["again"].toBool();
      a.act_type = (int32_t)ctx->saved_data["act"].toInt();
      a.act_alpha = (float)ctx->saved_data["slope"].toDouble();
      a.k = (int32_t)shape.back();
      Tensor third;
      Rows pre;
      if (saved[2].defined() && a.from_inputs && (a.act_type == CUMM_HIP_ACT_RELU || a.act_type == CUMM_HIP_ACT_LEAKY_RELU)) {
        const int64_t bytes = std::max<int64_t>(g.rows * CUMM_HIP_LINEAR_GATE_BYTES(g.cols), 256);
        a.gate = (third = kept(saved[2], "gate", device, at::kByte, {bytes}).contiguous()).data_ptr();
      } else if (saved[2].defined() && a.from_inputs) {
        a.bias = (third = kept(saved[2], "bias", device, type, {g.cols}).contiguous()).data_ptr();
      } else if (saved[2].defined()) {
        // (the result has the call's leading dimensions, what the activation got has one)
        third = saved[2].dim() == 2 ? saved[2] : saved[2].detach().reshape({-1, saved[2].size(-1)});
        pre = Rows(kept(third, "the activation's argument", device, type, {g.rows, g.cols}));
        a.pre_act = pre.at();
        a.ld_pre_act = pre.pitch;
      }
      if (saved[1].defined()) {
        w = Rows(kept(saved[1], "weight", device, type, {g.cols, shape.back()}));
        a.weight = w.at();
        a.ld_weight = w.pitch;
      }
      if (saved[0].defined()) {
        x = Rows(kept(saved[0], "x", device, type, shape));
        a.x = x.at();
        a.ld_x = x.pitch;
      }
      if (need[0]) {
        result[0] = at::empty(shape, options);
        a.grad_x = result[0].data_ptr();
      }
      if (need[1]) {
        result[1] = at::empty({g.cols, (int64_t)a.k}, options);
        a.grad_weight = result[1].data_ptr();
      }
      if (need[2]) {
        result[2] = at::empty({g.cols}, options);
        a.grad_bias = result[2].data_ptr();
      }
      with_workspace(a, api.linear_backward_workspace, api.linear_backward, device);
    }
    return once(std::move(result));
  }
};

// what the calls below cannot be made in
bool traced() { return c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing(); }
bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }

// each: the result, or an undefined tensor where the call is Python's
Tensor linear_of(const Tensor &x, const Tensor &w, const Tensor &bias, const Tensor &residual, int64_t act, double slope) {
  const c10::Device device = x.device();
  const at::ScalarType type = x.scalar_type();
  if (!device.is_cuda() || tv_type(type) < 0 || x.dim() < 1 || w.dim() != 2 || !simple(x, device, type) || !simple(w, device, type) || w.size(1) != x.size(-1) || w.size(0) > INT32_MAX || w.size(1) > INT32_MAX ||
      (bias.defined() && (!simple(bias, device, type) || bias.dim() != 1 || bias.size(0) != w.size(0))) ||
      (residual.defined() && (!simple(residual, device, type) || residual.sizes() != c10::IntArrayRef(with_last(x, w.size(0))))) || traced())
    return Tensor();
  const c10::DeviceGuard guard(device);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(bias) || wants_grad(residual)))
    return LinearLayer::apply(x, w, maybe(bias), maybe(residual), act, slope, wants_grad(w), wants_grad(x));
  at::AutoGradMode no_grad(false);
  return linear_result(x, w, bias, residual, act, slope, type, false, Tensor(), Tensor()).first;
}

Tensor linear_s8_of(const Tensor &x, const Tensor &x_scale, const Tensor &w, const Tensor &w_scale, const Tensor &bias, const Tensor &residual, int64_t act,
                    double slope, at::ScalarType out_type) {
  const c10::Device device = x.device();
  if (!device.is_cuda() || tv_type(out_type) < 0 || x.dim() < 1 || w.dim() != 2 || !simple(x, device, at::kChar) || !simple(w, device, at::kChar) ||
      w.size(1) != x.size(-1) || w.size(0) > INT32_MAX || w.size(1) > INT32_MAX || !simple(x_scale, device, at::kFloat) || !simple(w_scale, device, at::kFloat) ||
      x_scale.sizes() != x.sizes().slice(0, x.dim() - 1) || w_scale.dim() != 1 || w_scale.size(0) != w.size(0) ||
      (bias.defined() && (!simple(bias, device, at::kFloat) || bias.dim() != 1 || bias.size(0) != w.size(0))) ||
      (residual.defined() && (!simple(residual, device, out_type) || residual.sizes() != c10::IntArrayRef(with_last(x, w.size(0))))) || traced() ||
      (at::GradMode::is_enabled() && (wants_grad(x_scale) || wants_grad(w_scale) || wants_grad(bias) || wants_grad(residual))))
    return Tensor();
  const c10::DeviceGuard guard(device);
  at::AutoGradMode no_grad(false);
  return linear_result(x, w, bias, residual, act, slope, out_type, false, x_scale, w_scale).first;
}

struct NormResult {
  Tensor out, scale, total, inv;      // out: the codes where they are asked for
};
NormResult norm_result(const Tensor &x_, const Tensor &weight, const Tensor &residual, double eps, bool codes, bool want_inv) {
  const c10::Device device = x_.device();
  const Rows x(x_);
  NormResult got;
  got.out = at::empty(x_.sizes(), kind_of(codes ? at::kChar : x_.scalar_type(), device));
  CummHipRmsNormArgs a = {};
  a.dtype = layer_type(x_.scalar_type());
  a.m = x.rows;
  a.k = (int32_t)x.cols;
  a.eps = (float)eps;
  a.x = x.at();
  a.ld_x = x.pitch;
  Tensor w;
  if (weight.defined()) a.weight = (w = weight.contiguous()).data_ptr();
  Rows r;
  if (residual.defined()) {
    r = Rows(residual);
    got.total = at::empty(x_.sizes(), kind_of(x_.scalar_type(), device));
    a.residual = r.at();
    a.ld_residual = r.pitch;
    a.total = got.total.data_ptr();
  }
  if (codes) {
    got.scale = at::empty(x_.sizes().slice(0, x_.dim() - 1), kind_of(at::kFloat, device));
    a.codes = reinterpret_cast<int8_t *>(got.out.data_ptr());
    a.scale = got.scale.data_ptr<float>();
  } else {
    a.out = got.out.data_ptr();
  }
  if (want_inv) {
    got.inv = at::empty({x.rows}, kind_of(at::kFloat, device));
    a.inv_rms = got.inv.data_ptr<float>();
  }
  check(api.rms_norm(&a, current_stream().stream()));
  return got;
}

struct NormLayer : torch::autograd::Function<NormLayer> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &weight,
                                               const std::optional<Tensor> &residual_, double eps) {
    const Tensor residual = given(residual_);
    NormResult got = norm_result(x, weight, residual, eps, false, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({residual.defined() ? got.total : x, weight, got.inv});
    if (residual.defined()) return {got.out, got.total};
    return {got.out};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list result(4);
    const Tensor grad = grads[0], grad_total = grads.size() > 1 ? grads[1] : Tensor();
    if (!grad.defined() && !grad_total.defined()) return result;
    const bool need[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), grads.size() > 1 && ctx->needs_input_grad(2)};
    const auto saved = ctx->get_saved_variables();
    {
      at::AutoGradMode no_grad(false);
      const Tensor &any = grad.defined() ? grad : grad_total;      // (of the result's shape and type, as x)
      const c10::Device device = any.device();
      const c10::DeviceGuard guard(device);
      const Rows h(kept(saved[0], "the normed rows", device, any.scalar_type(), any.sizes()).detach());
      const Tensor w = kept(saved[1], "weight", device, any.scalar_type(), {h.cols}).detach().contiguous();
      const Tensor inv = kept(saved[2], "the rows' statistics", device, at::kFloat, {h.rows}).contiguous();
      Rows g, t;
      Tensor grad_x;
      CummHipRmsNormGradArgs a = {};
      a.dtype = layer_type(h.t.scalar_type());
      a.m = h.rows;
      a.k = (int32_t)h.cols;
      a.total = h.at();
      a.ld_total = h.pitch;
      a.weight = w.data_ptr();
      a.inv_rms = inv.data_ptr<float>();
      if (grad.defined()) {
        g = Rows(grad.detach());
        a.grad_out = g.at();
        a.ld_grad_out = g.pitch;
      }
      if (grad_total.defined()) {
        t = Rows(grad_total.detach());
        a.grad_total = t.at();
        a.ld_grad_total = t.pitch;
      }
      if (need[0] || need[2]) {
        grad_x = at::empty(saved[0].sizes(), kind_of(h.t.scalar_type(), device));
        a.grad_x = grad_x.data_ptr();
      }
      if (need[1]) {
        result[1] = at::empty({h.cols}, grad_x.defined() ? grad_x.options() : kind_of(h.t.scalar_type(), device));
        a.grad_weight = result[1].data_ptr();
      }
      with_workspace(a, api.rms_norm_backward_workspace, api.rms_norm_backward, device);
      if (need[0]) result[0] = grad_x;
      if (need[2]) result[2] = grad_x;
    }
    return once(std::move(result));
  }
};

bool norm_fits(const Tensor &x, const Tensor &weight, const Tensor &residual, double eps) {
  const c10::Device device = x.device();
  const at::ScalarType type = x.scalar_type();
  return device.is_cuda() && tv_type(type) >= 0 && x.dim() >= 1 && simple(x, device, type) && simple(weight, device, type) && weight.dim() == 1 &&
         weight.size(0) == x.size(-1) && x.size(-1) <= INT32_MAX && (!residual.defined() || (simple(residual, device, type) && residual.sizes() == x.sizes())) && eps > 0 && !traced();
}

// {out}, {out, total}, or nothing where the call is Python's
std::vector<Tensor> norm_of(const Tensor &x, const Tensor &weight, const Tensor &residual, double eps) {
  if (!norm_fits(x, weight, residual, eps)) return {};
  const c10::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(residual))) return NormLayer::apply(x, weight, maybe(residual), eps);
  at::AutoGradMode no_grad(false);
  NormResult got = norm_result(x, weight, residual, eps, false, false);
  if (residual.defined()) return {got.out, got.total};
  return {got.out};
}

// {codes, scale}, {codes, scale, total}, or nothing; weight undefined: rows in 8 bits without a norm
std::vector<Tensor> codes_of(const Tensor &x, const Tensor &weight, const Tensor &residual, double eps) {
  if (weight.defined() ? !norm_fits(x, weight, residual, eps)
                       : !(x.device().is_cuda() && x.dim() >= 1 && x.size(-1) <= INT32_MAX && (tv_type(x.scalar_type()) >= 0 || x.scalar_type() == at::kFloat) &&
                           simple(x, x.device(), x.scalar_type()) && !traced()))
    return {};
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(residual))) return {};
  const c10::DeviceGuard guard(x.device());
  at::AutoGradMode no_grad(false);
  NormResult got = norm_result(x, weight, residual, eps, true, false);
  if (residual.defined()) return {got.out, got.scale, got.total};
  return {got.out, got.scale};
}

// ---- as Python calls them: None where the call is its own
py::object layer_linear(const Tensor &x, const Tensor &w, const std::optional<Tensor> &bias, const std::optional<Tensor> &residual, int64_t act, double slope) {
  Tensor result;
  {
    py::gil_scoped_release release;
    result = linear_of(x, w, given(bias), given(residual), act, slope);
  }
  return result.defined() ? py::cast(result) : py::none();
}
py::object layer_linear_s8(const Tensor &x, const Tensor &x_scale, const Tensor &w, const Tensor &w_scale, const std::optional<Tensor> &bias,
                           const std::optional<Tensor> &residual, int64_t act, double slope, at::ScalarType type) {
  Tensor result;
  {
    py::gil_scoped_release release;
    result = linear_s8_of(x, x_scale, w, w_scale, given(bias), given(residual), act, slope, type);
  }
  return result.defined() ? py::cast(result) : py::none();
}
py::object tuple_of(const std::vector<Tensor> &v) {
  if (v.empty()) return py::none();
  if (v.size() == 1) return py::cast(v[0]);
  py::tuple t(v.size());
  for (size_t i = 0; i < v.size(); ++i) t[i] = py::cast(v[i]);
  return std::move(t);
}
py::object layer_norm_(const Tensor &x, const Tensor &weight, const std::optional<Tensor> &residual, double eps, bool codes) {
  std::vector<Tensor> result;
  {
    py::gil_scoped_release release;
    result = codes ? codes_of(x, weight, given(residual), eps) : norm_of(x, weight, given(residual), eps);
  }
  return tuple_of(result);
}
py::object layer_quantize(const Tensor &x) {
  std::vector<Tensor> result;
  {
    py::gil_scoped_release release;
    result = codes_of(x, Tensor(), Tensor(), 1.0);
  }
  return tuple_of(result);
}
