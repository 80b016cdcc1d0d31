// host_dense.cpp -- the geot_dense::* operators on dense rows: linear, segment_matmul, layer_norm (kernels: csrc/dense_mm.hip, csrc/row_norm.hip).
//
// The reference has no such operators (its models call torch.nn.Linear and torch.nn.LayerNorm around the aggregations); they live in a
// dispatcher namespace of their own, so that `geot` holds what the reference's layers define and expect there.  Each comes as
//   geot_dense::<op>            what a user calls: looks whether a gradient is asked for and goes to one of
//   geot_dense::<op>_forward    the kernel, nothing kept for a backward pass (inference stays out of Python altogether)
//   geot_dense::<op>_train      the differentiable form (autograd formulas below; fake-tensor rules in geot_amd/ops.py), over
//   geot_dense::<op>_backward   the gradients
// The formulas are C++ here, unlike the aggregations' in ops.py: a training step of a few rows is host time, and a Python formula was 60 us
// of its 90.
// Every call runs on its tensors' device and that device's current stream, allocates what it needs from torch's caching allocator (under
// capture: from the graph's own pool, so two captured graphs share no scratch) and neither synchronises nor remembers anything.
#include "host.h"

#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/custom_function.h>

namespace {
using namespace geot_host;

int activation_code(c10::string_view a) {
  if (a == "none") return GEOT_ACT_NONE;
  if (a == "relu") return GEOT_ACT_RELU;
  if (a == "gelu") return GEOT_ACT_GELU;
  if (a == "silu") return GEOT_ACT_SILU;
  TORCH_CHECK(false, "activation argument must be either none, relu, gelu or silu, got ", a);
}

int dense_dtype(const at::Tensor &t, const char *op) {
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::kFloat || s == at::kHalf || s == at::kBFloat16, "\"", op, "\" not implemented for '", toString(s), "'");
  return dtype_code(t, op);
}

bool given(const c10::optional<at::Tensor> &t) { return t.has_value() && t->defined(); }
const at::Tensor *ptr_of(const c10::optional<at::Tensor> &t) { return given(t) ? &*t : nullptr; }
const void *data_of(const c10::optional<at::Tensor> &t) { return given(t) ? t->data_ptr() : nullptr; }
c10::optional<at::Tensor> dense(const c10::optional<at::Tensor> &t) { return given(t) ? c10::optional<at::Tensor>(t->contiguous()) : c10::nullopt; }

// [..., width] as rows: a 2-D tensor whose rows are dense keeps its row stride, anything else is laid out
struct Rows {
  at::Tensor t;
  int64_t rows, ld;
};
Rows as_rows(const at::Tensor &x) {
  const int64_t width = x.size(-1);
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  if (x.dim() == 2 && (x.stride(1) == 1 || width <= 1) && (x.stride(0) >= width || rows <= 1)) return {x, rows, rows <= 1 ? width : x.stride(0)};
  return {x.contiguous(), rows, width};
}
std::vector<int64_t> with_width(const at::Tensor &x, int64_t width) {
  auto s = x.sizes().vec();
  s.back() = width;
  return s;
}
at::Tensor scratch(const at::Tensor &like, size_t bytes) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }
// (a tangent would get lost without a word: the kernels know nothing of it)
void reverse_mode_only(const char *op, std::initializer_list<const at::Tensor *> ts) {
  for (const at::Tensor *t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->_fw_grad(/*level=*/0).defined(), op, ": forward-mode gradients (jvp, dual tensors) are not supported");
}
bool wants_grad(std::initializer_list<const at::Tensor *> ts) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const at::Tensor *t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}

// ---- linear ------------------------------------------------------------------------------------------------------------------------
void check_linear(const at::Tensor &x, const at::Tensor &w, const c10::optional<at::Tensor> &bias, const c10::optional<at::Tensor> &residual) {
  TORCH_CHECK(x.dim() >= 1, "linear: x must be at least 1 dimensional");
  TORCH_CHECK(w.dim() == 2, "linear: weight must be 2 dimensional ([out, in])");
  TORCH_CHECK(x.size(-1) == w.size(1), "linear: x has ", x.size(-1), " features a row, weight takes ", w.size(1));
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), "expected weight of dtype ", toString(x.scalar_type()), " but found ", toString(w.scalar_type()));
  if (given(bias)) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == w.size(0), "linear: bias must have one value per output feature (", w.size(0), ")");
    TORCH_CHECK(bias->scalar_type() == x.scalar_type(), "expected bias of dtype ", toString(x.scalar_type()), " but found ", toString(bias->scalar_type()));
  }
  if (given(residual)) {
    TORCH_CHECK(residual->sizes().vec() == with_width(x, w.size(0)), "linear: residual must have the output's shape ", with_width(x, w.size(0)), ", got ", residual->sizes());
    TORCH_CHECK(residual->scalar_type() == x.scalar_type(), "expected residual of dtype ", toString(x.scalar_type()), " but found ", toString(residual->scalar_type()));
  }
}

std::tuple<at::Tensor, at::Tensor> linear_forward_op(const at::Tensor &x_in, const at::Tensor &w_in, const c10::optional<at::Tensor> &bias_in,
                                                     const c10::optional<at::Tensor> &residual_in, c10::string_view activation, bool save) {
  check_linear(x_in, w_in, bias_in, residual_in);
  const int act = activation_code(activation);
  require_gpu("linear", {&x_in, &w_in, ptr_of(bias_in), ptr_of(residual_in)});
  const int dt = dense_dtype(x_in, "linear");
  GEOT_DEVICE_GUARD(x_in);
  const Rows x = as_rows(x_in);
  const at::Tensor w = w_in.contiguous();
  const auto bias = dense(bias_in);
  const int64_t in = w.size(1), out = w.size(0);
  at::Tensor y = at::empty(with_width(x_in, out), x_in.options());
  // what the activation's gradient needs: z, except that relu without a residual has its answer in y, and that narrow layers compute it again
  const bool keep = save && geot_linear_keeps_preactivation(in, act, given(residual_in), dt);
  at::Tensor z = keep ? at::empty_like(y) : at::empty({0}, x_in.options());
  Rows r{at::Tensor(), 0, 0};
  if (given(residual_in)) r = as_rows(*residual_in);
  const at::Tensor ws = scratch(x_in, geot_linear_workspace_bytes(x.rows, in, out, dt));
  GEOT_CALL(geot_linear(x.t.data_ptr(), x.ld, w.data_ptr(), data_of(bias), r.t.defined() ? r.t.data_ptr() : nullptr, r.ld, keep ? z.data_ptr() : nullptr,
                        y.data_ptr(), x.rows, in, out, act, dt, ws.data_ptr(), ws.numel(), stream_of(x_in)));
  return std::make_tuple(y, z);
}
std::tuple<at::Tensor, at::Tensor> linear_train_op(const at::Tensor &x, const at::Tensor &w, const c10::optional<at::Tensor> &bias,
                                                   const c10::optional<at::Tensor> &residual, c10::string_view activation) {
  return linear_forward_op(x, w, bias, residual, activation, true);
}

// z: what the forward kept ([0]: nothing - no activation, or one whose z is computed again)
std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_backward_op(const at::Tensor &grad_in, const at::Tensor &x_in, const at::Tensor &w_in,
                                                                  const c10::optional<at::Tensor> &bias_in, const at::Tensor &z_in, c10::string_view activation,
                                                                  bool need_x, bool need_w, bool need_b) {
  check_linear(x_in, w_in, bias_in, grad_in);
  const int act = activation_code(activation);
  const bool has_z = z_in.sizes() == grad_in.sizes() && z_in.numel() > 0;
  TORCH_CHECK(!has_z || z_in.scalar_type() == grad_in.scalar_type(), "linear: the backward pass needs what the differentiable forward (geot_dense::linear_train) saved");
  require_gpu("linear", {&grad_in, &x_in, &w_in, ptr_of(bias_in), &z_in});
  const int dt = dense_dtype(x_in, "linear");
  GEOT_DEVICE_GUARD(x_in);
  void *st = stream_of(x_in);
  const Rows x = as_rows(x_in);
  const at::Tensor w = w_in.contiguous();
  const int64_t in = w.size(1), out = w.size(0);
  at::Tensor dz = grad_in.contiguous(), dx, dw, db;
  if (act != GEOT_ACT_NONE) {
    const at::Tensor dy = dz, z = has_z ? z_in.contiguous() : at::Tensor();
    const auto bias = dense(bias_in);
    dz = at::empty_like(dy);
    if (need_b) db = x.rows > 0 ? at::empty({out}, w.options()) : at::zeros({out}, w.options());
    const at::Tensor ws = scratch(x_in, need_b ? geot_linear_grad_preactivation_workspace_bytes(x.rows, out) : 0);
    GEOT_CALL(geot_linear_grad_preactivation(dy.data_ptr(), has_z ? z.data_ptr() : nullptr, x.t.data_ptr(), x.ld, w.data_ptr(), data_of(bias), dz.data_ptr(),
                                             need_b ? db.data_ptr() : nullptr, x.rows, in, out, act, dt, ws.data_ptr(), ws.numel(), st));
  }
  if (need_x) {
    dx = at::empty(x_in.sizes(), x_in.options());
    const at::Tensor ws = scratch(x_in, geot_linear_grad_input_workspace_bytes(x.rows, in, out, dt));
    GEOT_CALL(geot_linear_grad_input(dz.data_ptr(), w.data_ptr(), dx.data_ptr(), x.rows, in, out, dt, ws.data_ptr(), ws.numel(), st));
  }
  const bool sums = need_b && act == GEOT_ACT_NONE;
  if (need_w || sums) {
    const int64_t cols = need_w ? in : 0; // (the bias's gradient alone: column sums beside a product of width 0)
    if (need_w) dw = at::empty_like(w);
    if (sums) db = at::empty({out}, w.options());
    const at::Tensor ws = scratch(x_in, geot_linear_grad_weight_workspace_bytes(x.rows, cols, out, dt));
    GEOT_CALL(geot_linear_grad_weight(dz.data_ptr(), x.t.data_ptr(), x.ld, need_w ? dw.data_ptr() : nullptr, sums ? db.data_ptr() : nullptr, x.rows, cols, out, dt,
                                      ws.data_ptr(), ws.numel(), st));
  }
  const at::Tensor none = at::empty({0}, x_in.options());
  return std::make_tuple(dx.defined() ? dx : none, dw.defined() ? dw : none, db.defined() ? db : none);
}

at::Tensor linear_op(const at::Tensor &x, const at::Tensor &w, const c10::optional<at::Tensor> &bias, const c10::optional<at::Tensor> &residual,
                     c10::string_view activation) {
  reverse_mode_only("linear", {&x, &w, ptr_of(bias), ptr_of(residual)});
  if (wants_grad({&x, &w, ptr_of(bias), ptr_of(residual)})) {
    static const auto train = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::linear_train", "").typed<decltype(linear_train_op)>();
    return std::get<0>(train.call(x, w, bias, residual, activation));
  }
  static const auto fwd = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::linear_forward", "").typed<decltype(linear_forward_op)>();
  return std::get<0>(fwd.call(x, w, bias, residual, activation, false));
}

// ---- segment_matmul ------------------------------------------------------------------------------------------------------------------
void check_segment(const at::Tensor &x, const at::Tensor &ptr, const at::Tensor &w, const c10::optional<at::Tensor> &bias) {
  TORCH_CHECK(x.dim() == 2, "segment_matmul: x must be 2 dimensional ([rows, in])");
  TORCH_CHECK(w.dim() == 3, "segment_matmul: weight must be 3 dimensional ([groups, in, out])");
  TORCH_CHECK(ptr.dim() == 1 && ptr.size(0) == w.size(0) + 1, "segment_matmul: ptr must hold groups + 1 = ", w.size(0) + 1, " row offsets");
  TORCH_CHECK(ptr.scalar_type() == at::kLong, "expected scalar type Long but found ", toString(ptr.scalar_type()), " (ptr)");
  TORCH_CHECK(w.size(0) <= 65535, "segment_matmul: at most 65535 groups, got ", w.size(0));
  TORCH_CHECK(x.size(1) == w.size(1), "segment_matmul: x has ", x.size(1), " features a row, weight takes ", w.size(1));
  TORCH_CHECK(w.scalar_type() == x.scalar_type(), "expected weight of dtype ", toString(x.scalar_type()), " but found ", toString(w.scalar_type()));
  if (given(bias)) {
    TORCH_CHECK(bias->dim() == 2 && bias->size(0) == w.size(0) && bias->size(1) == w.size(2), "segment_matmul: bias must be [groups, out]");
    TORCH_CHECK(bias->scalar_type() == x.scalar_type(), "expected bias of dtype ", toString(x.scalar_type()), " but found ", toString(bias->scalar_type()));
  }
}

at::Tensor segment_matmul_forward_op(const at::Tensor &x_in, const at::Tensor &ptr_in, const at::Tensor &w_in, const c10::optional<at::Tensor> &bias_in) {
  check_segment(x_in, ptr_in, w_in, bias_in);
  require_gpu("segment_matmul", {&x_in, &ptr_in, &w_in, ptr_of(bias_in)});
  const int dt = dense_dtype(x_in, "segment_matmul");
  GEOT_DEVICE_GUARD(x_in);
  const Rows x = as_rows(x_in);
  const at::Tensor ptr = ptr_in.contiguous(), w = w_in.contiguous();
  const auto bias = dense(bias_in);
  at::Tensor y = at::empty({x.rows, w.size(2)}, x_in.options());
  const at::Tensor ws = scratch(x_in, geot_segment_matmul_workspace_bytes(x.rows, w.size(0), w.size(1), w.size(2), dt));
  GEOT_CALL(geot_segment_matmul(x.t.data_ptr(), x.ld, index_ptr(ptr), w.data_ptr(), data_of(bias), y.data_ptr(), x.rows, w.size(0), w.size(1), w.size(2), dt,
                                ws.data_ptr(), ws.numel(), stream_of(x_in)));
  return y;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> segment_matmul_backward_op(const at::Tensor &grad_in, const at::Tensor &x_in, const at::Tensor &ptr_in,
                                                                          const at::Tensor &w_in, bool need_x, bool need_w, bool need_b) {
  check_segment(x_in, ptr_in, w_in, c10::nullopt);
  TORCH_CHECK(grad_in.dim() == 2 && grad_in.size(0) == x_in.size(0) && grad_in.size(1) == w_in.size(2) && grad_in.scalar_type() == x_in.scalar_type(),
              "segment_matmul: the gradient must have the output's shape and dtype");
  require_gpu("segment_matmul", {&grad_in, &x_in, &ptr_in, &w_in});
  const int dt = dense_dtype(x_in, "segment_matmul");
  GEOT_DEVICE_GUARD(x_in);
  void *st = stream_of(x_in);
  const Rows x = as_rows(x_in);
  const at::Tensor ptr = ptr_in.contiguous(), w = w_in.contiguous(), dy = grad_in.contiguous();
  const int64_t groups = w.size(0), in = w.size(1), out = w.size(2);
  at::Tensor dx, dw, db;
  if (need_x) {
    dx = at::empty(x_in.sizes(), x_in.options());
    const at::Tensor ws = scratch(x_in, geot_segment_matmul_grad_input_workspace_bytes(x.rows, groups, in, out, dt));
    GEOT_CALL(geot_segment_matmul_grad_input(dy.data_ptr(), index_ptr(ptr), w.data_ptr(), dx.data_ptr(), x.rows, groups, in, out, dt, ws.data_ptr(), ws.numel(), st));
  }
  if (need_w || need_b) {
    const int64_t rows_p = need_w ? in : 0;
    dw = need_w ? at::empty_like(w) : at::Tensor();
    db = need_b ? at::empty({groups, out}, w.options()) : at::Tensor();
    const at::Tensor ws = scratch(x_in, geot_segment_matmul_grad_weight_workspace_bytes(x.rows, groups, rows_p, out, dt));
    GEOT_CALL(geot_segment_matmul_grad_weight(x.t.data_ptr(), x.ld, index_ptr(ptr), dy.data_ptr(), need_w ? dw.data_ptr() : nullptr, need_b ? db.data_ptr() : nullptr,
                                              x.rows, groups, rows_p, out, dt, ws.data_ptr(), ws.numel(), st));
  }
  const at::Tensor none = at::empty({0}, x_in.options());
  return std::make_tuple(dx.defined() ? dx : none, dw.defined() ? dw : none, db.defined() ? db : none);
}

at::Tensor segment_matmul_op(const at::Tensor &x, const at::Tensor &ptr, const at::Tensor &w, const c10::optional<at::Tensor> &bias) {
  static const auto train = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::segment_matmul_train", "").typed<decltype(segment_matmul_forward_op)>();
  static const auto fwd = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::segment_matmul_forward", "").typed<decltype(segment_matmul_forward_op)>();
  reverse_mode_only("segment_matmul", {&x, &w, ptr_of(bias)});
  return wants_grad({&x, &w, ptr_of(bias)}) ? train.call(x, ptr, w, bias) : fwd.call(x, ptr, w, bias);
}

// ---- layer_norm ----------------------------------------------------------------------------------------------------------------------
// the parameters' type (x's or float32)
at::ScalarType check_norm(const at::Tensor &x, const c10::optional<at::Tensor> &w, const c10::optional<at::Tensor> &b) {
  TORCH_CHECK(x.dim() >= 1, "layer_norm: x must be at least 1 dimensional");
  at::ScalarType p = x.scalar_type();
  for (const auto *t : {&w, &b})
    if (given(*t)) {
      TORCH_CHECK((*t)->dim() == 1 && (*t)->size(0) == x.size(-1), "layer_norm: weight and bias must have one value per feature (", x.size(-1), ")");
      p = (*t)->scalar_type();
      TORCH_CHECK(p == x.scalar_type() || p == at::kFloat, "layer_norm: expected weight and bias of dtype ", toString(x.scalar_type()), " or Float but found ", toString(p));
    }
  TORCH_CHECK(!given(w) || !given(b) || w->scalar_type() == b->scalar_type(), "layer_norm: weight and bias must have one dtype");
  return p;
}
int param_code(at::ScalarType p) { return p == at::kFloat ? GEOT_F32 : p == at::kHalf ? GEOT_F16 : GEOT_BF16; }

std::tuple<at::Tensor, at::Tensor> layer_norm_forward_op(const at::Tensor &x_in, const c10::optional<at::Tensor> &w_in, const c10::optional<at::Tensor> &b_in, double eps,
                                                         bool save) {
  const auto p = check_norm(x_in, w_in, b_in);
  require_gpu("layer_norm", {&x_in, ptr_of(w_in), ptr_of(b_in)});
  const int dt = dense_dtype(x_in, "layer_norm");
  GEOT_DEVICE_GUARD(x_in);
  const Rows x = as_rows(x_in);
  const auto w = dense(w_in), b = dense(b_in);
  at::Tensor y = at::empty(x_in.sizes(), x_in.options());
  at::Tensor stats = at::empty({save ? 3 : 0, x.rows}, x_in.options().dtype(at::kFloat));
  GEOT_CALL(geot_layer_norm(x.t.data_ptr(), x.ld, data_of(w), data_of(b), y.data_ptr(), save ? stats.data_ptr<float>() : nullptr, x.rows, x_in.size(-1), (float)eps, dt,
                            param_code(p), stream_of(x_in)));
  return std::make_tuple(y, stats);
}
std::tuple<at::Tensor, at::Tensor> layer_norm_train_op(const at::Tensor &x, const c10::optional<at::Tensor> &w, const c10::optional<at::Tensor> &b, double eps) {
  return layer_norm_forward_op(x, w, b, eps, true);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_backward_op(const at::Tensor &grad_in, const at::Tensor &x_in, const c10::optional<at::Tensor> &w_in,
                                                                      const c10::optional<at::Tensor> &b_in, const at::Tensor &stats, bool need_x, bool need_params) {
  const auto p = check_norm(x_in, w_in, b_in);
  TORCH_CHECK(grad_in.sizes() == x_in.sizes() && grad_in.scalar_type() == x_in.scalar_type(), "layer_norm: the gradient must have the output's shape and dtype");
  require_gpu("layer_norm", {&grad_in, &x_in, ptr_of(w_in), &stats});
  const int dt = dense_dtype(x_in, "layer_norm");
  GEOT_DEVICE_GUARD(x_in);
  const Rows x = as_rows(x_in);
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == 3 * x.rows, "layer_norm: the backward pass needs the forward's statistics");
  const at::Tensor dy = grad_in.contiguous();
  const auto w = dense(w_in);
  const int64_t feat = x_in.size(-1);
  at::Tensor dx = need_x ? at::empty(x_in.sizes(), x_in.options()) : at::empty({0}, x_in.options()), dw = at::empty({need_params ? feat : 0}, x_in.options().dtype(p)), db = at::empty_like(dw);
  const at::Tensor ws = scratch(x_in, need_params ? geot_layer_norm_backward_workspace_bytes(x.rows, feat) : 0);
  GEOT_CALL(geot_layer_norm_backward(x.t.data_ptr(), x.ld, data_of(w), stats.data_ptr<float>(), dy.data_ptr(), need_x ? dx.data_ptr() : nullptr, need_params ? dw.data_ptr() : nullptr,
                                     need_params ? db.data_ptr() : nullptr, x.rows, feat, dt, param_code(p), ws.data_ptr(), ws.numel(), stream_of(x_in)));
  return std::make_tuple(dx, dw, db);
}

at::Tensor layer_norm_op(const at::Tensor &x, const c10::optional<at::Tensor> &w, const c10::optional<at::Tensor> &b, double eps) {
  reverse_mode_only("layer_norm", {&x, ptr_of(w), ptr_of(b)});
  if (wants_grad({&x, ptr_of(w), ptr_of(b)})) {
    static const auto train = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::layer_norm_train", "").typed<decltype(layer_norm_train_op)>();
    return std::get<0>(train.call(x, w, b, eps));
  }
  static const auto fwd = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::layer_norm_forward", "").typed<decltype(layer_norm_forward_op)>();
  return std::get<0>(fwd.call(x, w, b, eps, false));
}

// ---- autograd ------------------------------------------------------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::Tensor or_undefined(const c10::optional<at::Tensor> &t) { return given(t) ? *t : at::Tensor(); }
c10::optional<at::Tensor> or_none(const at::Tensor &t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; }
at::Tensor if_needed(bool need, const at::Tensor &t) { return need ? t : at::Tensor(); }
// these backward passes have no gradient of their own; a caller that asks for one (create_graph) is told so
void first_order_only(const char *op) {
  TORCH_CHECK_NOT_IMPLEMENTED(!c10::GradMode::is_enabled(), op, ": the backward pass is not differentiable (create_graph=True is not supported)");
}

// y = act(z) + residual, z = x W^T + b:  dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = column sums of dz;  dresidual = dy
struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &w, const c10::optional<at::Tensor> &bias, const c10::optional<at::Tensor> &residual,
                               std::string act) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::linear_train", "").typed<decltype(linear_train_op)>();
    auto [y, z] = op.call(x, w, bias, residual, act);
    // relu without a residual: y has z's sign, nothing else is kept
    ctx->save_for_backward({x, w, or_undefined(bias), act == "relu" && !given(residual) ? y : z});
    ctx->saved_data["bias"] = given(bias);
    ctx->saved_data["residual"] = given(residual);
    ctx->saved_data["activation"] = act;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({z});
    return {y, z};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(5);
    const at::Tensor &dy = grads[0];
    if (!dy.defined()) return out;
    first_order_only("linear");
    const auto saved = ctx->get_saved_variables();
    size_t at = 2; // (inputs that were not given are not counted)
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    const bool nb = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(at++), nr = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(at);
    if (nx || nw || nb) {
      static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::linear_backward", "").typed<decltype(linear_backward_op)>();
      const std::string act = ctx->saved_data["activation"].toStringRef();
      auto [dx, dw, db] = op.call(dy, saved[0], saved[1], or_none(saved[2]), saved[3], act, nx, nw, nb);
      out[0] = if_needed(nx, dx);
      out[1] = if_needed(nw, dw);
      out[2] = if_needed(nb, db);
    }
    out[3] = if_needed(nr, dy);
    return out;
  }
};
std::tuple<at::Tensor, at::Tensor> linear_train_autograd(const at::Tensor &x, const at::Tensor &w, const c10::optional<at::Tensor> &bias,
                                                         const c10::optional<at::Tensor> &residual, c10::string_view activation) {
  auto r = LinearFunction::apply(x, w, bias, residual, std::string(activation));
  return std::make_tuple(r[0], r[1]);
}

// per group g:  dx = dy W[g]^T;  dW[g] = x_g^T dy_g;  db[g] = column sums of dy_g
struct SegmentMatmulFunction : torch::autograd::Function<SegmentMatmulFunction> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &ptr, const at::Tensor &w, const c10::optional<at::Tensor> &bias) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::segment_matmul_train", "").typed<decltype(segment_matmul_forward_op)>();
    ctx->save_for_backward({x, ptr, w});
    ctx->saved_data["bias"] = given(bias);
    ctx->set_materialize_grads(false);
    return op.call(x, ptr, w, bias);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    first_order_only("segment_matmul");
    const auto saved = ctx->get_saved_variables();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(2);
    const bool nb = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3);
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::segment_matmul_backward", "").typed<decltype(segment_matmul_backward_op)>();
    auto [dx, dw, db] = op.call(grads[0], saved[0], saved[1], saved[2], nx, nw, nb);
    out[0] = if_needed(nx, dx);
    out[2] = if_needed(nw, dw);
    out[3] = if_needed(nb, db);
    return out;
  }
};
at::Tensor segment_matmul_train_autograd(const at::Tensor &x, const at::Tensor &ptr, const at::Tensor &w, const c10::optional<at::Tensor> &bias) {
  return SegmentMatmulFunction::apply(x, ptr, w, bias);
}

// h = (x - mean) rstd, g = dy w:  dx = rstd (g - mean g - h mean(g h));  dw = sum over rows of dy h;  db = sum over rows of dy
struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
  static variable_list forward(AutogradContext *ctx, const at::Tensor &x, const c10::optional<at::Tensor> &w, const c10::optional<at::Tensor> &b, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::layer_norm_train", "").typed<decltype(layer_norm_train_op)>();
    auto [y, stats] = op.call(x, w, b, eps);
    ctx->save_for_backward({x, or_undefined(w), or_undefined(b), stats});
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({stats});
    return {y, stats};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    first_order_only("layer_norm");
    const auto saved = ctx->get_saved_variables();
    size_t at = 1; // (inputs that were not given are not counted)
    const bool nx = ctx->needs_input_grad(0), nw = saved[1].defined() && ctx->needs_input_grad(at++), nb = saved[2].defined() && ctx->needs_input_grad(at);
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("geot_dense::layer_norm_backward", "").typed<decltype(layer_norm_backward_op)>();
    auto [dx, dw, db] = op.call(grads[0], saved[0], or_none(saved[1]), or_none(saved[2]), saved[3], nx, nw || nb);
    out[0] = if_needed(nx, dx);
    out[1] = if_needed(nw, dw);
    out[2] = if_needed(nb, db);
    return out;
  }
};
std::tuple<at::Tensor, at::Tensor> layer_norm_train_autograd(const at::Tensor &x, const c10::optional<at::Tensor> &w, const c10::optional<at::Tensor> &b, double eps) {
  auto r = LayerNormFunction::apply(x, w, b, eps);
  return std::make_tuple(r[0], r[1]);
}

} // namespace

TORCH_LIBRARY_FRAGMENT(geot_dense, m) {
  m.def("linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, str activation) -> Tensor", linear_op);
  m.def("linear_forward(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, str activation, bool save) -> (Tensor, Tensor)");
  m.def("linear_train(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, str activation) -> (Tensor, Tensor)");
  m.def("linear_backward(Tensor grad, Tensor x, Tensor weight, Tensor? bias, Tensor z, str activation, bool need_x, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)");
  m.def("segment_matmul(Tensor x, Tensor ptr, Tensor weight, Tensor? bias) -> Tensor", segment_matmul_op);
  m.def("segment_matmul_forward(Tensor x, Tensor ptr, Tensor weight, Tensor? bias) -> Tensor");
  m.def("segment_matmul_train(Tensor x, Tensor ptr, Tensor weight, Tensor? bias) -> Tensor");
  m.def("segment_matmul_backward(Tensor grad, Tensor x, Tensor ptr, Tensor weight, bool need_x, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)");
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", layer_norm_op);
  m.def("layer_norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps, bool save) -> (Tensor, Tensor)");
  m.def("layer_norm_train(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, bool need_x, bool need_params) -> (Tensor, Tensor, Tensor)");
}

// (the CPU key runs the argument checks and then refuses CPU tensors, as the package's other GPU-only operators do)
#define GEOT_DENSE_IMPLS(m)                                            \
  m.impl("linear_forward", linear_forward_op);                         \
  m.impl("linear_train", linear_train_op);                             \
  m.impl("linear_backward", linear_backward_op);                       \
  m.impl("segment_matmul_forward", segment_matmul_forward_op);         \
  m.impl("segment_matmul_train", segment_matmul_forward_op);           \
  m.impl("segment_matmul_backward", segment_matmul_backward_op);       \
  m.impl("layer_norm_forward", layer_norm_forward_op);                 \
  m.impl("layer_norm_train", layer_norm_train_op);                     \
  m.impl("layer_norm_backward", layer_norm_backward_op)
TORCH_LIBRARY_IMPL(geot_dense, CUDA, m) { GEOT_DENSE_IMPLS(m); }
TORCH_LIBRARY_IMPL(geot_dense, CPU, m) { GEOT_DENSE_IMPLS(m); }
TORCH_LIBRARY_IMPL(geot_dense, Autograd, m) {
  m.impl("linear_train", linear_train_autograd);
  m.impl("segment_matmul_train", segment_matmul_train_autograd);
  m.impl("layer_norm_train", layer_norm_train_autograd);
}
