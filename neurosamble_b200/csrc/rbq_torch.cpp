// torch.ops.rbq.linear, layer_norm and softmax_loss over the C ABI of librbq.so: definitions, checks
// of arguments, shapes for meta and fake tensors, and gradients.
//
// They are registered from C++ because a training step calls them hundreds of times on small inputs
// and is then bound by the host: through Python's custom operators a forward and backward pair took the
// host 230 us, through Python autograd functions 160 us, whatever the sizes.
//
// The kernel behind every operator is registered for all devices and refuses what is not on CUDA, so
// that a host tensor gets the library's message.  Work goes to the current stream of the input's device;
// nothing synchronises.  Inputs are made dense and moved to a 16-byte boundary where they are not.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <array>
#include <initializer_list>
#include <memory>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/rbq.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void call(int status)
{
  static const char* kNames[] = {"ok", "invalid argument", "CUDA error", "out of device memory", "I/O error",
                                 "wrong call order", "malformed index file"};
  TORCH_CHECK(status == RBQ_OK, "rbq error ", status, " (", status >= 0 && status < 7 ? kNames[status] : "?", "): ",
              rbq_last_error());
}

std::string type_name(at::ScalarType t)
{
  switch (t) {
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kFloat: return "torch.float32";
    case at::kDouble: return "torch.float64";
    case at::kLong: return "torch.int64";
    case at::kInt: return "torch.int32";
    default: return std::string("torch.") + c10::toString(t);
  }
}

int type_code(at::ScalarType t) { return t == at::kHalf ? RBQ_F16 : t == at::kBFloat16 ? RBQ_BF16 : RBQ_F32; }

void check_type(const Tensor& t, at::ScalarType type, const char* name)
{
  TORCH_CHECK(t.scalar_type() == type, "rbq: ", name, " must be ", type_name(type), ", got ", type_name(t.scalar_type()));
}
void check_first_type(const Tensor& t, bool f32_too, const char* name)
{
  const auto s = t.scalar_type();
  TORCH_CHECK(s == at::kHalf || s == at::kBFloat16 || (f32_too && s == at::kFloat), "rbq: ", name,
              " must be torch.float16 or torch.bfloat16", f32_too ? " or torch.float32" : "", ", got ", type_name(s));
}

// t of the given type on like's device, dense and on a 16-byte boundary.
Tensor operand(const Tensor& t, const Tensor& like, at::ScalarType type, const char* name)
{
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), "rbq: ", name, " must be a CUDA tensor on ", like.device(),
              ", got ", t.device());
  check_type(t, type, name);
  Tensor d = t.contiguous();
  return reinterpret_cast<uintptr_t>(d.const_data_ptr()) % 16 == 0 ? d : d.clone();
}

Tensor first(const Tensor& t, bool f32_too, const char* name)
{
  TORCH_CHECK(t.is_cuda(), "rbq: ", name, " must be a CUDA tensor");
  check_first_type(t, f32_too, name);
  return operand(t, t, t.scalar_type(), name);
}

void check_shape(const Tensor& t, at::IntArrayRef want, const char* name)
{
  TORCH_CHECK(t.sizes() == want, "rbq: ", name, " must have shape ", want, ", got ", t.sizes());
}

// The same checks for meta and fake tensors, whose sizes may be symbols.
void check_meta(const Tensor& t, at::ScalarType type, c10::SymIntArrayRef want, const char* name)
{
  check_type(t, type, name);
  TORCH_CHECK(t.dim() == (int64_t)want.size(), "rbq: ", name, " must have shape ", want, ", got ", t.sym_sizes());
  for (size_t i = 0; i < want.size(); ++i)
    TORCH_SYM_CHECK(t.sym_size(i).sym_eq(want[i]), "rbq: ", name, " must have shape ", want, ", got ", t.sym_sizes());
}
c10::SymDimVector rows_of(const Tensor& x) { return c10::SymDimVector(x.sym_sizes().begin(), x.sym_sizes().end() - 1); }

void* data(const Tensor& t) { return t.defined() ? const_cast<void*>(t.const_data_ptr()) : nullptr; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
Tensor scratch(const Tensor& like, int64_t bytes)
{
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
// Outputs for meta and fake tensors: dense rows whatever the input's strides, as the kernels write them.
Tensor dense_meta(const Tensor& like) { return at::empty_symint(like.sym_sizes(), like.options()); }
Tensor dense_meta_if(bool need, const Tensor& like) { return need ? dense_meta(like) : at::empty({0}, like.options()); }
Tensor empty_if(bool need, const Tensor& like) { return need ? at::empty_like(like) : at::empty({0}, like.options()); }

bool wants_grad(std::initializer_list<Tensor> ts)
{
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// There are no forward-mode derivatives: an input that carries a tangent is refused, since the tangent would be
// dropped below autograd (and taken as zero by the caller).
void no_tangents(std::initializer_list<Tensor> ts, const char* name)
{
  for (const Tensor& t : ts)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), "rbq: ", name, " has no forward-mode derivative");
}

// Outputs of a backward pass, whose own gradient is refused.  The refusal hangs on what the pass read, so that
// every way back from the outputs to one of those meets it: from a node with no way on, autograd.grad with such an
// input would skip it and take its part of the derivative as zero.
template <size_t N>
std::array<Tensor, N> once(std::array<Tensor, N> out, const char* name, std::initializer_list<Tensor> read)
{
  if (!wants_grad(read)) return out;
  variable_list in;
  for (const Tensor& t : out)
    if (t.defined() && t.numel() > 0) in.push_back(t.detach());
  if (in.empty()) return out;
  for (const Tensor& t : read)
    if (t.defined() && t.requires_grad()) in.push_back(t);
  auto fn = std::make_shared<torch::autograd::DelayedError>(
      std::string("rbq: the gradient of ") + name + " cannot be differentiated again", (int64_t)in.size());
  variable_list wrapped = (*fn)(std::move(in));
  size_t i = 0;
  for (Tensor& t : out)
    if (t.defined() && t.numel() > 0) t = wrapped[i++];
  return out;
}

// ---- linear ------------------------------------------------------------------------------------
struct LinearArgs {
  Tensor x, w, bias;
  int64_t m, k, n;
  int act, type;
};

int activation(c10::string_view act)
{
  if (act == "none") return RBQ_ACT_NONE;
  if (act == "relu") return RBQ_ACT_RELU;
  if (act == "gelu") return RBQ_ACT_GELU;
  TORCH_CHECK(false, "rbq: act must be one of none, relu, gelu, got '", std::string(act), "'");
}

LinearArgs linear_args(const Tensor& x, const Tensor& w, const OptTensor& bias, c10::string_view act)
{
  LinearArgs a;
  a.x = first(x, false, "x");
  a.w = operand(w, a.x, a.x.scalar_type(), "w");
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1), "rbq: linear takes x [..., k] and w [n, k], got ",
              x.sizes(), " and ", w.sizes());
  a.n = w.size(0);
  a.k = w.size(1);
  TORCH_CHECK(a.n >= 1 && a.k >= 1, "rbq: linear needs k >= 1 and n >= 1");
  TORCH_CHECK(a.n < (1ll << 31) && a.k < (1ll << 31), "rbq: linear: bad sizes");
  if (bias.has_value() && bias->defined()) {
    a.bias = operand(*bias, a.x, a.x.scalar_type(), "bias");
    check_shape(a.bias, {a.n}, "bias");
  }
  a.act = activation(act);
  a.m = a.x.numel() / a.k;
  a.type = type_code(a.x.scalar_type());
  return a;
}

std::vector<int64_t> with_last(const Tensor& x, int64_t n)
{
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = n;
  return s;
}

Tensor linear_kernel(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, c10::string_view act)
{
  const LinearArgs a = linear_args(x, w, bias, act);
  const auto out = with_last(a.x, a.n);
  Tensor r;
  if (residual.has_value() && residual->defined()) {
    r = operand(*residual, a.x, a.x.scalar_type(), "residual");
    check_shape(r, out, "residual");
  }
  const c10::cuda::CUDAGuard guard(a.x.device());
  int64_t bytes = 0;
  call(rbq_linear_workspace(a.m, a.k, a.n, a.type, a.act, 0, &bytes));
  Tensor y = at::empty(out, a.x.options()), ws = scratch(a.x, bytes);
  call(rbq_linear(data(a.x), data(a.w), data(a.bias), data(r), data(y), a.m, a.k, a.n, a.type, a.act, data(ws), bytes,
                  stream_of(a.x)));
  return y;
}

c10::SymDimVector check_linear_meta(const Tensor& x, const Tensor& w, const OptTensor& bias, c10::string_view act)
{
  check_first_type(x, false, "x");
  check_type(w, x.scalar_type(), "w");
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 2, "rbq: linear takes x [..., k] and w [n, k], got ", x.sym_sizes(), " and ",
              w.sym_sizes());
  TORCH_SYM_CHECK(x.sym_size(-1).sym_eq(w.sym_size(1)), "rbq: linear takes x [..., k] and w [n, k], got ", x.sym_sizes(),
                  " and ", w.sym_sizes());
  if (bias.has_value() && bias->defined()) check_meta(*bias, x.scalar_type(), {w.sym_size(0)}, "bias");
  activation(act);
  c10::SymDimVector out = rows_of(x);
  out.push_back(w.sym_size(0));
  return out;
}

Tensor linear_meta(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, c10::string_view act)
{
  const auto out = check_linear_meta(x, w, bias, act);
  if (residual.has_value() && residual->defined()) check_meta(*residual, x.scalar_type(), out, "residual");
  return at::empty_symint(out, x.options());
}

std::tuple<Tensor, Tensor, Tensor> linear_backward_kernel(const Tensor& g, const Tensor& x, const Tensor& w,
                                                          const OptTensor& bias, c10::string_view act, bool need_x,
                                                          bool need_w, bool need_bias)
{
  const LinearArgs a = linear_args(x, w, bias, act);
  const Tensor gd = operand(g, a.x, a.x.scalar_type(), "g");
  check_shape(gd, with_last(a.x, a.n), "g");
  const c10::cuda::CUDAGuard guard(a.x.device());
  Tensor dx = empty_if(need_x, a.x), dw = empty_if(need_w, a.w), db = at::empty({need_bias ? a.n : 0}, a.x.options());
  int64_t bytes = 0;
  call(rbq_linear_workspace(a.m, a.k, a.n, a.type, a.act, 1, &bytes));
  Tensor ws = scratch(a.x, bytes);
  call(rbq_linear_backward(data(gd), data(a.x), data(a.w), data(a.bias), need_x ? data(dx) : nullptr,
                           need_w ? data(dw) : nullptr, need_bias ? data(db) : nullptr, a.m, a.k, a.n, a.type, a.act,
                           data(ws), bytes, stream_of(a.x)));
  return {dx, dw, db};
}

std::tuple<Tensor, Tensor, Tensor> linear_backward_meta(const Tensor& g, const Tensor& x, const Tensor& w,
                                                        const OptTensor& bias, c10::string_view act, bool need_x, bool need_w,
                                                        bool need_bias)
{
  check_meta(g, x.scalar_type(), check_linear_meta(x, w, bias, act), "g");
  return {dense_meta_if(need_x, x), dense_meta_if(need_w, w),
          need_bias ? at::empty_symint({w.sym_size(0)}, x.options()) : at::empty({0}, x.options())};
}

c10::TypedOperatorHandle<decltype(linear_kernel)>& linear_op()
{
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("rbq::linear", "").typed<decltype(linear_kernel)>();
  return op;
}

c10::TypedOperatorHandle<decltype(linear_backward_kernel)>& linear_backward_op()
{
  static auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("rbq::linear_backward", "").typed<decltype(linear_backward_kernel)>();
  return op;
}

// Refuses forward-mode and second derivatives; LinearFunction's backward pass and direct calls come here.
std::tuple<Tensor, Tensor, Tensor> linear_backward_autograd(const Tensor& g, const Tensor& x, const Tensor& w,
                                                            const OptTensor& bias, c10::string_view act, bool need_x,
                                                            bool need_w, bool need_bias)
{
  const Tensor b = bias.value_or(Tensor());
  no_tangents({g, x, w, b}, "linear_backward");
  std::array<Tensor, 3> d;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    std::tie(d[0], d[1], d[2]) = linear_backward_op().call(g, x, w, bias, act, need_x, need_w, need_bias);
  }
  d = once(std::move(d), "linear", {g, x, w, b});
  return {d[0], d[1], d[2]};
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  // Absent optional inputs have no edge: those of bias and residual are numbered without them.
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias,
                        const OptTensor& residual, const std::string& act)
  {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({x, w, bias.value_or(Tensor())});
    ctx->saved_data["act"] = act;
    ctx->saved_data["residual"] = residual.has_value();
    return linear_op().call(x, w, bias, residual, act);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads)
  {
    const auto saved = ctx->get_saved_variables();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    const bool has_bias = saved[2].defined(), nb = has_bias && ctx->needs_input_grad(2);
    const bool nr = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(has_bias ? 3 : 2);
    Tensor dx, dw, db;
    if (nx || nw || nb)
      std::tie(dx, dw, db) = linear_backward_autograd(grads[0], saved[0], saved[1], has_bias ? OptTensor(saved[2]) : OptTensor(),
                                                      ctx->saved_data["act"].toStringRef(), nx, nw, nb);
    return {nx ? dx : Tensor(), nw ? dw : Tensor(), nb ? db : Tensor(), nr ? grads[0] : Tensor(), Tensor()};
  }
};

Tensor linear_autograd(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual,
                       c10::string_view act)
{
  no_tangents({x, w, bias.value_or(Tensor()), residual.value_or(Tensor())}, "linear");
  if (!wants_grad({x, w, bias.value_or(Tensor()), residual.value_or(Tensor())})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return linear_op().call(x, w, bias, residual, act);
  }
  return LinearFunction::apply(x, w, bias, residual, std::string(act));
}

// ---- layer norm --------------------------------------------------------------------------------
struct NormArgs {
  Tensor x, w;
  int64_t rows, d;
  int type, param_type;
};

void check_param_type(const Tensor& x, const Tensor& w)
{
  TORCH_CHECK(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, "rbq: w must be ",
              type_name(x.scalar_type()), " or torch.float32, got ", type_name(w.scalar_type()));
}

NormArgs norm_args(const Tensor& x, const Tensor& w)
{
  NormArgs a;
  a.x = first(x, true, "x");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "rbq: layer_norm takes x [..., d] with d >= 1, got ", x.sizes());
  check_param_type(x, w);
  a.w = operand(w, a.x, w.scalar_type(), "w");
  a.d = a.x.size(-1);
  TORCH_CHECK(a.d < (1ll << 31), "rbq: layer norm: bad sizes");
  check_shape(a.w, {a.d}, "w");
  a.rows = a.x.numel() / a.d;
  a.type = type_code(a.x.scalar_type());
  a.param_type = type_code(a.w.scalar_type());
  return a;
}

using Three = std::tuple<Tensor, Tensor, Tensor>;

Three layer_norm_kernel(const Tensor& x, const Tensor& w, const Tensor& b, double eps)
{
  const NormArgs a = norm_args(x, w);
  const Tensor bd = operand(b, a.x, a.w.scalar_type(), "b");
  check_shape(bd, {a.d}, "b");
  const c10::cuda::CUDAGuard guard(a.x.device());
  Tensor y = at::empty_like(a.x);
  Tensor mean = at::empty(a.x.sizes().slice(0, a.x.dim() - 1), a.x.options().dtype(at::kFloat)), rstd = at::empty_like(mean);
  call(rbq_layer_norm(data(a.x), data(a.w), data(bd), data(y), (float*)data(mean), (float*)data(rstd), a.rows, a.d, (float)eps,
                      a.type, a.param_type, stream_of(a.x)));
  return {y, mean, rstd};
}

void check_norm_meta(const Tensor& x, const Tensor& w)
{
  check_first_type(x, true, "x");
  TORCH_CHECK(x.dim() >= 1, "rbq: layer_norm takes x [..., d] with d >= 1, got ", x.sym_sizes());
  check_param_type(x, w);
  check_meta(w, w.scalar_type(), {x.sym_size(-1)}, "w");
}

Three layer_norm_meta(const Tensor& x, const Tensor& w, const Tensor& b, double)
{
  check_norm_meta(x, w);
  check_meta(b, w.scalar_type(), {x.sym_size(-1)}, "b");
  Tensor mean = at::empty_symint(rows_of(x), x.options().dtype(at::kFloat));
  return {dense_meta(x), mean, at::empty_like(mean)};
}

Three layer_norm_backward_kernel(const Tensor& g, const Tensor& x, const Tensor& w, const Tensor& mean, const Tensor& rstd,
                                 bool need_x, bool need_w, bool need_b)
{
  const NormArgs a = norm_args(x, w);
  const Tensor gd = operand(g, a.x, a.x.scalar_type(), "g");
  check_shape(gd, a.x.sizes(), "g");
  const auto rows = a.x.sizes().slice(0, a.x.dim() - 1);
  const Tensor md = operand(mean, a.x, at::kFloat, "mean"), rd = operand(rstd, a.x, at::kFloat, "rstd");
  check_shape(md, rows, "mean");
  check_shape(rd, rows, "rstd");
  const c10::cuda::CUDAGuard guard(a.x.device());
  Tensor dx = empty_if(need_x, a.x);
  Tensor dw = at::empty({need_w ? a.d : 0}, a.w.options()), db = at::empty({need_b ? a.d : 0}, a.w.options());
  int64_t bytes = 0;
  if (need_w || need_b) call(rbq_layer_norm_backward_workspace(a.rows, a.d, &bytes));
  Tensor ws = scratch(a.x, bytes);
  call(rbq_layer_norm_backward(data(gd), data(a.x), data(a.w), (float*)data(md), (float*)data(rd), need_x ? data(dx) : nullptr,
                               need_w ? data(dw) : nullptr, need_b ? data(db) : nullptr, a.rows, a.d, a.type, a.param_type,
                               data(ws), bytes, stream_of(a.x)));
  return {dx, dw, db};
}

Three layer_norm_backward_meta(const Tensor& g, const Tensor& x, const Tensor& w, const Tensor& mean, const Tensor& rstd,
                               bool need_x, bool need_w, bool need_b)
{
  check_norm_meta(x, w);
  check_meta(g, x.scalar_type(), x.sym_sizes(), "g");
  check_meta(mean, at::kFloat, rows_of(x), "mean");
  check_meta(rstd, at::kFloat, rows_of(x), "rstd");
  return {dense_meta_if(need_x, x), dense_meta_if(need_w, w), dense_meta_if(need_b, w)};
}

c10::TypedOperatorHandle<decltype(layer_norm_kernel)>& layer_norm_op()
{
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("rbq::layer_norm", "").typed<decltype(layer_norm_kernel)>();
  return op;
}

c10::TypedOperatorHandle<decltype(layer_norm_backward_kernel)>& layer_norm_backward_op()
{
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("rbq::layer_norm_backward", "")
                       .typed<decltype(layer_norm_backward_kernel)>();
  return op;
}

Three layer_norm_backward_autograd(const Tensor& g, const Tensor& x, const Tensor& w, const Tensor& mean, const Tensor& rstd,
                                   bool need_x, bool need_w, bool need_b)
{
  no_tangents({g, x, w, mean, rstd}, "layer_norm_backward");
  std::array<Tensor, 3> d;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    std::tie(d[0], d[1], d[2]) = layer_norm_backward_op().call(g, x, w, mean, rstd, need_x, need_w, need_b);
  }
  d = once(std::move(d), "layer_norm", {g, x, w, mean, rstd});
  return {d[0], d[1], d[2]};
}

struct LayerNormFunction : torch::autograd::Function<LayerNormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& b, double eps)
  {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, mean, rstd] = layer_norm_op().call(x, w, b, eps);
    ctx->save_for_backward({x, w, mean, rstd});
    ctx->mark_non_differentiable({mean, rstd});
    ctx->set_materialize_grads(false);
    return {y, mean, rstd};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads)
  {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = ctx->needs_input_grad(2);
    auto [dx, dw, db] = layer_norm_backward_autograd(grads[0], s[0], s[1], s[2], s[3], nx, nw, nb);
    return {nx ? dx : Tensor(), nw ? dw : Tensor(), nb ? db : Tensor(), Tensor()};
  }
};

Three layer_norm_autograd(const Tensor& x, const Tensor& w, const Tensor& b, double eps)
{
  no_tangents({x, w, b}, "layer_norm");
  if (!wants_grad({x, w, b})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return layer_norm_op().call(x, w, b, eps);
  }
  auto out = LayerNormFunction::apply(x, w, b, eps);
  return {out[0], out[1], out[2]};
}

// ---- softmax loss ------------------------------------------------------------------------------
struct LossArgs {
  Tensor q, bank, target;
  int64_t n, v, d;
  int type;
};

LossArgs loss_args(const Tensor& q, const Tensor& bank, const Tensor& target)
{
  LossArgs a;
  a.q = first(q, false, "q");
  a.bank = operand(bank, a.q, a.q.scalar_type(), "bank");
  TORCH_CHECK(q.dim() == 2 && bank.dim() == 2 && q.size(1) == bank.size(1) && bank.size(0) >= 1 && q.size(1) >= 1,
              "rbq: softmax_loss takes q [n, d] and bank [v, d] with v, d >= 1, got ", q.sizes(), " and ", bank.sizes());
  a.target = operand(target, a.q, at::kLong, "target");
  a.n = q.size(0);
  a.v = bank.size(0);
  a.d = q.size(1);
  TORCH_CHECK(a.d < (1ll << 31), "rbq: softmax loss: bad sizes");
  check_shape(a.target, {a.n}, "target");
  a.type = type_code(a.q.scalar_type());
  return a;
}

using Two = std::tuple<Tensor, Tensor>;

Two softmax_loss_kernel(const Tensor& q, const Tensor& bank, const Tensor& target, double scale)
{
  const LossArgs a = loss_args(q, bank, target);
  const c10::cuda::CUDAGuard guard(a.q.device());
  Tensor loss = at::empty({a.n}, a.q.options().dtype(at::kFloat)), lse = at::empty_like(loss);
  int64_t bytes = 0;
  call(rbq_softmax_loss_workspace(a.n, a.v, a.d, a.type, 0, &bytes));
  Tensor ws = scratch(a.q, bytes);
  call(rbq_softmax_loss(data(a.q), data(a.bank), (int64_t*)data(a.target), a.n, a.v, a.d, (float)scale, a.type,
                        (float*)data(loss), (float*)data(lse), data(ws), bytes, stream_of(a.q)));
  return {loss, lse};
}

void check_loss_meta(const Tensor& q, const Tensor& bank, const Tensor& target)
{
  check_first_type(q, false, "q");
  check_type(bank, q.scalar_type(), "bank");
  TORCH_CHECK(q.dim() == 2 && bank.dim() == 2, "rbq: softmax_loss takes q [n, d] and bank [v, d] with v, d >= 1, got ",
              q.sym_sizes(), " and ", bank.sym_sizes());
  TORCH_SYM_CHECK(q.sym_size(1).sym_eq(bank.sym_size(1)), "rbq: softmax_loss takes q [n, d] and bank [v, d] with v, d >= 1, got ",
                  q.sym_sizes(), " and ", bank.sym_sizes());
  check_meta(target, at::kLong, {q.sym_size(0)}, "target");
}

Two softmax_loss_meta(const Tensor& q, const Tensor& bank, const Tensor& target, double)
{
  check_loss_meta(q, bank, target);
  Tensor loss = at::empty_symint({q.sym_size(0)}, q.options().dtype(at::kFloat));
  return {loss, at::empty_like(loss)};
}

Two softmax_loss_backward_kernel(const Tensor& g, const Tensor& q, const Tensor& bank, const Tensor& target,
                                 const Tensor& loss, const Tensor& lse, double scale, bool need_q, bool need_bank)
{
  const LossArgs a = loss_args(q, bank, target);
  const Tensor gd = operand(g, a.q, at::kFloat, "g"), ld = operand(loss, a.q, at::kFloat, "loss"),
               sd = operand(lse, a.q, at::kFloat, "lse");
  check_shape(gd, {a.n}, "g");
  check_shape(ld, {a.n}, "loss");
  check_shape(sd, {a.n}, "lse");
  const c10::cuda::CUDAGuard guard(a.q.device());
  Tensor dq = empty_if(need_q, a.q), dbank = empty_if(need_bank, a.bank);
  int64_t bytes = 0;
  call(rbq_softmax_loss_workspace(a.n, a.v, a.d, a.type, 1, &bytes));
  Tensor ws = scratch(a.q, bytes);
  call(rbq_softmax_loss_backward((float*)data(gd), data(a.q), data(a.bank), (int64_t*)data(a.target), (float*)data(ld),
                                 (float*)data(sd), a.n, a.v, a.d, (float)scale, a.type, need_q ? data(dq) : nullptr,
                                 need_bank ? data(dbank) : nullptr, data(ws), bytes, stream_of(a.q)));
  return {dq, dbank};
}

Two softmax_loss_backward_meta(const Tensor& g, const Tensor& q, const Tensor& bank, const Tensor& target, const Tensor& loss,
                               const Tensor& lse, double, bool need_q, bool need_bank)
{
  check_loss_meta(q, bank, target);
  check_meta(g, at::kFloat, {q.sym_size(0)}, "g");
  check_meta(loss, at::kFloat, {q.sym_size(0)}, "loss");
  check_meta(lse, at::kFloat, {q.sym_size(0)}, "lse");
  return {dense_meta_if(need_q, q), dense_meta_if(need_bank, bank)};
}

c10::TypedOperatorHandle<decltype(softmax_loss_kernel)>& softmax_loss_op()
{
  static auto op = c10::Dispatcher::singleton().findSchemaOrThrow("rbq::softmax_loss", "").typed<decltype(softmax_loss_kernel)>();
  return op;
}

c10::TypedOperatorHandle<decltype(softmax_loss_backward_kernel)>& softmax_loss_backward_op()
{
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("rbq::softmax_loss_backward", "")
                       .typed<decltype(softmax_loss_backward_kernel)>();
  return op;
}

Two softmax_loss_backward_autograd(const Tensor& g, const Tensor& q, const Tensor& bank, const Tensor& target,
                                   const Tensor& loss, const Tensor& lse, double scale, bool need_q, bool need_bank)
{
  no_tangents({g, q, bank, loss, lse}, "softmax_loss_backward");
  std::array<Tensor, 2> d;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    std::tie(d[0], d[1]) = softmax_loss_backward_op().call(g, q, bank, target, loss, lse, scale, need_q, need_bank);
  }
  d = once(std::move(d), "softmax_loss", {g, q, bank, loss, lse});
  return {d[0], d[1]};
}

struct SoftmaxLossFunction : torch::autograd::Function<SoftmaxLossFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& bank, const Tensor& target, double scale)
  {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [loss, lse] = softmax_loss_op().call(q, bank, target, scale);
    ctx->save_for_backward({q, bank, target, loss, lse});
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    return {loss, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads)
  {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    const bool nq = ctx->needs_input_grad(0), nk = ctx->needs_input_grad(1);
    auto [dq, dbank] = softmax_loss_backward_autograd(grads[0], s[0], s[1], s[2], s[3], s[4], ctx->saved_data["scale"].toDouble(),
                                                      nq, nk);
    return {nq ? dq : Tensor(), nk ? dbank : Tensor(), Tensor(), Tensor()};
  }
};

Two softmax_loss_autograd(const Tensor& q, const Tensor& bank, const Tensor& target, double scale)
{
  no_tangents({q, bank}, "softmax_loss");
  if (!wants_grad({q, bank})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return softmax_loss_op().call(q, bank, target, scale);
  }
  auto out = SoftmaxLossFunction::apply(q, bank, target, scale);
  return {out[0], out[1]};
}

TORCH_LIBRARY_FRAGMENT(rbq, m)
{
  m.def("linear(Tensor x, Tensor w, Tensor? bias=None, Tensor? residual=None, str act='none') -> Tensor");
  m.def(
      "linear_backward(Tensor g, Tensor x, Tensor w, Tensor? bias, str act, bool need_x, bool need_w, bool need_bias) -> "
      "(Tensor, Tensor, Tensor)");
  m.def("layer_norm(Tensor x, Tensor w, Tensor b, float eps=1e-5) -> (Tensor, Tensor, Tensor)");
  m.def(
      "layer_norm_backward(Tensor g, Tensor x, Tensor w, Tensor mean, Tensor rstd, bool need_x, bool need_w, bool need_b) -> "
      "(Tensor, Tensor, Tensor)");
  m.def("softmax_loss(Tensor q, Tensor bank, Tensor target, float scale) -> (Tensor, Tensor)");
  m.def(
      "softmax_loss_backward(Tensor g, Tensor q, Tensor bank, Tensor target, Tensor loss, Tensor lse, float scale, "
      "bool need_q, bool need_bank) -> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(rbq, CompositeExplicitAutograd, m)
{
  m.impl("linear", linear_kernel);
  m.impl("linear_backward", linear_backward_kernel);
  m.impl("layer_norm", layer_norm_kernel);
  m.impl("layer_norm_backward", layer_norm_backward_kernel);
  m.impl("softmax_loss", softmax_loss_kernel);
  m.impl("softmax_loss_backward", softmax_loss_backward_kernel);
}
TORCH_LIBRARY_IMPL(rbq, Meta, m)
{
  m.impl("linear", linear_meta);
  m.impl("linear_backward", linear_backward_meta);
  m.impl("layer_norm", layer_norm_meta);
  m.impl("layer_norm_backward", layer_norm_backward_meta);
  m.impl("softmax_loss", softmax_loss_meta);
  m.impl("softmax_loss_backward", softmax_loss_backward_meta);
}
TORCH_LIBRARY_IMPL(rbq, Autograd, m)
{
  m.impl("linear", linear_autograd);
  m.impl("linear_backward", linear_backward_autograd);
  m.impl("layer_norm", layer_norm_autograd);
  m.impl("layer_norm_backward", layer_norm_backward_autograd);
  m.impl("softmax_loss", softmax_loss_autograd);
  m.impl("softmax_loss_backward", softmax_loss_backward_autograd);
}

}  // namespace
