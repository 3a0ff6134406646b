// torch operators over the C ABI (include/msda.h) for the operators around the attention:
// unipercept::counter_dropout, unipercept::dropout_add_layer_norm, unipercept::level_group_norm.
//
// Each is a composite operator: it checks its arguments, and either runs the opaque forward
// operator or, where a gradient is wanted, records a node that runs the opaque backward operator.
// The opaque operators have a kernel on the GPU and shapes on the meta device (so torch.compile
// sees them), and refuse to be differentiated themselves.
//
// The layer is C++ because short calls are bound by the host: on MI355X's host a training step of
// dropout on 600 x 256 elements (two launches of a few microseconds each) took 148 us through
// Python's custom operators and autograd functions, most of it in the backward, where a Python
// node runs on the engine's own thread and has to take the interpreter's lock.
//
// libmsda.so is loaded, with its symbols global, before this library.
#include <ATen/ATen.h>
#include <ATen/functorch/BatchedTensorImpl.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/msda.h"

namespace {

using at::IntArrayRef;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kMaxRowBytes = 16384;  // a row of the normalising kernels
constexpr int64_t kMaxLevels = 16;
constexpr int64_t kMaxDropElements = int64_t(1) << 35;
constexpr int64_t kMaxRows = INT32_MAX;
constexpr int64_t kMaxMaps = int64_t(1) << 21;  // samples x levels x tiles of 32 groups

// ---- argument checks ------------------------------------------------------------------------------

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MSDA_F32;
    case at::kDouble: return MSDA_F64;
    case at::kBFloat16: return MSDA_BF16;
    case at::kHalf: return MSDA_F16;
    default: return -1;
  }
}
// Sizes as plain numbers.  Under a trace with symbolic shapes the numbers of this call are taken and
// guarded: a call of other sizes is traced again.
at::DimVector dims(const Tensor& t) {
  if (!t.unsafeGetTensorImpl()->has_symbolic_sizes_strides()) return at::DimVector(t.sizes());
  at::DimVector out;
  for (const c10::SymInt& s : t.sym_sizes()) out.push_back(s.guard_int(__FILE__, __LINE__));
  return out;
}
int64_t count(const at::DimVector& d) {
  int64_t n = 1;
  for (int64_t v : d) n *= v;
  return n;
}
IntArrayRef shown(const at::DimVector& d) { return IntArrayRef(d.data(), d.size()); }

bool half_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
at::ScalarType compute_type(at::ScalarType t) { return t == at::kDouble ? at::kDouble : at::kFloat; }

void check_tensor(const char* what, const Tensor& t) {
  TORCH_CHECK_TYPE(dtype_code(t.scalar_type()) >= 0, what, ": unsupported dtype ", t.scalar_type());
  TORCH_CHECK(t.is_cuda() || t.is_meta(), what,
              " runs only on a ROCm GPU (HIP kernels); got a tensor on ", t.device());
}

int activation_code(const char* what, const std::string& name, bool relu_only) {
  if (name == "none") return MSDA_ACT_NONE;
  if (name == "relu") return MSDA_ACT_RELU;
  if (!relu_only && name == "silu") return MSDA_ACT_SILU;
  if (!relu_only && name == "gelu") return MSDA_ACT_GELU;
  TORCH_CHECK_VALUE(false, what, ": activation must be one of ",
                    relu_only ? "'none', 'relu'" : "'none', 'relu', 'silu', 'gelu'", ", got '", name, "'");
}

void check_rng(const char* what, double p, int64_t site, const Tensor& state, const Tensor& x) {
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, what, ": p must lie in [0, 1], got ", p);
  TORCH_CHECK_VALUE(site >= 0 && site <= INT32_MAX, what, ": site must lie in [0, 2**31), got ", site);
  if (p == 0.0) return;
  TORCH_CHECK_VALUE(state.defined(), what, ": p > 0 needs rng_state (see new_rng_state)");
  const at::DimVector sd = dims(state);
  TORCH_CHECK_VALUE(state.scalar_type() == at::kLong && sd.size() == 1 && sd[0] == 2, what,
                    ": rng_state must be an int64 tensor (seed, offset), got ", shown(sd), " ",
                    state.scalar_type());
  TORCH_CHECK(state.device() == x.device(), what, ": rng_state lives on ", state.device(),
              ", the input on ", x.device());
  const int64_t n = count(dims(x));
  TORCH_CHECK_VALUE(n <= kMaxDropElements, what, ": at most 2**35 elements, got ", n);
}

void check_row(const char* what, int64_t columns, const Tensor& t) {
  const int64_t most = kMaxRowBytes / static_cast<int64_t>(t.element_size());
  TORCH_CHECK_VALUE(columns >= 1 && columns <= most, what, ": rows of 1 to ", most, " columns of ",
                    t.scalar_type(), ", got ", columns);
}

void check_params(const char* what, const Tensor& weight, const Tensor& bias, const Tensor& x,
                  at::ScalarType dtype) {
  TORCH_CHECK_VALUE(dims(weight) == dims(bias) && weight.scalar_type() == bias.scalar_type(), what,
                    ": weight and bias must agree in shape and dtype");
  TORCH_CHECK_TYPE(weight.scalar_type() == dtype ||
                       (half_type(x.scalar_type()) && weight.scalar_type() == at::kFloat),
                   what, ": parameters must be ", dtype,
                   " (or float32 next to a 16-bit input), got ", weight.scalar_type());
  TORCH_CHECK(weight.device() == x.device() && bias.device() == x.device(), what,
              ": all tensors must live on the same device");
}

constexpr const char* kDrop = "counter_dropout";
constexpr const char* kNorm = "dropout_add_layer_norm";
constexpr const char* kGroup = "level_group_norm";

void check_add_norm(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias,
                    const Tensor& state, double p, int64_t site, double eps) {
  check_tensor(kNorm, x);
  check_tensor(kNorm, residual);
  const at::DimVector xd = dims(x), wd = dims(weight);
  TORCH_CHECK_VALUE(!xd.empty() && xd == dims(residual), kNorm,
                    ": x and residual must agree in shape, got ", shown(xd), " and ",
                    shown(dims(residual)));
  TORCH_CHECK_TYPE(residual.scalar_type() == x.scalar_type() ||
                       (half_type(x.scalar_type()) && residual.scalar_type() == at::kFloat),
                   kNorm, ": residual must have x's dtype (or float32 next to a 16-bit x), got ",
                   residual.scalar_type(), " next to ", x.scalar_type());
  TORCH_CHECK(residual.device() == x.device(), kNorm, ": all tensors must live on the same device");
  const int64_t columns = xd.back();
  check_row(kNorm, columns, residual);
  TORCH_CHECK_VALUE(wd.size() == 1 && wd[0] == columns, kNorm, ": weight and bias must be (", columns,
                    ",), got ", shown(wd));
  check_params(kNorm, weight, bias, x, residual.scalar_type());
  TORCH_CHECK_VALUE(eps >= 0.0, kNorm, ": eps must not be negative, got ", eps);
  TORCH_CHECK_VALUE(count(xd) / columns <= kMaxRows, kNorm, ": at most 2**31 - 1 rows, got ",
                    count(xd) / columns);
  check_rng(kNorm, p, site, state, x);
}

// rows of the levels; one level of all positions without a list
std::vector<int64_t> level_rows(const Tensor& x, IntArrayRef rows) {
  const at::DimVector xd = dims(x);
  TORCH_CHECK_VALUE(xd.size() >= 2, kGroup, ": expected (N, ..., C), got ", shown(xd));
  int64_t positions = 1;
  for (size_t d = 1; d + 1 < xd.size(); ++d) positions *= xd[d];
  if (rows.empty()) return {positions};
  TORCH_CHECK_VALUE(static_cast<int64_t>(rows.size()) <= kMaxLevels, kGroup, ": 1 to ", kMaxLevels,
                    " levels, got ", rows.size());
  int64_t sum = 0;
  for (int64_t r : rows) {
    TORCH_CHECK_VALUE(r >= 1 || positions == 0, kGroup, ": levels must be positive, got ", rows);
    sum += r;
  }
  TORCH_CHECK_VALUE(sum == positions, kGroup, ": x has ", positions, " positions but the levels cover ",
                    sum);
  return rows.vec();
}

void check_group_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups,
                      const std::vector<int64_t>& rows, double eps) {
  check_tensor(kGroup, x);
  const at::DimVector xd = dims(x), wd = dims(weight);
  const int64_t samples = xd[0], columns = xd.back(), levels = static_cast<int64_t>(rows.size());
  check_row(kGroup, columns, x);
  TORCH_CHECK_VALUE(groups >= 1 && columns % groups == 0, kGroup, ": ", columns,
                    " channels do not divide into ", groups, " groups");
  const bool shared = wd.size() == 1 && wd[0] == columns;
  const bool each = wd.size() == 2 && wd[0] == levels && wd[1] == columns;
  TORCH_CHECK_VALUE(shared || each, kGroup, ": weight and bias must be (", columns, ",) or (", levels,
                    ", ", columns, "), got ", shown(wd));
  check_params(kGroup, weight, bias, x, x.scalar_type());
  TORCH_CHECK_VALUE(eps >= 0.0, kGroup, ": eps must not be negative, got ", eps);
  int64_t positions = 0;
  for (int64_t r : rows) positions += r;
  TORCH_CHECK_VALUE(positions == 0 || samples <= kMaxRows / positions, kGroup,
                    ": at most 2**31 - 1 positions, got ", samples, " x ", positions);
  TORCH_CHECK_VALUE(samples <= kMaxMaps / levels / ((groups + 31) / 32), kGroup,
                    ": at most 2**21 samples x levels (x tiles of 32 groups), got ", samples, " x ",
                    levels, " with ", groups, " groups");
}

void check_grad(const char* what, const Tensor& grad, const Tensor& like) {
  TORCH_CHECK_VALUE(grad.sizes() == like.sizes() && grad.device() == like.device(), what,
                    ": grad_output must be ", like.sizes(), " on ", like.device(), ", got ",
                    grad.sizes(), " on ", grad.device());
}

// ---- calls --------------------------------------------------------------------------------------------

Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
const void* in(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.mutable_data_ptr() : nullptr; }
const int64_t* state_ptr(const Tensor& t) { return static_cast<const int64_t*>(in(t)); }

Tensor fresh(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
// a gradient's buffer, or an empty tensor where it is not wanted
Tensor fresh_if(const Tensor& t, bool wanted) {
  return wanted ? fresh(t) : at::empty({0}, t.options());
}
Tensor bytes(const Tensor& like, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}
void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}
void check_call(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", msda_error_string(rc));
}

Tensor dropout_fwd(const Tensor& x_, const OptTensor& state_, double p, int64_t site,
                   const std::string& activation) {
  const int act = activation_code(kDrop, activation, true);
  check_tensor(kDrop, x_);
  check_rng(kDrop, p, site, given(state_), x_);
  const Tensor x = x_.contiguous();
  Tensor y = fresh(x);
  if (x.numel() == 0) return y;
  const Tensor state = p > 0.0 ? given(state_).contiguous() : Tensor();
  c10::DeviceGuard guard(x.device());
  check_call(msda_dropout_forward(in(x), out(y), state_ptr(state), x.numel(), p, static_cast<int>(site),
                                  act, dtype_code(x.scalar_type()), stream_of(x)),
             "msda_dropout_forward");
  return y;
}

Tensor dropout_bwd(const Tensor& grad_, const OptTensor& y_, const OptTensor& state_, double p,
                   int64_t site, const std::string& activation) {
  const int act = activation_code(kDrop, activation, true);
  check_tensor(kDrop, grad_);
  const Tensor grad = grad_.contiguous();
  Tensor y, state;
  if (act == MSDA_ACT_RELU) {
    y = given(y_);
    TORCH_CHECK_VALUE(y.defined() && y.scalar_type() == grad.scalar_type(), kDrop,
                      ": the ReLU's gradient needs the forward's output");
    check_grad(kDrop, grad, y);
    y = y.contiguous();
  } else if (p > 0.0) {
    check_rng(kDrop, p, site, given(state_), grad);
    state = given(state_).contiguous();
  }
  Tensor gx = fresh(grad);
  if (grad.numel() == 0) return gx;
  c10::DeviceGuard guard(grad.device());
  check_call(msda_dropout_backward(in(grad), in(y), out(gx), state_ptr(state), grad.numel(), p,
                                   static_cast<int>(site), act, dtype_code(grad.scalar_type()),
                                   stream_of(grad)),
             "msda_dropout_backward");
  return gx;
}

using Three = std::tuple<Tensor, Tensor, Tensor>;
using Four = std::tuple<Tensor, Tensor, Tensor, Tensor>;

Three add_norm_fwd(const Tensor& x_, const Tensor& residual_, const Tensor& weight_, const Tensor& bias_,
                   const OptTensor& state_, double p, int64_t site, double eps, bool stats) {
  check_add_norm(x_, residual_, weight_, bias_, given(state_), p, site, eps);
  const Tensor x = x_.contiguous(), residual = residual_.contiguous();
  const Tensor weight = weight_.contiguous(), bias = bias_.contiguous();
  const int64_t columns = x.size(-1), rows = x.numel() / columns;
  Tensor y = fresh(residual);
  const auto wide = residual.options().dtype(compute_type(residual.scalar_type()));
  Tensor mean = at::empty({stats ? rows : 0}, wide), rstd = at::empty({stats ? rows : 0}, wide);
  if (rows == 0) return {y, mean, rstd};
  const Tensor state = p > 0.0 ? given(state_).contiguous() : Tensor();
  c10::DeviceGuard guard(x.device());
  check_call(msda_dropout_add_norm_forward(
                 in(x), in(residual), in(weight), in(bias), out(y), out(mean), out(rstd),
                 state_ptr(state), rows, static_cast<int>(columns), p, static_cast<int>(site), eps,
                 dtype_code(x.scalar_type()), dtype_code(residual.scalar_type()),
                 dtype_code(weight.scalar_type()), stream_of(x)),
             "msda_dropout_add_norm_forward");
  return {y, mean, rstd};
}

Four add_norm_bwd(const Tensor& grad_, const Tensor& x_, const Tensor& residual_, const Tensor& weight_,
                  const Tensor& mean, const Tensor& rstd, const OptTensor& state_, double p,
                  int64_t site, bool want_x, bool want_residual, bool want_params) {
  check_add_norm(x_, residual_, weight_, weight_, given(state_), p, site, 0.0);
  check_grad(kNorm, grad_, residual_);
  const Tensor x = x_.contiguous(), residual = residual_.contiguous(), weight = weight_.contiguous();
  const Tensor grad = grad_.to(residual.scalar_type()).contiguous();
  const int64_t columns = x.size(-1), rows = x.numel() / columns;
  TORCH_CHECK_VALUE(mean.numel() == rows && rstd.numel() == rows && mean.is_contiguous() &&
                        rstd.is_contiguous() && mean.device() == x.device() && rstd.device() == x.device() &&
                        mean.scalar_type() == compute_type(residual.scalar_type()) &&
                        rstd.scalar_type() == mean.scalar_type(),
                    kNorm, ": the backward needs the forward's row statistics");
  Tensor gx = fresh_if(x, want_x), gr = fresh_if(residual, want_residual);
  Tensor gw = fresh_if(weight, want_params), gb = fresh_if(weight, want_params);
  if (rows == 0) return {gx, gr, gw.zero_(), gb.zero_()};
  const int xc = dtype_code(x.scalar_type()), rc = dtype_code(residual.scalar_type());
  const size_t need =
      want_params ? msda_dropout_add_norm_workspace_bytes(rows, static_cast<int>(columns), xc, rc) : 0;
  const Tensor workspace = bytes(x, need);
  const Tensor state = p > 0.0 ? given(state_).contiguous() : Tensor();
  c10::DeviceGuard guard(x.device());
  check_call(msda_dropout_add_norm_backward(
                 in(grad), in(x), in(residual), in(weight), in(mean), in(rstd), out(gx), out(gr), out(gw),
                 out(gb), out(workspace), need, state_ptr(state), rows, static_cast<int>(columns), p,
                 static_cast<int>(site), xc, rc, dtype_code(weight.scalar_type()), stream_of(x)),
             "msda_dropout_add_norm_backward");
  return {gx, gr, gw, gb};
}

Three group_norm_fwd(const Tensor& x_, const Tensor& weight_, const Tensor& bias_, int64_t groups,
                     IntArrayRef rows_, double eps, const std::string& activation, bool stats) {
  const int act = activation_code(kGroup, activation, false);
  const std::vector<int64_t> rows = level_rows(x_, rows_);
  check_group_norm(x_, weight_, bias_, groups, rows, eps);
  const Tensor x = x_.contiguous(), weight = weight_.contiguous(), bias = bias_.contiguous();
  const int levels = static_cast<int>(rows.size()), n = static_cast<int>(x.size(0));
  const int c = static_cast<int>(x.size(-1)), g = static_cast<int>(groups);
  Tensor y = fresh(x);
  const auto wide = x.options().dtype(compute_type(x.scalar_type()));
  const std::vector<int64_t> shape =
      stats ? std::vector<int64_t>{n, levels, g} : std::vector<int64_t>{0};
  Tensor mean = at::empty(shape, wide), rstd = at::empty(shape, wide);
  if (x.numel() == 0) return {y, mean, rstd};
  const int s = static_cast<int>(x.numel() / n / c), code = dtype_code(x.scalar_type());
  const size_t need = msda_group_norm_workspace_bytes(rows.data(), n, s, c, g, levels, code, 0);
  const Tensor workspace = bytes(x, need);
  c10::DeviceGuard guard(x.device());
  check_call(msda_group_norm_forward(in(x), in(weight), in(bias), out(y), out(mean), out(rstd),
                                     out(workspace), need, rows.data(), n, s, c, g, levels,
                                     weight.dim() == 2 ? levels : 1, eps, act, code,
                                     dtype_code(weight.scalar_type()), stream_of(x)),
             "msda_group_norm_forward");
  return {y, mean, rstd};
}

Three group_norm_bwd(const Tensor& grad_, const Tensor& x_, const Tensor& weight_, const Tensor& bias_,
                     const Tensor& mean, const Tensor& rstd, int64_t groups, IntArrayRef rows_,
                     const std::string& activation, bool want_x, bool want_params) {
  const int act = activation_code(kGroup, activation, false);
  const std::vector<int64_t> rows = level_rows(x_, rows_);
  check_group_norm(x_, weight_, bias_, groups, rows, 0.0);
  check_grad(kGroup, grad_, x_);
  const Tensor x = x_.contiguous(), weight = weight_.contiguous(), bias = bias_.contiguous();
  const Tensor grad = grad_.to(x.scalar_type()).contiguous();
  const int levels = static_cast<int>(rows.size()), n = static_cast<int>(x.size(0));
  const int c = static_cast<int>(x.size(-1)), g = static_cast<int>(groups);
  TORCH_CHECK_VALUE(mean.numel() == int64_t(n) * levels * g && rstd.numel() == mean.numel() &&
                        mean.is_contiguous() && rstd.is_contiguous() && mean.device() == x.device() &&
                        rstd.device() == x.device() &&
                        mean.scalar_type() == compute_type(x.scalar_type()) &&
                        rstd.scalar_type() == mean.scalar_type(),
                    kGroup, ": the backward needs the forward's statistics");
  Tensor gx = fresh_if(x, want_x), gw = fresh_if(weight, want_params), gb = fresh_if(bias, want_params);
  if (x.numel() == 0) return {gx, gw.zero_(), gb.zero_()};
  const int s = static_cast<int>(x.numel() / n / c), code = dtype_code(x.scalar_type());
  const size_t need = msda_group_norm_workspace_bytes(rows.data(), n, s, c, g, levels, code, 1);
  const Tensor workspace = bytes(x, need);
  c10::DeviceGuard guard(x.device());
  check_call(msda_group_norm_backward(in(grad), in(x), in(weight), in(bias), in(mean), in(rstd), out(gx),
                                      out(gw), out(gb), out(workspace), need, rows.data(), n, s, c, g,
                                      levels, weight.dim() == 2 ? levels : 1, act, code,
                                      dtype_code(weight.scalar_type()), stream_of(x)),
             "msda_group_norm_backward");
  return {gx, gw, gb};
}

// ---- shapes (meta device) ---------------------------------------------------------------------------

Tensor dropout_fwd_meta(const Tensor& x, const OptTensor&, double, int64_t, const std::string&) {
  return at::empty_symint(x.sym_sizes(), x.options());
}
Tensor dropout_bwd_meta(const Tensor& grad, const OptTensor&, const OptTensor&, double, int64_t,
                        const std::string&) {
  return at::empty_symint(grad.sym_sizes(), grad.options());
}
Tensor like_meta(const Tensor& t, bool wanted) {
  return wanted ? at::empty_symint(t.sym_sizes(), t.options()) : at::empty({0}, t.options());
}
Three add_norm_fwd_meta(const Tensor& x, const Tensor& residual, const Tensor&, const Tensor&,
                        const OptTensor&, double, int64_t, double, bool stats) {
  const auto wide = residual.options().dtype(compute_type(residual.scalar_type()));
  const c10::SymInt rows = stats ? x.sym_numel() / x.sym_size(-1) : c10::SymInt(0);
  return {at::empty_symint(residual.sym_sizes(), residual.options()), at::empty_symint({rows}, wide),
          at::empty_symint({rows}, wide)};
}
Four add_norm_bwd_meta(const Tensor&, const Tensor& x, const Tensor& residual, const Tensor& weight,
                       const Tensor&, const Tensor&, const OptTensor&, double, int64_t, bool want_x,
                       bool want_residual, bool want_params) {
  return {like_meta(x, want_x), like_meta(residual, want_residual), like_meta(weight, want_params),
          like_meta(weight, want_params)};
}
Three group_norm_fwd_meta(const Tensor& x, const Tensor&, const Tensor&, int64_t groups,
                          IntArrayRef rows, double, const std::string&, bool stats) {
  const auto wide = x.options().dtype(compute_type(x.scalar_type()));
  const int64_t levels = rows.empty() ? 1 : static_cast<int64_t>(rows.size());
  std::vector<c10::SymInt> shape{c10::SymInt(0)};
  if (stats) shape = {x.sym_size(0), c10::SymInt(levels), c10::SymInt(groups)};
  return {at::empty_symint(x.sym_sizes(), x.options()), at::empty_symint(shape, wide),
          at::empty_symint(shape, wide)};
}
Three group_norm_bwd_meta(const Tensor&, const Tensor& x, const Tensor& weight, const Tensor& bias,
                          const Tensor&, const Tensor&, int64_t, IntArrayRef, const std::string&,
                          bool want_x, bool want_params) {
  return {like_meta(x, want_x), like_meta(weight, want_params), like_meta(bias, want_params)};
}

// ---- dispatch -----------------------------------------------------------------------------------------

template <typename F>
c10::TypedOperatorHandle<F> find(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

Tensor call_dropout_fwd(const Tensor& x, const OptTensor& state, double p, int64_t site,
                        const std::string& act) {
  static const auto op = find<decltype(dropout_fwd)>("unipercept::counter_dropout_fwd");
  return op.call(x, state, p, site, act);
}
Tensor call_dropout_bwd(const Tensor& grad, const OptTensor& y, const OptTensor& state, double p,
                        int64_t site, const std::string& act) {
  static const auto op = find<decltype(dropout_bwd)>("unipercept::counter_dropout_bwd");
  return op.call(grad, y, state, p, site, act);
}
Three call_add_norm_fwd(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& bias,
                        const OptTensor& state, double p, int64_t site, double eps, bool stats) {
  static const auto op = find<decltype(add_norm_fwd)>("unipercept::dropout_add_norm_fwd");
  return op.call(x, residual, weight, bias, state, p, site, eps, stats);
}
Three call_group_norm_fwd(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups,
                          IntArrayRef rows, double eps, const std::string& act, bool stats) {
  static const auto op = find<decltype(group_norm_fwd)>("unipercept::level_group_norm_fwd");
  return op.call(x, weight, bias, groups, rows, eps, act, stats);
}

// A backward operator is called below autograd, unless the caller builds a graph of the gradient:
// then it goes through the operator's autograd kernel, which refuses to be differentiated.
struct BelowAutograd {
  std::optional<at::AutoDispatchBelowADInplaceOrView> guard;
  explicit BelowAutograd(bool on = !at::GradMode::is_enabled()) {
    if (on) guard.emplace();
  }
};

// The operators have no forward-mode derivatives: a tangent would be dropped without a word below
// autograd, and a missing tangent counts as zero.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(/*level=*/0).defined(), what,
                                ": forward-mode derivatives are not implemented");
}

OptTensor optional_of(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct DropoutNode : torch::autograd::Function<DropoutNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& state, double p,
                        int64_t site, const std::string& act) {
    BelowAutograd below(true);
    Tensor y = call_dropout_fwd(x, state, p, site, act);
    const bool relu = act == "relu";  // the ReLU's gradient needs y, which the next layer keeps anyway
    ctx->save_for_backward({relu ? y : Tensor(), relu ? Tensor() : given(state)});
    ctx->saved_data["p"] = p;
    ctx->saved_data["site"] = site;
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    refuse_tangents(kDrop, {&grads[0]});
    BelowAutograd below;
    Tensor gx = call_dropout_bwd(grads[0], optional_of(saved[0]), optional_of(saved[1]),
                                 ctx->saved_data["p"].toDouble(), ctx->saved_data["site"].toInt(),
                                 ctx->saved_data["act"].toStringRef());
    return {gx, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct AddNormNode : torch::autograd::Function<AddNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual,
                        const Tensor& weight, const Tensor& bias, const OptTensor& state, double p,
                        int64_t site, double eps) {
    BelowAutograd below(true);
    Tensor y, mean, rstd;
    std::tie(y, mean, rstd) =
        call_add_norm_fwd(x, residual, weight, bias, state, p, site, eps, true);
    ctx->save_for_backward({x, residual, weight, mean, rstd, given(state)});
    ctx->saved_data["p"] = p;
    ctx->saved_data["site"] = site;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = find<decltype(add_norm_bwd)>("unipercept::dropout_add_norm_bwd");
    const variable_list saved = ctx->get_saved_variables();
    const double p = ctx->saved_data["p"].toDouble();
    const bool need_x = ctx->needs_input_grad(0), need_r = ctx->needs_input_grad(1);
    const bool need_w = ctx->needs_input_grad(2), need_b = ctx->needs_input_grad(3);
    // nothing dropped and one type: both gradients are the same tensor
    const bool shared = p == 0.0 && saved[0].scalar_type() == saved[1].scalar_type();
    refuse_tangents(kNorm, {&grads[0]});
    BelowAutograd below;
    Tensor gx, gr, gw, gb;
    std::tie(gx, gr, gw, gb) =
        op.call(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4], optional_of(saved[5]), p,
                ctx->saved_data["site"].toInt(), need_x && !shared, need_r || (shared && need_x),
                need_w || need_b);
    if (shared) gx = gr;
    return {need_x ? gx : Tensor(), need_r ? gr : Tensor(), need_w ? gw : Tensor(),
            need_b ? gb : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct GroupNormNode : torch::autograd::Function<GroupNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& bias,
                        int64_t groups, IntArrayRef rows, double eps, const std::string& act) {
    BelowAutograd below(true);
    Tensor y, mean, rstd;
    std::tie(y, mean, rstd) = call_group_norm_fwd(x, weight, bias, groups, rows, eps, act, true);
    ctx->save_for_backward({x, weight, bias, mean, rstd});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["rows"] = rows.vec();
    ctx->saved_data["act"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = find<decltype(group_norm_bwd)>("unipercept::level_group_norm_bwd");
    const variable_list saved = ctx->get_saved_variables();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = ctx->needs_input_grad(2);
    refuse_tangents(kGroup, {&grads[0]});
    BelowAutograd below;
    Tensor gx, gw, gb;
    std::tie(gx, gw, gb) = op.call(
        grads[0], saved[0], saved[1], saved[2], saved[3], saved[4], ctx->saved_data["groups"].toInt(),
        ctx->saved_data["rows"].toIntVector(), ctx->saved_data["act"].toStringRef(), need_x,
        need_w || need_b);
    return {need_x ? gx : Tensor(), need_w ? gw : Tensor(), need_b ? gb : Tensor(),
            Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

bool grad_wanted(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->requires_grad()) return true;
  return false;
}

// ---- the operators --------------------------------------------------------------------------------------

Tensor counter_dropout(const Tensor& x, double p, const OptTensor& state_, int64_t site,
                       const std::string& activation) {
  check_tensor(kDrop, x);
  activation_code(kDrop, activation, true);
  check_rng(kDrop, p, site, given(state_), x);
  if (p == 0.0 && activation == "none") return x;
  refuse_tangents(kDrop, {&x});
  const OptTensor state = p > 0.0 ? state_ : OptTensor();
  if (grad_wanted({&x})) return DropoutNode::apply(x, state, p, site, activation);
  BelowAutograd below(true);
  return call_dropout_fwd(x, state, p, site, activation);
}

Tensor dropout_add_layer_norm(const Tensor& x, const Tensor& residual, const Tensor& weight,
                              const Tensor& bias, double p, const OptTensor& state_, int64_t site,
                              double eps) {
  check_add_norm(x, residual, weight, bias, given(state_), p, site, eps);
  refuse_tangents(kNorm, {&x, &residual, &weight, &bias});
  const OptTensor state = p > 0.0 ? state_ : OptTensor();
  if (grad_wanted({&x, &residual, &weight, &bias}))
    return AddNormNode::apply(x, residual, weight, bias, state, p, site, eps);
  BelowAutograd below(true);
  return std::get<0>(
      call_add_norm_fwd(x, residual, weight, bias, state, p, site, eps, false));
}

Tensor level_group_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups,
                        IntArrayRef rows_, double eps, const std::string& activation) {
  activation_code(kGroup, activation, false);
  const std::vector<int64_t> rows = level_rows(x, rows_);
  check_group_norm(x, weight, bias, groups, rows, eps);
  refuse_tangents(kGroup, {&x, &weight, &bias});
  if (grad_wanted({&x, &weight, &bias}))
    return GroupNormNode::apply(x, weight, bias, groups, IntArrayRef(rows), eps, activation);
  BelowAutograd below(true);
  return std::get<0>(call_group_norm_fwd(x, weight, bias, groups, rows, eps, activation, false));
}

// ---- vmap ---------------------------------------------------------------------------------------------

// Levels of torch.func.vmap that a tensor is mapped at.
std::vector<int64_t> mapped_levels(const Tensor& t) {
  std::vector<int64_t> levels;
  const at::functorch::BatchedTensorImpl* batched = at::functorch::maybeGetBatchedImpl(t);
  for (; batched != nullptr; batched = at::functorch::maybeGetBatchedImpl(batched->value()))
    levels.push_back(batched->level());
  return levels;
}

// vmap runs an operator sample by sample, each from element 0 of the same state: every sample would
// drop the same elements.  Right where the caller asks for that (randomness "same") or maps the states
// with the samples; refused otherwise.
void check_vmap(const char* what, double p, const Tensor& state, std::initializer_list<const Tensor*> tensors) {
  if (p == 0.0) return;
  std::vector<int64_t> repeated;
  for (const Tensor* t : tensors)
    for (int64_t level : mapped_levels(*t)) repeated.push_back(level);
  if (repeated.empty()) return;
  for (int64_t level : mapped_levels(state))
    repeated.erase(std::remove(repeated.begin(), repeated.end(), level), repeated.end());
  if (repeated.empty()) return;
  // torch's own random operators know the mode: no numbers at all are drawn here, which raises in mode
  // "error" and returns a mapped tensor in mode "different"
  for (int64_t level : mapped_levels(at::rand({0}, at::TensorOptions(at::kCPU))))
    TORCH_CHECK(std::find(repeated.begin(), repeated.end(), level) == repeated.end(), what,
                ": every sample of this vmap would get the same mask; map rng_state with the samples, or "
                "call the operator on the batch");
}

// Under vmap: checked, then sample by sample (the *_each operators have no kernel here).
Tensor counter_dropout_vmap(const Tensor& x, double p, const OptTensor& state, int64_t site,
                            const std::string& activation) {
  check_vmap(kDrop, p, given(state), {&x});
  static const auto op = find<decltype(counter_dropout)>("unipercept::counter_dropout_each");
  return op.call(x, p, state, site, activation);
}

Tensor dropout_add_layer_norm_vmap(const Tensor& x, const Tensor& residual, const Tensor& weight,
                                   const Tensor& bias, double p, const OptTensor& state, int64_t site,
                                   double eps) {
  check_vmap(kNorm, p, given(state), {&x, &residual, &weight, &bias});
  static const auto op = find<decltype(dropout_add_layer_norm)>("unipercept::dropout_add_layer_norm_each");
  return op.call(x, residual, weight, bias, p, state, site, eps);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(unipercept, m) {
  m.def("counter_dropout(Tensor x, float p, Tensor? rng_state, int site, str activation) -> Tensor");
  m.def("counter_dropout_each(Tensor x, float p, Tensor? rng_state, int site, str activation) -> Tensor");
  m.def(
      "dropout_add_layer_norm_each(Tensor x, Tensor residual, Tensor weight, Tensor bias, float p, "
      "Tensor? rng_state, int site, float eps) -> Tensor");
  m.def("counter_dropout_fwd(Tensor x, Tensor? rng_state, float p, int site, str activation) -> Tensor");
  m.def(
      "counter_dropout_bwd(Tensor grad_output, Tensor? out, Tensor? rng_state, float p, int site, "
      "str activation) -> Tensor");
  m.def(
      "dropout_add_layer_norm(Tensor x, Tensor residual, Tensor weight, Tensor bias, float p, "
      "Tensor? rng_state, int site, float eps) -> Tensor");
  m.def(
      "dropout_add_norm_fwd(Tensor x, Tensor residual, Tensor weight, Tensor bias, Tensor? rng_state, "
      "float p, int site, float eps, bool stats) -> (Tensor, Tensor, Tensor)");
  m.def(
      "dropout_add_norm_bwd(Tensor grad_output, Tensor x, Tensor residual, Tensor weight, Tensor mean, "
      "Tensor rstd, Tensor? rng_state, float p, int site, bool want_x, bool want_residual, "
      "bool want_params) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "level_group_norm(Tensor x, Tensor weight, Tensor bias, int num_groups, int[] rows, float eps, "
      "str activation) -> Tensor");
  m.def(
      "level_group_norm_fwd(Tensor x, Tensor weight, Tensor bias, int num_groups, int[] rows, float eps, "
      "str activation, bool stats) -> (Tensor, Tensor, Tensor)");
  m.def(
      "level_group_norm_bwd(Tensor grad_output, Tensor x, Tensor weight, Tensor bias, Tensor mean, "
      "Tensor rstd, int num_groups, int[] rows, str activation, bool want_x, bool want_params) -> "
      "(Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(unipercept, CompositeImplicitAutograd, m) {
  m.impl("counter_dropout", counter_dropout);
  m.impl("dropout_add_layer_norm", dropout_add_layer_norm);
  m.impl("level_group_norm", level_group_norm);
  m.impl("counter_dropout_each", counter_dropout);
  m.impl("dropout_add_layer_norm_each", dropout_add_layer_norm);
}

TORCH_LIBRARY_IMPL(unipercept, FuncTorchBatched, m) {
  m.impl("counter_dropout", counter_dropout_vmap);
  m.impl("dropout_add_layer_norm", dropout_add_layer_norm_vmap);
}

TORCH_LIBRARY_IMPL(unipercept, CUDA, m) {
  m.impl("counter_dropout_fwd", dropout_fwd);
  m.impl("counter_dropout_bwd", dropout_bwd);
  m.impl("dropout_add_norm_fwd", add_norm_fwd);
  m.impl("dropout_add_norm_bwd", add_norm_bwd);
  m.impl("level_group_norm_fwd", group_norm_fwd);
  m.impl("level_group_norm_bwd", group_norm_bwd);
}

TORCH_LIBRARY_IMPL(unipercept, Meta, m) {
  m.impl("counter_dropout_fwd", dropout_fwd_meta);
  m.impl("counter_dropout_bwd", dropout_bwd_meta);
  m.impl("dropout_add_norm_fwd", add_norm_fwd_meta);
  m.impl("dropout_add_norm_bwd", add_norm_bwd_meta);
  m.impl("level_group_norm_fwd", group_norm_fwd_meta);
  m.impl("level_group_norm_bwd", group_norm_bwd_meta);
}

TORCH_LIBRARY_IMPL(unipercept, Autograd, m) {
  for (const char* name : {"counter_dropout_fwd", "counter_dropout_bwd", "dropout_add_norm_fwd",
                           "dropout_add_norm_bwd", "level_group_norm_fwd", "level_group_norm_bwd"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
