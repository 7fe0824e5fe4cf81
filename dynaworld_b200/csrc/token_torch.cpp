// torch binding of the token-side operators: argument checks, outputs, workspaces and the autograd
// nodes of linear and rms_norm around the C entry points of libgsb200 (bound by address, so that this
// file needs the library's header only).
//
// The render stages are bound in Python (ctypes, torch.autograd.Function): a frame is milliseconds.
// These operators take microseconds, and one product of a single token spent 3 us on the GPU and
// 12.5 on the host that way, a norm with its gradients 107, most of it in the Python halves of the
// autograd engine.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <string>

#include "gsb200.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ---- the C entry points -----------------------------------------------------------------------

#define GSB_TOKEN_ENTRIES(X)                                                                       \
  X(gsb_rms_norm_fwd) X(gsb_rms_norm_bwd_workspace) X(gsb_rms_norm_bwd) X(gsb_rms_norm_fp8)        \
  X(gsb_quantize_rows_fp8) X(gsb_linear_fwd_workspace) X(gsb_linear_fwd) X(gsb_linear_bwd_workspace) \
  X(gsb_linear_bwd)

struct Entries {
#define X(name) decltype(&::name) name = nullptr;
  GSB_TOKEN_ENTRIES(X)
#undef X
} lib;

void bind(const std::map<std::string, uintptr_t>& addresses) {
#define X(name) lib.name = reinterpret_cast<decltype(lib.name)>(addresses.at(#name));
  GSB_TOKEN_ENTRIES(X)
#undef X
}

// Raises as every other call of the library does.
void check_status(const char* name, int status) {
  if (status == GSB_OK) return;
  py::gil_scoped_acquire gil;
  py::module_::import("dynaworld_b200._lib").attr("check")(name, status);
}

// The stage's NVTX range and events, when tracing was on at the forward call.
class Stage {
 public:
  Stage(const char* name, bool traced) {
    if (!traced) return;
    py::gil_scoped_acquire gil;
    stage_ = py::module_::import("dynaworld_b200.render").attr("_stage")(name);
    stage_.attr("__enter__")();
  }
  ~Stage() {
    if (!stage_) return;
    py::gil_scoped_acquire gil;
    try {
      stage_.attr("__exit__")(py::none(), py::none(), py::none());
    } catch (py::error_already_set& e) {
      e.discard_as_unraisable("token stage");
    }
    stage_ = py::object();
  }

 private:
  py::object stage_;
};

// ---- arguments --------------------------------------------------------------------------------

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return GSB_F32;
    case at::kBFloat16: return GSB_BF16;
    case at::kHalf: return GSB_F16;
    default: return -1;
  }
}

// As Python prints it.
std::string name_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kDouble: return "torch.float64";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kFloat8_e4m3fn: return "torch.float8_e4m3fn";
    default: return at::toString(t);
  }
}

int check_input(const char* what, const Tensor& x) {
  const int code = type_code(x.scalar_type());
  TORCH_CHECK_TYPE(code >= 0, what, " takes float32, bfloat16 or float16 tensors, got ", name_of(x.scalar_type()));
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, what, " needs rows of at least one element, got shape ",
                    x.sizes());
  return code;
}

void check_like(const char* what, const char* name, const Tensor& t, at::IntArrayRef shape, at::ScalarType type,
                const Tensor& x) {
  TORCH_CHECK_VALUE(t.sizes() == shape, what, ": ", name, " must have shape ", shape, ", got ", t.sizes());
  TORCH_CHECK_TYPE(t.scalar_type() == type, what, ": ", name, " must be ", name_of(type), ", got ",
                   name_of(t.scalar_type()));
  TORCH_CHECK(t.device() == x.device(), what, ": ", name, " is on ", t.device(), ", the input on ", x.device());
}

void check_device(const char* what, const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "the b200 ", what, " runs on CUDA devices only (got a tensor on ", x.device(), ")");
}

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t && t->requires_grad(); }

bool has_tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }

// Forward-mode derivatives have no formula here: a dual tensor (which need not require a gradient) would
// lose its tangent silently.
template <typename... T>
void refuse_tangent(const char* what, const T&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && (has_tangent(t) || ...)), what,
                              " has no forward-mode derivative; unpack its dual tensors or use reverse mode.");
}

template <typename... T>
void refuse_grad(const char* what, const T&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(at::GradMode::is_enabled() && (wants_grad(t) || ...)), what,
                              " is not differentiable; call it under torch.no_grad() or detach its inputs.");
}

// [..., width] as [rows, width] with adjacent row elements: a view where the strides allow it (any
// positive row stride), else a copy.
Tensor rows_of(const Tensor& t, int64_t width) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, width});
  if ((r.stride(1) != 1 && width > 1) || (r.stride(0) < 1 && r.size(0) > 1)) r = r.contiguous();
  return r.is_neg() ? r.resolve_neg() : r;  // a view may stand for the negative of what its memory holds
}
OptTensor rows_of(const OptTensor& t, int64_t width) {
  return t ? OptTensor(rows_of(*t, width)) : std::nullopt;
}

// [n] with adjacent elements.
Tensor line_of(const Tensor& t) { return t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous(); }
OptTensor line_of(const OptTensor& t) { return t ? OptTensor(line_of(*t)) : std::nullopt; }

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* address(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

// A new tensor on like's device, past the dispatcher: half the time of at::empty, and a call makes
// one to three.
Tensor empty(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
  return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}
Tensor workspace(const Tensor& like, size_t bytes) {
  return bytes ? empty(like, {int64_t(bytes)}, at::kByte) : Tensor();
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

at::DimVector with_last(at::IntArrayRef shape, int64_t last) {
  at::DimVector s(shape.begin(), shape.end());
  s.back() = last;
  return s;
}

// A backward that built a graph would lose the second derivatives silently: its outputs raise when
// they are differentiated.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that is differentiable once", int64_t(grads.size()));
  return (*error)(std::move(grads));
}

// ---- linear -----------------------------------------------------------------------------------

int activation_code(const std::string& name) {
  static const char* names[] = {"none", "relu", "gelu", "gelu_tanh", "silu"};
  for (int i = 0; i < 5; ++i)
    if (name == names[i]) return i;
  TORCH_CHECK_VALUE(false, "Unknown activation: '", name, "' (one of none, relu, gelu, gelu_tanh, silu)");
}

gsb_linear linear_spec(const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& residual, int act,
                       int code, int out_code) {
  gsb_linear p{};
  p.m = x.size(0);
  p.n = int32_t(w.size(0));
  p.k = int32_t(w.size(1));
  p.dtype = code;
  p.out_dtype = out_code;
  p.activation = act;
  p.x = address(x);
  p.x_stride = x.stride(0);
  p.weight = address(w);
  p.weight_stride = w.stride(0);
  p.bias = address(bias);
  p.residual = address(residual);
  p.residual_stride = residual ? residual->stride(0) : 0;
  return p;
}

void linear_forward(const gsb_linear& p, const Tensor& y, const Tensor& preact, bool traced) {
  const c10::cuda::CUDAGuard guard(y.device());
  Stage stage("linear", traced);
  const size_t bytes = lib.gsb_linear_fwd_workspace(&p);
  const Tensor ws = workspace(y, bytes);
  check_status("gsb_linear_fwd", lib.gsb_linear_fwd(&p, address(y), address(preact), address(ws), bytes, stream_of(y)));
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias,
                        const OptTensor& residual, int64_t act, int64_t code, bool traced) {
    const Tensor y = empty(x, {x.size(0), w.size(0)}, x.scalar_type());
    Tensor preact;
    if (act != GSB_ACT_NONE && (x.requires_grad() || w.requires_grad() || wants_grad(bias)))
      preact = empty(x, y.sizes(), code == GSB_F32 ? at::kFloat : at::kHalf);
    linear_forward(linear_spec(x, w, bias, residual, int(act), int(code), int(code)), y, preact, traced);
    ctx->save_for_backward({x, w, preact});
    ctx->saved_data["how"] = c10::List<int64_t>({act, code, traced, bias.has_value(), residual.has_value()});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &preact = saved[2];
    const auto how = ctx->saved_data["how"].toIntVector();
    const bool has_bias = how[3], has_residual = how[4];
    // edges: x, w, then the optional ones that are there
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_b = has_bias && ctx->needs_input_grad(2);
    const bool need_r = has_residual && ctx->needs_input_grad(2 + has_bias);
    Tensor dx, dw, db;
    const Tensor& dy = grads[0];
    if (dy.defined() && (need_x || need_w || need_b)) {
      const c10::cuda::CUDAGuard guard(x.device());
      Stage stage("linear_bwd", how[2]);
      const Tensor g = rows_of(dy, w.size(0));
      if (need_x) dx = empty(x, {x.size(0), w.size(1)}, x.scalar_type());
      if (need_w) dw = empty(x, {w.size(0), w.size(1)}, x.scalar_type());
      if (need_b) db = empty(x, {w.size(0)}, x.scalar_type());
      const gsb_linear p = linear_spec(x, w, std::nullopt, std::nullopt, int(how[0]), int(how[1]), int(how[1]));
      const size_t bytes = lib.gsb_linear_bwd_workspace(&p, address(g), g.stride(0));
      const Tensor ws = workspace(x, bytes);
      check_status("gsb_linear_bwd", lib.gsb_linear_bwd(&p, address(preact), address(g), g.stride(0), address(dx),
                                                        address(dw), address(db), address(ws), bytes, stream_of(x)));
    }
    variable_list out = once({dx, dw, db, need_r ? dy : Tensor()});
    out.resize(7);
    return out;
  }
};

int64_t check_shapes(const char* what, const Tensor& x, const Tensor& w, const OptTensor& bias,
                     const OptTensor& residual, at::ScalarType type) {
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == x.size(-1) && w.size(0) >= 1, what, ": weight must be [n, ",
                    x.size(-1), "], got ", w.sizes());
  TORCH_CHECK_VALUE(w.size(0) <= (1 << 24) && w.size(1) <= (1 << 24), what, ": weight ", w.sizes(),
                    " is larger than 2^24 on a side");
  TORCH_CHECK_TYPE(w.scalar_type() == x.scalar_type(), what, ": weight must be ", name_of(x.scalar_type()), ", got ",
                   name_of(w.scalar_type()));
  TORCH_CHECK(w.device() == x.device(), what, ": weight is on ", w.device(), ", the input on ", x.device());
  const int64_t n = w.size(0);
  if (bias) check_like(what, "bias", *bias, {n}, type, x);
  if (residual) check_like(what, "residual", *residual, with_last(x.sizes(), n), type, x);
  return n;
}

Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
              const std::string& activation, bool traced) {
  const int code = check_input("linear", x);
  const int act = activation_code(activation);
  const int64_t n = check_shapes("linear", x, weight, bias, residual, x.scalar_type());
  refuse_tangent("linear", x, weight, bias, residual);
  check_device("linear", x);
  const Tensor x2 = rows_of(x, x.size(-1)), w2 = rows_of(weight, weight.size(1));
  const OptTensor r2 = rows_of(residual, n), b = line_of(bias);
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || wants_grad(bias) || wants_grad(residual))) {
    const Tensor y = LinearNode::apply(x2, w2, b, r2, int64_t(act), int64_t(code), traced);
    return x.dim() == 2 ? y : y.view(with_last(x.sizes(), n));
  }
  const Tensor y = empty(x, with_last(x.sizes(), n), x.scalar_type());
  linear_forward(linear_spec(x2, w2, b, r2, act, code, code), y, Tensor(), traced);
  return y;
}

Tensor linear_fp8(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& weight_scale,
                  const OptTensor& bias, const OptTensor& residual, const std::string& activation,
                  const py::object& dtype, bool traced) {
  const char* what = "linear_fp8";
  TORCH_CHECK_TYPE(x.scalar_type() == at::kFloat8_e4m3fn, what, " takes torch.float8_e4m3fn codes, got ",
                   name_of(x.scalar_type()));
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, what, " needs rows of at least one element, got shape ",
                    x.sizes());
  TORCH_CHECK_TYPE(THPDtype_Check(dtype.ptr()), what, ": dtype must be a torch.dtype");
  const at::ScalarType type = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
  const int out_code = type_code(type);
  TORCH_CHECK_TYPE(out_code >= 0, what, " gives float32, bfloat16 or float16, not ", name_of(type));
  const int act = activation_code(activation);
  const int64_t n = check_shapes(what, x, weight, bias, residual, type);
  check_like(what, "x_scale", x_scale, x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
  check_like(what, "weight_scale", weight_scale, {n}, at::kFloat, x);
  refuse_tangent(what, x, x_scale, weight, weight_scale, bias, residual);
  refuse_grad(what, x, x_scale, weight, weight_scale, bias, residual);
  check_device(what, x);
  const Tensor x2 = rows_of(x, x.size(-1)), w2 = rows_of(weight, weight.size(1));
  const OptTensor r2 = rows_of(residual, n), b = line_of(bias);
  const Tensor xs = line_of(x_scale), ws = line_of(weight_scale);
  gsb_linear p = linear_spec(x2, w2, b, r2, act, GSB_E4M3, out_code);
  p.x_scale = static_cast<const float*>(address(xs));
  p.weight_scale = static_cast<const float*>(address(ws));
  const Tensor y = empty(x, with_last(x.sizes(), n), type);
  linear_forward(p, y, Tensor(), traced);
  return y;
}

// ---- norm -------------------------------------------------------------------------------------

gsb_norm norm_spec(const Tensor& x, int code, double eps, const OptTensor& residual, const OptTensor& weight) {
  gsb_norm n{};
  n.rows = x.size(0);
  n.dim = int32_t(x.size(1));
  n.dtype = code;
  n.eps = float(eps);
  n.x = address(x);
  n.x_stride = x.stride(0);
  n.residual = address(residual);
  n.residual_stride = residual ? residual->stride(0) : 0;
  n.weight = address(weight);
  return n;
}

void norm_forward(const gsb_norm& n, const Tensor& y, const Tensor& summed, const Tensor& rstd, bool traced) {
  const c10::cuda::CUDAGuard guard(y.device());
  Stage stage("rms_norm", traced);
  check_status("gsb_rms_norm_fwd", lib.gsb_rms_norm_fwd(&n, address(y), address(summed),
                                                        static_cast<float*>(address(rstd)), stream_of(y)));
}

struct RmsNormNode : torch::autograd::Function<RmsNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual,
                               double eps, int64_t code, bool traced) {
    const Tensor y = empty(x, x.sizes(), x.scalar_type());
    const Tensor summed = residual ? empty(x, x.sizes(), x.scalar_type()) : Tensor();
    const Tensor rstd = empty(x, {x.size(0)}, at::kFloat);
    norm_forward(norm_spec(x, int(code), eps, residual, weight), y, summed, rstd, traced);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, residual.value_or(Tensor()), rstd});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["how"] = c10::List<int64_t>({code, traced});
    if (residual) return {y, summed};
    return {y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &rstd = saved[3];
    const bool has_residual = saved[2].defined();
    const OptTensor residual = has_residual ? OptTensor(saved[2]) : std::nullopt;
    const auto how = ctx->saved_data["how"].toIntVector();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_r = has_residual && ctx->needs_input_grad(2);
    const Tensor none, &dy = grads[0], &dsummed = grads.size() > 1 ? grads[1] : none;
    Tensor dx, dw;
    if (dy.defined()) {
      const c10::cuda::CUDAGuard guard(x.device());
      Stage stage("rms_norm_bwd", how[1]);
      const int64_t dim = x.size(1);
      const Tensor g = rows_of(dy, dim), ds = dsummed.defined() ? rows_of(dsummed, dim) : Tensor();
      dx = empty(x, x.sizes(), x.scalar_type());
      if (need_w) dw = empty(x, {dim}, x.scalar_type());
      const gsb_norm n = norm_spec(x, int(how[0]), ctx->saved_data["eps"].toDouble(), residual, weight);
      const size_t bytes = lib.gsb_rms_norm_bwd_workspace(&n);
      const Tensor ws = workspace(x, bytes);
      check_status("gsb_rms_norm_bwd",
                   lib.gsb_rms_norm_bwd(&n, static_cast<const float*>(address(rstd)), address(g), g.stride(0),
                                        address(ds), ds.defined() ? ds.stride(0) : 0, address(dx), address(dw),
                                        address(ws), bytes, stream_of(x)));
    } else {  // only the stream was used
      dx = dsummed;
      if (need_w) dw = at::zeros_like(weight);
    }
    variable_list out = once({need_x ? dx : Tensor(), dw, need_r ? dx : Tensor()});
    out.resize(6);
    return out;
  }
};

int check_norm(const char* what, const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
  const int code = check_input(what, x);
  TORCH_CHECK_VALUE(x.size(-1) <= (1 << 24), what, ": rows of ", x.size(-1), " values are too long");
  if (weight) check_like(what, "weight", *weight, {x.size(-1)}, x.scalar_type(), x);
  if (residual) check_like(what, "residual", *residual, x.sizes(), x.scalar_type(), x);
  TORCH_CHECK_VALUE(eps >= 0.0, what, ": eps must not be negative, got ", eps);
  refuse_tangent(what, x, weight, residual);
  check_device(what, x);
  return code;
}

py::object rms_norm(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps, bool traced) {
  const int code = check_norm("rms_norm", x, weight, residual, eps);
  const int64_t dim = x.size(-1);
  const Tensor x2 = rows_of(x, dim), w = line_of(weight);
  const OptTensor r2 = rows_of(residual, dim);
  Tensor y, h;
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || wants_grad(residual))) {
    const variable_list out = RmsNormNode::apply(x2, w, r2, eps, int64_t(code), traced);
    y = out[0];
    if (residual) h = out[1];
    if (x.dim() != 2) {
      y = y.view(x.sizes());
      if (residual) h = h.view(x.sizes());
    }
  } else {
    y = empty(x, x.sizes(), x.scalar_type());
    if (residual) h = empty(x, x.sizes(), x.scalar_type());
    norm_forward(norm_spec(x2, code, eps, r2, w), y, h, Tensor(), traced);
  }
  if (residual) return py::make_tuple(y, h);
  return py::cast(y);
}

py::object rms_norm_fp8(const Tensor& x, const Tensor& weight, const OptTensor& residual, double eps, bool traced) {
  const int code = check_norm("rms_norm_fp8", x, weight, residual, eps);
  refuse_grad("rms_norm_fp8", x, weight, residual);
  const int64_t dim = x.size(-1);
  const Tensor x2 = rows_of(x, dim), w = line_of(weight);
  const OptTensor r2 = rows_of(residual, dim);
  const Tensor q = empty(x, x.sizes(), at::kFloat8_e4m3fn);
  const Tensor scale = empty(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
  const Tensor h = residual ? empty(x, x.sizes(), x.scalar_type()) : Tensor();
  {
    const c10::cuda::CUDAGuard guard(x.device());
    Stage stage("rms_norm_fp8", traced);
    const gsb_norm n = norm_spec(x2, code, eps, r2, w);
    check_status("gsb_rms_norm_fp8", lib.gsb_rms_norm_fp8(&n, address(q), static_cast<float*>(address(scale)),
                                                          address(h), stream_of(x)));
  }
  if (residual) return py::make_tuple(q, scale, h);
  return py::make_tuple(q, scale);
}

py::object quantize_rows_fp8(const Tensor& x, bool traced) {
  const int code = check_norm("quantize_rows_fp8", x, std::nullopt, std::nullopt, 0.0);
  refuse_grad("quantize_rows_fp8", x);
  const Tensor x2 = rows_of(x, x.size(-1));
  const Tensor q = empty(x, x.sizes(), at::kFloat8_e4m3fn);
  const Tensor scale = empty(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
  const c10::cuda::CUDAGuard guard(x.device());
  Stage stage("quantize_rows_fp8", traced);
  const gsb_norm n = norm_spec(x2, code, 0.0, std::nullopt, std::nullopt);
  check_status("gsb_quantize_rows_fp8",
               lib.gsb_quantize_rows_fp8(&n, address(q), static_cast<float*>(address(scale)), stream_of(x)));
  return py::make_tuple(q, scale);
}

}  // namespace

PYBIND11_MODULE(_token_torch, m) {
  m.def("bind", &bind);
  m.def("linear", &linear);
  m.def("linear_fp8", &linear_fp8);
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_fp8", &rms_norm_fp8);
  m.def("quantize_rows_fp8", &quantize_rows_fp8);
}
