// binding.cpp -- torch side of pyramid_group_norm, rotary and adamw_step:
// argument checks, allocation, autograd nodes and calls through the C ABI
// (include/msda_b200.h).
//
// These calls take 5 to 50 us on the device at ordinary sizes, and a step of
// many tensors has hundreds of arguments, so the host side is native: a
// forward and backward through a Python autograd function took 133 to 175 us
// where the device work was 18 to 120 us (0.4 us a tensor for the optimizer).
// The functions come from the library that _lib.py has loaded, by address.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/python.h>

#include <algorithm>
#include <array>
#include <string>
#include <vector>

#include "../../include/msda_b200.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------------ the library
struct Api {
  decltype(&msda_status_string) status_string;
  decltype(&msda_last_error) last_error;
  decltype(&msda_group_norm_workspace_bytes) norm_workspace;
  decltype(&msda_group_norm_fwd) norm_fwd;
  decltype(&msda_group_norm_bwd) norm_bwd;
  decltype(&msda_rotary) rotary;
  decltype(&msda_adamw_step) adamw_step;
  decltype(&msda_adamw_values) adamw_values;
} api;

void bind(const std::vector<uintptr_t>& at) {
  TORCH_CHECK(at.size() * sizeof(void*) == sizeof(Api), "binding: one address per function");
  memcpy(&api, at.data(), sizeof(api));
}

// The exception that Python gets for a C status: as _core.check_status.
void check(int code) {
  if (code == MSDA_SUCCESS) return;
  const std::string msg = api.last_error();
  switch (code) {
    case MSDA_ERROR_UNSUPPORTED_DTYPE: TORCH_CHECK_NOT_IMPLEMENTED(false, msg);
    case MSDA_ERROR_INVALID_ARGUMENT:
    case MSDA_ERROR_SHAPE_MISMATCH:
    case MSDA_ERROR_TOO_MANY_LEVELS:
    case MSDA_ERROR_INT32_OVERFLOW:
    case MSDA_ERROR_MISALIGNED:
    case MSDA_ERROR_WORKSPACE:
    case MSDA_ERROR_UNSUPPORTED_CHANNELS: TORCH_CHECK_VALUE(false, msg);
    default: TORCH_CHECK(false, api.status_string(code), ": ", msg);
  }
}

int dtype_code(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return MSDA_FLOAT32;
    case at::kHalf: return MSDA_FLOAT16;
    case at::kBFloat16: return MSDA_BFLOAT16;
    default:
      TORCH_CHECK_NOT_IMPLEMENTED(false, what, " only supports fp32, fp16, and bf16. Got ",
                                  torch::getTHPDtype(t.scalar_type())->name, ".");
  }
}

void* current_stream(const Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

void* ptr(const optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }

Tensor empty(at::IntArrayRef shape, const Tensor& like, at::ScalarType dtype) {
  return at::detail::empty_cuda(shape, dtype, like.device(), at::MemoryFormat::Contiguous);
}
Tensor empty(at::IntArrayRef shape, const Tensor& like) {
  return empty(shape, like, like.scalar_type());
}

const Tensor& tensor_of(PyObject* o, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be tensors, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

// The gradients of a backward have none themselves: under create_graph they
// say so where they are differentiated, instead of passing for constants.
void once_differentiable(const variable_list& grads, variable_list& out) {
  if (!at::GradMode::is_enabled()) return;
  auto node = std::make_shared<torch::autograd::Error>(
      "this operator's backward has no derivative", torch::autograd::collect_next_edges(grads));
  for (Tensor& t : out)
    if (t.defined()) torch::autograd::set_history(t, node);
}

// Forward-mode derivatives there are none of either, and a dual tensor may not
// require a gradient: its tangent would be dropped beside the autograd function.
// Looking for a tangent takes 20 ns a tensor, so callers ask once whether there
// can be any.
bool dual_level() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what,
                              " has no forward-mode derivative");
}

// ------------------------------------------------------------------ group norm
struct Norm {
  bool maps;
  std::vector<int64_t> rows;
  int64_t groups;
  double eps;
  int activation;
};

int activation_code(const std::string& name) {
  static const char* const kNames[] = {"none", "relu", "silu", "gelu"};
  for (int i = 0; i < 4; ++i)
    if (name == kNames[i]) return i;
  TORCH_CHECK_VALUE(false, "activation must be one of ['gelu', 'none', 'relu', 'silu'], got '",
                    name, "'");
}

using Sizes = std::vector<std::vector<int64_t>>;

Sizes level_sizes(const py::object& shapes) {
  if (!THPVariable_Check(shapes.ptr())) return shapes.cast<Sizes>();
  Tensor t = THPVariable_Unpack(shapes.ptr());
  TORCH_CHECK_VALUE(!t.is_floating_point() && t.scalar_type() != at::kBool && !t.is_complex(),
                    "spatial_shapes must be an integer tensor, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == 2, "spatial_shapes must be (L, d), got ", t.sizes());
  t = t.to(at::kCPU, at::kLong).contiguous();
  Sizes out(t.size(0));
  const int64_t* p = t.const_data_ptr<int64_t>();
  for (auto& s : out) {
    s.assign(p, p + t.size(1));
    p += t.size(1);
  }
  return out;
}

variable_list norm_inputs(const py::object& x) {
  if (THPVariable_Check(x.ptr())) return {THPVariable_Unpack(x.ptr())};
  variable_list xs;
  for (const auto& o : py::reinterpret_borrow<py::sequence>(x))
    xs.push_back(tensor_of(o.ptr(), "levels"));
  return xs;
}

Norm norm_check(const variable_list& xs, bool maps, const py::object& spatial_shapes,
                int64_t groups, const optional<Tensor>& weight, const optional<Tensor>& bias,
                double eps, const std::string& activation) {
  TORCH_CHECK_VALUE(!xs.empty(), "pyramid_group_norm needs at least one level");
  const Tensor& first = xs[0];
  TORCH_CHECK_VALUE(first.is_cuda(),
                    "pyramid_group_norm requires CUDA tensors. Got CPU tensors instead.");
  dtype_code(first, "pyramid_group_norm");
  if (dual_level()) {
    for (const Tensor& t : xs) no_tangent(t, "pyramid_group_norm");
    for (const auto* p : {&weight, &bias})
      if (*p) no_tangent(**p, "pyramid_group_norm");
  }
  for (const Tensor& t : xs) {
    TORCH_CHECK_VALUE(maps ? t.dim() >= 3 : t.dim() == 3,
                      "x must be (B, K, C), or levels of (B, *spatial, C); got ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == first.device() && t.scalar_type() == first.scalar_type() &&
                          t.size(0) == first.size(0) && t.size(-1) == first.size(-1),
                      "levels must share their device, dtype, batch and channels; got ", t.sizes(),
                      " ", t.scalar_type(), " beside ", first.sizes(), " ", first.scalar_type());
  }
  Norm n{maps, {}, groups, eps, activation_code(activation)};
  if (maps) {
    for (const Tensor& t : xs) {
      int64_t rows = 1;
      for (int64_t s : t.sizes().slice(1, t.dim() - 2)) rows *= s;
      n.rows.push_back(rows);
    }
    if (!spatial_shapes.is_none()) {
      const Sizes sizes = level_sizes(spatial_shapes);
      bool same = sizes.size() == xs.size();
      for (size_t l = 0; same && l < xs.size(); ++l)
        same = at::IntArrayRef(sizes[l]) == xs[l].sizes().slice(1, xs[l].dim() - 2);
      TORCH_CHECK_VALUE(same, "spatial_shapes do not match the levels' sizes");
    }
  } else {
    TORCH_CHECK_VALUE(!spatial_shapes.is_none(),
                      "spatial_shapes is required for a flattened pyramid");
    int64_t sum = 0;
    for (const auto& s : level_sizes(spatial_shapes)) {
      int64_t rows = 1;
      for (int64_t k : s) {
        TORCH_CHECK_VALUE(k >= 0, "negative spatial shape: ", s);
        TORCH_CHECK_VALUE(!__builtin_mul_overflow(rows, k, &rows), "spatial shape too large: ", s);
      }
      n.rows.push_back(rows);
      TORCH_CHECK_VALUE(!__builtin_add_overflow(sum, rows, &sum), "spatial shapes too large");
    }
    TORCH_CHECK_VALUE(sum == first.size(1), "K=", first.size(1),
                      " does not match sum of spatial shapes ", sum);
  }
  const int64_t channels = first.size(-1), levels = static_cast<int64_t>(n.rows.size());
  TORCH_CHECK_VALUE(groups >= 1 && channels >= 1 && channels % groups == 0, "channels (", channels,
                    ") must be a positive multiple of num_groups (", groups, ")");
  for (const auto* p : {&weight, &bias}) {
    if (!*p) continue;
    const char* name = p == &weight ? "weight" : "bias";
    const Tensor& t = **p;
    TORCH_CHECK_VALUE(t.device() == first.device(), name, " must be on ", first.device(), ", got ",
                      t.device());
    dtype_code(t, name);
    TORCH_CHECK_VALUE((t.dim() == 1 && t.size(0) == channels) ||
                          (t.dim() == 2 && t.size(0) == levels && t.size(1) == channels),
                      name, " must be (", channels, ",) or (", levels, ", ", channels, "), got ",
                      t.sizes());
  }
  TORCH_CHECK_VALUE(!weight || !bias || weight->sizes() == bias->sizes(), "weight ",
                    weight->sizes(), " and bias ", bias->sizes(), " differ in shape");
  return n;
}

// Elements between neighbouring rows of (B, *spatial, C), or -1 where no one step serves them all.
int64_t row_stride(const Tensor& t) {
  if (t.numel() == 0) return 0;
  if (t.stride(-1) != 1 && t.size(-1) > 1) return -1;
  int64_t step = 0, rows = 1;
  for (int64_t d = t.dim() - 2; d >= 1; --d) {
    if (t.size(d) == 1) continue;
    if (rows == 1) step = t.stride(d);
    else if (t.stride(d) != step * rows) return -1;
    rows *= t.size(d);
  }
  return step;
}

// Host tables of the levels' addresses and (batch, row) strides; copies what
// has no evenly spaced rows of dense channels.
struct Levels {
  std::vector<void*> at;
  std::vector<int64_t> strides;
  variable_list copies;
  Levels(bool maps, const variable_list& xs, const std::vector<int64_t>& rows) {
    auto add = [&](const Tensor& t) -> std::pair<Tensor, int64_t> {
      const int64_t step = row_stride(t);
      if (step >= 0) return {t, step};
      copies.push_back(t.contiguous());
      return {copies.back(), row_stride(copies.back())};
    };
    if (maps) {
      for (const Tensor& x : xs) {
        const auto [t, step] = add(x);
        at.push_back(t.data_ptr());
        strides.insert(strides.end(), {t.stride(0), step});
      }
    } else {
      const auto [t, step] = add(xs[0]);
      char* p = static_cast<char*>(t.data_ptr());
      for (int64_t n : rows) {
        at.push_back(p);
        p += n * step * t.element_size();
        strides.insert(strides.end(), {t.stride(0), step});
      }
    }
  }
};

struct Affine {
  optional<Tensor> weight, bias;
  int dtype = MSDA_FLOAT32, per_level = 0;
  Affine(optional<Tensor> w, optional<Tensor> b) {
    if (w && b && w->scalar_type() != b->scalar_type()) {
      w = w->to(at::kFloat);
      b = b->to(at::kFloat);
    }
    if (w) weight = w->contiguous();
    if (b) bias = b->contiguous();
    if (weight || bias) {
      const Tensor& one = weight ? *weight : *bias;
      dtype = dtype_code(one, "affine map");
      per_level = one.dim() == 2;
    }
  }
};

// y, and the statistics with the workspace behind them.
std::pair<Tensor, Tensor> norm_forward(const Norm& n, const variable_list& xs,
                                       const optional<Tensor>& weight,
                                       const optional<Tensor>& bias) {
  at::NoGradGuard no_grad;
  const Tensor& first = xs[0];
  const c10::cuda::CUDAGuard guard(first.device());
  const int64_t batch = first.size(0), channels = first.size(-1);
  const int64_t levels = static_cast<int64_t>(n.rows.size());
  const int code = dtype_code(first, "pyramid_group_norm");
  int64_t keys = 0;
  for (int64_t r : n.rows) keys += r;
  const Levels x(n.maps, xs, n.rows);
  const Affine affine(weight, bias);
  const size_t ws = api.norm_workspace(code, batch, channels, n.groups, levels, n.rows.data(), 0);
  const int64_t front = (batch * levels * n.groups * 2 + 63) / 64 * 64;  // 256-byte boundary
  Tensor y = empty({batch, keys, channels}, first);
  Tensor stats = empty({front + static_cast<int64_t>(ws / 4)}, first, at::kFloat);
  float* s = stats.data_ptr<float>();
  check(api.norm_fwd(code, batch, channels, n.groups, levels, n.rows.data(), x.at.data(),
                     x.strides.data(), ptr(affine.weight), ptr(affine.bias), affine.dtype,
                     affine.per_level, n.eps, n.activation, y.data_ptr(), s, s + front, ws,
                     current_stream(first)));
  return {y, stats};
}

// Gradients of xs, then of weight and bias (undefined where there is none).
variable_list norm_backward(const Norm& n, const variable_list& xs, const optional<Tensor>& weight,
                            const optional<Tensor>& bias, const Tensor& stats,
                            const Tensor& grad_y) {
  if (dual_level()) no_tangent(grad_y, "pyramid_group_norm's backward");
  at::NoGradGuard no_grad;
  const Tensor& first = xs[0];
  const c10::cuda::CUDAGuard guard(first.device());
  const int64_t batch = first.size(0), channels = first.size(-1);
  const int64_t levels = static_cast<int64_t>(n.rows.size());
  const int code = dtype_code(first, "pyramid_group_norm");
  const Tensor gy = grad_y.to(first.scalar_type()).contiguous();
  const Levels x(n.maps, xs, n.rows);
  const Affine affine(weight, bias);
  variable_list out;
  for (const Tensor& t : xs) out.push_back(empty(t.sizes(), t));
  const Levels gx(n.maps, out, n.rows);
  Tensor gw, gb;
  if (affine.weight) gw = at::empty_like(*affine.weight);
  if (affine.bias) gb = at::empty_like(*affine.bias);
  const size_t bytes =
      api.norm_workspace(code, batch, channels, n.groups, levels, n.rows.data(), 1);
  Tensor ws = empty({static_cast<int64_t>(bytes)}, first, at::kByte);
  check(api.norm_bwd(code, batch, channels, n.groups, levels, n.rows.data(), x.at.data(),
                     x.strides.data(), ptr(affine.weight), ptr(affine.bias), affine.dtype,
                     affine.per_level, n.activation, stats.data_ptr<float>(), gy.data_ptr(),
                     gx.at.data(), gx.strides.data(), gw.defined() ? gw.data_ptr() : nullptr,
                     gb.defined() ? gb.data_ptr() : nullptr, ws.data_ptr(), bytes,
                     current_stream(first)));
  out.push_back(gw.defined() ? gw.to(weight->scalar_type()) : gw);
  out.push_back(gb.defined() ? gb.to(bias->scalar_type()) : gb);
  return out;
}

class PyramidGroupNormFn : public torch::autograd::Function<PyramidGroupNormFn> {
 public:
  static Tensor forward(AutogradContext* ctx, at::TensorList xs, const optional<Tensor>& weight,
                        const optional<Tensor>& bias, const Norm& n) {
    variable_list saved(xs.begin(), xs.end());
    auto [y, stats] = norm_forward(n, saved, weight, bias);
    saved.push_back(stats);
    saved.push_back(weight.value_or(Tensor()));
    saved.push_back(bias.value_or(Tensor()));
    ctx->save_for_backward(saved);
    ctx->saved_data["maps"] = n.maps;
    ctx->saved_data["rows"] = n.rows;
    ctx->saved_data["groups"] = n.groups;
    ctx->saved_data["activation"] = static_cast<int64_t>(n.activation);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list saved = ctx->get_saved_variables();
    const Tensor bias = saved.back();
    saved.pop_back();
    const Tensor weight = saved.back();
    saved.pop_back();
    const Tensor stats = saved.back();
    saved.pop_back();
    const Norm n{ctx->saved_data["maps"].toBool(), ctx->saved_data["rows"].toIntVector(),
                 ctx->saved_data["groups"].toInt(), 0.0,
                 static_cast<int>(ctx->saved_data["activation"].toInt())};
    auto some = [](const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; };
    variable_list out = norm_backward(n, saved, some(weight), some(bias), stats, grads[0]);
    once_differentiable(grads, out);
    out.push_back(Tensor());  // the sizes
    return out;
  }
};

bool wants_grad(at::TensorList ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

Tensor pyramid_group_norm(const py::object& x, const py::object& spatial_shapes, int64_t groups,
                          const optional<Tensor>& weight, const optional<Tensor>& bias, double eps,
                          const std::string& activation) {
  const bool maps = !THPVariable_Check(x.ptr());
  const variable_list xs = norm_inputs(x);
  const Norm n = norm_check(xs, maps, spatial_shapes, groups, weight, bias, eps, activation);
  if (wants_grad(xs) || wants_grad({weight.value_or(Tensor()), bias.value_or(Tensor())}))
    return PyramidGroupNormFn::apply(at::TensorList(xs), weight, bias, n);
  return norm_forward(n, xs, weight, bias).first;
}

// For the traced operators: (y, statistics) and (gradients...).
std::pair<Tensor, Tensor> pyramid_group_norm_forward(const variable_list& xs, bool maps,
                                                     const py::object& spatial_shapes,
                                                     int64_t groups,
                                                     const optional<Tensor>& weight,
                                                     const optional<Tensor>& bias, double eps,
                                                     const std::string& activation) {
  const Norm n = norm_check(xs, maps, spatial_shapes, groups, weight, bias, eps, activation);
  auto [y, stats] = norm_forward(n, xs, weight, bias);
  const int64_t used = y.size(0) * static_cast<int64_t>(n.rows.size()) * groups * 2;
  return {y, stats.slice(0, 0, used)};
}

variable_list pyramid_group_norm_backward(const Tensor& grad_y, const Tensor& stats,
                                          const variable_list& xs, bool maps,
                                          const py::object& spatial_shapes, int64_t groups,
                                          const optional<Tensor>& weight,
                                          const optional<Tensor>& bias,
                                          const std::string& activation) {
  const Norm n = norm_check(xs, maps, spatial_shapes, groups, weight, bias, 0.0, activation);
  return norm_backward(n, xs, weight, bias, stats, grad_y);
}

// ------------------------------------------------------------------ rotary
constexpr int64_t kMaxAxes = 4, kMaxPairs = 2048;

// The positions as (1 or B, Q, A).
Tensor rotary_check(at::TensorList xs, const Tensor& positions, const Tensor& inv_freq,
                    const Tensor& axis_index) {
  const Tensor& first = xs[0];
  TORCH_CHECK_VALUE(first.is_cuda(), "rotary requires CUDA tensors. Got CPU tensors instead.");
  dtype_code(first, "rotary");
  if (dual_level()) {
    for (const Tensor& x : xs) no_tangent(x, "rotary");
    no_tangent(positions, "rotary");
    no_tangent(inv_freq, "rotary");
  }
  TORCH_CHECK(!at::GradMode::is_enabled() || !inv_freq.requires_grad(),
              "rotary forms no gradient for inv_freq: detach it");
  TORCH_CHECK_VALUE(first.dim() == 4, "expected (B, Q, H, C), got ", first.sizes());
  const int64_t B = first.size(0), Q = first.size(1), C = first.size(3);
  for (const Tensor& x : xs)
    TORCH_CHECK_VALUE(x.device() == first.device() && x.scalar_type() == first.scalar_type() &&
                          x.dim() == 4 && x.size(0) == B && x.size(1) == Q && x.size(3) == C,
                      "queries and keys must share their device, dtype, batch, tokens and "
                      "channels; got ", x.sizes(), " ", x.scalar_type(), " beside ",
                      first.sizes(), " ", first.scalar_type());
  const Tensor p = positions.dim() == 2 ? positions.unsqueeze(0) : positions;
  TORCH_CHECK_VALUE(p.dim() == 3 && (p.size(0) == 1 || p.size(0) == B) && p.size(1) == Q,
                    "positions must be (Q, A) or (1 or B, Q, A) with B=", B, ", Q=", Q, "; got ",
                    positions.sizes());
  TORCH_CHECK_VALUE(p.size(2) >= 1 && p.size(2) <= kMaxAxes, "positions must have 1 to ", kMaxAxes,
                    " axes, got ", p.size(2));
  TORCH_CHECK_VALUE(p.scalar_type() != at::kBool && !p.is_complex(),
                    "positions must be numbers, got ", p.scalar_type());
  TORCH_CHECK_VALUE(inv_freq.dim() == 1 && inv_freq.scalar_type() == at::kFloat &&
                        axis_index.sizes() == inv_freq.sizes() &&
                        axis_index.scalar_type() == at::kInt,
                    "inv_freq must be (pairs,) fp32 and axis_index (pairs,) int32, got ",
                    inv_freq.sizes(), " ", inv_freq.scalar_type(), " and ", axis_index.sizes(),
                    " ", axis_index.scalar_type());
  const int64_t pairs = inv_freq.size(0);
  TORCH_CHECK_VALUE(2 * pairs <= C && pairs <= kMaxPairs, pairs, " pairs do not fit ", C,
                    " channels (and at most ", kMaxPairs, ")");
  TORCH_CHECK_VALUE(p.device() == first.device() && inv_freq.device() == first.device() &&
                        axis_index.device() == first.device(),
                    "positions, inv_freq and axis_index must be on ", first.device(), ", got ",
                    p.device(), ", ", inv_freq.device(), " and ", axis_index.device());
  return p;
}

// In a dtype and layout that the kernel reads.
Tensor kernel_positions(const Tensor& p) {
  const auto t = p.scalar_type();
  if (t == at::kFloat || t == at::kInt || t == at::kLong) return p.contiguous();
  return p.to(p.is_floating_point() ? at::kFloat : at::kLong).contiguous();
}

Tensor dense_channels(const Tensor& x) {
  return x.stride(3) == 1 || x.size(3) <= 1 ? x : x.contiguous();
}

struct Heads {
  std::array<int64_t, 2> heads{};
  std::array<void*, 2> at{};
  std::array<int64_t, 6> strides{};
  explicit Heads(at::TensorList ts) {
    for (size_t i = 0; i < ts.size(); ++i) {
      heads[i] = ts[i].size(2);
      at[i] = ts[i].data_ptr();
      for (int64_t d = 0; d < 3; ++d) strides[3 * i + d] = ts[i].stride(d);
    }
  }
};

// ys become the xs turned (or turned back); all in layouts that the kernel takes.
void turn(at::TensorList xs, at::TensorList ys, const Tensor& positions, const Tensor& inv_freq,
          const Tensor& axis_index, bool interleaved, bool inverse, at::TensorList inputs,
          const Tensor& gpos) {
  const Tensor& first = xs[0];
  const c10::cuda::CUDAGuard guard(first.device());
  const Heads x(xs), y(ys), in(inputs);
  const int64_t Q = first.size(1), axes = positions.size(2);
  const int pos_dtype = positions.scalar_type() == at::kFloat  ? MSDA_POSITION_FLOAT32
                        : positions.scalar_type() == at::kInt ? MSDA_POSITION_INT32
                                                               : MSDA_POSITION_INT64;
  check(api.rotary(dtype_code(first, "rotary"), first.size(0), Q, first.size(3),
                   static_cast<int>(xs.size()), x.heads.data(), x.at.data(), x.strides.data(),
                   y.at.data(), y.strides.data(), positions.data_ptr(), pos_dtype,
                   positions.size(0) == 1 ? 0 : Q * axes, axes, inv_freq.data_ptr<float>(),
                   axis_index.data_ptr<int32_t>(), inv_freq.size(0), interleaved, inverse,
                   inputs.empty() ? nullptr : in.at.data(),
                   inputs.empty() ? nullptr : in.strides.data(),
                   gpos.defined() ? gpos.data_ptr<float>() : nullptr, current_stream(first)));
}

variable_list rotary_forward(at::TensorList xs, const Tensor& positions, const Tensor& inv_freq,
                             const Tensor& axis_index, bool interleaved) {
  at::NoGradGuard no_grad;
  variable_list in, out;
  for (const Tensor& x : xs) {
    in.push_back(dense_channels(x));
    out.push_back(empty(x.sizes(), x));
  }
  turn(in, out, kernel_positions(positions), inv_freq.contiguous(), axis_index.contiguous(),
       interleaved, false, {}, Tensor());
  return out;
}

// Gradients of the tensors and, with their inputs given, of the positions.
variable_list rotary_backward(at::TensorList grads, at::TensorList inputs, const Tensor& positions,
                              const Tensor& inv_freq, const Tensor& axis_index, bool interleaved) {
  if (dual_level())
    for (const Tensor& g : grads) no_tangent(g, "rotary's backward");
  at::NoGradGuard no_grad;
  variable_list gys, gxs, ins;
  for (const Tensor& g : grads) {
    gys.push_back(dense_channels(g));
    gxs.push_back(empty(g.sizes(), g));
  }
  for (const Tensor& x : inputs) ins.push_back(dense_channels(x));
  const Tensor pos = kernel_positions(positions);
  Tensor gpos;
  if (!inputs.empty())
    gpos = empty({grads[0].size(0), grads[0].size(1), pos.size(2)}, grads[0], at::kFloat);
  turn(gys, gxs, pos, inv_freq.contiguous(), axis_index.contiguous(), interleaved, true, ins, gpos);
  if (gpos.defined()) {
    if (pos.size(0) != gpos.size(0)) gpos = gpos.sum(0, true);  // one set for the whole batch
    gxs.push_back(gpos.to(positions.scalar_type()));
  }
  return gxs;
}

class RotaryFn : public torch::autograd::Function<RotaryFn> {
 public:
  static variable_list forward(AutogradContext* ctx, at::TensorList xs,
                               const Tensor& positions, const Tensor& inv_freq,
                               const Tensor& axis_index, bool interleaved) {
    variable_list out = rotary_forward(xs, positions, inv_freq, axis_index, interleaved);
    variable_list saved{positions, inv_freq, axis_index};
    if (positions.requires_grad()) saved.insert(saved.end(), xs.begin(), xs.end());
    ctx->save_for_backward(saved);
    ctx->saved_data["interleaved"] = interleaved;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::TensorList inputs = at::TensorList(saved).slice(3);
    variable_list out = rotary_backward(grads, inputs, saved[0], saved[1], saved[2],
                                        ctx->saved_data["interleaved"].toBool());
    once_differentiable(grads, out);
    if (inputs.empty()) out.push_back(Tensor());  // the positions
    out.insert(out.end(), 3, Tensor());           // inv_freq, axis_index, interleaved
    return out;
  }
};

variable_list rotary(const variable_list& xs, const Tensor& positions, const Tensor& inv_freq,
                     const Tensor& axis_index, bool interleaved) {
  const Tensor p = rotary_check(xs, positions, inv_freq, axis_index);
  if (wants_grad(xs) || wants_grad(p))
    return RotaryFn::apply(at::TensorList(xs), p, inv_freq, axis_index, interleaved);
  return rotary_forward(xs, p, inv_freq, axis_index, interleaved);
}

Tensor rotary_one(const Tensor& x, const Tensor& positions, const Tensor& inv_freq,
                  const Tensor& axis_index, bool interleaved) {
  return rotary({x}, positions, inv_freq, axis_index, interleaved)[0];
}

std::pair<Tensor, Tensor> rotary_qk(const Tensor& q, const Tensor& k, const Tensor& positions,
                                    const Tensor& inv_freq, const Tensor& axis_index,
                                    bool interleaved) {
  variable_list out = rotary({q, k}, positions, inv_freq, axis_index, interleaved);
  return {out[0], out[1]};
}

// Whether some n_d, each of its range, give sum n_d stride_d = goal: whether two
// elements lie at one address, the n_d being what their indexes differ by.
// Ranges are tried from the widest stride on, and of each only what the others
// can still make up for: one or two where strides hold each other's rows.  Past
// `tries` the answer is yes.
struct Step {
  int64_t stride, lo, hi;
};
using Steps = std::array<Step, 7>;  // three of each tensor, and one within a run

bool meets(const Step* at, const Step* end, int64_t goal, int& tries) {
  if (at == end) return goal == 0;
  if (--tries < 0) return true;
  int64_t lo = 0, hi = 0;  // what the steps behind can add
  for (const Step* s = at + 1; s != end; ++s) {
    lo += s->lo * s->stride;
    hi += s->hi * s->stride;
  }
  auto floor_div = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
  const int64_t from = std::max(at->lo, -floor_div(hi - goal, at->stride)),
                to = std::min(at->hi, floor_div(goal - lo, at->stride));
  for (int64_t n = from; n <= to; ++n)
    if (meets(at + 1, end, goal - n * at->stride, tries)) return true;
  return false;
}

void sort_steps(Steps& steps, size_t count) {
  std::sort(steps.begin(), steps.begin() + count,
            [](const Step& x, const Step& y) { return x.stride > y.stride; });
}

// Whether two elements of (B, Q, H) runs of `run` bytes lie at one address.
bool overlaps_itself(const Tensor& x, int64_t run) {
  Steps steps{{{1, 1 - run, run - 1}}};
  size_t count = 1;
  for (int64_t d = 0; d < 3; ++d)
    if (const int64_t n = x.size(d) - 1; n > 0)
      steps[count++] = {x.stride(d) * x.element_size(), -n, n};
  sort_steps(steps, count);
  int tries = 1 << 12;
  for (size_t i = 0; i + 1 < count; ++i) {  // the first index that differs
    steps[i].lo = 1;
    if (meets(&steps[i], &steps[0] + count, 0, tries)) return true;
  }
  return false;
}

// Whether an element of a's runs lies at the address of one of b's.
bool overlap(const Tensor& a, const Tensor& b, int64_t run) {
  Steps steps{{{1, 1 - run, run - 1}}};
  size_t all = 1, count = 1;
  for (int64_t d = 0; d < 3; ++d) {
    if (a.size(d) > 1) steps[all++] = {a.stride(d) * a.element_size(), 0, a.size(d) - 1};
    if (b.size(d) > 1) steps[all++] = {b.stride(d) * b.element_size(), 1 - b.size(d), 0};
  }
  sort_steps(steps, all);
  for (size_t i = 1; i < all; ++i) {  // those of one stride are one
    if (steps[count - 1].stride == steps[i].stride) {
      steps[count - 1].lo += steps[i].lo;
      steps[count - 1].hi += steps[i].hi;
    } else {
      steps[count++] = steps[i];
    }
  }
  int tries = 1 << 12;
  return meets(&steps[0], &steps[0] + count,
               static_cast<char*>(b.data_ptr()) - static_cast<char*>(a.data_ptr()), tries);
}

// Refuses tensors whose heads' first `run` bytes lie twice in memory, within one
// tensor or in both: several threads of the launch would read and write them.
void no_overlap(const variable_list& xs, int64_t run) {
  if (run == 0) return;
  for (size_t i = 0; i < xs.size(); ++i) {
    if (xs[i].numel() == 0) continue;
    TORCH_CHECK_VALUE(!overlaps_itself(xs[i], run),
                      "rotary_qk_ cannot write to a tensor that overlaps itself, strides ",
                      xs[i].strides(), " for ", xs[i].sizes());
    for (size_t j = 0; j < i; ++j)
      TORCH_CHECK_VALUE(xs[j].numel() == 0 || !overlap(xs[j], xs[i], run),
                        "rotary_qk_ cannot write to queries and keys that share memory");
  }
}

void rotary_in_place(const variable_list& xs, const Tensor& positions, const Tensor& inv_freq,
                     const Tensor& axis_index, bool interleaved) {
  const Tensor p = rotary_check(xs, positions, inv_freq, axis_index);
  TORCH_CHECK(!wants_grad(xs) && !wants_grad(p),
              "rotary_qk_ has no gradient: use rotary_qk, or torch.no_grad()");
  for (const Tensor& x : xs) {
    TORCH_CHECK_VALUE(x.stride(3) == 1 || x.size(3) <= 1, "rotary_qk_ needs dense channels");
    for (int64_t d = 0; d < 4; ++d)
      TORCH_CHECK_VALUE(x.stride(d) != 0 || x.size(d) <= 1,
                        "rotary_qk_ cannot write to an expanded tensor");
  }
  no_overlap(xs, 2 * inv_freq.size(0) * xs[0].element_size());
  at::NoGradGuard no_grad;
  turn(xs, xs, kernel_positions(p), inv_freq.contiguous(), axis_index.contiguous(), interleaved,
       false, {}, Tensor());
  for (const Tensor& x : xs) x.unsafeGetTensorImpl()->bump_version();
}

// ------------------------------------------------------------------ AdamW
constexpr int64_t kAdamBlock = 128;

struct AdamState {
  Tensor exp_avg, exp_avg_sq, exp_avg_exponent, exp_avg_sq_exponent, master;
  int bits = 0;
  int64_t elements = 0;
  std::vector<Tensor> all;
};

AdamState adam_state(const py::dict& state, at::ScalarType dtype, at::Device device) {
  AdamState s;
  const std::pair<const char*, Tensor*> names[] = {
      {"exp_avg", &s.exp_avg},
      {"exp_avg_sq", &s.exp_avg_sq},
      {"exp_avg_exponent", &s.exp_avg_exponent},
      {"exp_avg_sq_exponent", &s.exp_avg_sq_exponent},
      {"master", &s.master}};
  for (const auto& [name, to] : names)
    if (PyObject* o = PyDict_GetItemString(state.ptr(), name)) *to = tensor_of(o, "states");
  TORCH_CHECK_VALUE(s.exp_avg.defined() && s.exp_avg_sq.defined(),
                    "the state has no 'exp_avg' or no 'exp_avg_sq'");
  const auto kind = s.exp_avg.scalar_type();
  TORCH_CHECK_VALUE(kind == at::kFloat || kind == at::kByte,
                    "states must be fp32 or uint8 codes, got ", kind);
  s.bits = kind == at::kFloat ? 32 : 8;
  s.elements = s.exp_avg.numel();
  const bool small = s.bits == 8;
  TORCH_CHECK_VALUE(!s.master.defined() || dtype != at::kFloat,
                    "fp32 parameters take no master copy");
  TORCH_CHECK_VALUE(s.exp_avg_exponent.defined() == small &&
                        s.exp_avg_sq_exponent.defined() == small,
                    "states of ", s.bits, " bits have ", small ? "" : "no ", "exponents");
  for (const auto& [name, to] : names) {
    if (!to->defined()) continue;
    const bool exponent = to == &s.exp_avg_exponent || to == &s.exp_avg_sq_exponent;
    const auto want = to == &s.master ? at::kFloat : kind;
    const int64_t n = exponent ? s.elements / kAdamBlock : s.elements;
    TORCH_CHECK_VALUE(to->scalar_type() == want && to->dim() == 1 && to->numel() == n &&
                          to->device() == device && to->is_contiguous(),
                      "state '", name, "' must be dense ", want, " of ", n, " elements on ",
                      device, ", got ", to->scalar_type(), " ", to->sizes(), " on ", to->device());
    s.all.push_back(*to);
  }
  TORCH_CHECK_VALUE(static_cast<size_t>(py::len(state)) == s.all.size(),
                    "the state holds something else than moments, exponents and a master copy");
  TORCH_CHECK_VALUE(!small || s.elements % kAdamBlock == 0,
                    "8-bit states have a multiple of 128 elements, got ", s.elements);
  return s;
}

// g in p's memory order, for tensors that are not both dense in the usual order.
Tensor laid_out(const Tensor& p, const Tensor& g) {
  TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(),
                    "a parameter's elements must fill one range of memory, got strides ",
                    p.strides(), " for ", p.sizes());
  for (int64_t d = 0; d < p.dim(); ++d)
    if (p.size(d) > 1 && p.stride(d) != g.stride(d)) return at::empty_like(p).copy_(g);
  return g;
}

// Refuses a parameter whose elements lie in another order than when its states
// were made; the stride of an axis of one element says nothing.
void same_order(const Tensor& p, const Tensor& then) {
  if (p.strides() == then.strides()) return;
  for (int64_t d = 0; d < p.dim(); ++d)
    TORCH_CHECK_VALUE(p.size(d) <= 1 || p.stride(d) == then.stride(d), "a parameter ", p.sizes(),
                      " has strides ", p.strides(), " and had ", then.strides(),
                      " when its states were made: change its memory format before the first step");
}

// layouts: None, or for each parameter a tensor of the strides that its states were made for.
void adamw_step(const py::object& params, const py::object& grads, const py::dict& state,
                const py::object& step, double lr, double beta1, double beta2, double eps,
                double weight_decay, int64_t seed, const optional<Tensor>& grad_scale,
                const py::object& layouts) {
  at::NoGradGuard no_grad;
  const py::object ps = py::reinterpret_steal<py::object>(
      PySequence_Fast(params.ptr(), "params must be a sequence of tensors"));
  if (!ps) throw py::error_already_set();
  const py::object gs = py::reinterpret_steal<py::object>(
      PySequence_Fast(grads.ptr(), "grads must be a sequence of tensors"));
  if (!gs) throw py::error_already_set();
  const int64_t n = PySequence_Fast_GET_SIZE(ps.ptr());
  TORCH_CHECK_VALUE(PySequence_Fast_GET_SIZE(gs.ptr()) == n, n, " tensors and ",
                    PySequence_Fast_GET_SIZE(gs.ptr()), " gradients");
  if (n == 0) return;
  const Tensor first = tensor_of(PySequence_Fast_GET_ITEM(ps.ptr(), 0), "params");
  TORCH_CHECK_VALUE(first.is_cuda(), "AdamW requires CUDA tensors. Got CPU tensors instead.");
  const int code = dtype_code(first, "AdamW");
  const auto dtype = first.scalar_type();
  const auto device = first.device();
  const AdamState s = adam_state(state, dtype, device);
  const c10::cuda::CUDAGuard guard(device);
  TORCH_CHECK(at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None,
              "adamw_step cannot be captured in a CUDA graph: the step's bias corrections are "
              "computed on the host");
  std::vector<void*> p_at(n);
  std::vector<const void*> g_at(n);
  std::vector<int64_t> counts(n), steps(n);
  std::vector<Tensor> kept, changed;
  changed.reserve(n);
  const bool dual = dual_level();
  TORCH_CHECK(layouts.is_none() ||
                  (PyList_Check(layouts.ptr()) && PyList_GET_SIZE(layouts.ptr()) == n),
              "layouts must be a list of ", n, " tensors");
  for (int64_t i = 0; i < n; ++i) {
    const Tensor& p = tensor_of(PySequence_Fast_GET_ITEM(ps.ptr(), i), "params");
    PyObject* o = PySequence_Fast_GET_ITEM(gs.ptr(), i);
    TORCH_CHECK_VALUE(p.scalar_type() == dtype && p.device() == device,
                      "the tensors of a step must share their dtype and device");
    if (dual) no_tangent(p, "adamw_step");
    if (!layouts.is_none())
      same_order(p, tensor_of(PyList_GET_ITEM(layouts.ptr(), i), "layouts"));
    p_at[i] = p.data_ptr();
    counts[i] = p.numel();
    g_at[i] = nullptr;
    const bool dense = p.is_contiguous();
    TORCH_CHECK_VALUE(dense || p.is_non_overlapping_and_dense(),
                      "a parameter's elements must fill one range of memory, got strides ",
                      p.strides(), " for ", p.sizes());
    if (o == Py_None) continue;
    const Tensor& g = tensor_of(o, "grads");
    TORCH_CHECK_VALUE(g.layout() == at::kStrided, "gradients must be dense, got ", g.layout());
    TORCH_CHECK_VALUE(g.scalar_type() == dtype && g.device() == device, "gradients must be ",
                      dtype, " on ", device, ", as the tensors");
    if (dual) no_tangent(g, "adamw_step");
    TORCH_CHECK_VALUE(g.sizes() == p.sizes(), "gradient ", g.sizes(), " for a tensor ", p.sizes());
    if (dense && g.is_contiguous()) {
      g_at[i] = g.data_ptr();
    } else {
      kept.push_back(laid_out(p, g));
      g_at[i] = kept.back().data_ptr();
    }
    if (counts[i] > 0) changed.push_back(p);
  }
  if (PyLong_Check(step.ptr())) {
    std::fill(steps.begin(), steps.end(), step.cast<int64_t>());
  } else {
    steps = step.cast<std::vector<int64_t>>();
    TORCH_CHECK_VALUE(static_cast<int64_t>(steps.size()) == n, n, " tensors and ", steps.size(),
                      " steps");
  }
  TORCH_CHECK_VALUE(!grad_scale || (grad_scale->scalar_type() == at::kFloat &&
                                    grad_scale->numel() == 1 && grad_scale->device() == device),
                    "grad_scale must be one fp32 value on ", device);
  auto at = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  check(api.adamw_step(code, s.bits, n, p_at.data(), g_at.data(), counts.data(), steps.data(), lr,
                       beta1, beta2, eps, weight_decay, static_cast<uint32_t>(seed),
                       static_cast<const float*>(ptr(grad_scale)), at(s.exp_avg),
                       at(s.exp_avg_sq), static_cast<uint8_t*>(at(s.exp_avg_exponent)),
                       static_cast<uint8_t*>(at(s.exp_avg_sq_exponent)),
                       static_cast<float*>(at(s.master)), s.elements, current_stream(first)));
  for (const Tensor& t : changed) t.unsafeGetTensorImpl()->bump_version();
  for (const Tensor& t : s.all) t.unsafeGetTensorImpl()->bump_version();
}

std::pair<Tensor, Tensor> adamw_values(const py::dict& state) {
  at::NoGradGuard no_grad;
  PyObject* o = PyDict_GetItemString(state.ptr(), "exp_avg");
  TORCH_CHECK_VALUE(o != nullptr, "the state has no 'exp_avg' or no 'exp_avg_sq'");
  const Tensor m = tensor_of(o, "states");
  TORCH_CHECK_VALUE(m.is_cuda(), "AdamW requires CUDA tensors. Got CPU tensors instead.");
  const AdamState s = adam_state(state, at::kBFloat16, m.device());
  if (s.bits == 32) return {s.exp_avg, s.exp_avg_sq};
  const c10::cuda::CUDAGuard guard(m.device());
  Tensor mo = empty({s.elements}, m, at::kBFloat16), vo = empty({s.elements}, m, at::kBFloat16);
  check(api.adamw_values(s.exp_avg.data_ptr<uint8_t>(), s.exp_avg_exponent.data_ptr<uint8_t>(),
                         s.exp_avg_sq.data_ptr<uint8_t>(),
                         s.exp_avg_sq_exponent.data_ptr<uint8_t>(), s.elements, mo.data_ptr(),
                         vo.data_ptr(), current_stream(m)));
  return {mo, vo};
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
  using torch::wrap_pybind_function;
  m.def("bind", wrap_pybind_function(bind));
  m.def("pyramid_group_norm", wrap_pybind_function(pyramid_group_norm));
  m.def("pyramid_group_norm_forward", wrap_pybind_function(pyramid_group_norm_forward));
  m.def("pyramid_group_norm_backward", wrap_pybind_function(pyramid_group_norm_backward));
  m.def("rotary", wrap_pybind_function(rotary_one));
  m.def("rotary_qk", wrap_pybind_function(rotary_qk));
  m.def("rotary_in_place", wrap_pybind_function(rotary_in_place));
  m.def("no_overlap", wrap_pybind_function(no_overlap));
  m.def("rotary_check", wrap_pybind_function([](const variable_list& xs, const Tensor& p,
                                                const Tensor& f, const Tensor& a) {
          return rotary_check(xs, p, f, a);
        }));
  m.def("rotary_forward", wrap_pybind_function([](const variable_list& xs, const Tensor& p,
                                                  const Tensor& f, const Tensor& a, bool i) {
          return rotary_forward(xs, rotary_check(xs, p, f, a), f, a, i);
        }));
  m.def("rotary_backward",
        wrap_pybind_function([](const variable_list& grads, const variable_list& inputs,
                                const Tensor& p, const Tensor& f, const Tensor& a, bool i) {
          return rotary_backward(grads, inputs, p, f, a, i);
        }));
  m.def("adamw_step", wrap_pybind_function(adamw_step));
  m.def("adamw_values", wrap_pybind_function(adamw_values));
}
