// The eager calls of the mixer's operators (layer norm, rotary positions,
// decayed linear attention) on PyTorch tensors: argument checks, layouts,
// buffers, autograd nodes and the calls into libdwarf_dsqg.so's C ABI.
//
// They are C++ because the kernels are short: from Python, with ctypes and
// Python autograd nodes, a forward and backward cost 175 to 280 us of host time
// around 40 to 200 us of kernels, and a single-token step 24 us; here 65 to 120
// (30 of them PyTorch's engine for the gradient of a view) and 4.6.
// Loaded as the module _mixer (Python: _launch.native()).
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>
#include <pybind11/stl.h>

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>

#include "dwarf_mixer.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kHd = 64;

// A status that is neither success nor an invalid argument (the Python side's NativeLibraryError).
struct StatusError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check_status(int rc, const char* what) {
  if (rc == DWARF_OK) return;
  const std::string text = std::string(what) + ": " + dwarf_last_error();
  TORCH_CHECK_VALUE(rc != DWARF_ERR_INVALID_ARGUMENT, text);
  throw StatusError(text);
}

// The entry point on the tensor's device and that device's current stream.
template <typename F, typename A>
void launch(F fn, const A& args, const Tensor& on, const char* what) {
  const c10::DeviceGuard guard(on.device());
  check_status(fn(&args, reinterpret_cast<dwarf_stream_t>(c10::hip::getCurrentHIPStream(on.device().index()).stream())), what);
}

// What a launch on raw pointers would go past: tensors without memory of their own (fake, batched, wrapped by a transform),
// those that stand for other values than their memory holds (negated, zero tensors), and whatever watches the dispatcher
// (modes, traces).  An eager call or backward node that meets any of them goes through the custom ops, which the dispatcher
// knows.
constexpr c10::DispatchKeySet kWatched{
    c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::PythonDispatcher,
    c10::DispatchKey::PreDispatch, c10::DispatchKey::Functionalize, c10::DispatchKey::Tracer, c10::DispatchKey::Batched,
    c10::DispatchKey::VmapMode, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchVmapMode,
    c10::DispatchKey::FuncTorchBatchedDecomposition, c10::DispatchKey::FuncTorchGradWrapper,
    c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode,
    c10::DispatchKey::Negative, c10::DispatchKey::Conjugate, c10::DispatchKey::ZeroTensor};

c10::DispatchKeySet keys_of(const Tensor& t) { return t.defined() ? t.key_set() : c10::DispatchKeySet(); }
c10::DispatchKeySet keys_of(const OptTensor& t) { return t ? keys_of(*t) : c10::DispatchKeySet(); }
template <typename... T>
bool watched(const T&... t) {
  const c10::impl::LocalDispatchKeySet local = c10::impl::tls_local_dispatch_key_set();
  return (((keys_of(t) | ...) | local.included_) - local.excluded_).has_any(kWatched);
}

// The custom op `name` through the dispatcher.
template <typename... T>
std::vector<Tensor> dispatched(const char* name, const T&... args) {
  torch::jit::Stack stack{c10::IValue(args)...};
  c10::Dispatcher::singleton().findSchemaOrThrow(name, "").callBoxed(&stack);
  std::vector<Tensor> out;
  for (const c10::IValue& v : stack) out.push_back(v.toTensor());
  return out;
}

// Derivatives in forward mode: there are none, and a result without a tangent would count as a constant.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }
template <typename... T>
void refuse_tangents(const char* what, const T&... t) {
  TORCH_CHECK(!(has_tangent(t) || ...), what, " has no derivative in forward mode: differentiate it backward");
}

int dtype_of(const Tensor& x, const char* what) {
  switch (x.scalar_type()) {
    case at::kBFloat16: return DWARF_BF16;
    case at::kHalf: return DWARF_F16;
    case at::kFloat: return DWARF_F32;
    default: TORCH_CHECK_VALUE(false, what, " must be bf16, fp16 or fp32, got ", x.scalar_type());
  }
}

// A size as the C ABI takes it.
int32_t size32(int64_t n) {
  TORCH_CHECK(n <= INT32_MAX, "dimensions must stay below 2^31, got ", n);
  return static_cast<int32_t>(n);
}

void check_cuda(const Tensor& x) { TORCH_CHECK(x.is_cuda(), "the mixer's HIP kernels require device tensors"); }
void check_beside(const char* name, const Tensor& t, const Tensor& x) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", expected ", x.device());
}
void check_beside(const char* name, const OptTensor& t, const Tensor& x) {
  if (t) check_beside(name, *t, x);
}
bool is_index(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

Tensor empty_like_dtype(at::IntArrayRef shape, const Tensor& like, at::ScalarType dtype) {
  return at::empty(shape, like.options().dtype(dtype));
}
Tensor empty_f32(at::IntArrayRef shape, const Tensor& like) { return empty_like_dtype(shape, like, at::kFloat); }
// An empty [B,H,N,D] tensor in [B,N,H,D] memory; no view, which made without gradients could not be changed in place with them.
Tensor token_major(int64_t B, int64_t H, int64_t N, int64_t D, const Tensor& like) {
  const int64_t row = std::max<int64_t>(H, 1) * D;
  return at::empty_strided({B, H, N, D}, {std::max<int64_t>(N, 1) * row, D, row, 1}, like.options());
}
Tensor workspace(size_t nbytes, const Tensor& like) {
  return nbytes ? empty_like_dtype({static_cast<int64_t>(nbytes)}, like, at::kByte) : Tensor();
}

template <int N>
void put_strides(int64_t (&to)[N], const Tensor& t) {
  const auto s = t.strides();
  for (int i = 0; i < N; ++i) to[i] = s[i];
}

bool aligned(const Tensor& t, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }

// Unit last stride and 16-byte aligned rows.
bool rows_ok(const Tensor& t) {
  const auto s = t.strides();
  const int64_t per16 = 16 / t.element_size();
  if (s.back() != 1 || !aligned(t, 16)) return false;
  for (size_t i = 0; i + 1 < s.size(); ++i)
    if (s[i] % per16) return false;
  return true;
}
// A contiguous copy: contiguous() alone gives a dense tensor back as it is, at whatever address it begins.
Tensor dense_copy(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
Tensor kernel_rows(const Tensor& t) { return rows_ok(t) ? t : dense_copy(t); }

// Gradients whose own derivative raises: the backward nodes are first order.
variable_list first_order(variable_list grads, const char* what) {
  if (!c10::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const Tensor& g : grads)
    if (g.defined()) in.push_back(g.detach().requires_grad_(true));
  const auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + ": trying to differentiate twice a backward that is first order only", static_cast<int64_t>(in.size()));
  const variable_list out = node->apply(std::move(in));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// ---- layer norm --------------------------------------------------------------------------------
struct NormRows {
  Tensor x;
  int64_t row, group;   // strides
};

// x as [rows][groups][D]; copied where its leading dimensions do not collapse into one row stride.
NormRows norm_rows(const Tensor& x, int64_t groups) {
  auto strides = [&](const Tensor& t, NormRows& r) {
    const auto n = t.sizes();
    const auto s = t.strides();
    int64_t last = t.dim() - 1;
    if (n[last] > 1 && s[last] != 1) return false;
    r.group = groups > 1 ? s[--last] : 0;
    r.row = 0;
    int64_t span = -1;   // stride of the dimension in front that collapses with the ones behind
    for (int64_t i = last - 1; i >= 0; --i) {
      if (n[i] == 1) continue;
      if (span < 0) r.row = s[i];
      else if (s[i] != span) return false;
      span = s[i] * n[i];
    }
    return true;
  };
  NormRows r{x, 0, 0};
  if (!strides(x, r)) {
    r.x = x.contiguous();
    strides(r.x, r);
  }
  return r;
}

Tensor table(const OptTensor& t) {
  if (!t) return Tensor();
  return t->scalar_type() == at::kFloat && t->is_contiguous() ? *t : t->to(at::kFloat).contiguous();
}
const float* f32_ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
float* f32_out(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

void norm_fill(dwarf_layer_norm_fwd_args& a, const NormRows& r, int64_t groups, const Tensor& w, double eps) {
  const int64_t D = r.x.size(-1);
  a.rows = r.x.numel() / (groups * D);
  a.groups = size32(groups);
  a.D = size32(D);
  a.dtype = dtype_of(r.x, "x");
  a.eps = static_cast<float>(eps);
  a.x = r.x.const_data_ptr();
  a.x_stride[0] = r.row;
  a.x_stride[1] = r.group;
  a.weight = f32_ptr(w);
}

// What the launches take for granted, for callers that come without layer_norm's own checks (the custom ops).
void check_norm_launch(const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t groups) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must have a last dimension to normalise, got ", x.sizes());
  TORCH_CHECK_VALUE(groups == 1 || (groups > 1 && x.dim() >= 2 && x.size(-2) == groups), "groups=", groups, " does not fit x ",
                    x.sizes());
  for (const auto& [name, t] : {std::make_pair("weight", &weight), std::make_pair("bias", &bias)}) {
    if (!*t) continue;
    TORCH_CHECK_VALUE((*t)->is_floating_point() && (*t)->numel() == groups * x.size(-1), name, " must hold ", groups, " x ",
                      x.size(-1), " floating values, got ", (*t)->sizes(), " ", (*t)->scalar_type());
  }
  dtype_of(x, "x");
  check_cuda(x);
  check_beside("weight", weight, x);
  check_beside("bias", bias, x);
}

Tensor norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t groups, double eps) {
  const NormRows r = norm_rows(x, groups);
  const Tensor w = table(weight), b = table(bias);
  const Tensor y = at::empty(x.sizes(), x.options());
  dwarf_layer_norm_fwd_args a{};
  norm_fill(a, r, groups, w, eps);
  a.bias = f32_ptr(b);
  a.y = y.data_ptr();
  a.y_stride[0] = groups * a.D;
  a.y_stride[1] = a.D;
  launch(dwarf_layer_norm_fwd, a, x, "dwarf_layer_norm_fwd");
  return y;
}

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& dy, const Tensor& x, const OptTensor& weight, int64_t groups,
                                                 double eps, bool need_dx, bool need_dw, bool need_db) {
  const NormRows r = norm_rows(x, groups), g = norm_rows(dy.to(x.scalar_type()), groups);
  const Tensor w = table(weight);
  Tensor dx, dw, db;
  dwarf_layer_norm_bwd_args a{};
  norm_fill(a.fwd, r, groups, w, eps);
  a.dy = g.x.const_data_ptr();
  a.dy_stride[0] = g.row;
  a.dy_stride[1] = g.group;
  if (need_dx) {
    dx = at::empty(x.sizes(), x.options());
    a.dx = dx.data_ptr();
    a.dx_stride[0] = groups * a.fwd.D;
    a.dx_stride[1] = a.fwd.D;
  }
  if (need_dw) dw = empty_f32({groups * a.fwd.D}, x);
  if (need_db) db = empty_f32({groups * a.fwd.D}, x);
  a.dweight = f32_out(dw);
  a.dbias = f32_out(db);
  a.workspace_bytes = dwarf_layer_norm_bwd_workspace_bytes(&a);
  const Tensor ws = workspace(a.workspace_bytes, x);
  if (ws.defined()) a.workspace = ws.data_ptr();
  launch(dwarf_layer_norm_bwd, a, x, "dwarf_layer_norm_bwd");
  return {dx, dw, db};
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                        int64_t groups, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({x, weight.value_or(Tensor())});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["weight"] = weight.has_value();
    if (bias) {
      ctx->saved_data["bias_shape"] = bias->sizes();
      ctx->saved_data["bias_dtype"] = bias->scalar_type();
    }
    return norm_forward(x, weight, bias, groups, eps);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const bool has_w = ctx->saved_data["weight"].toBool(), has_b = ctx->saved_data.count("bias_shape") > 0;
    const bool need_w = has_w && ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
    variable_list out(5);
    {
      const at::NoGradGuard no_grad;
      const OptTensor weight = has_w ? OptTensor(saved[1]) : std::nullopt;
      const int64_t groups = ctx->saved_data["groups"].toInt();
      const double eps = ctx->saved_data["eps"].toDouble();
      const bool need_x = ctx->needs_input_grad(0);
      Tensor dx, dw, db;
      refuse_tangents("layer_norm", grads[0], saved[0], weight);
      if (watched(grads[0], saved[0], weight)) {
        const auto r = dispatched("dwarf::layer_norm_bwd", grads[0], saved[0], weight, groups, eps, need_x, need_w, need_b);
        dx = r[0], dw = r[1], db = r[2];
      } else {
        std::tie(dx, dw, db) = norm_backward(grads[0], saved[0], weight, groups, eps, need_x, need_w, need_b);
      }
      if (need_x) out[0] = dx;
      if (need_w) out[1] = dw.view(saved[1].sizes()).to(saved[1].scalar_type());
      if (need_b) out[2] = db.view(ctx->saved_data["bias_shape"].toIntVector()).to(ctx->saved_data["bias_dtype"].toScalarType());
    }
    return first_order(std::move(out), "layer_norm");
  }
};

// Nothing: the call goes through the custom ops (see kWatched).
OptTensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  refuse_tangents("layer_norm", x, weight, bias);
  if (watched(x, weight, bias)) return std::nullopt;
  TORCH_CHECK_VALUE(std::isfinite(eps) && eps >= 0, "eps must be finite and not negative");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must have a last dimension to normalise, got ", x.sizes());
  int64_t groups = 1;
  for (const auto& [name, t] : {std::make_pair("weight", &weight), std::make_pair("bias", &bias)}) {
    if (!*t) continue;
    const Tensor& v = **t;
    TORCH_CHECK_VALUE((v.dim() == 1 || v.dim() == 2) && v.dim() <= x.dim() && v.sizes() == x.sizes().slice(x.dim() - v.dim()),
                      name, " must hold the last one or two dimensions of x ", x.sizes(), ", got ", v.sizes());
    TORCH_CHECK_VALUE(v.is_floating_point(), name, " must be floating point, got ", v.scalar_type());
    if (v.dim() == 2) groups = v.size(0);
  }
  TORCH_CHECK_VALUE(!weight || !bias || weight->sizes() == bias->sizes(), "weight and bias must share a shape");
  TORCH_CHECK_VALUE(groups >= 1, "weight and bias need at least one group");
  dtype_of(x, "x");
  check_cuda(x);
  check_beside("weight", weight, x);
  check_beside("bias", bias, x);
  if (at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad())))
    return LayerNormFn::apply(x, weight, bias, groups, eps);
  return norm_forward(x, weight, bias, groups, eps);
}

// ---- rotary positions --------------------------------------------------------------------------
Tensor pair_rows(const Tensor& x, bool interleaved) {
  const auto s = x.strides();
  bool ok = s[3] == 1;
  if (interleaved) ok = ok && aligned(x, 2 * x.element_size()) && s[0] % 2 == 0 && s[1] % 2 == 0 && s[2] % 2 == 0;
  return ok ? x : dense_copy(x);
}

std::tuple<Tensor, Tensor> rotate(const Tensor& q_, const OptTensor& k_, const Tensor& positions, const Tensor& turns,
                                  bool interleaved, bool inverse, double magnitude) {
  const Tensor q = pair_rows(q_, interleaved);
  dwarf_rotary_args a{};
  a.B = size32(q.size(0));
  a.H = size32(q.size(1));
  a.N = size32(q.size(2));
  a.D = size32(q.size(3));
  a.pairs = size32(turns.numel());
  a.dtype = dtype_of(q, "q");
  a.interleaved = interleaved;
  a.inverse = inverse;
  a.magnitude = static_cast<float>(magnitude);
  const Tensor q_out = token_major(a.B, a.H, a.N, a.D, q);
  a.q = q.const_data_ptr();
  put_strides(a.q_stride, q);
  a.q_out = q_out.data_ptr();
  put_strides(a.q_out_stride, q_out);
  Tensor k, k_out;
  if (k_) {
    k = pair_rows(*k_, interleaved);
    a.H_kv = size32(k.size(1));
    k_out = token_major(a.B, a.H_kv, a.N, a.D, k);
    a.k = k.const_data_ptr();
    put_strides(a.k_stride, k);
    a.k_out = k_out.data_ptr();
    put_strides(a.k_out_stride, k_out);
  }
  a.positions = positions.const_data_ptr();
  a.position_bytes = static_cast<int32_t>(positions.element_size());
  a.position_stride[0] = positions.dim() == 2 ? positions.stride(0) : 0;
  a.position_stride[1] = positions.stride(-1);
  a.turns = static_cast<const uint64_t*>(turns.const_data_ptr());
  launch(dwarf_rotary, a, q, "dwarf_rotary");
  return {q_out, k_out};
}

struct RotaryFn : torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& positions,
                               const Tensor& turns, bool interleaved, double magnitude) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, turns});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["q"] = q.sizes();
    if (k) ctx->saved_data["k"] = k->sizes();
    auto [q_out, k_out] = rotate(q, k, positions, turns, interleaved, false, magnitude);
    return k ? variable_list{q_out, k_out} : variable_list{q_out};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const bool has_k = ctx->saved_data.count("k") > 0;
    variable_list out(6);
    Tensor dq = grads[0], dk = has_k ? grads[1] : Tensor();
    if (!dq.defined() && !dk.defined()) return out;
    {
      const at::NoGradGuard no_grad;
      refuse_tangents("rotary_embed", dq, dk);
      const bool interleaved = ctx->saved_data["interleaved"].toBool();
      const double magnitude = ctx->saved_data["magnitude"].toDouble();
      // a single one is turned alone: its heads take q's place
      const Tensor& first = dq.defined() ? dq : dk;
      const OptTensor second = dq.defined() && dk.defined() ? OptTensor(dk) : std::nullopt;
      Tensor a, b;
      if (watched(dq, dk, saved[0], saved[1])) {
        const auto r = dispatched("dwarf::rotary", first, second, saved[0], saved[1], interleaved, true, magnitude);
        a = r[0], b = r[1];
      } else {
        std::tie(a, b) = rotate(first, second, saved[0], saved[1], interleaved, true, magnitude);
      }
      if (dq.defined()) out[0] = a;
      if (dk.defined()) out[1] = dq.defined() ? b : a;
    }
    return first_order(std::move(out), "rotary_embed");
  }
};

void check_rotary(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& turns) {
  TORCH_CHECK_VALUE(q.dim() == 4, "q must be [B,H,N,D], got ", q.sizes());
  const int64_t B = q.size(0), N = q.size(2), D = q.size(3);
  if (k)
    TORCH_CHECK_VALUE(k->dim() == 4 && k->size(0) == B && k->size(2) == N && k->size(3) == D && k->scalar_type() == q.scalar_type(),
                      "k must be [B,H_kv,N,D] like q ", q.sizes(), " ", q.scalar_type(), ", got ", k->sizes(), " ", k->scalar_type());
  TORCH_CHECK_VALUE(D % 2 == 0 && 2 * turns.numel() <= D, "D=", D, " must be even and at least the plan's rotary_dim ", 2 * turns.numel());
  TORCH_CHECK_VALUE(q.size(1) >= 1 && (!k || k->size(1) >= 1), "q and k need at least one head");
  TORCH_CHECK_VALUE(is_index(positions), "positions must be int32 or int64, got ", positions.scalar_type());
  TORCH_CHECK_VALUE((positions.dim() == 1 && positions.size(0) == N) ||
                        (positions.dim() == 2 && positions.size(0) == B && positions.size(1) == N),
                    "positions must be [", N, "] or [", B, ",", N, "], got ", positions.sizes());
  TORCH_CHECK_VALUE(turns.scalar_type() == at::kLong && turns.is_contiguous(), "the plan's turns must be contiguous int64, got ",
                    turns.scalar_type(), " strides ", turns.strides());
  dtype_of(q, "q");
  check_cuda(q);
  check_beside("k", k, q);
  check_beside("positions", positions, q);
  check_beside("plan", turns, q);
}

// Nothing: the call goes through the custom ops (see kWatched).
std::optional<std::tuple<Tensor, OptTensor>> rotary_embed(const Tensor& q, const OptTensor& k, const Tensor& positions,
                                                          const Tensor& turns, bool interleaved, double magnitude) {
  using Result = std::tuple<Tensor, OptTensor>;
  refuse_tangents("rotary_embed", q, k);
  if (watched(q, k, positions, turns)) return std::nullopt;
  check_rotary(q, k, positions, turns);
  if (at::GradMode::is_enabled() && (q.requires_grad() || (k && k->requires_grad()))) {
    const variable_list r = RotaryFn::apply(q, k, positions, turns, interleaved, magnitude);
    return Result{r[0], k ? OptTensor(r[1]) : std::nullopt};
  }
  auto [q_out, k_out] = rotate(q, k, positions, turns, interleaved, false, magnitude);
  return Result{q_out, k ? OptTensor(k_out) : std::nullopt};
}

// ---- decayed linear attention ------------------------------------------------------------------
// [B,H,N,64] as the kernels read it: 16-byte aligned rows that do not overlap, less than 2^22 elements apart.
Tensor token_rows(const Tensor& t) {
  if (t.size(2) > 1 && (t.stride(2) < kHd || t.stride(2) >= (int64_t(1) << 22))) return dense_copy(t);
  return kernel_rows(t);
}
Tensor aligned_f32(const Tensor& t) {
  const Tensor c = t.to(at::kFloat).contiguous();
  return aligned(c, 16) ? c : dense_copy(c);
}
Tensor decay_table(const Tensor& log_decay) {
  return log_decay.scalar_type() == at::kFloat && log_decay.is_contiguous() ? log_decay : log_decay.to(at::kFloat).contiguous();
}
// 64-bit values beyond 32 bits stay what they mean, below every slot and length or above them all.
Tensor index_table(const OptTensor& t) {
  if (!t) return Tensor();
  if (t->scalar_type() != at::kInt) return t->clamp(-1, INT32_MAX).to(at::kInt).contiguous();
  return t->contiguous();
}
const int32_t* i32_ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr<int32_t>() : nullptr; }

// What both directions read, in the kernels' layouts; held until the launches are queued.
struct Operands {
  Tensor q, k, v, decay, initial, lengths;
  Operands(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay, const OptTensor& initial_,
           const OptTensor& lengths_)
      : q(token_rows(q_)), k(token_rows(k_)), v(token_rows(v_)), decay(decay_table(log_decay)),
        initial(initial_ ? aligned_f32(*initial_) : Tensor()), lengths(index_table(lengths_)) {}
  void fill(dwarf_linear_attention_fwd_args& a, double scale) const {
    a.B = size32(q.size(0));
    a.H = size32(q.size(1));
    a.H_kv = size32(k.size(1));
    a.N = size32(q.size(2));
    a.head_dim = size32(q.size(3));
    a.dtype = dtype_of(q, "q");
    a.scale = static_cast<float>(scale);
    a.q = q.const_data_ptr();
    put_strides(a.q_stride, q);
    a.k = k.const_data_ptr();
    put_strides(a.k_stride, k);
    a.v = v.const_data_ptr();
    put_strides(a.v_stride, v);
    a.log_decay = f32_ptr(decay);
    a.lengths = i32_ptr(lengths);
    a.initial = f32_ptr(initial);
  }
};

// (out, the final state or undefined, the segments' states: undefined where there are none, unless `shaped`)
std::tuple<Tensor, Tensor, Tensor> attention_forward(const Tensor& q, const Tensor& k, const Tensor& v,
                                                     const Tensor& log_decay, const OptTensor& initial,
                                                     const OptTensor& lengths, double scale, bool want_state,
                                                     bool shaped) {
  const Operands in(q, k, v, log_decay, initial, lengths);
  dwarf_linear_attention_fwd_args a{};
  in.fill(a, scale);
  const Tensor out = token_major(a.B, a.H, a.N, kHd, q);
  const Tensor state = want_state ? empty_f32({a.B, a.H, kHd, kHd}, q) : Tensor();
  a.states_bytes = dwarf_linear_attention_states_bytes(&a);
  const int64_t per = static_cast<int64_t>(a.B) * a.H * kHd * kHd;
  const int64_t segs = per ? static_cast<int64_t>(a.states_bytes / sizeof(float)) / per : 0;
  const Tensor states = segs || shaped ? empty_f32({a.B, a.H, segs, kHd, kHd}, q) : Tensor();
  a.out = out.data_ptr();
  put_strides(a.out_stride, out);
  a.final = f32_out(state);
  a.states = f32_out(states);
  launch(dwarf_linear_attention_fwd, a, q, "dwarf_linear_attention_fwd");
  return {out, state, states};
}

// (dq, dk, dv, dlog_decay, dinitial), undefined where not needed
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> attention_backward(
    const Tensor& dout_, const OptTensor& dstate_, const Tensor& q, const Tensor& k, const Tensor& v,
    const Tensor& log_decay, const OptTensor& initial, const OptTensor& lengths, double scale, const Tensor& states,
    const OptTensor& state, bool need_decay, bool need_initial) {
  const Operands in(q, k, v, log_decay, initial, lengths);
  const Tensor dout = token_rows(dout_.to(q.scalar_type()));
  const Tensor dstate = dstate_ ? aligned_f32(*dstate_) : Tensor();
  dwarf_linear_attention_bwd_args a{};
  in.fill(a.fwd, scale);
  const int64_t B = a.fwd.B, H = a.fwd.H, Hkv = a.fwd.H_kv, N = a.fwd.N;
  a.fwd.states = const_cast<float*>(f32_ptr(states));
  a.fwd.states_bytes = states.defined() ? static_cast<size_t>(states.numel()) * sizeof(float) : 0;
  a.fwd.final = state ? const_cast<float*>(state->const_data_ptr<float>()) : nullptr;
  a.dout = dout.const_data_ptr();
  put_strides(a.dout_stride, dout);
  a.dfinal = f32_ptr(dstate);
  const Tensor dq = token_major(B, H, N, kHd, q), dk = token_major(B, Hkv, N, kHd, q), dv = token_major(B, Hkv, N, kHd, q);
  a.dq = dq.data_ptr();
  put_strides(a.dq_stride, dq);
  a.dk = dk.data_ptr();
  put_strides(a.dk_stride, dk);
  a.dv = dv.data_ptr();
  put_strides(a.dv_stride, dv);
  const Tensor dlog = need_decay ? empty_f32({H}, q) : Tensor();
  const Tensor dinitial = need_initial ? empty_f32({B, H, kHd, kHd}, q) : Tensor();
  a.dlog_decay = f32_out(dlog);
  a.dinitial = f32_out(dinitial);
  a.workspace_bytes = dwarf_linear_attention_bwd_workspace_bytes(&a);
  const Tensor ws = workspace(a.workspace_bytes, q);
  if (ws.defined()) a.workspace = ws.data_ptr();
  launch(dwarf_linear_attention_bwd, a, q, "dwarf_linear_attention_bwd");
  return {dq, dk, dv, dlog, dinitial};
}

struct LinearAttentionFn : torch::autograd::Function<LinearAttentionFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& log_decay, const OptTensor& initial, const OptTensor& lengths, double scale,
                               bool want_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    auto [out, state, states] = attention_forward(q, k, v, log_decay, initial, lengths, scale, want_state, false);
    // the final state serves the decay's gradient
    const Tensor kept = want_state && log_decay.requires_grad() ? state : Tensor();
    ctx->save_for_backward({q, k, v, log_decay, initial.value_or(Tensor()), lengths.value_or(Tensor()), states, kept});
    ctx->saved_data["scale"] = scale;
    return want_state ? variable_list{out, state} : variable_list{out};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    variable_list result(8);
    Tensor dout = grads[0];
    const Tensor dstate = grads.size() > 1 ? grads[1] : Tensor();
    if (!dout.defined() && !dstate.defined()) return result;
    {
      const at::NoGradGuard no_grad;
      refuse_tangents("linear_attention", dout, dstate, s[0], s[1], s[2], s[3], s[4]);
      if (!dout.defined()) dout = at::zeros_like(s[0]);
      auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
      const double scale = ctx->saved_data["scale"].toDouble();
      const bool need_decay = ctx->needs_input_grad(3), need_initial = s[4].defined() && ctx->needs_input_grad(4);
      Tensor dq, dk, dv, dlog, dinitial;
      if (watched(dout, dstate, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7])) {
        const Tensor states = s[6].defined() ? s[6] : empty_f32({0}, s[0]);
        const auto r = dispatched("dwarf::linear_attention_bwd", dout, opt(dstate), s[0], s[1], s[2], s[3], opt(s[4]),
                                  opt(s[5]), scale, states, opt(s[7]), need_decay, need_initial);
        dq = r[0], dk = r[1], dv = r[2];
        if (need_decay) dlog = r[3];
        if (need_initial) dinitial = r[4];
      } else {
        std::tie(dq, dk, dv, dlog, dinitial) = attention_backward(dout, opt(dstate), s[0], s[1], s[2], s[3], opt(s[4]),
                                                                  opt(s[5]), scale, s[6], opt(s[7]), need_decay, need_initial);
      }
      if (ctx->needs_input_grad(0)) result[0] = dq;
      if (ctx->needs_input_grad(1)) result[1] = dk;
      if (ctx->needs_input_grad(2)) result[2] = dv;
      if (dlog.defined()) result[3] = dlog.view(s[3].sizes()).to(s[3].scalar_type());
      if (dinitial.defined()) result[4] = dinitial;
    }
    return first_order(std::move(result), "linear_attention");
  }
};

double scale_or_default(const std::optional<double>& scale) {
  TORCH_CHECK_VALUE(!scale || std::isfinite(*scale), "scale must be finite");
  return scale ? *scale : 0.125;
}

void check_heads(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const char* dims) {
  const int64_t H = q.size(1), Hkv = k.size(1);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
                    "k and v must share a shape and q's dtype ", q.scalar_type(), "; got ", k.sizes(), " ", k.scalar_type(),
                    ", ", v.sizes(), " ", v.scalar_type());
  TORCH_CHECK_VALUE(q.size(0) == k.size(0) && q.sizes().slice(2) == k.sizes().slice(2), "k ", k.sizes(), " does not match q ",
                    q.sizes(), " (", dims, ")");
  TORCH_CHECK_VALUE(Hkv >= 1 && H >= 1 && H % Hkv == 0, "num query heads H=", H, " must be divisible by KV heads H_kv=", Hkv);
  TORCH_CHECK_VALUE(log_decay.numel() == H && log_decay.is_floating_point(), "log_decay must hold one floating value per head (",
                    H, "), got ", log_decay.sizes(), " ", log_decay.scalar_type());
  dtype_of(q, "q");
}

void check_state(const char* name, const OptTensor& t, const Tensor& q) {
  if (!t) return;
  TORCH_CHECK_VALUE(q.dim() == 4, "q must be [B,H,N,64], got ", q.sizes());
  const int64_t B = q.size(0), H = q.size(1), hd = q.size(3);
  TORCH_CHECK_VALUE(t->sizes() == at::IntArrayRef({B, H, hd, hd}) && t->scalar_type() == at::kFloat, name, " must be fp32 [", B,
                    ",", H, ",", hd, ",", hd, "], got ", t->sizes(), " ", t->scalar_type());
}

void check_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptTensor& initial,
                     const OptTensor& lengths) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k and v must be [B,H,N,64], got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  check_heads(q, k, v, log_decay, "[B,H,N,64]");
  const int64_t B = q.size(0), hd = q.size(3);
  check_state("initial_state", initial, q);
  if (lengths)
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == B && is_index(*lengths), "lengths must be [", B,
                      "] int32 or int64, got ", lengths->sizes(), " ", lengths->scalar_type());
  check_cuda(q);
  check_beside("k", k, q);
  check_beside("v", v, q);
  check_beside("log_decay", log_decay, q);
  check_beside("initial_state", initial, q);
  check_beside("lengths", lengths, q);
  TORCH_CHECK(hd == kHd, "linear attention is built for head_dim 64, got ", hd);
}

// None: the call goes through the custom ops (see kWatched).
py::object linear_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                            const std::optional<double>& scale_, const OptTensor& initial, const OptTensor& lengths,
                            bool return_state) {
  refuse_tangents("linear_attention", q, k, v, log_decay, initial);
  if (watched(q, k, v, log_decay, initial, lengths)) return py::none();
  const double scale = scale_or_default(scale_);
  check_attention(q, k, v, log_decay, initial, lengths);
  Tensor out, state;
  {
    const py::gil_scoped_release release;
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || log_decay.requires_grad() ||
                                       (initial && initial->requires_grad()))) {
      const variable_list r = LinearAttentionFn::apply(q, k, v, log_decay, initial, lengths, scale, return_state);
      out = r[0];
      if (return_state) state = r[1];
    } else {
      Tensor states;
      std::tie(out, state, states) = attention_forward(q, k, v, log_decay, initial, lengths, scale, return_state, false);
    }
  }
  return return_state ? py::object(py::make_tuple(out, state)) : py::cast(out);
}

bool pool_ok(const Tensor& t, int64_t H) {
  return t.dim() == 4 && t.scalar_type() == at::kFloat && t.size(1) == H && t.size(2) == kHd && t.size(3) == kHd &&
         (t.size(0) <= 1 || (t.stride(0) >= H * kHd * kHd && t.stride(0) % 4 == 0)) && t.stride(1) == kHd * kHd &&
         t.stride(2) == kHd && t.stride(3) == 1 && aligned(t, 16);
}

void check_pools(const Tensor& state, const OptTensor& new_state, int64_t H) {
  TORCH_CHECK_VALUE(pool_ok(state, H), "state must be an fp32 [P,", H, ",64,64] pool with contiguous, 16-byte aligned slots, got ",
                    state.sizes(), " ", state.scalar_type(), " strides ", state.strides());
  if (new_state) {
    TORCH_CHECK_VALUE(pool_ok(*new_state, H), "new_state must be an fp32 [P,", H,
                      ",64,64] pool with contiguous, 16-byte aligned slots, got ", new_state->sizes(), " ",
                      new_state->scalar_type(), " strides ", new_state->strides());
    TORCH_CHECK_VALUE(new_state->sizes() == state.sizes() && (state.size(0) <= 1 || new_state->strides() == state.strides()),
                      "new_state must have state's shape and strides");
  }
}

Tensor attention_step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& log_decay, const Tensor& state,
                      const OptTensor& new_state, const OptTensor& slots_, double scale, const OptTensor& out_) {
  const Tensor q = kernel_rows(q_), k = kernel_rows(k_), v = kernel_rows(v_);
  const Tensor decay = decay_table(log_decay), slots = index_table(slots_);
  const Tensor out = out_ ? *out_ : at::empty(q.sizes(), q.options());
  dwarf_linear_attention_step_args a{};
  a.S = size32(q.size(0));
  a.H = size32(q.size(1));
  a.H_kv = size32(k.size(1));
  a.pool = size32(state.size(0));
  a.head_dim = size32(q.size(2));
  a.dtype = dtype_of(q, "q");
  a.scale = static_cast<float>(scale);
  a.q = q.const_data_ptr();
  put_strides(a.q_stride, q);
  a.k = k.const_data_ptr();
  put_strides(a.k_stride, k);
  a.v = v.const_data_ptr();
  put_strides(a.v_stride, v);
  a.log_decay = f32_ptr(decay);
  a.slots = i32_ptr(slots);
  a.state = state.const_data_ptr<float>();
  a.new_state = (new_state ? *new_state : state).data_ptr<float>();
  a.slot_stride = a.pool > 1 ? state.stride(0) : static_cast<int64_t>(a.H) * kHd * kHd;
  a.out = out.data_ptr();
  put_strides(a.out_stride, out);
  launch(dwarf_linear_attention_step, a, q, "dwarf_linear_attention_step");
  // written behind autograd's back: a graph that saved the pool has to notice
  for (const Tensor& t : {new_state ? *new_state : state, out_ ? *out_ : Tensor()})
    if (t.defined() && !t.is_inference()) torch::autograd::impl::bump_version(t);
  return out;
}

// The step's tensors in memory, in bytes: n0 rows of n1 runs of `run` bytes ([S,H,64], or a pool whose slots are whole).
struct Runs {
  int64_t at, n0, s0, n1, s1, run;
  explicit Runs(const Tensor& t) {
    const bool pool = t.dim() == 4;
    const int64_t es = static_cast<int64_t>(t.element_size());
    at = static_cast<int64_t>(reinterpret_cast<intptr_t>(t.const_data_ptr()));
    n0 = t.size(0), s0 = t.stride(0) * es;
    n1 = pool ? 1 : t.size(1), s1 = pool ? 0 : t.stride(1) * es;
    run = (pool ? t.size(1) * kHd * kHd : kHd) * es;
  }
  int64_t end() const { return at + (n0 - 1) * s0 + (n1 - 1) * s1 + run; }
};
int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b != 0 && a < 0); }

// Whether some n in [low, high] has n step + e inside (-behind, ahead).
bool steps_into(int64_t low, int64_t high, int64_t step, int64_t e, int64_t behind, int64_t ahead) {
  if (step == 0) return -behind < e && e < ahead;
  low = std::max(low, -floor_div(e + behind - 1, step));
  high = std::min(high, floor_div(ahead - 1 - e, step));
  return low <= high;
}

// Whether a byte belongs to both.  Rows of one stride, which slices of a fused buffer have, need no loop over them.
bool meet(Runs a, Runs b) {
  if (a.end() <= b.at || b.end() <= a.at) return false;
  if (a.s0 == 0) a.n0 = 1;   // expanded: one row, one head
  if (b.s0 == 0) b.n0 = 1;
  if (a.s1 == 0) a.n1 = 1;
  if (b.s1 == 0) b.n1 = 1;
  if (a.n0 > 1 && b.n0 > 1 && a.s0 != b.s0) {
    Runs row = a;
    row.n0 = 1;
    for (int64_t i = 0; i < a.n0; ++i, row.at += a.s0)
      if (meet(row, b)) return true;
    return false;
  }
  const int64_t s0 = b.n0 > 1 ? b.s0 : a.s0, d = b.at - a.at;
  auto heads = [&](int64_t e) { return steps_into(1 - a.n0, b.n0 - 1, s0, e, b.run, a.run); };
  if (a.s1 == b.s1 || a.n1 == 1 || b.n1 == 1) {
    const int64_t s1 = b.n1 > 1 ? b.s1 : a.s1;
    for (int64_t m = 1 - a.n1; m < b.n1; ++m)
      if (heads(d + m * s1)) return true;
    return false;
  }
  for (int64_t i = 0; i < a.n1; ++i)
    for (int64_t j = 0; j < b.n1; ++j)
      if (heads(d + j * b.s1 - i * a.s1)) return true;
  return false;
}
bool meets_itself(const Runs& a) {
  if ((a.n0 > 1 && a.s0 < a.run) || (a.n1 > 1 && a.s1 < a.run)) return true;
  for (int64_t m = 1; m < a.n1; ++m)   // the other sign is the same pair
    if (steps_into(1 - a.n0, a.n0 - 1, a.s0, m * a.s1, a.run, a.run)) return true;
  return false;
}

void check_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state,
                const OptTensor& slots, const OptTensor& new_state, const OptTensor& out) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k and v must be [S,H,64], got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  check_heads(q, k, v, log_decay, "[S,H,64]");
  const int64_t S = q.size(0), H = q.size(1);
  TORCH_CHECK(q.size(2) == kHd, "linear attention is built for head_dim 64, got ", q.size(2));
  check_pools(state, new_state, H);
  TORCH_CHECK_VALUE(slots || state.size(0) >= S, "a pool of ", state.size(0), " states does not hold the ", S, " rows");
  if (slots)
    TORCH_CHECK_VALUE(slots->dim() == 1 && slots->size(0) == S && is_index(*slots), "slots must be [", S,
                      "] int32 or int64, got ", slots->sizes(), " ", slots->scalar_type());
  if (out)
    TORCH_CHECK_VALUE(out->sizes() == q.sizes() && out->scalar_type() == q.scalar_type() && rows_ok(*out), "out must be [", S,
                      ",", H, ",64] ", q.scalar_type(), " with 16-byte aligned rows");
  if (out)
    for (const auto& [name, t] : {std::make_pair("out", &*out), std::make_pair("q", &q), std::make_pair("k", &k),
                                  std::make_pair("v", &v), std::make_pair("state", &state),
                                  std::make_pair("new_state", new_state ? &*new_state : &state)}) {
      if (!out->numel() || !t->numel()) continue;
      TORCH_CHECK_VALUE(!(t == &*out ? meets_itself(Runs(*t)) : meet(Runs(*out), Runs(*t))), "out shares memory with ", name);
    }
  check_cuda(q);
  check_beside("k", k, q);
  check_beside("v", v, q);
  check_beside("log_decay", log_decay, q);
  check_beside("state", state, q);
  check_beside("slots", slots, q);
  check_beside("new_state", new_state, q);
  check_beside("out", out, q);
  TORCH_CHECK_VALUE(!S || state.size(0), "the pool is empty");
}

// Nothing: the call goes through the custom ops (see kWatched).
OptTensor linear_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state,
                                const OptTensor& slots, const OptTensor& new_state, const std::optional<double>& scale_,
                                const OptTensor& out) {
  refuse_tangents("linear_attention_step", q, k, v, log_decay, state, new_state, out);
  if (watched(q, k, v, log_decay, state, slots, new_state, out)) return std::nullopt;
  const double scale = scale_or_default(scale_);
  check_step(q, k, v, log_decay, state, slots, new_state, out);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad() ||
                                               log_decay.requires_grad() || state.requires_grad() ||
                                               (new_state && new_state->requires_grad()) || (out && out->requires_grad())),
              "linear_attention_step has no gradients: call it under torch.no_grad(), or linear_attention");
  return attention_step(q, k, v, log_decay, state, new_state, slots, scale, out);
}

}  // namespace

PYBIND11_MODULE(_mixer, m) {
  m.doc() = "Eager calls of the mixer's operators (C++ side of norm.py, rotary.py and linattn.py)";
  m.attr("abi_version") = DWARF_ABI_VERSION;
  // the Python class of failed launches
  static PyObject* error_class = nullptr;
  m.def("set_error_class", [](py::object cls) {
    Py_XDECREF(error_class);
    error_class = cls.release().ptr();
  });
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const StatusError& e) {
      PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what());
    }
  });
  const auto no_gil = py::call_guard<py::gil_scoped_release>();
  m.def("layer_norm", &layer_norm, no_gil);
  m.def("rotary_embed", &rotary_embed, no_gil);
  m.def("linear_attention", &linear_attention);
  m.def("linear_attention_step", &linear_attention_step, no_gil);
  // the custom ops' launches: the same, checked here
  m.def("norm_forward", [](const Tensor& x, const OptTensor& weight, const OptTensor& bias, int64_t groups, double eps) {
    refuse_tangents("layer_norm", x, weight, bias);
    check_norm_launch(x, weight, bias, groups);
    return norm_forward(x, weight, bias, groups, eps);
  }, no_gil);
  m.def("norm_backward", [](const Tensor& dy, const Tensor& x, const OptTensor& weight, int64_t groups, double eps, bool need_dx,
                            bool need_dw, bool need_db) {
    refuse_tangents("layer_norm", dy, x, weight);
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "dy must have x's shape ", x.sizes(), ", got ", dy.sizes());
    check_norm_launch(x, weight, std::nullopt, groups);
    check_beside("dy", dy, x);
    return norm_backward(dy, x, weight, groups, eps, need_dx, need_dw, need_db);
  }, no_gil);
  m.def("rotate", [](const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& turns, bool interleaved,
                     bool inverse, double magnitude) {
    refuse_tangents("rotary_embed", q, k);
    check_rotary(q, k, positions, turns);
    return rotate(q, k, positions, turns, interleaved, inverse, magnitude);
  }, no_gil);
  m.def("attention_forward", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                const OptTensor& initial, const OptTensor& lengths, double scale, bool want_state) {
    refuse_tangents("linear_attention", q, k, v, log_decay, initial);
    check_attention(q, k, v, log_decay, initial, lengths);
    return attention_forward(q, k, v, log_decay, initial, lengths, scale, want_state, true);
  }, no_gil);
  m.def("attention_backward", [](const Tensor& dout, const OptTensor& dstate, const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& log_decay, const OptTensor& initial, const OptTensor& lengths, double scale,
                                 const Tensor& states, const OptTensor& state, bool need_decay, bool need_initial) {
    refuse_tangents("linear_attention", dout, dstate, q, k, v, log_decay, initial);
    TORCH_CHECK_VALUE(dout.sizes() == q.sizes(), "dout must have q's shape ", q.sizes(), ", got ", dout.sizes());
    check_state("dstate", dstate, q);
    check_state("state", state, q);
    TORCH_CHECK_VALUE(!state || (state->is_contiguous() && aligned(*state, 16)), "state must be contiguous and 16-byte aligned");
    TORCH_CHECK_VALUE(states.scalar_type() == at::kFloat && states.is_contiguous(), "states must be the forward's");
    check_attention(q, k, v, log_decay, initial, lengths);
    check_beside("dout", dout, q);
    check_beside("dstate", dstate, q);
    check_beside("state", state, q);
    check_beside("states", states, q);
    return attention_backward(dout, dstate, q, k, v, log_decay, initial, lengths, scale, states, state, need_decay, need_initial);
  }, no_gil);
  m.def("attention_step", [](const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state,
                             const OptTensor& new_state, const OptTensor& slots, double scale, const OptTensor& out) {
    refuse_tangents("linear_attention_step", q, k, v, log_decay, state, new_state, out);
    check_step(q, k, v, log_decay, state, slots, new_state, out);
    return attention_step(q, k, v, log_decay, state, new_state, slots, scale, out);
  }, no_gil);
}
