// What the eager calls on PyTorch tensors share (mixer_torch.cpp,
// selective_torch.cpp): statuses and launches, the tensors that go through the
// custom ops instead, argument checks, buffers, first-order gradients.
#pragma once

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
#include <optional>
#include <string>

#include "dwarf_mixer.h"

namespace dwarf_torch {

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// A status that is neither success nor an invalid argument (the Python side's NativeLibraryError).
struct StatusError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

inline void check_status(int rc, const char* what) {
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

inline c10::DispatchKeySet keys_of(const Tensor& t) { return t.defined() ? t.key_set() : c10::DispatchKeySet(); }
inline c10::DispatchKeySet keys_of(const OptTensor& t) { return t ? keys_of(*t) : c10::DispatchKeySet(); }
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
inline bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
inline bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }
template <typename... T>
void refuse_tangents(const char* what, const T&... t) {
  TORCH_CHECK(!(has_tangent(t) || ...), what, " has no derivative in forward mode: differentiate it backward");
}

inline int dtype_of(const Tensor& x, const char* what) {
  switch (x.scalar_type()) {
    case at::kBFloat16: return DWARF_BF16;
    case at::kHalf: return DWARF_F16;
    case at::kFloat: return DWARF_F32;
    default: TORCH_CHECK_VALUE(false, what, " must be bf16, fp16 or fp32, got ", x.scalar_type());
  }
}

// A size as the C ABI takes it.
inline int32_t size32(int64_t n) {
  TORCH_CHECK(n <= INT32_MAX, "dimensions must stay below 2^31, got ", n);
  return static_cast<int32_t>(n);
}

inline void check_cuda(const Tensor& x) { TORCH_CHECK(x.is_cuda(), "the mixer's HIP kernels require device tensors"); }
inline void check_beside(const char* name, const Tensor& t, const Tensor& x) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", expected ", x.device());
}
inline void check_beside(const char* name, const OptTensor& t, const Tensor& x) {
  if (t) check_beside(name, *t, x);
}
inline bool is_index(const Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong; }

inline Tensor empty_like_dtype(at::IntArrayRef shape, const Tensor& like, at::ScalarType dtype) {
  return at::empty(shape, like.options().dtype(dtype));
}
inline Tensor empty_f32(at::IntArrayRef shape, const Tensor& like) { return empty_like_dtype(shape, like, at::kFloat); }
inline Tensor workspace(size_t nbytes, const Tensor& like) {
  return nbytes ? empty_like_dtype({static_cast<int64_t>(nbytes)}, like, at::kByte) : Tensor();
}

template <int N>
void put_strides(int64_t (&to)[N], const Tensor& t) {
  const auto s = t.strides();
  for (int i = 0; i < N; ++i) to[i] = s[i];
}

inline bool aligned(const Tensor& t, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }

// Unit last stride and 16-byte aligned rows.
inline bool rows_ok(const Tensor& t) {
  const auto s = t.strides();
  const int64_t per16 = 16 / t.element_size();
  if (s.back() != 1 || !aligned(t, 16)) return false;
  for (size_t i = 0; i + 1 < s.size(); ++i)
    if (s[i] % per16) return false;
  return true;
}
// A contiguous copy: contiguous() alone gives a dense tensor back as it is, at whatever address it begins.
inline Tensor dense_copy(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
inline Tensor kernel_rows(const Tensor& t) { return rows_ok(t) ? t : dense_copy(t); }

// Gradients whose own derivative raises: the backward nodes are first order.
inline variable_list first_order(variable_list grads, const char* what) {
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

inline Tensor table(const OptTensor& t) {
  if (!t) return Tensor();
  return t->scalar_type() == at::kFloat && t->is_contiguous() ? *t : t->to(at::kFloat).contiguous();
}
inline const float* f32_ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
inline float* f32_out(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

inline Tensor aligned_f32(const Tensor& t) {
  const Tensor c = t.to(at::kFloat).contiguous();
  return aligned(c, 16) ? c : dense_copy(c);
}
// 64-bit values beyond 32 bits stay what they mean, below every slot and length or above them all.
inline Tensor index_table(const OptTensor& t) {
  if (!t) return Tensor();
  if (t->scalar_type() != at::kInt) return t->clamp(-1, INT32_MAX).to(at::kInt).contiguous();
  return t->contiguous();
}
inline const int32_t* i32_ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr<int32_t>() : nullptr; }

// Rows that a norm runs over.
struct NormRows {
  Tensor x;
  int64_t row, group;   // strides
};

// x as [rows][groups][D]; copied where its leading dimensions do not collapse into one row stride.
inline NormRows norm_rows(const Tensor& x, int64_t groups) {
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

// selective_torch.cpp's part of the module.
void register_selective(py::module_& m);

}  // namespace dwarf_torch
