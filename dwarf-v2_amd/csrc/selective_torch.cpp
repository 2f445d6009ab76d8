// The eager calls of the selective mixer's operators (RMS norm with the
// residual, short causal convolution, selective scan) on PyTorch tensors:
// argument checks, layouts, buffers, autograd nodes and the calls into
// libdwarf_dsqg.so's C ABI.  Part of the module _mixer, for mixer_torch.cpp's
// reasons.
#include "torch_calls.h"

#include "dwarf_selective.h"

namespace {

using namespace dwarf_torch;

OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t && t->requires_grad(); }
template <typename... T>
bool any_grad(const T&... t) { return at::GradMode::is_enabled() && (wants_grad(t) || ...); }

// Whether each of a node's tensor inputs needs its gradient; the engine counts the inputs that were given.
struct Needs {
  AutogradContext* ctx;
  size_t at = 0;
  bool next(bool given) { return given && ctx->needs_input_grad(at++); }
};

// ---- RMS norm ----------------------------------------------------------------------------------
struct RmsResult {
  Tensor y, sum, scale;   // sum: with a residual; scale: in 8 bits
};

RmsResult rms_forward(const Tensor& x, const OptTensor& weight, const OptTensor& residual, int64_t groups, double eps, bool eights) {
  const NormRows r = norm_rows(x, groups);
  const Tensor w = table(weight);
  RmsResult out;
  dwarf_rms_norm_fwd_args a{};
  const int64_t D = x.size(-1);
  a.rows = x.numel() / (groups * D);
  a.groups = size32(groups);
  a.D = size32(D);
  a.dtype = dtype_of(x, "x");
  a.eps = static_cast<float>(eps);
  a.x = r.x.const_data_ptr();
  a.x_stride[0] = r.row;
  a.x_stride[1] = r.group;
  a.weight = f32_ptr(w);
  NormRows rr;
  if (residual) {
    rr = norm_rows(*residual, groups);
    out.sum = at::empty(x.sizes(), residual->options());
    a.residual_dtype = dtype_of(*residual, "residual");
    a.residual = rr.x.const_data_ptr();
    a.residual_stride[0] = rr.row;
    a.residual_stride[1] = rr.group;
    a.sum = out.sum.data_ptr();
    a.sum_stride[0] = groups * D;
    a.sum_stride[1] = D;
  }
  out.y = empty_like_dtype(x.sizes(), x, eights ? at::kFloat8_e4m3fn : x.scalar_type());
  a.y = out.y.data_ptr();
  a.y_stride[0] = groups * D;
  a.y_stride[1] = D;
  if (eights) {
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = 1;
    out.scale = empty_f32(shape, x);
    a.scale = f32_out(out.scale);
  }
  launch(dwarf_rms_norm_fwd, a, x, "dwarf_rms_norm_fwd");
  return out;
}

// (dx of dy's dtype, dresidual of the stream's, dweight fp32 [groups * D]); undefined where not needed
std::tuple<Tensor, Tensor, Tensor> rms_backward(const Tensor& dy, const OptTensor& dsum, const Tensor& stream, const OptTensor& weight,
                                                int64_t groups, double eps, bool need_dx, bool need_dr, bool need_dw) {
  const NormRows r = norm_rows(stream, groups), g = norm_rows(dy, groups);
  const Tensor w = table(weight);
  NormRows u;
  Tensor dx, dr, dw;
  dwarf_rms_norm_bwd_args a{};
  const int64_t D = stream.size(-1);
  a.rows = stream.numel() / (groups * D);
  a.groups = size32(groups);
  a.D = size32(D);
  a.dtype = dtype_of(dy, "dy");
  a.stream_dtype = dtype_of(stream, "stream");
  a.eps = static_cast<float>(eps);
  a.stream = r.x.const_data_ptr();
  a.stream_stride[0] = r.row;
  a.stream_stride[1] = r.group;
  a.weight = f32_ptr(w);
  a.dy = g.x.const_data_ptr();
  a.dy_stride[0] = g.row;
  a.dy_stride[1] = g.group;
  if (dsum) {
    u = norm_rows(dsum->to(stream.scalar_type()), groups);
    a.dsum = u.x.const_data_ptr();
    a.dsum_stride[0] = u.row;
    a.dsum_stride[1] = u.group;
  }
  const bool same = a.dtype == a.stream_dtype;   // one gradient serves both
  if (need_dx || (same && need_dr)) {
    dx = at::empty(stream.sizes(), dy.options());
    a.dx = dx.data_ptr();
    a.dx_stride[0] = groups * D;
    a.dx_stride[1] = D;
    if (same && need_dr) dr = dx;
  }
  if (need_dr && !same) {
    dr = at::empty(stream.sizes(), stream.options());
    a.dresidual = dr.data_ptr();
    a.dresidual_stride[0] = groups * D;
    a.dresidual_stride[1] = D;
  }
  if (need_dw) dw = empty_f32({groups * D}, stream);
  a.dweight = f32_out(dw);
  a.workspace_bytes = dwarf_rms_norm_bwd_workspace_bytes(&a);
  const Tensor ws = workspace(a.workspace_bytes, stream);
  if (ws.defined()) a.workspace = ws.data_ptr();
  launch(dwarf_rms_norm_bwd, a, stream, "dwarf_rms_norm_bwd");
  return {need_dx ? dx : Tensor(), dr, dw};
}

struct RmsNormFn : torch::autograd::Function<RmsNormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& residual,
                               int64_t groups, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    const RmsResult r = rms_forward(x, weight, residual, groups, eps, false);
    ctx->save_for_backward({residual ? r.sum : x, weight.value_or(Tensor())});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["dtype"] = x.scalar_type();
    return residual ? variable_list{r.y, r.sum} : variable_list{r.y};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    variable_list out(5);
    const bool added = ctx->saved_data["residual"].toBool();
    Tensor dy = grads[0];
    const Tensor dsum = added ? grads[1] : Tensor();
    if (!dy.defined() && !dsum.defined()) return out;
    {
      const at::NoGradGuard no_grad;
      refuse_tangents("rms_norm", dy, dsum, s[0], s[1]);
      const at::ScalarType dtype = ctx->saved_data["dtype"].toScalarType();
      Needs needs{ctx};
      const bool need_x = needs.next(true), need_w = needs.next(s[1].defined()), need_r = needs.next(added);
      // the sum alone was used: its gradient is the inputs', and the weight's is zero
      if (!dy.defined()) dy = at::zeros_like(s[0], s[0].options().dtype(dtype));
      dy = dy.to(dtype);
      const int64_t groups = ctx->saved_data["groups"].toInt();
      const double eps = ctx->saved_data["eps"].toDouble();
      Tensor dx, dr, dw;
      if (watched(dy, dsum, s[0], s[1])) {
        const auto r = dispatched("dwarf::rms_norm_bwd", dy, optional(dsum), s[0], optional(s[1]), groups, eps, need_x, need_r, need_w);
        dx = r[0], dr = r[1], dw = r[2];
      } else {
        std::tie(dx, dr, dw) = rms_backward(dy, optional(dsum), s[0], optional(s[1]), groups, eps, need_x, need_r, need_w);
      }
      if (need_x) out[0] = dx;
      if (need_w) out[1] = dw.view(s[1].sizes()).to(s[1].scalar_type());
      if (need_r) out[2] = dr;
    }
    return first_order(std::move(out), "rms_norm");
  }
};

// Checks a call and returns the groups.
int64_t check_rms(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
  TORCH_CHECK_VALUE(std::isfinite(eps) && eps >= 0, "eps must be finite and not negative");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must have a last dimension to normalise, got ", x.sizes());
  int64_t groups = 1;
  if (weight) {
    const Tensor& v = *weight;
    TORCH_CHECK_VALUE((v.dim() == 1 || v.dim() == 2) && v.dim() <= x.dim() && v.sizes() == x.sizes().slice(x.dim() - v.dim()),
                      "weight must hold the last one or two dimensions of x ", x.sizes(), ", got ", v.sizes());
    TORCH_CHECK_VALUE(v.is_floating_point(), "weight must be floating point, got ", v.scalar_type());
    if (v.dim() == 2) groups = v.size(0);
  }
  TORCH_CHECK_VALUE(groups >= 1, "weight needs at least one group");
  dtype_of(x, "x");
  if (residual)
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && (residual->scalar_type() == x.scalar_type() || residual->scalar_type() == at::kFloat),
                      "residual must have x's shape ", x.sizes(), " and its dtype ", x.scalar_type(), " or fp32, got ",
                      residual->sizes(), " ", residual->scalar_type());
  check_cuda(x);
  check_beside("weight", weight, x);
  check_beside("residual", residual, x);
  return groups;
}

// None: the call goes through the custom ops (see kWatched).
py::object rms_norm(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
  refuse_tangents("rms_norm", x, weight, residual);
  if (watched(x, weight, residual)) return py::none();
  const int64_t groups = check_rms(x, weight, residual, eps);
  Tensor y, sum;
  {
    const py::gil_scoped_release release;
    if (any_grad(x, weight, residual)) {
      const variable_list r = RmsNormFn::apply(x, weight, residual, groups, eps);
      y = r[0];
      if (residual) sum = r[1];
    } else {
      const RmsResult r = rms_forward(x, weight, residual, groups, eps, false);
      y = r.y, sum = r.sum;
    }
  }
  return residual ? py::object(py::make_tuple(y, sum)) : py::cast(y);
}

py::object rms_norm_fp8(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
  refuse_tangents("rms_norm_fp8", x, weight, residual);
  if (watched(x, weight, residual)) return py::none();
  const int64_t groups = check_rms(x, weight, residual, eps);
  TORCH_CHECK(!any_grad(x, weight, residual), "rms_norm_fp8 has no gradients: call it under torch.no_grad(), or rms_norm");
  RmsResult r;
  {
    const py::gil_scoped_release release;
    r = rms_forward(x, weight, residual, groups, eps, true);
  }
  return residual ? py::object(py::make_tuple(r.y, r.scale, r.sum)) : py::object(py::make_tuple(r.y, r.scale));
}

// What the launches take for granted, for the custom ops.
void check_rms_launch(const Tensor& x, const OptTensor& weight, const OptTensor& residual, int64_t groups, double eps) {
  check_rms(x, std::nullopt, residual, eps);
  TORCH_CHECK_VALUE(groups == 1 || (groups > 1 && x.dim() >= 2 && x.size(-2) == groups), "groups=", groups, " does not fit x ", x.sizes());
  if (weight)
    TORCH_CHECK_VALUE(weight->is_floating_point() && weight->numel() == groups * x.size(-1), "weight must hold ", groups, " x ",
                      x.size(-1), " floating values, got ", weight->sizes(), " ", weight->scalar_type());
  check_beside("weight", weight, x);
}

// ---- sequences ---------------------------------------------------------------------------------
// Rows whose elements lie side by side, as they are; others copied.
Tensor unit_rows(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

void check_lengths(const OptTensor& lengths, int64_t B) {
  if (lengths)
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == B && is_index(*lengths), "lengths must be [", B,
                      "] int32 or int64, got ", lengths->sizes(), " ", lengths->scalar_type());
}
void check_slots(const OptTensor& slots, int64_t rows) {
  if (slots)
    TORCH_CHECK_VALUE(slots->dim() == 1 && slots->size(0) == rows && is_index(*slots), "slots must be [", rows,
                      "] int32 or int64, got ", slots->sizes(), " ", slots->scalar_type());
}
// A table of one floating value for each channel.
void check_channels(const char* name, const OptTensor& t, int64_t D) {
  if (t)
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == D && t->is_floating_point(), name, " must be [", D, "] floating point, got ",
                      t->sizes(), " ", t->scalar_type());
}
void check_like(const char* name, const OptTensor& t, const Tensor& x) {
  if (t)
    TORCH_CHECK_VALUE(t->sizes() == x.sizes() && t->scalar_type() == x.scalar_type(), name, " must be ", x.sizes(), " ",
                      x.scalar_type(), " as x is, got ", t->sizes(), " ", t->scalar_type());
}

// The bytes from a tensor's first to its last element.
std::pair<intptr_t, intptr_t> extent(const Tensor& t) {
  const intptr_t at = reinterpret_cast<intptr_t>(t.const_data_ptr());
  if (!t.numel()) return {at, at};
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return {at, at + (last + 1) * static_cast<int64_t>(t.element_size())};
}
// A step writes a pool's slots while other workgroups read the rows.
void check_apart(const char* name, const OptTensor& t, const Tensor& pool) {
  if (!t || !t->numel() || !pool.numel()) return;
  const auto a = extent(*t), b = extent(pool);
  TORCH_CHECK_VALUE(a.second <= b.first || b.second <= a.first, name, " shares memory with the states");
}

// A pool [P, rows, cols] with contiguous slots, and the one that the new states go to.
void check_pool(const char* name, const Tensor& t, int64_t rows, int64_t cols, at::ScalarType dtype) {
  const bool ok = t.dim() == 3 && t.scalar_type() == dtype && t.size(1) == rows && t.size(2) == cols &&
                  (rows * cols == 0 || ((t.size(0) <= 1 || t.stride(0) >= rows * cols) && (rows <= 1 || t.stride(1) == cols) &&
                                        (cols <= 1 || t.stride(2) == 1)));
  TORCH_CHECK_VALUE(ok, name, " must be a ", dtype, " [P,", rows, ",", cols, "] pool with contiguous slots, got ", t.sizes(), " ",
                    t.scalar_type(), " strides ", t.strides());
}
void check_pools(const Tensor& state, const OptTensor& new_state, const OptTensor& slots, int64_t R, int64_t rows, int64_t cols,
                 at::ScalarType dtype) {
  check_pool("state", state, rows, cols, dtype);
  if (new_state) {
    check_pool("new_state", *new_state, rows, cols, dtype);
    TORCH_CHECK_VALUE(new_state->sizes() == state.sizes() && (state.size(0) <= 1 || new_state->stride(0) == state.stride(0)),
                      "new_state must have state's shape and strides");
  }
  TORCH_CHECK_VALUE(slots || state.size(0) >= R, "a pool of ", state.size(0), " states does not hold the ", R, " rows");
  TORCH_CHECK_VALUE(!R || state.size(0), "the pool is empty");
}
int64_t slot_stride(const Tensor& state) { return state.size(0) > 1 ? state.stride(0) : state.size(1) * state.size(2); }
// Written behind autograd's back: a graph that saved the pool has to notice.
void written(const Tensor& t) {
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

// ---- short causal convolution ------------------------------------------------------------------
struct ConvOperands {
  Tensor x, weight, bias, initial, lengths;
  ConvOperands(const Tensor& x_, const Tensor& weight_, const OptTensor& bias_, const OptTensor& initial_, const OptTensor& lengths_)
      : x(unit_rows(x_)), weight(table(weight_)), bias(table(bias_)), initial(initial_ ? initial_->contiguous() : Tensor()),
        lengths(index_table(lengths_)) {}
  void fill(dwarf_causal_conv_fwd_args& a, bool silu) const {
    a.B = size32(x.size(0));
    a.N = size32(x.size(1));
    a.D = size32(x.size(2));
    a.W = size32(weight.size(1));
    a.dtype = dtype_of(x, "x");
    a.silu = silu;
    a.x = x.const_data_ptr();
    a.x_stride[0] = x.stride(0);
    a.x_stride[1] = x.stride(1);
    a.weight = f32_ptr(weight);
    a.bias = f32_ptr(bias);
    a.lengths = i32_ptr(lengths);
    a.initial = initial.defined() ? initial.const_data_ptr() : nullptr;
  }
};

std::tuple<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& initial,
                                        const OptTensor& lengths, bool silu, bool want_state) {
  const ConvOperands in(x, weight, bias, initial, lengths);
  dwarf_causal_conv_fwd_args a{};
  in.fill(a, silu);
  const Tensor y = at::empty(x.sizes(), x.options());
  const Tensor state = want_state ? at::empty({a.B, a.W - 1, a.D}, x.options()) : Tensor();
  a.y = y.data_ptr();
  a.y_stride[0] = static_cast<int64_t>(a.N) * a.D;
  a.y_stride[1] = a.D;
  // where W is 1 there are no rows to keep
  if (want_state && state.numel()) a.final = state.data_ptr();
  launch(dwarf_causal_conv_fwd, a, x, "dwarf_causal_conv_fwd");
  return {y, state};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> conv_backward(const Tensor& dy_, const OptTensor& dstate, const Tensor& x,
                                                         const Tensor& weight, const OptTensor& bias, const OptTensor& initial,
                                                         const OptTensor& lengths, bool silu, bool need_w, bool need_b,
                                                         bool need_initial) {
  const ConvOperands in(x, weight, bias, initial, lengths);
  const Tensor dy = unit_rows(dy_.to(x.scalar_type()));
  const Tensor df = dstate && dstate->numel() ? dstate->to(x.scalar_type()).contiguous() : Tensor();
  dwarf_causal_conv_bwd_args a{};
  in.fill(a.fwd, silu);
  const int64_t B = a.fwd.B, D = a.fwd.D, W = a.fwd.W;
  a.dy = dy.const_data_ptr();
  a.dy_stride[0] = dy.stride(0);
  a.dy_stride[1] = dy.stride(1);
  a.dfinal = df.defined() ? df.const_data_ptr() : nullptr;
  const Tensor dx = at::empty(x.sizes(), x.options());
  a.dx = dx.data_ptr();
  a.dx_stride[0] = a.fwd.N * D;
  a.dx_stride[1] = D;
  const Tensor dw = need_w ? empty_f32({D, W}, x) : Tensor(), db = need_b ? empty_f32({D}, x) : Tensor();
  const Tensor di = need_initial ? at::empty({B, W - 1, D}, x.options()) : Tensor();
  a.dweight = f32_out(dw);
  a.dbias = f32_out(db);
  if (need_initial && di.numel()) a.dinitial = di.data_ptr();
  a.workspace_bytes = dwarf_causal_conv_bwd_workspace_bytes(&a);
  const Tensor ws = workspace(a.workspace_bytes, x);
  if (ws.defined()) a.workspace = ws.data_ptr();
  launch(dwarf_causal_conv_bwd, a, x, "dwarf_causal_conv_bwd");
  return {dx, dw, db, di};
}

struct CausalConvFn : torch::autograd::Function<CausalConvFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                               const OptTensor& initial, const OptTensor& lengths, bool silu, bool want_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    auto [y, state] = conv_forward(x, weight, bias, initial, lengths, silu, want_state);
    ctx->save_for_backward({x, weight, bias.value_or(Tensor()), initial.value_or(Tensor()), lengths.value_or(Tensor())});
    ctx->saved_data["silu"] = silu;
    return want_state ? variable_list{y, state} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    variable_list out(7);
    Tensor dy = grads[0];
    const Tensor dstate = grads.size() > 1 ? grads[1] : Tensor();
    if (!dy.defined() && !dstate.defined()) return out;
    {
      const at::NoGradGuard no_grad;
      refuse_tangents("causal_conv", dy, dstate, s[0], s[1], s[2], s[3]);
      if (!dy.defined()) dy = at::zeros_like(s[0]);
      const bool silu = ctx->saved_data["silu"].toBool();
      Needs needs{ctx};
      const bool need_x = needs.next(true), need_w = needs.next(true), need_b = needs.next(s[2].defined()),
                 need_i = needs.next(s[3].defined());
      Tensor dx, dw, db, di;
      if (watched(dy, dstate, s[0], s[1], s[2], s[3], s[4])) {
        const auto r = dispatched("dwarf::causal_conv_bwd", dy, optional(dstate), s[0], s[1], optional(s[2]), optional(s[3]),
                                  optional(s[4]), silu, need_w, need_b, need_i);
        dx = r[0], dw = r[1], db = r[2], di = r[3];
      } else {
        std::tie(dx, dw, db, di) = conv_backward(dy, optional(dstate), s[0], s[1], optional(s[2]), optional(s[3]), optional(s[4]),
                                                 silu, need_w, need_b, need_i);
      }
      if (need_x) out[0] = dx;
      if (need_w) out[1] = dw.to(s[1].scalar_type());
      if (need_b) out[2] = db.to(s[2].scalar_type());
      if (need_i) out[3] = di;
    }
    return first_order(std::move(out), "causal_conv");
  }
};

void check_taps(const Tensor& weight, const OptTensor& bias, int64_t D) {
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) == D && weight.size(1) >= 1 && weight.is_floating_point(), "weight must be [",
                    D, ",W] floating point, got ", weight.sizes(), " ", weight.scalar_type());
  TORCH_CHECK(weight.size(1) <= 8, "the convolution is built for W up to 8, got ", weight.size(1));
  check_channels("bias", bias, D);
}

void check_conv(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& initial, const OptTensor& lengths) {
  TORCH_CHECK_VALUE(x.dim() == 3 && x.size(2) >= 1, "x must be [B,N,D], got ", x.sizes());
  dtype_of(x, "x");
  check_taps(weight, bias, x.size(2));
  if (initial)
    TORCH_CHECK_VALUE(initial->sizes() == at::IntArrayRef({x.size(0), weight.size(1) - 1, x.size(2)}) &&
                          initial->scalar_type() == x.scalar_type(),
                      "initial_state must be ", x.scalar_type(), " [", x.size(0), ",", weight.size(1) - 1, ",", x.size(2), "], got ",
                      initial->sizes(), " ", initial->scalar_type());
  check_lengths(lengths, x.size(0));
  check_cuda(x);
  check_beside("weight", weight, x);
  check_beside("bias", bias, x);
  check_beside("initial_state", initial, x);
  check_beside("lengths", lengths, x);
}

// None: the call goes through the custom ops (see kWatched).
py::object causal_conv(const Tensor& x, const Tensor& weight, const OptTensor& bias, bool silu, const OptTensor& initial,
                       const OptTensor& lengths, bool return_state) {
  refuse_tangents("causal_conv", x, weight, bias, initial);
  if (watched(x, weight, bias, initial, lengths)) return py::none();
  check_conv(x, weight, bias, initial, lengths);
  Tensor y, state;
  {
    const py::gil_scoped_release release;
    if (any_grad(x, weight, bias, initial)) {
      const variable_list r = CausalConvFn::apply(x, weight, bias, initial, lengths, silu, return_state);
      y = r[0];
      if (return_state) state = r[1];
    } else {
      std::tie(y, state) = conv_forward(x, weight, bias, initial, lengths, silu, return_state);
    }
  }
  return return_state ? py::object(py::make_tuple(y, state)) : py::cast(y);
}

Tensor conv_step(const Tensor& x_, const Tensor& weight_, const OptTensor& bias_, const Tensor& state, const OptTensor& new_state,
                 const OptTensor& slots_, bool silu) {
  const Tensor x = unit_rows(x_), weight = table(weight_), bias = table(bias_), slots = index_table(slots_);
  const Tensor out = at::empty(x.sizes(), x.options());
  dwarf_causal_conv_step_args a{};
  a.R = size32(x.size(0));
  a.D = size32(x.size(1));
  a.W = size32(weight.size(1));
  a.pool = size32(state.size(0));
  a.dtype = dtype_of(x, "x");
  a.silu = silu;
  a.x = x.const_data_ptr();
  a.x_stride = x.stride(0);
  a.weight = f32_ptr(weight);
  a.bias = f32_ptr(bias);
  a.slots = i32_ptr(slots);
  a.state = state.const_data_ptr();
  a.new_state = (new_state ? *new_state : state).data_ptr();
  a.slot_stride = slot_stride(state);
  a.out = out.data_ptr();
  a.out_stride = a.D;
  launch(dwarf_causal_conv_step, a, x, "dwarf_causal_conv_step");
  written(new_state ? *new_state : state);
  return out;
}

void check_conv_step(const Tensor& x, const Tensor& weight, const OptTensor& bias, const Tensor& state, const OptTensor& new_state,
                     const OptTensor& slots) {
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) >= 1, "x must be [rows,D], got ", x.sizes());
  dtype_of(x, "x");
  check_taps(weight, bias, x.size(1));
  check_slots(slots, x.size(0));
  check_pools(state, new_state, slots, x.size(0), weight.size(1) - 1, x.size(1), x.scalar_type());
  check_cuda(x);
  check_beside("weight", weight, x);
  check_beside("bias", bias, x);
  check_beside("state", state, x);
  check_beside("new_state", new_state, x);
  check_beside("slots", slots, x);
  check_apart("x", x, new_state ? *new_state : state);
}

// Nothing: the call goes through the custom ops (see kWatched).
OptTensor causal_conv_step(const Tensor& x, const Tensor& weight, const OptTensor& bias, const Tensor& state, bool silu,
                           const OptTensor& slots, const OptTensor& new_state) {
  refuse_tangents("causal_conv_step", x, weight, bias, state, new_state);
  if (watched(x, weight, bias, state, slots, new_state)) return std::nullopt;
  check_conv_step(x, weight, bias, state, new_state, slots);
  TORCH_CHECK(!any_grad(x, weight, bias, state, new_state),
              "causal_conv_step has no gradients: call it under torch.no_grad(), or causal_conv");
  return conv_step(x, weight, bias, state, new_state, slots, silu);
}

// ---- selective scan ----------------------------------------------------------------------------
// B or C [..., G, S]; without groups, [..., S] is one.
Tensor grouped(const Tensor& t, const Tensor& x) { return t.dim() == x.dim() ? t.unsqueeze(-2) : t; }

// Rows of a sequence as the scan takes them: elements side by side, tokens less than 2^22 elements apart; others copied.
Tensor scan_rows(const Tensor& t) {
  const Tensor u = unit_rows(t);
  return u.size(1) > 1 && u.stride(1) >= (int64_t(1) << 22) ? u.clone(at::MemoryFormat::Contiguous) : u;
}
int64_t step_along(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

struct ScanOperands {
  Tensor x, delta, gate, B, C, A, skip, bias, initial, lengths;
  ScanOperands(const Tensor& x_, const Tensor& delta_, const Tensor& A_, const Tensor& B_, const Tensor& C_, const OptTensor& skip_,
               const OptTensor& gate_, const OptTensor& bias_, const OptTensor& initial_, const OptTensor& lengths_)
      : x(scan_rows(x_)), delta(scan_rows(delta_)), gate(gate_ ? scan_rows(*gate_) : Tensor()), B(scan_rows(grouped(B_, x_))),
        C(scan_rows(grouped(C_, x_))), A(table(A_)), skip(table(skip_)), bias(table(bias_)),
        initial(initial_ ? initial_->contiguous() : Tensor()), lengths(index_table(lengths_)) {}
  void fill(dwarf_selective_scan_fwd_args& a, bool softplus) const {
    a.B = size32(x.size(0));
    a.N = size32(x.size(1));
    a.D = size32(x.size(2));
    a.G = size32(B.size(2));
    a.S = size32(B.size(3));
    a.dtype = dtype_of(x, "x");
    a.softplus = softplus;
    a.x = x.const_data_ptr();
    a.x_stride[0] = step_along(x, 0), a.x_stride[1] = step_along(x, 1);
    a.delta = delta.const_data_ptr();
    a.delta_stride[0] = step_along(delta, 0), a.delta_stride[1] = step_along(delta, 1);
    if (gate.defined()) {
      a.gate = gate.const_data_ptr();
      a.gate_stride[0] = step_along(gate, 0), a.gate_stride[1] = step_along(gate, 1);
    }
    a.Bm = B.const_data_ptr();
    a.Cm = C.const_data_ptr();
    for (int i = 0; i < 3; ++i) a.B_stride[i] = step_along(B, i), a.C_stride[i] = step_along(C, i);
    a.A = f32_ptr(A);
    a.skip = f32_ptr(skip);
    a.delta_bias = f32_ptr(bias);
    a.lengths = i32_ptr(lengths);
    a.initial = f32_ptr(initial);
  }
};

// (y, the final state or undefined, the backward's checkpoints or undefined)
std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B,
                                                const Tensor& C, const OptTensor& skip, const OptTensor& gate, const OptTensor& bias,
                                                const OptTensor& initial, const OptTensor& lengths, bool softplus, bool want_state,
                                                bool want_checkpoints) {
  const ScanOperands in(x, delta, A, B, C, skip, gate, bias, initial, lengths);
  dwarf_selective_scan_fwd_args a{};
  in.fill(a, softplus);
  const Tensor y = at::empty(x.sizes(), x.options());
  const Tensor state = want_state ? empty_f32({a.B, a.D, a.S}, x) : Tensor();
  Tensor checkpoints;
  if (want_checkpoints) {
    a.checkpoint_bytes = dwarf_selective_scan_checkpoint_bytes(&a);
    checkpoints = empty_f32({static_cast<int64_t>(a.checkpoint_bytes / sizeof(float))}, x);
    if (a.checkpoint_bytes) a.checkpoints = f32_out(checkpoints);
  }
  a.y = y.data_ptr();
  a.y_stride[0] = static_cast<int64_t>(a.N) * a.D, a.y_stride[1] = a.D;
  a.final = f32_out(state);
  a.workspace_bytes = dwarf_selective_scan_fwd_workspace_bytes(&a);
  const Tensor ws = workspace(a.workspace_bytes, x);
  if (ws.defined()) a.workspace = ws.data_ptr();
  launch(dwarf_selective_scan_fwd, a, x, "dwarf_selective_scan_fwd");
  return {y, state, checkpoints};
}

struct ScanGrads {
  Tensor dx, ddelta, dA, dB, dC, dskip, dgate, dbias, dinitial;   // undefined where not needed
};

ScanGrads scan_backward(const Tensor& dy_, const OptTensor& dstate, const Tensor& x, const Tensor& delta, const Tensor& A,
                        const Tensor& B, const Tensor& C, const OptTensor& skip, const OptTensor& gate, const OptTensor& bias,
                        const OptTensor& initial, const OptTensor& lengths, const Tensor& checkpoints, bool softplus, bool need_A,
                        bool need_skip, bool need_bias, bool need_initial) {
  const ScanOperands in(x, delta, A, B, C, skip, gate, bias, initial, lengths);
  const Tensor dy = scan_rows(dy_.to(x.scalar_type()));
  const Tensor df = dstate ? dstate->to(at::kFloat).contiguous() : Tensor();
  dwarf_selective_scan_bwd_args a{};
  in.fill(a.fwd, softplus);
  const int64_t N = a.fwd.N, D = a.fwd.D, S = a.fwd.S;
  a.fwd.checkpoints = const_cast<float*>(checkpoints.const_data_ptr<float>());
  a.fwd.checkpoint_bytes = static_cast<size_t>(checkpoints.numel()) * sizeof(float);
  a.dy = dy.const_data_ptr();
  a.dy_stride[0] = step_along(dy, 0), a.dy_stride[1] = step_along(dy, 1);
  a.dfinal = f32_ptr(df);
  ScanGrads g;
  g.dx = at::empty(x.sizes(), x.options());
  g.ddelta = at::empty(x.sizes(), x.options());
  g.dB = at::empty(B.sizes(), x.options());
  g.dC = at::empty(C.sizes(), x.options());
  a.dx = g.dx.data_ptr();
  a.ddelta = g.ddelta.data_ptr();
  a.dx_stride[0] = a.ddelta_stride[0] = a.dgate_stride[0] = N * D;
  a.dx_stride[1] = a.ddelta_stride[1] = a.dgate_stride[1] = D;
  if (gate) {
    g.dgate = at::empty(x.sizes(), x.options());
    a.dgate = g.dgate.data_ptr();
  }
  a.dB = g.dB.data_ptr();
  a.dC = g.dC.data_ptr();
  if (need_A) g.dA = empty_f32({D, S}, x);
  if (need_skip) g.dskip = empty_f32({D}, x);
  if (need_bias) g.dbias = empty_f32({D}, x);
  if (need_initial) g.dinitial = empty_f32({a.fwd.B, D, S}, x);
  a.dA = f32_out(g.dA);
  a.dskip = f32_out(g.dskip);
  a.ddelta_bias = f32_out(g.dbias);
  a.dinitial = f32_out(g.dinitial);
  a.workspace_bytes = dwarf_selective_scan_bwd_workspace_bytes(&a);
  const Tensor ws = workspace(a.workspace_bytes, x);
  if (ws.defined()) a.workspace = ws.data_ptr();
  launch(dwarf_selective_scan_bwd, a, x, "dwarf_selective_scan_bwd");
  return g;
}

struct SelectiveScanFn : torch::autograd::Function<SelectiveScanFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B,
                               const Tensor& C, const OptTensor& skip, const OptTensor& gate, const OptTensor& bias,
                               const OptTensor& initial, const OptTensor& lengths, bool softplus, bool want_state) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    auto [y, state, checkpoints] = scan_forward(x, delta, A, B, C, skip, gate, bias, initial, lengths, softplus, want_state, true);
    ctx->save_for_backward({x, delta, A, B, C, skip.value_or(Tensor()), gate.value_or(Tensor()), bias.value_or(Tensor()),
                            initial.value_or(Tensor()), lengths.value_or(Tensor()), checkpoints});
    ctx->saved_data["softplus"] = softplus;
    return want_state ? variable_list{y, state} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    variable_list out(12);
    Tensor dy = grads[0];
    const Tensor dstate = grads.size() > 1 ? grads[1] : Tensor();
    if (!dy.defined() && !dstate.defined()) return out;
    {
      const at::NoGradGuard no_grad;
      refuse_tangents("selective_scan", dy, dstate, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8]);
      if (!dy.defined()) dy = at::zeros_like(s[0]);
      const bool softplus = ctx->saved_data["softplus"].toBool();
      Needs needs{ctx};
      bool need[9];
      for (int i = 0; i < 9; ++i) need[i] = needs.next(s[i].defined());
      ScanGrads g;
      if (watched(dy, dstate, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], s[10])) {
        const auto r = dispatched("dwarf::selective_scan_bwd", dy, optional(dstate), s[0], s[1], s[2], s[3], s[4], optional(s[5]),
                                  optional(s[6]), optional(s[7]), optional(s[8]), optional(s[9]), s[10], softplus, need[2], need[5],
                                  need[7], need[8]);
        g = ScanGrads{r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7], r[8]};
      } else {
        g = scan_backward(dy, optional(dstate), s[0], s[1], s[2], s[3], s[4], optional(s[5]), optional(s[6]), optional(s[7]),
                          optional(s[8]), optional(s[9]), s[10], softplus, need[2], need[5], need[7], need[8]);
      }
      if (need[0]) out[0] = g.dx;
      if (need[1]) out[1] = g.ddelta;
      if (need[2]) out[2] = g.dA.to(s[2].scalar_type());
      if (need[3]) out[3] = g.dB;
      if (need[4]) out[4] = g.dC;
      if (need[5]) out[5] = g.dskip.to(s[5].scalar_type());
      if (need[6]) out[6] = g.dgate;
      if (need[7]) out[7] = g.dbias.to(s[7].scalar_type());
      if (need[8]) out[8] = g.dinitial;
    }
    return first_order(std::move(out), "selective_scan");
  }
};

// The checks that sequences and steps share; dims: what x is.
void check_scan_inputs(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& skip,
                       const OptTensor& gate, const OptTensor& bias, const char* dims) {
  const int64_t D = x.size(-1);
  dtype_of(x, "x");
  check_like("delta", delta, x);
  check_like("gate", gate, x);
  TORCH_CHECK_VALUE(A.dim() == 2 && A.size(0) == D && A.size(1) >= 1 && A.is_floating_point(), "A must be [", D,
                    ",S] floating point, got ", A.sizes(), " ", A.scalar_type());
  const int64_t S = A.size(1), lead = x.dim() - 1;
  for (const auto& [name, t] : {std::make_pair("B", &B), std::make_pair("C", &C)}) {
    const bool ok = (t->dim() == lead + 1 || t->dim() == lead + 2) && t->sizes().slice(0, lead) == x.sizes().slice(0, lead) &&
                    t->size(-1) == S && t->scalar_type() == x.scalar_type();
    TORCH_CHECK_VALUE(ok, name, " must be ", x.scalar_type(), " [", dims, ",G,", S, "] or [", dims, ",", S, "] for x ", x.sizes(),
                      ", got ", t->sizes(), " ", t->scalar_type());
  }
  TORCH_CHECK_VALUE(B.sizes() == C.sizes(), "B and C must share a shape, got ", B.sizes(), " and ", C.sizes());
  const int64_t G = B.dim() == lead + 2 ? B.size(-2) : 1;
  TORCH_CHECK_VALUE(G >= 1 && D % G == 0, "D=", D, " channels must be divisible by G=", G, " groups");
  TORCH_CHECK(S <= 64, "the scan is built for up to 64 states, got ", S);
  check_channels("skip", skip, D);
  check_channels("delta_bias", bias, D);
}
void check_scan_devices(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& skip,
                        const OptTensor& gate, const OptTensor& bias) {
  check_cuda(x);
  check_beside("delta", delta, x);
  check_beside("A", A, x);
  check_beside("B", B, x);
  check_beside("C", C, x);
  check_beside("skip", skip, x);
  check_beside("gate", gate, x);
  check_beside("delta_bias", bias, x);
}

void check_scan(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& skip,
                const OptTensor& gate, const OptTensor& bias, const OptTensor& initial, const OptTensor& lengths) {
  TORCH_CHECK_VALUE(x.dim() == 3 && x.size(2) >= 1, "x must be [B,N,D], got ", x.sizes());
  check_scan_inputs(x, delta, A, B, C, skip, gate, bias, "B,N");
  if (initial)
    TORCH_CHECK_VALUE(initial->sizes() == at::IntArrayRef({x.size(0), x.size(2), A.size(1)}) && initial->scalar_type() == at::kFloat,
                      "initial_state must be fp32 [", x.size(0), ",", x.size(2), ",", A.size(1), "], got ", initial->sizes(), " ",
                      initial->scalar_type());
  check_lengths(lengths, x.size(0));
  check_scan_devices(x, delta, A, B, C, skip, gate, bias);
  check_beside("initial_state", initial, x);
  check_beside("lengths", lengths, x);
}

// None: the call goes through the custom ops (see kWatched).
py::object selective_scan(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                          const OptTensor& skip, const OptTensor& gate, const OptTensor& bias, bool softplus,
                          const OptTensor& initial, const OptTensor& lengths, bool return_state) {
  refuse_tangents("selective_scan", x, delta, A, B, C, skip, gate, bias, initial);
  if (watched(x, delta, A, B, C, skip, gate, bias, initial, lengths)) return py::none();
  check_scan(x, delta, A, B, C, skip, gate, bias, initial, lengths);
  Tensor y, state;
  {
    const py::gil_scoped_release release;
    if (any_grad(x, delta, A, B, C, skip, gate, bias, initial)) {
      const variable_list r = SelectiveScanFn::apply(x, delta, A, B, C, skip, gate, bias, initial, lengths, softplus, return_state);
      y = r[0];
      if (return_state) state = r[1];
    } else {
      Tensor checkpoints;
      std::tie(y, state, checkpoints) =
          scan_forward(x, delta, A, B, C, skip, gate, bias, initial, lengths, softplus, return_state, false);
    }
  }
  return return_state ? py::object(py::make_tuple(y, state)) : py::cast(y);
}

Tensor scan_step(const Tensor& x_, const Tensor& delta_, const Tensor& A_, const Tensor& B_, const Tensor& C_, const Tensor& state,
                 const OptTensor& new_state, const OptTensor& skip_, const OptTensor& gate_, const OptTensor& bias_,
                 const OptTensor& slots_, bool softplus) {
  const Tensor x = unit_rows(x_), delta = unit_rows(delta_), B = unit_rows(grouped(B_, x_)), C = unit_rows(grouped(C_, x_));
  const Tensor gate = gate_ ? unit_rows(*gate_) : Tensor(), A = table(A_), skip = table(skip_), bias = table(bias_);
  const Tensor slots = index_table(slots_), out = at::empty(x.sizes(), x.options());
  dwarf_selective_scan_step_args a{};
  a.R = size32(x.size(0));
  a.D = size32(x.size(1));
  a.G = size32(B.size(1));
  a.S = size32(B.size(2));
  a.pool = size32(state.size(0));
  a.dtype = dtype_of(x, "x");
  a.softplus = softplus;
  a.x = x.const_data_ptr();
  a.x_stride = x.stride(0);
  a.delta = delta.const_data_ptr();
  a.delta_stride = delta.stride(0);
  if (gate.defined()) {
    a.gate = gate.const_data_ptr();
    a.gate_stride = gate.stride(0);
  }
  a.Bm = B.const_data_ptr();
  a.Cm = C.const_data_ptr();
  for (int i = 0; i < 2; ++i) a.B_stride[i] = B.stride(i), a.C_stride[i] = C.stride(i);
  a.A = f32_ptr(A);
  a.skip = f32_ptr(skip);
  a.delta_bias = f32_ptr(bias);
  a.slots = i32_ptr(slots);
  a.state = state.const_data_ptr<float>();
  a.new_state = (new_state ? *new_state : state).data_ptr<float>();
  a.slot_stride = slot_stride(state);
  a.out = out.data_ptr();
  a.out_stride = a.D;
  launch(dwarf_selective_scan_step, a, x, "dwarf_selective_scan_step");
  written(new_state ? *new_state : state);
  return out;
}

void check_scan_step(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& state,
                     const OptTensor& new_state, const OptTensor& skip, const OptTensor& gate, const OptTensor& bias,
                     const OptTensor& slots) {
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) >= 1, "x must be [rows,D], got ", x.sizes());
  check_scan_inputs(x, delta, A, B, C, skip, gate, bias, "rows");
  check_slots(slots, x.size(0));
  check_pools(state, new_state, slots, x.size(0), x.size(1), A.size(1), at::kFloat);
  check_scan_devices(x, delta, A, B, C, skip, gate, bias);
  check_beside("state", state, x);
  check_beside("new_state", new_state, x);
  check_beside("slots", slots, x);
  const Tensor& pool = new_state ? *new_state : state;
  check_apart("x", x, pool);
  check_apart("delta", delta, pool);
  check_apart("gate", gate, pool);
  check_apart("B", B, pool);
  check_apart("C", C, pool);
}

// Nothing: the call goes through the custom ops (see kWatched).
OptTensor selective_scan_step(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                              const Tensor& state, const OptTensor& skip, const OptTensor& gate, const OptTensor& bias, bool softplus,
                              const OptTensor& slots, const OptTensor& new_state) {
  refuse_tangents("selective_scan_step", x, delta, A, B, C, state, skip, gate, bias, new_state);
  if (watched(x, delta, A, B, C, state, skip, gate, bias, slots, new_state)) return std::nullopt;
  check_scan_step(x, delta, A, B, C, state, new_state, skip, gate, bias, slots);
  TORCH_CHECK(!any_grad(x, delta, A, B, C, state, skip, gate, bias, new_state),
              "selective_scan_step has no gradients: call it under torch.no_grad(), or selective_scan");
  return scan_step(x, delta, A, B, C, state, new_state, skip, gate, bias, slots, softplus);
}

}  // namespace

void dwarf_torch::register_selective(py::module_& m) {
  const auto no_gil = py::call_guard<py::gil_scoped_release>();
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_fp8", &rms_norm_fp8);
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step, no_gil);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step, no_gil);
  // the custom ops' launches: the same, checked here
  m.def("rms_forward", [](const Tensor& x, const OptTensor& weight, const OptTensor& residual, int64_t groups, double eps, bool eights) {
    refuse_tangents("rms_norm", x, weight, residual);
    check_rms_launch(x, weight, residual, groups, eps);
    const RmsResult r = rms_forward(x, weight, residual, groups, eps, eights);
    return std::make_tuple(r.y, optional(r.sum), optional(r.scale));
  }, no_gil);
  m.def("rms_backward", [](const Tensor& dy, const OptTensor& dsum, const Tensor& stream, const OptTensor& weight, int64_t groups,
                           double eps, bool need_dx, bool need_dr, bool need_dw) {
    refuse_tangents("rms_norm", dy, dsum, stream, weight);
    TORCH_CHECK_VALUE(dy.sizes() == stream.sizes(), "dy must have the rows' shape ", stream.sizes(), ", got ", dy.sizes());
    TORCH_CHECK_VALUE(!dsum || dsum->sizes() == stream.sizes(), "dsum must have the rows' shape ", stream.sizes());
    TORCH_CHECK_VALUE(stream.scalar_type() == dy.scalar_type() || stream.scalar_type() == at::kFloat, "the rows must have dy's dtype ",
                      dy.scalar_type(), " or fp32, got ", stream.scalar_type());
    check_rms_launch(stream, weight, std::nullopt, groups, eps);
    dtype_of(dy, "dy");
    check_beside("dy", dy, stream);
    check_beside("dsum", dsum, stream);
    const auto [dx, dr, dw] = rms_backward(dy, dsum, stream, weight, groups, eps, need_dx, need_dr, need_dw);
    return std::make_tuple(optional(dx), optional(dr), optional(dw));
  }, no_gil);
  m.def("conv_forward", [](const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& initial,
                           const OptTensor& lengths, bool silu, bool want_state) {
    refuse_tangents("causal_conv", x, weight, bias, initial);
    check_conv(x, weight, bias, initial, lengths);
    const auto [y, state] = conv_forward(x, weight, bias, initial, lengths, silu, want_state);
    return std::make_tuple(y, optional(state));
  }, no_gil);
  m.def("conv_backward", [](const Tensor& dy, const OptTensor& dstate, const Tensor& x, const Tensor& weight, const OptTensor& bias,
                            const OptTensor& initial, const OptTensor& lengths, bool silu, bool need_w, bool need_b, bool need_initial) {
    refuse_tangents("causal_conv", dy, dstate, x, weight, bias, initial);
    check_conv(x, weight, bias, initial, lengths);
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "dy must have x's shape ", x.sizes(), ", got ", dy.sizes());
    TORCH_CHECK_VALUE(!dstate || dstate->sizes() == at::IntArrayRef({x.size(0), weight.size(1) - 1, x.size(2)}),
                      "dstate must have the state's shape");
    check_beside("dy", dy, x);
    check_beside("dstate", dstate, x);
    const auto [dx, dw, db, di] = conv_backward(dy, dstate, x, weight, bias, initial, lengths, silu, need_w, need_b, need_initial);
    return std::make_tuple(dx, optional(dw), optional(db), optional(di));
  }, no_gil);
  m.def("conv_step", [](const Tensor& x, const Tensor& weight, const OptTensor& bias, const Tensor& state, const OptTensor& new_state,
                        const OptTensor& slots, bool silu) {
    refuse_tangents("causal_conv_step", x, weight, bias, state, new_state);
    check_conv_step(x, weight, bias, state, new_state, slots);
    return conv_step(x, weight, bias, state, new_state, slots, silu);
  }, no_gil);
  m.def("scan_forward", [](const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                           const OptTensor& skip, const OptTensor& gate, const OptTensor& bias, const OptTensor& initial,
                           const OptTensor& lengths, bool softplus, bool want_state, bool want_checkpoints) {
    refuse_tangents("selective_scan", x, delta, A, B, C, skip, gate, bias, initial);
    check_scan(x, delta, A, B, C, skip, gate, bias, initial, lengths);
    const auto [y, state, checkpoints] =
        scan_forward(x, delta, A, B, C, skip, gate, bias, initial, lengths, softplus, want_state, want_checkpoints);
    return std::make_tuple(y, optional(state), optional(checkpoints));
  }, no_gil);
  m.def("scan_backward", [](const Tensor& dy, const OptTensor& dstate, const Tensor& x, const Tensor& delta, const Tensor& A,
                            const Tensor& B, const Tensor& C, const OptTensor& skip, const OptTensor& gate, const OptTensor& bias,
                            const OptTensor& initial, const OptTensor& lengths, const Tensor& checkpoints, bool softplus, bool need_A,
                            bool need_skip, bool need_bias, bool need_initial) {
    refuse_tangents("selective_scan", dy, dstate, x, delta, A, B, C, skip, gate, bias, initial);
    check_scan(x, delta, A, B, C, skip, gate, bias, initial, lengths);
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes(), "dy must have x's shape ", x.sizes(), ", got ", dy.sizes());
    TORCH_CHECK_VALUE(!dstate || dstate->sizes() == at::IntArrayRef({x.size(0), x.size(2), A.size(1)}),
                      "dstate must have the state's shape");
    TORCH_CHECK_VALUE(checkpoints.scalar_type() == at::kFloat && checkpoints.is_contiguous() && aligned(checkpoints, 16),
                      "checkpoints must be the forward's");
    check_beside("dy", dy, x);
    check_beside("dstate", dstate, x);
    check_beside("checkpoints", checkpoints, x);
    const ScanGrads g = scan_backward(dy, dstate, x, delta, A, B, C, skip, gate, bias, initial, lengths, checkpoints, softplus, need_A,
                                      need_skip, need_bias, need_initial);
    return std::make_tuple(g.dx, g.ddelta, optional(g.dA), g.dB, g.dC, optional(g.dskip), optional(g.dgate), optional(g.dbias),
                           optional(g.dinitial));
  }, no_gil);
  m.def("scan_step", [](const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& state,
                        const OptTensor& new_state, const OptTensor& skip, const OptTensor& gate, const OptTensor& bias,
                        const OptTensor& slots, bool softplus) {
    refuse_tangents("selective_scan_step", x, delta, A, B, C, state, skip, gate, bias, new_state);
    check_scan_step(x, delta, A, B, C, state, new_state, skip, gate, bias, slots);
    return scan_step(x, delta, A, B, C, state, new_state, skip, gate, bias, slots, softplus);
  }, no_gil);
}
