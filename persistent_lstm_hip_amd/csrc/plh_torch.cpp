// plh_torch.cpp -- the torch front end of the block operators (module plh_torch, behind persistent_lstm_hip_amd/ops.py).
//
// Checks the arguments, allocates the outputs, calls the C ABI on the device's current stream and is the operators'
// autograd node.  It is C++ because a call's host time bounds the small ones: through ctypes and a Python autograd
// function a layer norm of one row took 11 us, and a training step of a small one, whose kernels run for 25 us, 125 us.
// No kernel is in this file, and the library itself does not depend on torch.
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/persistent_lstm_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

// ---- arguments ----------------------------------------------------------------------------------

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return PLH_F16;
    case at::kBFloat16: return PLH_BF16;
    case at::kFloat: return PLH_F32;
    default: return -1;
  }
}

// A dual tensor of forward-mode differentiation need not have requires_grad: its tangent would be dropped.
void check_no_tangent(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(!t._fw_grad(/*level=*/0).defined(), name,
                    " carries a forward-mode tangent: the block operators have reverse-mode gradients only");
}

int check_tensor(const Tensor& t, const char* name, int64_t dims = -1) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be on a HIP device: this library has no CPU path");
  const int code = dtype_code(t.scalar_type());
  TORCH_CHECK_VALUE(code >= 0, name, " must be float16, bfloat16 or float32, not ", t.scalar_type());
  TORCH_CHECK_VALUE(dims < 0 || t.dim() == dims, name, " must have ", dims, " dimensions, not ", t.dim());
  check_no_tangent(t, name);
  return code;
}

void check_like(const Tensor& t, const char* name, at::IntArrayRef shape, at::Device device) {
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be a tensor of shape ", shape, ", not ", t.sizes());
  TORCH_CHECK_VALUE(t.device() == device, name, " must be on ", device);
  check_no_tangent(t, name);
}

void check(int rc, const char* what) {
  if (rc == PLH_OK) return;
  const std::string msg = std::string(what) + ": " + plh_last_error();
  TORCH_CHECK_VALUE(rc != PLH_ERR_INVALID && rc != PLH_ERR_UNSUPPORTED, msg);
  TORCH_CHECK(false, msg);
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}

Tensor given(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

bool tracks(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Without the way through the dispatcher (a call that returns 48 tensors 50 -> 40 us).
Tensor empty(at::IntArrayRef shape, at::ScalarType type, at::Device device) {
  return at::detail::empty_cuda(shape, type, device, std::nullopt);
}
Tensor empty_strided(at::IntArrayRef shape, at::IntArrayRef strides, at::ScalarType type, at::Device device) {
  return at::detail::empty_strided_cuda(shape, strides, type, device);
}

// t with its values in its storage (torch may hold a real tensor as the storage's negative, as the imaginary part of a
// conjugate) and contiguous.
Tensor values(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor dense(const Tensor& t) { return values(t).contiguous(); }

// A gradient as the kernels read it: of the output's type, contiguous.
Tensor incoming(const Tensor& grad, at::ScalarType type) {
  check_no_tangent(grad, "an incoming gradient");
  return dense(grad.to(type));
}

// In a node below, needs_input_grad counts the tensors that it was given (an optional that holds none is not counted).

// What the backward pass of the node that runs returns can be differentiated no further: asked for a second derivative it
// raises.  Gradients depend on the incoming ones and, where the node is not linear in its first input, on its first
// `inputs` inputs: with a loss that is linear in the output only those are tracked.  The raising node is linked to all of
// them, as a derivative's own would be: the engine leaves out what does not lead to the tensors that it is asked for.
// Where nothing is tracked the gradients are constants.
variable_list once_over(variable_list grads, const variable_list& incoming, uint32_t inputs, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::edge_list edges = torch::autograd::collect_next_edges(incoming);
  const auto node = torch::autograd::get_current_node();
  for (uint32_t i = 0; i < inputs; ++i) edges.push_back(node->next_edge(i));
  bool any = false;
  for (const auto& e : edges) any = any || e.is_valid();
  if (!any) return grads;
  const auto raises =
      std::make_shared<torch::autograd::Error>(std::string(what) + " is differentiable once only", std::move(edges));
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    g = g.detach();
    torch::autograd::create_gradient_edge(g, raises);
  }
  return grads;
}

// The same of a node that is linear in all but its first input.
variable_list once(variable_list grads, const variable_list& incoming, uint32_t inputs, const char* what) {
  const auto node = torch::autograd::get_current_node();
  return once_over(std::move(grads), incoming, inputs > 0 && node->next_edge(0).is_valid() ? inputs : 0, what);
}

// Refuses a state that a step may not overwrite.
void check_inplace(const Tensor& state, const char* name, bool inplace) {
  if (!inplace) return;
  TORCH_CHECK_VALUE(state.is_contiguous() && !state.is_neg(), name,
                    " must be contiguous (and no lazily negated view) to be updated in place");
  // (before the kernel runs: torch would raise for the version only after it)
  TORCH_CHECK_VALUE(!state.is_inference() || c10::InferenceMode::is_enabled(), name,
                    " is an inference tensor: it can be updated in place in inference mode only");
}

// ---- gated linear recurrence --------------------------------------------------------------------

int64_t hidden_of(const Tensor& gates, bool output_gate) {
  const int64_t width = gates.size(-1), parts = output_gate ? 3 : 2;
  TORCH_CHECK_VALUE(width > 0 && width % parts == 0, "gates needs ", parts, " * hidden columns (f, g",
                    output_gate ? ", o" : "", "), not ", width);
  const int64_t hidden = width / parts;  // (an int in the C ABI, which checks what fits one)
  TORCH_CHECK_VALUE(hidden <= 1 << 24, "hidden must not exceed 2^24, not ", hidden);
  return hidden;
}

// gates itself where its last dimension is dense (any other strides), else a copy.
Tensor dense_rows(const Tensor& gates) {
  return gates.stride(-1) == 1 || gates.size(-1) == 1 ? values(gates) : gates.contiguous();
}

// int32 on the device.  Host lengths are checked; lengths on the device are not (that would synchronise the stream):
// the kernels take them as if clamped to [0, seq_len].
Tensor device_lengths(const MaybeTensor& lengths, int64_t batch, int64_t seq_len, at::Device device) {
  if (!lengths.has_value()) return Tensor();
  Tensor n = *lengths;
  if (n.numel() == 0) n = n.to(at::kInt);  // (an empty list has no integer type)
  TORCH_CHECK_VALUE(n.dim() == 1 && n.numel() == batch && at::isIntegralType(n.scalar_type(), /*includeBool=*/false),
                    "lengths must be a 1-D integer tensor with one entry per batch row");
  if (n.device().is_cpu()) {
    hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
    TORCH_CHECK(hipStreamIsCapturing(c10::hip::getCurrentHIPStream(device.index()), &capturing) == hipSuccess,
                "the stream's capture status is not known");
    TORCH_CHECK_VALUE(capturing == hipStreamCaptureStatusNone, "lengths must be on ", device,
                      " while a graph is captured: its replays would copy them from host memory that is freed by then");
    n = n.to(at::kLong).contiguous();
    const int64_t* v = n.const_data_ptr<int64_t>();
    for (int64_t i = 0; i < batch; ++i)
      TORCH_CHECK_VALUE(v[i] >= 0 && v[i] <= seq_len, "lengths must lie in [0, ", seq_len, "]");
    return n.to(at::kInt).pin_memory().to(device, /*non_blocking=*/true);
  }
  TORCH_CHECK_VALUE(n.device() == device, "lengths must be on the host or on ", device);
  if (n.scalar_type() == at::kLong) n = n.clamp(0, seq_len);
  return n.to(at::kInt).contiguous();
}

Tensor scan_workspace(int64_t B, int64_t T, int64_t H, at::Device device) {
  const int64_t n = plh_gated_scan_workspace_bytes(B, T, (int)H);
  return n > 0 ? empty({n}, at::kByte, device) : Tensor();
}

struct ScanOut {
  Tensor out, c_n, states;
};

ScanOut scan_forward(const Tensor& gates, const Tensor& c0, const Tensor& lengths, bool output_gate, bool keep) {
  const int64_t B = gates.size(0), T = gates.size(1), H = gates.size(2) / (output_gate ? 3 : 2);
  const at::Device device = gates.device();
  ScanOut r{empty({B, T, H}, gates.scalar_type(), device), empty({B, H}, at::kFloat, device), Tensor()};
  if (keep) r.states = empty({plh_gated_scan_states(T), B, H}, at::kFloat, device);
  const Tensor ws = scan_workspace(B, T, H, device);
  check(plh_gated_scan_forward(dtype_code(gates.scalar_type()), output_gate, ptr(gates), gates.stride(0),
                               gates.stride(1), B, T, (int)H, ptr<int32_t>(lengths), ptr<float>(c0), ptr(r.out),
                               ptr<float>(r.c_n), ptr<float>(r.states), ptr(ws), ws.defined() ? ws.numel() : 0,
                               stream_of(gates)),
        "gated_scan");
  return r;
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& gates, const MaybeTensor& c0,
                               const MaybeTensor& lengths, bool output_gate) {
    const ScanOut r = scan_forward(gates, given(c0), given(lengths), output_gate, true);
    ctx->save_for_backward({gates, given(lengths), r.states});
    ctx->saved_data["output_gate"] = output_gate;
    ctx->saved_data["has_c0"] = c0.has_value();
    ctx->set_materialize_grads(false);
    return {r.out, r.c_n};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &gates = saved[0], &lengths = saved[1], &states = saved[2];
    const bool output_gate = ctx->saved_data["output_gate"].toBool();
    const int64_t B = gates.size(0), T = gates.size(1), H = states.size(2);
    const at::Device device = gates.device();
    const c10::DeviceGuard guard(device);
    const auto like_gates = at::TensorOptions().dtype(gates.scalar_type()).device(device);
    const Tensor d_out = grads[0].defined() ? incoming(grads[0], gates.scalar_type()) : at::zeros({B, T, H}, like_gates);
    const Tensor d_cn = grads[1].defined() ? incoming(grads[1], at::kFloat) : Tensor();
    Tensor d_gates = empty(gates.sizes(), gates.scalar_type(), device), d_c0;
    if (ctx->saved_data["has_c0"].toBool() && ctx->needs_input_grad(1)) d_c0 = empty({B, H}, at::kFloat, device);
    const Tensor ws = scan_workspace(B, T, H, device);
    check(plh_gated_scan_backward(dtype_code(gates.scalar_type()), output_gate, ptr(gates), gates.stride(0),
                                  gates.stride(1), B, T, (int)H, ptr<int32_t>(lengths), ptr<float>(states), ptr(d_out),
                                  ptr<float>(d_cn), ptr(d_gates), ptr<float>(d_c0), ptr(ws),
                                  ws.defined() ? ws.numel() : 0, stream_of(gates)),
          "gated_scan backward");
    // (linear in c0 alone)
    return once({d_gates, d_c0, Tensor(), Tensor()}, grads, ctx->saved_data["has_c0"].toBool() ? 2 : 1, "gated_scan");
  }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& gates_in, const MaybeTensor& c0_in, const MaybeTensor& lengths,
                                      bool output_gate) {
  check_tensor(gates_in, "gates", 3);
  const int64_t H = hidden_of(gates_in, output_gate), B = gates_in.size(0), T = gates_in.size(1);
  const at::Device device = gates_in.device();
  const c10::DeviceGuard guard(device);
  MaybeTensor c0;
  if (c0_in.has_value()) {
    check_tensor(*c0_in, "c0");
    check_like(*c0_in, "c0", {B, H}, device);
    c0 = dense(c0_in->to(at::kFloat));
  }
  const Tensor n = device_lengths(lengths, B, T, device), gates = dense_rows(gates_in);
  if (at::GradMode::is_enabled() && (tracks(gates) || tracks(given(c0)))) {
    const variable_list r = GatedScan::apply(gates, c0, maybe(n), output_gate);
    return {r[0], r[1]};
  }
  const ScanOut r = scan_forward(gates, given(c0), n, output_gate, false);
  return {r.out, r.c_n};
}

std::tuple<Tensor, Tensor> gated_scan_step(const Tensor& gates_in, const Tensor& c_in, bool output_gate, bool inplace) {
  const int code = check_tensor(gates_in, "gates", 2);
  const int64_t H = hidden_of(gates_in, output_gate), B = gates_in.size(0);
  const at::Device device = gates_in.device();
  check_like(c_in, "c", {B, H}, device);
  TORCH_CHECK_VALUE(c_in.scalar_type() == at::kFloat, "c must be float32, not ", c_in.scalar_type());
  check_inplace(c_in, "c", inplace);
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !(tracks(gates_in) || tracks(c_in)),
                    "gated_scan_step is not differentiable: call it under torch.no_grad(), or gated_scan");
  const c10::DeviceGuard guard(device);
  const Tensor c = dense(c_in), gates = dense_rows(gates_in);
  Tensor out = empty({B, H}, gates.scalar_type(), device), c_n = inplace ? c_in : empty({B, H}, at::kFloat, device);
  check(plh_gated_scan_forward(code, output_gate, ptr(gates), gates.stride(0), 0, B, 1, (int)H, nullptr, ptr<float>(c),
                               ptr(out), ptr<float>(c_n), nullptr, nullptr, 0, stream_of(gates)),
        "gated_scan_step");
  if (inplace) c_n.unsafeGetTensorImpl()->bump_version();
  return {out, c_n};
}

// ---- layer norm ---------------------------------------------------------------------------------

// x as [rows, cols] with dense rows: a view where one row stride serves, else a copy.
Tensor matrix(const Tensor& x) {
  const int64_t cols = x.size(-1);
  if (x.dim() == 2 && (x.stride(1) == 1 || cols == 1)) return x;
  const Tensor m = x.reshape({x.numel() / cols, cols});
  return m.stride(1) == 1 || cols == 1 ? m : m.contiguous();
}

struct NormOut {
  Tensor y, stats;
};

NormOut norm_forward(const Tensor& x, const Tensor& m, const Tensor& weight, const Tensor& bias, double eps, bool keep) {
  const int64_t rows = m.size(0), cols = m.size(1);
  NormOut r{empty(x.sizes(), x.scalar_type(), x.device()), Tensor()};
  if (keep) r.stats = empty({2, rows}, at::kFloat, x.device());
  const Tensor& w = weight.defined() ? weight : bias;
  const int code = dtype_code(x.scalar_type());
  float* const mean = ptr<float>(r.stats);
  check(plh_layer_norm_forward(code, w.defined() ? dtype_code(w.scalar_type()) : code, ptr(m), m.stride(0), rows, cols,
                               ptr(weight), ptr(bias), (float)eps, ptr(r.y), mean, mean ? mean + rows : nullptr,
                               stream_of(x)),
        "layer_norm");
  return r;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias,
                        double eps) {
    const Tensor m = matrix(x), w = given(weight), b = given(bias);
    const NormOut r = norm_forward(x, m, w, b, eps, true);
    ctx->save_for_backward({m, w, r.stats});
    const Tensor& p = w.defined() ? w : b;
    ctx->saved_data["wdtype"] = (int64_t)(p.defined() ? p.scalar_type() : x.scalar_type());
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["has"] = (int64_t)(w.defined() + 2 * b.defined());
    return r.y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &m = saved[0], &w = saved[1], &stats = saved[2];
    const int64_t rows = m.size(0), cols = m.size(1), has = ctx->saved_data["has"].toInt();
    const auto wtype = (at::ScalarType)ctx->saved_data["wdtype"].toInt();
    const at::Device device = m.device();
    const c10::DeviceGuard guard(device);
    const Tensor d_y = incoming(grads[0], m.scalar_type());
    Tensor d_x, d_w, d_b, ws;
    if (ctx->needs_input_grad(0)) d_x = empty(ctx->saved_data["shape"].toIntVector(), m.scalar_type(), device);
    if ((has & 1) && ctx->needs_input_grad(1)) d_w = empty({cols}, wtype, device);
    if ((has & 2) && ctx->needs_input_grad(has == 3 ? 2 : 1)) d_b = empty({cols}, wtype, device);
    if (d_w.defined() || d_b.defined()) ws = empty({plh_layer_norm_workspace_bytes(rows, cols)}, at::kByte, device);
    const float* const mean = ptr<float>(stats);
    check(plh_layer_norm_backward(dtype_code(m.scalar_type()), dtype_code(wtype), ptr(m), m.stride(0), rows, cols,
                                  ptr(w), mean, mean ? mean + rows : nullptr, ptr(d_y), ptr(d_x), ptr(d_w), ptr(d_b),
                                  ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(m)),
          "layer_norm backward");
    // (linear in weight and bias alone; no gradient depends on the bias)
    return once({d_x, d_w, d_b, Tensor()}, grads, has & 1 ? 2 : 1, "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x_in, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
  check_tensor(x_in, "x");
  const Tensor x = values(x_in);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "x needs a last dimension of at least one element");
  const auto param = [&](const MaybeTensor& t, const char* name) -> MaybeTensor {
    if (!t.has_value()) return t;
    check_like(*t, name, {x.size(-1)}, x.device());
    TORCH_CHECK_VALUE(t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat, name, " must be ",
                      x.scalar_type(), " or float32, not ", t->scalar_type());
    return dense(*t);
  };
  const MaybeTensor w = param(weight, "weight"), b = param(bias, "bias");
  TORCH_CHECK_VALUE(!w.has_value() || !b.has_value() || w->scalar_type() == b->scalar_type(),
                    "weight and bias must have the same type");
  TORCH_CHECK_VALUE(eps >= 0.0, "eps must be non-negative");
  const c10::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() && (tracks(x) || tracks(given(w)) || tracks(given(b))))
    return LayerNorm::apply(x, w, b, eps);
  return norm_forward(x, matrix(x), given(w), given(b), eps, false).y;
}

// ---- dropout ------------------------------------------------------------------------------------

struct Mask {
  int threshold;
  uint64_t seed, offset;
};

Tensor dropout(const Tensor& x, const Tensor& residual, const Mask& m, const Tensor& offset) {
  Tensor out = empty(x.sizes(), x.scalar_type(), x.device());
  check(plh_dropout_add(dtype_code(x.scalar_type()), ptr(x), ptr(residual), ptr(out), x.numel(), m.threshold, m.seed,
                        m.offset, ptr<int64_t>(offset), stream_of(x)),
        "dropout_add");
  return out;
}

struct DropoutAdd : torch::autograd::Function<DropoutAdd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual, int64_t threshold,
                        int64_t seed, int64_t offset, const MaybeTensor& offset_dev) {
    const Tensor off = offset_dev.has_value() ? offset_dev->clone() : Tensor();  // the gradient's mask is that of now
    ctx->save_for_backward({off});
    ctx->saved_data["mask"] = std::vector<int64_t>{threshold, seed, offset};
    ctx->saved_data["has_residual"] = residual.has_value();
    ctx->saved_data["dtype"] = (int64_t)x.scalar_type();
    return dropout(x, given(residual), Mask{(int)threshold, (uint64_t)seed, (uint64_t)offset}, off);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const std::vector<int64_t> m = ctx->saved_data["mask"].toIntVector();
    const variable_list saved = ctx->get_saved_variables();
    const c10::DeviceGuard guard(grads[0].device());
    const Tensor d_out = incoming(grads[0], (at::ScalarType)ctx->saved_data["dtype"].toInt());
    Tensor d_x, d_r;
    if (ctx->needs_input_grad(0))
      d_x = dropout(d_out, Tensor(), Mask{(int)m[0], (uint64_t)m[1], (uint64_t)m[2]}, saved[0]);
    if (ctx->saved_data["has_residual"].toBool() && ctx->needs_input_grad(1)) d_r = d_out;
    return once({d_x, d_r, Tensor(), Tensor(), Tensor(), Tensor()}, grads, 0, "dropout_add");  // (linear in both)
  }
};

Tensor dropout_add(const Tensor& x_in, const MaybeTensor& residual_in, double p, uint64_t seed, uint64_t offset,
                   const MaybeTensor& offset_dev) {
  check_tensor(x_in, "x");
  const at::Device device = x_in.device();
  if (residual_in.has_value()) {
    check_like(*residual_in, "residual", x_in.sizes(), device);
    TORCH_CHECK_VALUE(residual_in->scalar_type() == x_in.scalar_type(), "residual must be ", x_in.scalar_type(), ", not ",
                      residual_in->scalar_type());
  }
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must lie in [0, 1]");
  TORCH_CHECK_VALUE(!offset_dev.has_value() || (offset_dev->numel() == 1 && offset_dev->scalar_type() == at::kLong &&
                                                offset_dev->device() == device),
                    "a tensor offset must be one int64 on ", device);
  const c10::DeviceGuard guard(device);
  const Mask m{(int)std::floor(p * 65536.0 + 0.5), seed, offset};
  const Tensor x = dense(x_in);
  MaybeTensor residual;
  if (residual_in.has_value()) residual = dense(*residual_in);
  if (at::GradMode::is_enabled() && (tracks(x) || tracks(given(residual))))
    return DropoutAdd::apply(x, residual, (int64_t)m.threshold, (int64_t)seed, (int64_t)offset, offset_dev);
  return dropout(x, given(residual), m, given(offset_dev));
}

// ---- causal convolution -------------------------------------------------------------------------

// weight [channels, width], bias [channels] or null: their type, checked.
int check_filter(const Tensor& weight, const MaybeTensor& bias, int64_t channels, const Tensor& x) {
  check_tensor(weight, "weight", 2);
  TORCH_CHECK_VALUE(weight.size(0) == channels, "weight must be [channels, width] with ", channels, " channels, not ",
                    weight.sizes());
  TORCH_CHECK_VALUE(weight.size(1) >= 1 && weight.size(1) <= 8, "weight must have a width of 1 to 8, not ", weight.size(1));
  check_like(weight, "weight", weight.sizes(), x.device());
  TORCH_CHECK_VALUE(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, "weight must be ",
                    x.scalar_type(), " or float32, not ", weight.scalar_type());
  if (bias.has_value()) {
    check_like(*bias, "bias", {channels}, x.device());
    TORCH_CHECK_VALUE(bias->scalar_type() == weight.scalar_type(), "weight and bias must have the same type");
  }
  return dtype_code(weight.scalar_type());
}

void check_conv_state(const Tensor& state, const Tensor& weight, int64_t batch, int64_t channels, const Tensor& x) {
  check_like(state, "state", {batch, weight.size(1) - 1, channels}, x.device());
  TORCH_CHECK_VALUE(state.scalar_type() == x.scalar_type(), "state must be ", x.scalar_type(), ", not ",
                    state.scalar_type());
}

std::tuple<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& state,
                                        const Tensor& lengths, bool silu) {
  const int64_t B = x.size(0), T = x.size(1), C = x.size(2), W = weight.size(1);
  Tensor y = empty({B, T, C}, x.scalar_type(), x.device()), state_n = empty({B, W - 1, C}, x.scalar_type(), x.device());
  check(plh_causal_conv_forward(dtype_code(x.scalar_type()), dtype_code(weight.scalar_type()), ptr(x), x.stride(0),
                                x.stride(1), B, T, C, (int)W, ptr(weight), ptr(bias), ptr(state),
                                ptr<int32_t>(lengths), silu, ptr(y), ptr(state_n), stream_of(x)),
        "causal_conv");
  return {y, state_n};
}

struct CausalConv : torch::autograd::Function<CausalConv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const MaybeTensor& bias,
                               const MaybeTensor& state, const MaybeTensor& lengths, bool silu) {
    const auto [y, state_n] = conv_forward(x, weight, given(bias), given(state), given(lengths), silu);
    ctx->save_for_backward({x, weight, given(bias), given(state), given(lengths)});
    ctx->saved_data["silu"] = silu;
    ctx->set_materialize_grads(false);
    return {y, state_n};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &state = saved[3], &lengths = saved[4];
    const bool silu = ctx->saved_data["silu"].toBool();
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2), W = weight.size(1);
    const at::Device device = x.device();
    const c10::DeviceGuard guard(device);
    const Tensor d_y = grads[0].defined() ? incoming(grads[0], x.scalar_type())
                                          : at::zeros({B, T, C}, at::TensorOptions().dtype(x.scalar_type()).device(device));
    const Tensor d_sn = grads[1].defined() ? incoming(grads[1], x.scalar_type()) : Tensor();
    const int at_state = bias.defined() ? 3 : 2;
    const bool wants_bias = bias.defined() && ctx->needs_input_grad(2);
    const bool wants_state = state.defined() && ctx->needs_input_grad(at_state);
    Tensor d_x, d_w, d_b, d_s, ws;
    if (ctx->needs_input_grad(0)) d_x = empty({B, T, C}, x.scalar_type(), device);
    if (ctx->needs_input_grad(1)) d_w = empty({C, W}, weight.scalar_type(), device);
    if (wants_bias) d_b = empty({C}, weight.scalar_type(), device);
    if (wants_state && T > 0) d_s = empty({B, W - 1, C}, x.scalar_type(), device);
    if (d_w.defined() || d_b.defined())
      ws = empty({plh_causal_conv_workspace_bytes(B, T, C, (int)W)}, at::kByte, device);
    check(plh_causal_conv_backward(dtype_code(x.scalar_type()), dtype_code(weight.scalar_type()), ptr(x), x.stride(0),
                                   x.stride(1), B, T, C, (int)W, ptr(weight), ptr(bias), ptr(state),
                                   ptr<int32_t>(lengths), silu, ptr(d_y), ptr(d_sn), ptr(d_x), ptr(d_w), ptr(d_b),
                                   ptr(d_s), ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(x)),
          "causal_conv backward");
    if (wants_state && T == 0)  // (no steps: the new state is the old one)
      d_s = d_sn.defined() ? d_sn : at::zeros({B, W - 1, C}, at::TensorOptions().dtype(x.scalar_type()).device(device));
    // With an activation no gradient is a constant; without one the operator is linear in its filter, and in what it
    // is applied to.
    const uint32_t inputs = 2 + bias.defined() + state.defined();
    const auto node = torch::autograd::get_current_node();
    const bool of_x = node->next_edge(0).is_valid() || (state.defined() && node->next_edge(at_state).is_valid());
    const bool depends = silu || (node->next_edge(1).is_valid() && of_x);
    return once_over({d_x, d_w, d_b, d_s, Tensor(), Tensor()}, grads, depends ? inputs : 0, "causal_conv");
  }
};

std::tuple<Tensor, Tensor> causal_conv(const Tensor& x_in, const Tensor& weight_in, const MaybeTensor& bias_in,
                                       const MaybeTensor& state_in, const MaybeTensor& lengths, bool silu) {
  check_tensor(x_in, "x", 3);
  const int64_t B = x_in.size(0), T = x_in.size(1), C = x_in.size(2);
  TORCH_CHECK_VALUE(C > 0, "x needs at least one channel");
  check_filter(weight_in, bias_in, C, x_in);
  const c10::DeviceGuard guard(x_in.device());
  const Tensor n = device_lengths(lengths, B, T, x_in.device()), x = dense_rows(x_in), weight = dense(weight_in);
  MaybeTensor bias, state;
  if (bias_in.has_value()) bias = dense(*bias_in);
  if (state_in.has_value()) {
    check_conv_state(*state_in, weight, B, C, x_in);
    state = dense(*state_in);
  }
  if (at::GradMode::is_enabled() && (tracks(x) || tracks(weight) || tracks(given(bias)) || tracks(given(state)))) {
    const variable_list r = CausalConv::apply(x, weight, bias, state, maybe(n), silu);
    return {r[0], r[1]};
  }
  return conv_forward(x, weight, given(bias), given(state), n, silu);
}

std::tuple<Tensor, Tensor> causal_conv_step(const Tensor& x_in, const Tensor& state_in, const Tensor& weight_in,
                                            const MaybeTensor& bias_in, bool silu, bool inplace) {
  const int code = check_tensor(x_in, "x", 2);
  const int64_t B = x_in.size(0), C = x_in.size(1);
  TORCH_CHECK_VALUE(C > 0, "x needs at least one channel");
  const int wcode = check_filter(weight_in, bias_in, C, x_in);
  check_conv_state(state_in, weight_in, B, C, x_in);
  check_inplace(state_in, "state", inplace);
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !(tracks(x_in) || tracks(state_in) || tracks(weight_in) ||
                                                     tracks(given(bias_in))),
                    "causal_conv_step is not differentiable: call it under torch.no_grad(), or causal_conv");
  const c10::DeviceGuard guard(x_in.device());
  const Tensor x = dense_rows(x_in), weight = dense(weight_in), state = dense(state_in);
  const Tensor bias = bias_in.has_value() ? dense(*bias_in) : Tensor();
  Tensor y = empty({B, C}, x.scalar_type(), x.device());
  Tensor state_n = inplace ? state_in : empty(state.sizes(), x.scalar_type(), x.device());
  check(plh_causal_conv_step(code, wcode, ptr(x), x.stride(0), B, C, (int)weight.size(1), ptr(weight), ptr(bias),
                             ptr(state), silu, ptr(y), ptr(state_n), stream_of(x)),
        "causal_conv_step");
  if (inplace) state_n.unsafeGetTensorImpl()->bump_version();
  return {y, state_n};
}

// ---- selective scan -----------------------------------------------------------------------------

// What a scan is given, checked; [batch, time, ...] or, of one step, [batch, ...].
struct Selective {
  Tensor u, dt, A, B, C, D, z, bias, lengths;
  bool softplus;

  bool step() const { return u.dim() == 2; }
  int64_t batch() const { return u.size(0); }
  int64_t steps() const { return step() ? 1 : u.size(1); }
  int64_t channels() const { return u.size(-1); }
  int64_t states() const { return A.size(1); }

  plh_selective_scan_args args() const {
    plh_selective_scan_args a = {};
    a.dtype = dtype_code(u.scalar_type()), a.wdtype = dtype_code(A.scalar_type());
    const auto put = [&](const Tensor& t, const void*& p, int64_t* stride) {
      if (!t.defined()) return;
      p = t.data_ptr(), stride[0] = t.stride(0), stride[1] = step() ? 0 : t.stride(1);
    };
    put(u, a.u, a.u_stride), put(dt, a.dt, a.dt_stride), put(z, a.z, a.z_stride);
    put(B, a.B, a.B_stride), put(C, a.C, a.C_stride);
    a.A = ptr(A), a.D = ptr(D), a.dt_bias = ptr(bias), a.lengths = ptr<int32_t>(lengths);
    a.batch = batch(), a.seq_len = steps(), a.channels = channels(), a.states = (int)states(), a.softplus = softplus;
    return a;
  }
};

Selective check_selective(int64_t dims, const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                          const MaybeTensor& D, const MaybeTensor& z, const MaybeTensor& bias, bool softplus) {
  check_tensor(u, "u", dims);
  const at::Device device = u.device();
  const int64_t channels = u.size(-1);
  TORCH_CHECK_VALUE(channels > 0, "u needs at least one channel");
  check_tensor(A, "A", 2);
  TORCH_CHECK_VALUE(A.size(0) == channels && A.size(1) >= 1 && A.size(1) <= 64, "A must be [channels, states] with ",
                    channels, " channels and 1 to 64 states, not ", A.sizes());
  check_like(A, "A", A.sizes(), device);
  const auto like_u = [&](const Tensor& t, const char* name, bool per_channel) {
    std::vector<int64_t> shape = u.sizes().vec();
    if (!per_channel) shape.back() = A.size(1);
    check_like(t, name, shape, device);
    TORCH_CHECK_VALUE(t.scalar_type() == u.scalar_type(), name, " must be ", u.scalar_type(), ", not ", t.scalar_type());
  };
  like_u(dt, "dt", true), like_u(B, "B", false), like_u(C, "C", false);
  if (z.has_value()) like_u(*z, "z", true);
  TORCH_CHECK_VALUE(A.scalar_type() == u.scalar_type() || A.scalar_type() == at::kFloat, "A must be ", u.scalar_type(),
                    " or float32, not ", A.scalar_type());
  const auto param = [&](const MaybeTensor& t, const char* name) -> Tensor {
    if (!t.has_value()) return Tensor();
    check_like(*t, name, {channels}, device);
    TORCH_CHECK_VALUE(t->scalar_type() == A.scalar_type(), name, " must have A's type, ", A.scalar_type(), ", not ",
                      t->scalar_type());
    return dense(*t);
  };
  const Tensor d = param(D, "D"), b = param(bias, "dt_bias");
  const c10::DeviceGuard guard(device);
  return {dense_rows(u), dense_rows(dt), dense(A), dense_rows(B), dense_rows(C),
          d, z.has_value() ? dense_rows(*z) : Tensor(), b, Tensor(), softplus};
}

Tensor selective_workspace(const Selective& s, bool backward) {
  const int64_t n = plh_selective_scan_workspace_bytes(s.batch(), s.steps(), s.channels(), (int)s.states(), backward);
  return n > 0 ? empty({n}, at::kByte, s.u.device()) : Tensor();
}

ScanOut selective_forward(const Selective& s, const Tensor& h0, bool keep) {
  const at::Device device = s.u.device();
  ScanOut r{empty({s.batch(), s.steps(), s.channels()}, s.u.scalar_type(), device),
            empty({s.batch(), s.channels(), s.states()}, at::kFloat, device), Tensor()};
  const plh_selective_scan_args args = s.args();
  if (keep)
    r.states = empty({plh_selective_scan_states(s.steps()), s.batch(), s.channels(), s.states()}, at::kFloat, device);
  const Tensor ws = selective_workspace(s, false);
  check(plh_selective_scan_forward(&args, ptr<float>(h0), ptr(r.out), ptr<float>(r.c_n), ptr<float>(r.states), ptr(ws),
                                   ws.defined() ? ws.numel() : 0, stream_of(s.u)),
        "selective_scan");
  return r;
}

struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B,
                               const Tensor& C, const MaybeTensor& D, const MaybeTensor& z, const MaybeTensor& h0,
                               const MaybeTensor& bias, const MaybeTensor& lengths, bool softplus) {
    const Selective s{u, dt, A, B, C, given(D), given(z), given(bias), given(lengths), softplus};
    const ScanOut r = selective_forward(s, given(h0), true);
    ctx->save_for_backward({u, dt, A, B, C, s.D, s.z, s.bias, s.lengths, r.states});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["has_h0"] = h0.has_value();
    ctx->set_materialize_grads(false);
    return {r.out, r.c_n};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Selective s{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], saved[7], saved[8],
                      ctx->saved_data["softplus"].toBool()};
    const bool has_h0 = ctx->saved_data["has_h0"].toBool();
    const at::Device device = s.u.device();
    const c10::DeviceGuard guard(device);
    const at::ScalarType type = s.u.scalar_type(), wtype = s.A.scalar_type();
    const std::vector<int64_t> shape = {s.batch(), s.steps(), s.channels()};
    const Tensor d_out = grads[0].defined() ? incoming(grads[0], type)
                                            : at::zeros(shape, at::TensorOptions().dtype(type).device(device));
    const Tensor d_hn = grads[1].defined() ? incoming(grads[1], at::kFloat) : Tensor();
    // the inputs that were given, in order: u, dt, A, B, C, then D, z, h0 and dt_bias where there are any
    uint32_t inputs = 5;
    const uint32_t at_D = s.D.defined() ? inputs++ : 0, at_z = s.z.defined() ? inputs++ : 0;
    const uint32_t at_h0 = has_h0 ? inputs++ : 0, at_bias = s.bias.defined() ? inputs++ : 0;
    const auto wants = [&](uint32_t i) { return i > 0 && ctx->needs_input_grad(i); };
    Tensor d_u = empty(shape, type, device), d_dt = empty(shape, type, device), d_z, d_B, d_C, d_A, d_D, d_bias, d_h0;
    if (s.z.defined()) d_z = empty(shape, type, device);
    if (wants(2)) d_A = empty(s.A.sizes(), wtype, device);
    if (wants(3)) d_B = empty(s.B.sizes(), type, device);
    if (wants(4)) d_C = empty(s.C.sizes(), type, device);
    if (wants(at_D)) d_D = empty(s.D.sizes(), wtype, device);
    if (wants(at_bias)) d_bias = empty(s.bias.sizes(), wtype, device);
    if (wants(at_h0)) d_h0 = empty({s.batch(), s.channels(), s.states()}, at::kFloat, device);
    const plh_selective_scan_args args = s.args();
    const plh_selective_scan_grads g = {ptr(d_u), ptr(d_dt), ptr(d_z), ptr(d_B), ptr(d_C),
                                        ptr(d_A), ptr(d_D), ptr(d_bias), ptr<float>(d_h0)};
    const Tensor ws = selective_workspace(s, true);
    check(plh_selective_scan_backward(&args, ptr<float>(saved[9]), ptr(d_out), ptr<float>(d_hn), &g, ptr(ws),
                                      ws.defined() ? ws.numel() : 0, stream_of(s.u)),
          "selective_scan backward");
    // The operator is not linear in dt, A, z and dt_bias, and it holds the products C B u, C h0 and D u.
    const auto node = torch::autograd::get_current_node();
    const auto of = [&](uint32_t i) { return node->next_edge(i).is_valid(); };
    const auto maybe_of = [&](uint32_t i) { return i > 0 && of(i); };
    const bool u = of(0), B = of(3), C = of(4);
    const bool depends = of(1) || of(2) || maybe_of(at_z) || maybe_of(at_bias) || (C && (B || u || maybe_of(at_h0))) ||
                         (u && (B || maybe_of(at_D)));
    return once_over({d_u, d_dt, d_A, d_B, d_C, d_D, d_z, d_h0, d_bias, Tensor(), Tensor()}, grads, depends ? inputs : 0,
                     "selective_scan");
  }
};

std::tuple<Tensor, Tensor> selective_scan(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B,
                                          const Tensor& C, const MaybeTensor& D, const MaybeTensor& z,
                                          const MaybeTensor& h0_in, const MaybeTensor& dt_bias, bool softplus,
                                          const MaybeTensor& lengths) {
  Selective s = check_selective(3, u, dt, A, B, C, D, z, dt_bias, softplus);
  const c10::DeviceGuard guard(u.device());
  MaybeTensor h0;
  if (h0_in.has_value()) {
    check_tensor(*h0_in, "h0");
    check_like(*h0_in, "h0", {s.batch(), s.channels(), s.states()}, u.device());
    h0 = dense(h0_in->to(at::kFloat));
  }
  s.lengths = device_lengths(lengths, s.batch(), s.steps(), u.device());
  bool tracked = tracks(given(h0));
  for (const Tensor* t : {&s.u, &s.dt, &s.A, &s.B, &s.C, &s.D, &s.z, &s.bias}) tracked = tracked || tracks(*t);
  if (at::GradMode::is_enabled() && tracked) {
    const variable_list r = SelectiveScan::apply(s.u, s.dt, s.A, s.B, s.C, maybe(s.D), maybe(s.z), h0, maybe(s.bias),
                                                 maybe(s.lengths), softplus);
    return {r[0], r[1]};
  }
  const ScanOut r = selective_forward(s, given(h0), false);
  return {r.out, r.c_n};
}

std::tuple<Tensor, Tensor> selective_scan_step(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B,
                                               const Tensor& C, const Tensor& h_in, const MaybeTensor& D,
                                               const MaybeTensor& z, const MaybeTensor& dt_bias, bool softplus,
                                               bool inplace) {
  const Selective s = check_selective(2, u, dt, A, B, C, D, z, dt_bias, softplus);
  check_like(h_in, "h", {s.batch(), s.channels(), s.states()}, u.device());
  TORCH_CHECK_VALUE(h_in.scalar_type() == at::kFloat, "h must be float32, not ", h_in.scalar_type());
  check_inplace(h_in, "h", inplace);
  bool tracked = tracks(h_in);
  for (const Tensor* t : {&s.u, &s.dt, &s.A, &s.B, &s.C, &s.D, &s.z, &s.bias}) tracked = tracked || tracks(*t);
  TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !tracked,
                    "selective_scan_step is not differentiable: call it under torch.no_grad(), or selective_scan");
  const c10::DeviceGuard guard(u.device());
  const Tensor h = dense(h_in);
  Tensor out = empty({s.batch(), s.channels()}, u.scalar_type(), u.device());
  Tensor h_n = inplace ? h_in : empty(h.sizes(), at::kFloat, u.device());
  const plh_selective_scan_args args = s.args();
  check(plh_selective_scan_step(&args, ptr<float>(h), ptr(out), ptr<float>(h_n), stream_of(u)), "selective_scan_step");
  if (inplace) h_n.unsafeGetTensorImpl()->bump_version();
  return {out, h_n};
}

// ---- gradient norm ------------------------------------------------------------------------------

std::tuple<std::vector<Tensor>, Tensor> clip_grad_norm(const std::vector<Tensor>& grads, double max_norm, bool inplace) {
  TORCH_CHECK_VALUE(!grads.empty(), "clip_grad_norm needs at least one tensor");
  TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm must be non-negative, not ", max_norm);
  const at::Device device = grads[0].device();
  const size_t count = grads.size();
  for (const Tensor& g : grads) {
    TORCH_CHECK_VALUE(g.layout() == at::kStrided, "a gradient must be a dense tensor, not ", g.layout());
    check_tensor(g, "a gradient");
    TORCH_CHECK_VALUE(g.device() == device, "all gradients must be on ", device, ", not ", g.device());
    TORCH_CHECK_VALUE(!at::GradMode::is_enabled() || !g.requires_grad(),
                      "clip_grad_norm is not differentiable: pass gradients that do not require one themselves (a "
                      "parameter's .grad), or call it under torch.no_grad()");
    TORCH_CHECK_VALUE(!inplace || !g.is_inference() || c10::InferenceMode::is_enabled(),
                      "a gradient is an inference tensor: it can be updated in place in inference mode only");
  }
  const c10::DeviceGuard guard(device);
  std::vector<Tensor> in(count), out(count), result(count);
  std::vector<const void*> src(count);
  std::vector<void*> dst(count);
  std::vector<int64_t> numel(count);
  std::vector<int> dtypes(count);
  std::vector<std::pair<const char*, const char*>> ranges;  // memory that is written in place
  for (size_t i = 0; i < count; ++i) {
    const Tensor& g = grads[i];
    const bool whole = g.is_non_overlapping_and_dense();  // its elements in some order: as good as contiguous
    if (inplace) {
      for (int64_t k = 0; !whole && k < g.dim(); ++k)
        TORCH_CHECK_VALUE(g.stride(k) != 0 || g.size(k) <= 1,
                          "a gradient is an expanded tensor, whose elements share memory: it cannot be updated in place");
      in[i] = whole ? g : g.contiguous();
      out[i] = in[i], result[i] = g;
      if (g.numel() > 0) {
        int64_t span = 1;
        for (int64_t k = 0; k < g.dim(); ++k) span += (g.size(k) - 1) * g.stride(k);
        const char* const begin = static_cast<const char*>(g.data_ptr());
        ranges.emplace_back(begin, begin + span * (int64_t)g.element_size());
      }
    } else {
      in[i] = whole ? values(g) : dense(g);
      out[i] = empty_strided(in[i].sizes(), in[i].strides(), in[i].scalar_type(), device), result[i] = out[i];
    }
    src[i] = ptr(in[i]), dst[i] = ptr(out[i]), numel[i] = g.numel(), dtypes[i] = dtype_code(g.scalar_type());
  }
  std::sort(ranges.begin(), ranges.end());
  for (size_t i = 1; i < ranges.size(); ++i)
    TORCH_CHECK_VALUE(ranges[i].first >= ranges[i - 1].second,
                      "two gradients share memory (or are the same, or lie in each other's gaps): they cannot be updated in place");
  Tensor norm = empty({}, at::kFloat, device);
  const Tensor ws = empty({plh_clip_grad_norm_workspace_bytes((int64_t)count, numel.data())}, at::kByte, device);
  check(plh_clip_grad_norm((int64_t)count, dtypes.data(), src.data(), dst.data(), numel.data(), max_norm,
                           ptr<float>(norm), ptr(ws), ws.numel(), stream_of(grads[0])),
        "clip_grad_norm");
  if (inplace) {
    const at::NoGradGuard no_grad;
    for (size_t i = 0; i < count; ++i) {
      if (!in[i].is_same(grads[i]))
        result[i].copy_(in[i]);
      else
        result[i].unsafeGetTensorImpl()->bump_version();
    }
  }
  return {result, norm};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  using release = py::call_guard<py::gil_scoped_release>;
  m.def("gated_scan", &gated_scan, release());
  m.def("gated_scan_step", &gated_scan_step, release());
  m.def("layer_norm", &layer_norm, release());
  m.def("dropout_add", &dropout_add, release());
  m.def("causal_conv", &causal_conv, release());
  m.def("causal_conv_step", &causal_conv_step, release());
  m.def("selective_scan", &selective_scan, release());
  m.def("selective_scan_step", &selective_scan_step, release());
  m.def("clip_grad_norm", &clip_grad_norm, release());
}
