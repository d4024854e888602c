// Python surface of the feed-forward operators (part of the `_cmpext3` module): tensor checks and
// outputs here, everything else through the C ABI of include/cmpext3_projection.h, on PyTorch's
// current stream of the tensors' device.
#include "projection_ops.h"

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <climits>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "../../include/cmpext3_projection.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return CMPEXT3_F16;
    case at::kBFloat16: return CMPEXT3_BF16;
    case at::kFloat: return CMPEXT3_F32;
    case at::kChar: return CMPEXT3_I8;
    default: return -1;
  }
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }
bool is16(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

void* current_stream(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check_status(int64_t st, const char* op) {
  TORCH_CHECK(st == CMPEXT3_OK, "cmpext3.", op, ": ", cmpext3_status_string((int)st));
}

void check_device(const Tensor& t, const Tensor& like, const char* op, const char* what) {
  TORCH_CHECK(t.is_cuda(), "cmpext3.", op, ": ", what, " must be on a GPU");
  TORCH_CHECK(t.device() == like.device(), "cmpext3.", op, ": device mismatch (", what, ")");
}

int checked_int(int64_t v, const char* op, const char* what) {
  TORCH_CHECK(v <= INT_MAX, "cmpext3.", op, ": ", what, " = ", v, " exceeds the supported range (2^31 - 1)");
  return (int)v;
}

int activation_code(const std::string& name, const char* op) {
  if (name == "silu") return CMPEXT3_ACT_SILU;
  if (name == "gelu") return CMPEXT3_ACT_GELU;
  if (name == "gelu_tanh") return CMPEXT3_ACT_GELU_TANH;
  if (name == "relu") return CMPEXT3_ACT_RELU;
  TORCH_CHECK(false, "cmpext3.", op, ": unknown activation '", name, "' (silu, gelu, gelu_tanh or relu)");
}

// The kernels' limit on row pitches; a view with a larger one is copied.
constexpr int64_t kMaxPitch = INT_MAX / (256 * 4);

// Rows of the last dimension, [product of the others, last]: read in place where rows have unit
// stride and one pitch, copied otherwise.
struct Rows {
  Tensor t;
  int64_t rows, cols, pitch;
};
Rows rows_of(const Tensor& in) {
  Rows r;
  r.cols = in.size(-1);
  r.rows = 1;
  for (int64_t d = 0; d + 1 < in.dim(); ++d) r.rows *= in.size(d);
  r.pitch = std::max<int64_t>(r.cols, 1);
  if (r.rows == 0 || r.cols == 0) {
    r.t = in;
    return r;
  }
  bool in_place = r.cols == 1 || in.stride(-1) == 1;
  // the dimensions before the last one, from the innermost that has more than one entry outwards
  int64_t pitch = 0, span = 0;
  for (int64_t d = in.dim() - 2; d >= 0 && in_place; --d) {
    if (in.size(d) == 1) continue;
    if (pitch == 0) {
      pitch = in.stride(d);
      in_place = pitch >= r.cols && pitch <= kMaxPitch;
    } else {
      in_place = in.stride(d) == span;
    }
    span = in.stride(d) * in.size(d);
  }
  if (in_place) {
    r.t = in;
    if (pitch > 0) r.pitch = pitch;
  } else {
    r.t = in.contiguous();
  }
  return r;
}

Tensor float_vector(const Tensor& t, int64_t size, const Tensor& like, const char* op, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kFloat, "cmpext3.", op, ": ", what, " must be float32, got ", t.scalar_type());
  TORCH_CHECK(t.numel() == size, "cmpext3.", op, ": ", what, " must have ", size, " elements, got ", t.numel());
  check_device(t, like, op, what);
  return t.contiguous();
}

std::tuple<Tensor, Tensor> quantize_int8(const Tensor& x) {
  const char* op = "quantize_int8";
  TORCH_CHECK(x.dim() >= 1, "cmpext3.", op, ": the input needs at least one dimension");
  TORCH_CHECK(is16(x) || x.scalar_type() == at::kFloat, "cmpext3.", op, ": unsupported dtype ", x.scalar_type(),
              " (float16, bfloat16 or float32)");
  TORCH_CHECK(x.is_cuda(), "cmpext3.", op, ": tensors must be on a GPU");
  c10::DeviceGuard guard(x.device());
  const Rows r = rows_of(x);
  Tensor codes = torch::empty(x.sizes(), x.options().dtype(at::kChar));
  Tensor scale = torch::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  cmpext3_quantize_int8_args a{};
  a.dtype = dtype_code(x.scalar_type());
  a.cols = checked_int(r.cols, op, "the row length");
  a.rows = r.rows;
  a.x = r.t.data_ptr();
  a.x_row = r.pitch;
  a.codes = (int8_t*)codes.data_ptr();
  a.codes_row = std::max<int64_t>(r.cols, 1);
  a.scale = (float*)scale.data_ptr();
  check_status(cmpext3_quantize_int8(&a, current_stream(x)), op);
  return {codes, scale};
}

// What all projections check: x's and the weights' shapes and devices.
void check_operands(const Tensor& x, std::initializer_list<const Tensor*> weights, const char* op) {
  TORCH_CHECK(x.dim() >= 1, "cmpext3.", op, ": the input needs at least one dimension");
  TORCH_CHECK(x.is_cuda(), "cmpext3.", op, ": tensors must be on a GPU");
  const Tensor& first = **weights.begin();
  for (const Tensor* w : weights) {
    TORCH_CHECK(w->dim() == 2, "cmpext3.", op, ": weights must be 2-D, got ", w->dim(), "-D");
    TORCH_CHECK(w->sizes() == first.sizes(), "cmpext3.", op, ": weight shape mismatch ", first.sizes(), " and ", w->sizes());
    TORCH_CHECK(w->size(1) == x.size(-1), "cmpext3.", op, ": shape mismatch ", x.sizes(), " and weight ", w->sizes());
    TORCH_CHECK(w->scalar_type() == first.scalar_type(), "cmpext3.", op, ": weight dtype mismatch");
    check_device(*w, x, op, "weight");
  }
}

void run_projection(const cmpext3_projection_args& a, const Tensor& like, const char* op) {
  const int64_t need = cmpext3_projection_workspace_size(&a);
  check_status(need < 0 ? need : CMPEXT3_OK, op);
  Tensor ws;
  if (need > 0) ws = torch::empty({need}, like.options().dtype(torch::kUInt8));
  check_status(cmpext3_projection(&a, ws.defined() ? ws.data_ptr() : nullptr, need, current_stream(like)), op);
}

void set_sizes(cmpext3_projection_args& a, const Rows& x, const Tensor& weight, const char* op) {
  a.M = checked_int(x.rows, op, "the number of rows");
  a.N = checked_int(weight.size(0), op, "the number of channels");
  a.K = checked_int(x.cols, op, "the row length");
}

std::vector<int64_t> with_last(const Tensor& x, int64_t n) {
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
  shape.push_back(n);
  return shape;
}

// Both 8-bit projections; w_up undefined: the plain one.
Tensor int8_projection(const Tensor& x, const Tensor& w_gate, const Tensor& gate_scale, const Tensor& w_up, const Tensor& up_scale,
                       const OptTensor& bias, const OptTensor& x_scale, c10::optional<at::ScalarType> dtype, int act, const char* op) {
  const bool gated = w_up.defined();
  if (gated)
    check_operands(x, {&w_gate, &w_up}, op);
  else
    check_operands(x, {&w_gate}, op);
  TORCH_CHECK(w_gate.scalar_type() == at::kChar, "cmpext3.", op, ": weights must be int8 codes, got ", w_gate.scalar_type());
  const bool codes = x.scalar_type() == at::kChar;
  TORCH_CHECK(codes || is16(x) || x.scalar_type() == at::kFloat, "cmpext3.", op, ": unsupported input dtype ", x.scalar_type(),
              " (int8 with x_scale, float16, bfloat16 or float32)");
  TORCH_CHECK(codes == given(x_scale), "cmpext3.", op, codes ? ": an int8 input needs x_scale" : ": only an int8 input has x_scale");
  const at::ScalarType out_type = dtype.has_value() ? *dtype : codes ? at::kBFloat16 : x.scalar_type();
  TORCH_CHECK(out_type == at::kHalf || out_type == at::kBFloat16 || out_type == at::kFloat, "cmpext3.", op,
              ": unsupported output dtype ", out_type, " (float16, bfloat16 or float32)");
  TORCH_CHECK(x.size(-1) <= CMPEXT3_I8_MAX_K, "cmpext3.", op, ": rows of ", x.size(-1), " codes could leave the 32-bit sums (at most ",
              CMPEXT3_I8_MAX_K, ")");
  c10::DeviceGuard guard(x.device());
  const int64_t N = w_gate.size(0);
  const Tensor gs = float_vector(gate_scale, N, x, op, gated ? "gate_scale" : "weight_scale");
  const Tensor us = gated ? float_vector(up_scale, N, x, op, "up_scale") : Tensor();
  Tensor bias_c;
  if (given(bias)) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N, "cmpext3.", op, ": the bias must have ", N, " elements, got ", bias->sizes());
    TORCH_CHECK(bias->scalar_type() == out_type, "cmpext3.", op, ": the bias must have the output's dtype ", out_type, ", got ",
                bias->scalar_type());
    check_device(*bias, x, op, "bias");
    bias_c = bias->contiguous();
  }
  const Rows rx = rows_of(x), rg = rows_of(w_gate), ru = gated ? rows_of(w_up) : rg;
  const Tensor xs = codes ? float_vector(*x_scale, rx.rows, x, op, "x_scale") : Tensor();
  Tensor out = torch::empty(with_last(x, N), x.options().dtype(out_type));
  cmpext3_projection_args a{};
  a.dtype = CMPEXT3_I8;
  a.x_dtype = dtype_code(x.scalar_type());
  a.out_dtype = dtype_code(out_type);
  a.activation = act;
  set_sizes(a, rx, w_gate, op);
  a.x = rx.t.data_ptr();
  a.x_row = rx.pitch;
  if (codes) a.x_scale = (const float*)xs.data_ptr();
  a.w_gate = rg.t.data_ptr();
  a.gate_row = rg.pitch;
  a.gate_scale = (const float*)gs.data_ptr();
  if (gated) {
    a.w_up = ru.t.data_ptr();
    a.up_row = ru.pitch;
    a.up_scale = (const float*)us.data_ptr();
    // an empty weight has no address, by which the gated form is known
    if (a.w_up == nullptr) a.w_up = a.up_scale;
  }
  if (bias_c.defined()) a.bias = bias_c.data_ptr();
  a.out = out.data_ptr();
  a.out_row = std::max<int64_t>(N, 1);
  if (out.numel() > 0) run_projection(a, x, op);
  return out;
}

Tensor int8_linear(const Tensor& x, const Tensor& weight, const Tensor& weight_scale, const OptTensor& bias, const OptTensor& x_scale,
                   c10::optional<at::ScalarType> dtype) {
  return int8_projection(x, weight, weight_scale, Tensor(), Tensor(), bias, x_scale, dtype, 0, "int8_linear");
}

Tensor int8_gated_linear(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& gate_scale, const Tensor& up_scale,
                         const std::string& activation, const OptTensor& x_scale, c10::optional<at::ScalarType> dtype) {
  const char* op = "int8_gated_linear";
  return int8_projection(x, w_gate, gate_scale, w_up, up_scale, c10::nullopt, x_scale, dtype, activation_code(activation, op), op);
}

// act(x w_gate^T) * (x w_up^T), and both products where `keep` asks for them: [2, rows, N rounded up to 8], so that
// kernels store and read whole pieces wherever N itself is odd.
std::tuple<Tensor, Tensor> gated_forward(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const std::string& activation,
                                                 bool keep) {
  const char* op = "gated_linear";
  check_operands(x, {&w_gate, &w_up}, op);
  TORCH_CHECK(is16(x), "cmpext3.", op, ": unsupported dtype ", x.scalar_type(), " (float16 or bfloat16)");
  TORCH_CHECK(w_gate.scalar_type() == x.scalar_type(), "cmpext3.", op, ": dtype mismatch ", x.scalar_type(), " and weight ",
              w_gate.scalar_type());
  const int act = activation_code(activation, op);
  c10::DeviceGuard guard(x.device());
  const Rows rx = rows_of(x), rg = rows_of(w_gate), ru = rows_of(w_up);
  const int64_t N = w_gate.size(0);
  Tensor out = torch::empty(with_last(x, N), x.options()), pre;
  cmpext3_projection_args a{};
  a.dtype = a.x_dtype = a.out_dtype = dtype_code(x.scalar_type());
  a.activation = act;
  set_sizes(a, rx, w_gate, op);
  a.x = rx.t.data_ptr();
  a.x_row = rx.pitch;
  a.w_gate = rg.t.data_ptr();
  a.gate_row = rg.pitch;
  a.w_up = ru.t.data_ptr();
  a.up_row = ru.pitch;
  if (a.w_up == nullptr) a.w_up = out.data_ptr();  // rows of no elements have no address
  a.out = out.data_ptr();
  a.out_row = std::max<int64_t>(N, 1);
  if (keep) {
    const int64_t pitch = (N + 7) / 8 * 8;
    pre = torch::empty({2, rx.rows, pitch}, x.options().dtype(at::kFloat));
    a.gate_out = (float*)pre.data_ptr();
    a.up_out = a.gate_out + rx.rows * pitch;
    a.pre_row = pitch;
  }
  if (out.numel() > 0) run_projection(a, x, op);
  return {out, pre};
}

// Gradients of x and of both weights, each only where asked for.
std::tuple<Tensor, Tensor, Tensor> gated_backward(const Tensor& grad, const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                                                  const Tensor& pre, const std::string& activation, bool want_x, bool want_gate,
                                                  bool want_up) {
  const char* op = "gated_linear (backward)";
  check_operands(x, {&w_gate, &w_up}, op);
  check_device(grad, x, op, "gradient");
  TORCH_CHECK(grad.scalar_type() == x.scalar_type(), "cmpext3.", op, ": dtype mismatch of the gradient, ", grad.scalar_type());
  c10::DeviceGuard guard(x.device());
  const Rows rx = rows_of(x), rd = rows_of(grad), rg = rows_of(w_gate), ru = rows_of(w_up);
  const int64_t N = w_gate.size(0), K = w_gate.size(1);
  TORCH_CHECK(rd.rows == rx.rows && rd.cols == N,
              "cmpext3.", op, ": shape mismatch of the gradient ", grad.sizes());
  Tensor dx, dgate, dup;
  cmpext3_gated_backward_args a{};
  a.dtype = dtype_code(x.scalar_type());
  a.activation = activation_code(activation, op);
  a.M = checked_int(rx.rows, op, "the number of rows");
  a.N = checked_int(N, op, "the number of channels");
  a.K = checked_int(K, op, "the row length");
  a.grad_out = rd.t.data_ptr();
  a.grad_row = rd.pitch;
  a.gate = (const float*)pre.data_ptr();
  a.up = a.gate + rx.rows * pre.size(2);
  a.pre_row = pre.size(2);
  a.x = rx.t.data_ptr();
  a.x_row = rx.pitch;
  a.w_gate = rg.t.data_ptr();
  a.gate_row = rg.pitch;
  a.w_up = ru.t.data_ptr();
  a.up_row = ru.pitch;
  if (want_x) {
    dx = N > 0 ? torch::empty(x.sizes(), x.options()) : torch::zeros(x.sizes(), x.options());
    a.dx = dx.data_ptr();
    a.dx_row = std::max<int64_t>(K, 1);
  }
  if (want_gate) {
    dgate = torch::empty({N, K}, x.options());
    a.dw_gate = dgate.data_ptr();
    a.dgate_row = std::max<int64_t>(K, 1);
  }
  if (want_up) {
    dup = torch::empty({N, K}, x.options());
    a.dw_up = dup.data_ptr();
    a.dup_row = std::max<int64_t>(K, 1);
  }
  if (N > 0 && K > 0) {
    const int64_t need = cmpext3_gated_backward_workspace_size(&a);
    check_status(need < 0 ? need : CMPEXT3_OK, op);
    Tensor ws;
    if (need > 0) ws = torch::empty({need}, x.options().dtype(torch::kUInt8));
    check_status(cmpext3_gated_backward(&a, ws.defined() ? ws.data_ptr() : nullptr, need, current_stream(x)), op);
  }
  return {dx, dgate, dup};
}

// Under graph capture the gradient of a leaf is added on the stream that its accumulating node was
// made on.  A node that an eager graph on another stream keeps alive would pull that stream into the
// capture, which ends the process from autograd's thread: refused here, before anything is recorded,
// for every leaf that the backward pass from this call would reach: an input, or what an input is a view or a result of.
void check_capture(std::initializer_list<const Tensor*> inputs) {
  using torch::autograd::AccumulateGrad;
  using torch::autograd::Node;
  const Tensor& first = **inputs.begin();
  if (!first.is_cuda()) return;
  const auto stream = c10::hip::getCurrentHIPStream(first.get_device());
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream.stream(), &capture) != hipSuccess || capture == hipStreamCaptureStatusNone) return;
  auto check = [&](Node* node) {
    const auto made_on = node->stream();
    TORCH_CHECK(made_on.has_value() && made_on->id() == stream.id(),
                "cmpext3.gated_linear: a graph that was made on another stream still holds an input of this captured call, or a leaf "
                "that one was made from; release it (or run it on the capturing stream) before the capture");
  };
  std::vector<Node*> left;
  for (const Tensor* input : inputs) {
    const Tensor& t = *input;
    if (!t.requires_grad()) continue;
    if (t.is_leaf()) {
      if (const auto node = torch::autograd::impl::try_get_grad_accumulator(t)) check(node.get());
    } else if (t.grad_fn() != nullptr) {
      left.push_back(t.grad_fn().get());
    }
  }
  std::unordered_set<Node*> seen(left.begin(), left.end());
  while (!left.empty()) {
    Node* node = left.back();
    left.pop_back();
    const auto* leaf = dynamic_cast<const AccumulateGrad*>(node);
    if (leaf != nullptr && leaf->variable.device() == first.device()) check(node);
    for (const auto& edge : node->next_edges())
      if (edge.function != nullptr && seen.insert(edge.function.get()).second) left.push_back(edge.function.get());
  }
}

// gated_linear with its gradients.  Saved for the backward pass: the inputs and, in fp32, both products.
struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                        const std::string& activation) {
    Tensor out, pre;
    std::tie(out, pre) = gated_forward(x, w_gate, w_up, activation, true);
    ctx->save_for_backward({x, w_gate, w_up, pre});
    ctx->saved_data["activation"] = activation;
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    Tensor dx, dgate, dup;
    std::tie(dx, dgate, dup) = gated_backward(grads[0], saved[0], saved[1], saved[2], saved[3],
                                              ctx->saved_data["activation"].toStringRef(), ctx->needs_input_grad(0),
                                              ctx->needs_input_grad(1), ctx->needs_input_grad(2));
    torch::autograd::variable_list out = {dx, dgate, dup};
    if (at::GradMode::is_enabled()) {
      // asked for a graph of the gradients: they have none, and say so when one is taken through them
      for (Tensor& t : out)
        if (t.defined()) t = t.detach().requires_grad_();
      out = (*std::make_shared<torch::autograd::DelayedError>("cmpext3.gated_linear: differentiable once only", 3))(std::move(out));
    }
    out.emplace_back();
    return out;
  }
};

// A dual tensor of forward-mode differentiation need not require a gradient: without this the result would have no
// tangent, which reads as a derivative of zero.
void refuse_forward_mode(std::initializer_list<const Tensor*> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), "cmpext3.gated_linear: no forward-mode derivative; it has a backward pass only");
}

Tensor gated_linear(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const std::string& activation) {
  refuse_forward_mode({&x, &w_gate, &w_up});
  if (!at::GradMode::is_enabled() || !(x.requires_grad() || w_gate.requires_grad() || w_up.requires_grad()))
    return std::get<0>(gated_forward(x, w_gate, w_up, activation, false));
  check_capture({&x, &w_gate, &w_up});
  return GatedLinear::apply(x, w_gate, w_up, activation);
}

}  // namespace

void register_projection_ops(py::module& m) {
  m.def("quantize_int8", &quantize_int8, "Rows as int8 codes with a scale for each", py::arg("x"));
  m.def("int8_linear", &int8_linear, "x @ weight.T for int8 codes with scales", py::arg("x"), py::arg("weight"), py::arg("weight_scale"),
        py::arg("bias") = py::none(), py::arg("x_scale") = py::none(), py::arg("dtype") = py::none());
  m.def("int8_gated_linear", &int8_gated_linear, "act(x @ w_gate.T) * (x @ w_up.T) for int8 codes with scales", py::arg("x"),
        py::arg("w_gate"), py::arg("w_up"), py::arg("gate_scale"), py::arg("up_scale"), py::arg("activation") = "silu",
        py::arg("x_scale") = py::none(), py::arg("dtype") = py::none());
  m.def("gated_linear", &gated_linear,
        R"(act(x @ w_gate.T) * (x @ w_up.T) in one kernel: x [..., K], weights [N, K], all float16 or all bfloat16; sums
and the activation in fp32, rounded once.

activation: "silu", "gelu" (by the error function), "gelu_tanh" or "relu".

Differentiable once in all three tensors, backwards only (forward mode is refused).  For the backward pass x, the weights and both products (in float32,
8 bytes for each result) are kept; where no input needs a gradient nothing is.  Weights may be the two halves of one
tensor.  Under graph capture the inputs' leaves must not be held by a graph of another stream (refused).)",
        py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("activation") = "silu");
}
