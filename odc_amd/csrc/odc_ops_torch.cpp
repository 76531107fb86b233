// odc_ops_torch.cpp — the host path between the calls of odc_amd.ops and the C ABI of include/odc_ops.h, as
// odc_torch.cpp is for the primitives: reads tensors and Python lists, checks them, allocates what a call
// returns, fills the C structures and makes the call on the tensors' device and its current stream. Layer norm's
// autograd node is here too. A CPython extension module, plain C++ against torch's headers; the entry points of
// libodc_ops.so are bound by address (bind()). The GIL is released around allocations and library calls.
#include <Python.h>

#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstring>
#include <memory>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "odc_ops.h"

#ifndef ODC_TORCH_VERSION
#error "ODC_TORCH_VERSION: the torch.__version__ that this is compiled against"
#endif

namespace {

// ------------------------------------------------------------------------------------------------
// the library
// ------------------------------------------------------------------------------------------------
decltype(&odc_layer_norm) p_layer_norm = nullptr;
decltype(&odc_layer_norm_backward) p_layer_norm_backward = nullptr;
decltype(&odc_layer_norm_backward_workspace) p_layer_norm_backward_workspace = nullptr;
decltype(&odc_squared_norm) p_squared_norm = nullptr;
decltype(&odc_squared_norm_workspace) p_squared_norm_workspace = nullptr;
decltype(&odc_adamw) p_adamw = nullptr;
decltype(&odc_adamw_check) p_adamw_check = nullptr;
decltype(&odc_dequantize_blocks) p_dequantize_blocks = nullptr;
decltype(&odc_ops_last_error) p_ops_last_error = nullptr;

// bind(name, address, ...): every entry point this module calls.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  for (Py_ssize_t i = 0; i + 1 < n; i += 2) {
    const char* name = PyUnicode_AsUTF8(args[i]);
    void* address = PyLong_AsVoidPtr(args[i + 1]);
    if (PyErr_Occurred()) return nullptr;
#define ODC_BIND(symbol) \
  if (!strcmp(name, "odc_" #symbol)) { p_##symbol = reinterpret_cast<decltype(p_##symbol)>(address); continue; }
    ODC_BIND(layer_norm)
    ODC_BIND(layer_norm_backward)
    ODC_BIND(layer_norm_backward_workspace)
    ODC_BIND(squared_norm)
    ODC_BIND(squared_norm_workspace)
    ODC_BIND(adamw)
    ODC_BIND(adamw_check)
    ODC_BIND(dequantize_blocks)
    ODC_BIND(ops_last_error)
#undef ODC_BIND
    PyErr_Format(PyExc_ValueError, "bind: unknown entry point %s", name);
    return nullptr;
  }
  if (!p_layer_norm || !p_layer_norm_backward || !p_layer_norm_backward_workspace || !p_squared_norm ||
      !p_squared_norm_workspace || !p_adamw || !p_adamw_check || !p_dequantize_blocks || !p_ops_last_error) {
    PyErr_SetString(PyExc_RuntimeError, "bind: an entry point is missing");
    return nullptr;
  }
  Py_RETURN_NONE;
}

// ------------------------------------------------------------------------------------------------
// Python values
// ------------------------------------------------------------------------------------------------
struct Failed {};  // a Python exception is set

template <class... Args>
[[noreturn]] void raise(PyObject* type, const char* format, Args... args) {
  PyErr_Format(type, format, args...);
  throw Failed();
}

// What `body` throws becomes the exception that torch's own functions raise (out of memory among them).
template <class F>
PyObject* guarded(F body) {
  HANDLE_TH_ERRORS
  try {
    return body();
  } catch (const Failed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

class WithoutGil {
 public:
  WithoutGil() : state_(PyEval_SaveThread()) {}
  ~WithoutGil() { PyEval_RestoreThread(state_); }
  WithoutGil(const WithoutGil&) = delete;
  WithoutGil& operator=(const WithoutGil&) = delete;

 private:
  PyThreadState* state_;
};

// The items of a sequence. They are held for as long as this is there: while a call has let go of the GIL, another thread
// may change the list that they came from.
class Sequence {
 public:
  Sequence(PyObject* o, const char* what) : items_(PySequence_Check(o) ? PySequence_Tuple(o) : nullptr) {
    if (items_) return;
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, what);
    throw Failed();
  }
  ~Sequence() { Py_DECREF(items_); }
  Sequence(const Sequence&) = delete;
  Sequence& operator=(const Sequence&) = delete;
  Py_ssize_t size() const { return PyTuple_GET_SIZE(items_); }
  PyObject* operator[](Py_ssize_t i) const { return PyTuple_GET_ITEM(items_, i); }

 private:
  PyObject* items_;
};

void expect_args(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) raise(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
}

const at::Tensor& as_tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s: expected a torch.Tensor, got %s", what, Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

at::Tensor as_optional_tensor(PyObject* o, const char* what) { return o == Py_None ? at::Tensor() : as_tensor(o, what); }

double as_double(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1 && PyErr_Occurred()) throw Failed();
  return v;
}

int64_t as_int(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Failed();
  return v;
}

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return ODC_OPS_BF16;
    case at::kHalf: return ODC_OPS_F16;
    case at::kFloat: return ODC_OPS_F32;
    default: return ODC_OPS_NONE;
  }
}

int32_t float_code(const char* what, const at::Tensor& t) {
  const int32_t code = dtype_code(t.scalar_type());
  if (code == ODC_OPS_NONE) raise(PyExc_TypeError, "%s: bf16, fp16 or fp32 is supported, not %s", what, at::toString(t.scalar_type()));
  return code;
}

void expect_gpu(const char* what, const at::Tensor& t) {
  if (!t.is_cuda() || t.layout() != at::kStrided) raise(PyExc_TypeError, "%s: expected a dense tensor on the GPU", what);
}

// `device` is a GPU. (A tensor that is not dense has no data pointer: asking for it raises.)
void expect_device(const char* what, const at::Tensor& t, const at::Device& device) {
  if (t.device() == device) return;
  expect_gpu(what, t);
  if (t.device() != device) raise(PyExc_ValueError, "%s is on %s, not on %s", what, t.device().str().c_str(), device.str().c_str());
}

// These calls are no operations to torch's dispatcher. A program that records operations would have recorded the
// allocation of their results alone.
void expect_no_tracing(const char* call) {
  if (at::tracer::impl::is_dispatch_enabled() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
    raise(PyExc_NotImplementedError, "%s cannot be traced: it is no operation of torch's", call);
}

// A tangent that the result would not have is one that is taken for zero.
class ForwardMode {
 public:
  ForwardMode() : on_(torch::autograd::ForwardADLevel::try_get_by_idx(0) && c10::AutogradState::get_tls_state().get_fw_grad_mode()) {}
  void expect_no_tangent(const char* what, const at::Tensor& t) const {
    if (on_ && t.defined() && t._fw_grad(0).defined()) raise(PyExc_NotImplementedError, "%s: forward-mode derivatives are not supported", what);
  }

 private:
  bool on_;  // whether any tensor can have one: of hundreds in a list, each is asked only then
};

void* current_stream(const at::Device& device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

// Of a call that is made without the GIL.
void check_status(int status) {
  TORCH_CHECK(status == ODC_OPS_OK, "libodc_ops: ", p_ops_last_error(), " (status ", status, ")");
}

// A kernel of this library wrote `t`: autograd sees that it changed, as after an operation of torch's own.
void mark_written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Memory that holds a tensor's values: torch puts a sign off (`x.conj().imag`), and the memory then has the other one.
at::Tensor contiguous(const at::Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }

// ------------------------------------------------------------------------------------------------
// layer norm
// ------------------------------------------------------------------------------------------------
// A tensor as rows of `width` neighbours at one stride. One that is not laid out so is copied first.
struct Rows {
  at::Tensor tensor;
  uint64_t stride = 0;

  Rows() = default;
  Rows(const at::Tensor& t, int64_t dims, int64_t width) {
    if (!t.defined()) return;
    tensor = t;
    if (!t.is_neg() && row_stride(t, dims, width, &stride)) return;
    tensor = contiguous(t);
    stride = (uint64_t)width;
  }

  const void* data() const { return tensor.defined() ? tensor.data_ptr() : nullptr; }

 private:
  // dims: how many of the last dimensions make a row
  static bool row_stride(const at::Tensor& t, int64_t dims, int64_t width, uint64_t* stride) {
    const auto sizes = t.sizes(), strides = t.strides();
    int64_t d = t.dim() - 1, next = 1;
    for (; d >= t.dim() - dims; --d) {
      if (sizes[(size_t)d] == 1) continue;
      if (strides[(size_t)d] != next) return false;
      next *= sizes[(size_t)d];
    }
    *stride = (uint64_t)width;
    bool known = false;
    for (; d >= 0; --d) {
      if (sizes[(size_t)d] == 1) continue;
      if (!known) *stride = (uint64_t)strides[(size_t)d];
      else if (strides[(size_t)d] != next) return false;
      known = true;
      next = strides[(size_t)d] * sizes[(size_t)d];
    }
    return true;
  }
};

struct NormShape {
  int64_t dims, width, rows;
};

struct NormOutputs {
  at::Tensor output, total, statistics;  // [2][rows]: means, and the reciprocals of the standard deviations
};

void* pointer(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

NormOutputs norm_forward(const at::Tensor& input, const at::Tensor& residual, const at::Tensor& weight, const at::Tensor& bias,
                         const NormShape& shape, double eps, bool keep_statistics) {
  const c10::DeviceGuard guard(input.device());
  const Rows x(input, shape.dims, shape.width), r(residual, shape.dims, shape.width);
  const at::Tensor w = contiguous(weight), b = contiguous(bias);
  NormOutputs out;
  out.output = at::empty(input.sizes(), input.options());
  if (residual.defined()) out.total = at::empty(input.sizes(), input.options());
  if (keep_statistics) {
    out.statistics = at::empty({2, shape.rows}, input.options().dtype(at::kFloat));
  }
  odc_norm_forward call = {};
  call.input = x.data();
  call.residual = r.data();
  call.weight = pointer(w);
  call.bias = pointer(b);
  call.output = out.output.data_ptr();
  call.total = pointer(out.total);
  call.mean = static_cast<float*>(pointer(out.statistics));
  call.rstd = call.mean ? call.mean + shape.rows : nullptr;
  call.rows = (uint64_t)shape.rows;
  call.width = (uint64_t)shape.width;
  call.input_stride = x.stride;
  call.residual_stride = r.stride;
  call.dtype = dtype_code(input.scalar_type());
  call.weight_dtype = w.defined() ? dtype_code(w.scalar_type()) : b.defined() ? dtype_code(b.scalar_type()) : call.dtype;
  call.eps = (float)eps;
  check_status(p_layer_norm(&call, current_stream(input.device())));
  return out;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

using Optional = std::optional<at::Tensor>;

Optional optional(const at::Tensor& t) { return t.defined() ? Optional(t) : std::nullopt; }

struct NormGradients {
  at::Tensor input, weight, bias;
};

struct Wanted {
  bool input, weight, bias;
};

NormGradients norm_backward(const at::Tensor& dy, const at::Tensor& dtotal, const at::Tensor& normalised, const at::Tensor& weight,
                            const at::Tensor& statistics, const NormShape& shape, at::ScalarType weight_type, Wanted wanted) {
  const c10::DeviceGuard guard(normalised.device());
  const Rows g(dy, shape.dims, shape.width), x(normalised, shape.dims, shape.width), t(dtotal, shape.dims, shape.width);
  const at::Tensor w = contiguous(weight);
  NormGradients out;
  at::Tensor workspace;
  odc_norm_backward call = {};
  call.rows = (uint64_t)shape.rows;
  call.width = (uint64_t)shape.width;
  call.dtype = dtype_code(normalised.scalar_type());
  call.weight_dtype = dtype_code(weight_type);
  call.grad_output = g.data();
  call.grad_output_stride = g.stride;
  call.grad_total = t.data();
  call.grad_total_stride = t.stride;
  call.normalised = x.data();
  call.normalised_stride = x.stride;
  call.weight = pointer(w);
  call.mean = static_cast<const float*>(statistics.data_ptr());
  call.rstd = call.mean + shape.rows;
  const auto row_shape = normalised.sizes().slice((size_t)(normalised.dim() - shape.dims));
  if (wanted.input) {
    out.input = at::empty(normalised.sizes(), normalised.options());
    call.grad_input = out.input.data_ptr();
  }
  if (wanted.weight) {
    out.weight = at::empty(row_shape, normalised.options().dtype(weight_type));
    call.grad_weight = out.weight.data_ptr();
  }
  if (wanted.bias) {
    out.bias = at::empty(row_shape, normalised.options().dtype(weight_type));
    call.grad_bias = out.bias.data_ptr();
  }
  if (wanted.weight || wanted.bias) {
    call.workspace_bytes = p_layer_norm_backward_workspace(call.rows, call.width, call.dtype);
    if (call.workspace_bytes) {
      workspace = at::empty({(int64_t)call.workspace_bytes}, normalised.options().dtype(at::kByte));
      call.workspace = workspace.data_ptr();
    }
  }
  check_status(p_layer_norm_backward(&call, current_stream(normalised.device())));
  return out;
}

// The backward pass as a node of its own, for callers that want a graph of it: a second derivative is refused when
// it is asked for, and not silently taken for zero.
class LayerNormBackward : public torch::autograd::Function<LayerNormBackward> {
 public:
  static variable_list forward(AutogradContext*, const at::Tensor& dy, const Optional& dtotal, const at::Tensor& normalised, const Optional& weight,
                               const at::Tensor& statistics, const NormShape& shape, at::ScalarType weight_type, Wanted wanted) {
    const NormGradients out =
        norm_backward(dy, dtotal.value_or(at::Tensor()), normalised, weight.value_or(at::Tensor()), statistics, shape, weight_type, wanted);
    variable_list list = {out.input, out.weight, out.bias};
    for (auto& t : list)
      if (!t.defined()) t = at::empty({0}, normalised.options());
    return list;
  }

  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "layer_norm: a second derivative is not supported");
    return {};
  }
};

class LayerNorm : public torch::autograd::Function<LayerNorm> {
 public:
  static variable_list forward(AutogradContext* ctx, const at::Tensor& input, const Optional& residual_, const Optional& weight_,
                               const Optional& bias_, const NormShape& shape, double eps) {
    const at::Tensor residual = residual_.value_or(at::Tensor()), weight = weight_.value_or(at::Tensor()), bias = bias_.value_or(at::Tensor());
    const NormOutputs out = norm_forward(input, residual, weight, bias, shape, eps, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({residual.defined() ? out.total : input, weight, out.statistics});
    const int64_t bias_dtype = bias.defined() ? (int64_t)bias.scalar_type() : int64_t(-1);
    ctx->saved_data["sizes"] = std::vector<int64_t>{shape.dims, shape.width, shape.rows, residual.defined(), bias_dtype};
    if (residual.defined()) return {out.output, out.total};
    return {out.output};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &normalised = saved[0], &weight = saved[1], &statistics = saved[2];
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const NormShape shape{sizes[0], sizes[1], sizes[2]};
    const bool residual = sizes[3] != 0;
    const int64_t bias_dtype = sizes[4];
    const at::Tensor& dy = grads[0];
    const at::Tensor dtotal = grads.size() > 1 ? grads[1] : at::Tensor();
    // (inputs that were not given have no number here)
    size_t input = 0;
    const bool wants_x = ctx->needs_input_grad(input++);
    const bool wants_r = residual && ctx->needs_input_grad(input++);
    const bool wants_w = weight.defined() && ctx->needs_input_grad(input++);
    const bool wants_b = bias_dtype >= 0 && ctx->needs_input_grad(input++);
    NormGradients out;
    if (!dy.defined()) {  // only the handed on total was used
      out.input = dtotal;
    } else {
      const at::ScalarType weight_type =
          weight.defined() ? weight.scalar_type() : bias_dtype >= 0 ? (at::ScalarType)bias_dtype : normalised.scalar_type();
      const Wanted wanted{wants_x || wants_r, wants_w, wants_b};
      if (at::GradMode::is_enabled()) {
        const variable_list list = LayerNormBackward::apply(dy, optional(dtotal), normalised, optional(weight), statistics, shape, weight_type, wanted);
        out = {list[0], list[1], list[2]};
      } else {
        out = norm_backward(dy, dtotal, normalised, weight, statistics, shape, weight_type, wanted);
      }
    }
    const auto given = [](bool wanted, const at::Tensor& t) { return wanted ? t : at::Tensor(); };
    // (the sizes and eps have no gradients)
    return {given(wants_x, out.input), given(wants_r, out.input), given(wants_w, out.weight), given(wants_b, out.bias), {}, {}};
  }
};

// layer_norm(input, residual or None, normalized_shape, weight or None, bias or None, eps) -> output, or with a
// residual (output, total)
PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 6);
    expect_no_tracing("layer_norm");
    const at::Tensor input = as_tensor(args[0], "input"), residual = as_optional_tensor(args[1], "residual");
    const at::Tensor weight = as_optional_tensor(args[3], "weight"), bias = as_optional_tensor(args[4], "bias");
    const double eps = as_double(args[5]);
    const ForwardMode forward_mode;
    forward_mode.expect_no_tangent("input", input);
    forward_mode.expect_no_tangent("residual", residual);
    forward_mode.expect_no_tangent("weight", weight);
    forward_mode.expect_no_tangent("bias", bias);
    std::vector<int64_t> shape;
    if (PyLong_Check(args[2])) {
      shape.push_back(as_int(args[2]));
    } else {
      const Sequence sizes(args[2], "normalized_shape is an int or a sequence of them");
      for (Py_ssize_t k = 0; k < sizes.size(); ++k) shape.push_back(as_int(sizes[k]));
    }
    expect_gpu("input", input);
    const int32_t code = float_code("input", input);
    const int64_t dims = (int64_t)shape.size();
    const at::IntArrayRef want(shape);
    if (!dims || input.dim() < dims || input.sizes().slice((size_t)(input.dim() - dims)) != want)
      raise(PyExc_ValueError, "the last dimensions of the input are not normalized_shape");
    if (residual.defined()) {
      expect_device("residual", residual, input.device());
      if (residual.scalar_type() != input.scalar_type()) raise(PyExc_TypeError, "residual: expected the dtype of the input");
      if (residual.sizes() != input.sizes()) raise(PyExc_ValueError, "residual: expected the shape of the input");
    }
    at::ScalarType weight_type = at::kByte;
    const std::pair<const char*, const at::Tensor*> parameters[] = {{"weight", &weight}, {"bias", &bias}};
    for (const auto& [name, t] : parameters) {
      if (!t->defined()) continue;
      expect_device(name, *t, input.device());
      const int32_t c = float_code(name, *t);
      if (c != code && c != ODC_OPS_F32) raise(PyExc_TypeError, "%s: expected the dtype of the input or fp32", name);
      if (t->sizes() != want) raise(PyExc_ValueError, "%s: expected the shape normalized_shape", name);
      if (weight_type != at::kByte && t->scalar_type() != weight_type) raise(PyExc_TypeError, "weight and bias have different dtypes");
      weight_type = t->scalar_type();
    }
    if (!(eps >= 0)) raise(PyExc_ValueError, "eps is not negative");
    NormShape rows{dims, 1, 1};
    for (int64_t d = 0; d < input.dim(); ++d) (d < input.dim() - dims ? rows.rows : rows.width) *= input.size(d);
    const bool needs_graph = at::GradMode::is_enabled() &&
                             (input.requires_grad() || (residual.defined() && residual.requires_grad()) ||
                              (weight.defined() && weight.requires_grad()) || (bias.defined() && bias.requires_grad()));
    at::Tensor output, total;
    {
      WithoutGil nobody;
      if (needs_graph) {
        const variable_list out = LayerNorm::apply(input, optional(residual), optional(weight), optional(bias), rows, eps);
        output = out[0];
        if (residual.defined()) total = out[1];
      } else {
        NormOutputs out = norm_forward(input, residual, weight, bias, rows, eps, false);
        output = std::move(out.output);
        total = std::move(out.total);
      }
    }
    PyObject* first = THPVariable_Wrap(std::move(output));
    if (!first || !residual.defined()) return first;
    PyObject* second = THPVariable_Wrap(std::move(total));
    PyObject* pair = second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_DECREF(first);
    Py_XDECREF(second);
    return pair;
  });
}

// ------------------------------------------------------------------------------------------------
// lists of tensors
// ------------------------------------------------------------------------------------------------
// squared_norm(tensors) -> a scalar tensor, or None where the dtypes differ
PyObject* squared_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 1);
    expect_no_tracing("squared_norm");
    const Sequence tensors(args[0], "tensors are a sequence");
    if (!tensors.size()) raise(PyExc_ValueError, "the squared norm of no tensors has no device to be on");
    std::vector<odc_span_item> items;
    std::vector<at::Tensor> copies;  // of what is not dense
    torch::autograd::edge_list inputs;  // a derivative that is asked for is refused, and not silently taken for zero
    items.reserve((size_t)tensors.size());
    const at::Tensor& first = as_tensor(tensors[0], "tensors");
    const ForwardMode forward_mode;
    forward_mode.expect_no_tangent("tensors", first);
    const bool graph = at::GradMode::is_enabled();
    expect_gpu("tensors", first);
    const int32_t code = float_code("tensors", first);
    for (Py_ssize_t k = 0; k < tensors.size(); ++k) {
      const at::Tensor& t = as_tensor(tensors[k], "tensors");
      forward_mode.expect_no_tangent("tensors", t);
      expect_device("tensors", t, first.device());
      if (float_code("tensors", t) != code) Py_RETURN_NONE;
      if (graph && t.requires_grad()) inputs.push_back(torch::autograd::impl::gradient_edge(t));
      if (t.is_non_overlapping_and_dense()) {
        items.push_back({t.data_ptr(), (uint64_t)t.numel()});
      } else {
        const c10::DeviceGuard guard(first.device());
        const at::AutoGradMode no_graph(false);
        copies.push_back(t.contiguous());
        items.push_back({copies.back().data_ptr(), (uint64_t)t.numel()});
      }
    }
    at::Tensor result;
    {
      WithoutGil nobody;
      const c10::DeviceGuard guard(first.device());
      const at::AutoGradMode no_graph(false);
      const uint32_t count = (uint32_t)items.size();
      const uint64_t bytes = p_squared_norm_workspace(items.data(), count, code);
      result = at::empty({}, first.options().dtype(at::kFloat));
      const at::Tensor workspace = at::empty({(int64_t)bytes}, first.options().dtype(at::kByte));
      check_status(p_squared_norm(items.data(), count, code, workspace.data_ptr(), bytes, static_cast<float*>(result.data_ptr()),
                                  current_stream(first.device())));
    }
    if (!inputs.empty())
      torch::autograd::set_history(result, std::shared_ptr<torch::autograd::Error>(
                                               new torch::autograd::Error("squared_norm: a derivative is not supported", std::move(inputs)),
                                               torch::autograd::deleteNode));
    return THPVariable_Wrap(std::move(result));
  });
}

// A tensor that is written is its memory (contiguous()).
void expect_no_sign_put_off(const char* name, const at::Tensor& t, Py_ssize_t k) {
  if (t.is_neg()) raise(PyExc_ValueError, "%s: tensor %zd is a view whose sign was put off: it cannot be written", name, k);
}

bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  if (a.dim() == 1 && b.dim() == 1) return a.numel() == b.numel() && a.is_contiguous() && b.is_contiguous();
  return a.sizes() == b.sizes() && (a.strides() == b.strides() || (a.is_contiguous() && b.is_contiguous()));
}

// The tensors of one list beside the parameters, which all have one dtype.
class Beside {
 public:
  Beside(PyObject* o, const char* name, Py_ssize_t n) : name_(name), given_(o != Py_None), items_(given_ ? o : empty(), "lists of tensors are sequences") {
    if (given_ && items_.size() != n) raise(PyExc_ValueError, "%s: %zd tensors for %zd parameters", name, items_.size(), n);
  }

  bool given() const { return given_; }
  at::ScalarType dtype() const { return dtype_; }

  const at::Tensor& at(Py_ssize_t k, const at::Device& device) {
    const at::Tensor& t = as_tensor(items_[k], name_);
    expect_device(name_, t, device);
    if (k == 0) dtype_ = t.scalar_type();
    if (t.scalar_type() != dtype_) raise(PyExc_TypeError, "%s: tensors of one call have one dtype", name_);
    return t;
  }

  // laid out as the parameter is
  void* like(Py_ssize_t k, const at::Tensor& param) {
    if (!given_) return nullptr;
    const at::Tensor& t = at(k, param.device());
    if (!same_layout(t, param)) raise(PyExc_ValueError, "%s: tensor %zd is not laid out as its parameter is", name_, k);
    expect_no_sign_put_off(name_, t, k);
    return t.data_ptr();
  }

  // the same, of what is only read
  const void* read_like(Py_ssize_t k, const at::Tensor& param) {
    if (!THPVariable_Check(items_[k]) || !THPVariable_Unpack(items_[k]).is_neg()) return like(k, param);
    resolved_.push_back(at(k, param.device()).resolve_neg());
    if (!same_layout(resolved_.back(), param)) raise(PyExc_ValueError, "%s: tensor %zd is not laid out as its parameter is", name_, k);
    return resolved_.back().data_ptr();
  }

  // `numel` values in the order of the memory
  void* flat(Py_ssize_t k, const at::Device& device, int64_t numel) {
    if (!given_) return nullptr;
    const at::Tensor& t = at(k, device);
    if (t.numel() != numel || !t.is_contiguous()) raise(PyExc_ValueError, "%s: tensor %zd: expected %lld contiguous elements", name_, k, (long long)numel);
    return t.data_ptr();
  }

  void expect(at::ScalarType dtype) const {
    if (given_ && items_.size() && dtype_ != dtype) raise(PyExc_TypeError, "%s: expected %s, not %s", name_, at::toString(dtype), at::toString(dtype_));
  }

  void mark() const {
    for (Py_ssize_t k = 0; given_ && k < items_.size(); ++k) mark_written(THPVariable_Unpack(items_[k]));
  }

 private:
  static PyObject* empty() {
    static PyObject* nothing = PyTuple_New(0);
    return nothing;
  }

  const char* name_;
  bool given_;
  Sequence items_;
  std::vector<at::Tensor> resolved_;
  at::ScalarType dtype_ = at::kByte;
};

constexpr int64_t kBlock = 32;

// A call of odc_adamw: its tensors, held and checked, and the structures that name them.
class AdamwCall {
 public:
  // params, grads, exp_avgs, exp_avg_scales or None, exp_avg_sqs or roots, their scales or None, copies or None,
  // squared_norm or None, step, lr, beta1, beta2, eps, weight_decay, grad_scale, max_norm, seed or None
  static constexpr Py_ssize_t kArguments = 17;

  explicit AdamwCall(PyObject* const* args)
      : params_(args[0], "params are a sequence"),
        count_(params_.size()),
        grads_(args[1], "grads", count_),
        m_(args[2], "exp_avgs", count_),
        m_scale_(args[3], "exp_avg_scales", count_),
        v_(args[4], args[3] == Py_None ? "exp_avg_sqs" : "exp_avg_roots", count_),
        v_scale_(args[5], "exp_avg_root_scales", count_),
        copies_(args[6], "copies", count_),
        squared_norm_(as_optional_tensor(args[7], "squared_norm")) {
    const bool eight = m_scale_.given();
    const int64_t step = as_int(args[8]);
    if (step < 1) raise(PyExc_ValueError, "the first step is 1");
    numbers_.step = (uint64_t)step;
    numbers_.lr = as_double(args[9]);
    numbers_.beta1 = as_double(args[10]);
    numbers_.beta2 = as_double(args[11]);
    numbers_.eps = as_double(args[12]);
    numbers_.weight_decay = as_double(args[13]);
    numbers_.grad_scale = as_double(args[14]);
    numbers_.max_norm = as_double(args[15]);
    if (args[16] != Py_None) {
      PyObject* masked = PyNumber_Index(args[16]);
      if (!masked) throw Failed();
      numbers_.seed = (uint32_t)PyLong_AsUnsignedLongLongMask(masked);  // its low 32 bits
      Py_DECREF(masked);
      numbers_.stochastic = 1;
    } else if (eight) {
      raise(PyExc_ValueError, "states in 8 bits are rounded by random numbers: give a seed, another one for every step");
    }
    if (!count_) return;
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    items_.reserve((size_t)count_);
    spans.reserve((size_t)count_);
    const at::Tensor& first = as_tensor(params_[0], "params");
    expect_gpu("params", first);
    for (Py_ssize_t k = 0; k < count_; ++k) {
      const at::Tensor& p = as_tensor(params_[k], "params");
      expect_device("params", p, first.device());
      if (p.scalar_type() != first.scalar_type()) raise(PyExc_TypeError, "params: tensors of one call have one dtype");
      if (!p.is_non_overlapping_and_dense()) raise(PyExc_ValueError, "params: tensor %zd is not dense", k);
      expect_no_sign_put_off("params", p, k);
      odc_adamw_item item = {};
      const int64_t numel = p.numel(), blocks = (numel + kBlock - 1) / kBlock;
      item.elems = (uint64_t)numel;
      item.param = p.data_ptr();
      item.grad = grads_.read_like(k, p);
      item.exp_avg = eight ? m_.flat(k, p.device(), numel) : m_.like(k, p);
      item.exp_avg_sq = eight ? v_.flat(k, p.device(), numel) : v_.like(k, p);
      item.exp_avg_scale = m_scale_.flat(k, p.device(), blocks);
      item.exp_avg_sq_scale = v_scale_.flat(k, p.device(), blocks);
      item.copy = copies_.like(k, p);
      items_.push_back(item);
      if (numel) spans.emplace_back((uintptr_t)item.param, (uintptr_t)item.param + (uintptr_t)numel * p.element_size());
    }
    if (!std::is_sorted(spans.begin(), spans.end())) std::sort(spans.begin(), spans.end());  // (the allocator's order, as a rule)
    for (size_t k = 1; k < spans.size(); ++k)
      if (spans[k].first < spans[k - 1].second) raise(PyExc_ValueError, "params: two tensors overlap");
    numbers_.param_dtype = float_code("params", first);
    if (numbers_.param_dtype == ODC_OPS_F16) raise(PyExc_TypeError, "params: fp32 or bf16 is supported, not Half");
    numbers_.grad_dtype = dtype_code(grads_.dtype());
    if (numbers_.grad_dtype == ODC_OPS_NONE) raise(PyExc_TypeError, "grads: bf16, fp16 or fp32 is supported, not %s", at::toString(grads_.dtype()));
    numbers_.copy_dtype = copies_.given() ? dtype_code(copies_.dtype()) : (int32_t)ODC_OPS_NONE;
    if (copies_.given() && (numbers_.copy_dtype < 0 || numbers_.copy_dtype == ODC_OPS_F32 || numbers_.param_dtype != ODC_OPS_F32))
      raise(PyExc_TypeError, "copies: bf16 or fp16, of fp32 parameters");
    numbers_.state_bits = eight ? 8 : 32;
    for (const Beside* states : {&m_, &v_}) states->expect(eight ? at::kFloat8_e4m3fn : at::kFloat);
    for (const Beside* scales : {&m_scale_, &v_scale_}) scales->expect(at::kFloat8_e8m0fnu);
    if (squared_norm_.defined()) {
      squared_norm_ = squared_norm_.resolve_neg();
      expect_device("squared_norm", squared_norm_, first.device());
      if (squared_norm_.numel() != 1 || squared_norm_.scalar_type() != at::kFloat) raise(PyExc_TypeError, "squared_norm: expected one fp32 value");
      numbers_.squared_norm = static_cast<const float*>(squared_norm_.data_ptr());
    }
  }

  // The checks of the C ABI's side.
  void check() const {
    if (count_) check_status(p_adamw_check(items_.data(), (uint32_t)count_, &numbers_));
  }

  void launch() const {
    if (!count_) return;
    {
      const at::Device device = THPVariable_Unpack(params_[0]).device();
      WithoutGil nobody;
      const c10::DeviceGuard guard(device);
      check_status(p_adamw(items_.data(), (uint32_t)count_, &numbers_, current_stream(device)));
    }
    for (Py_ssize_t k = 0; k < count_; ++k) mark_written(THPVariable_Unpack(params_[k]));
    for (const Beside* written : {&m_, &m_scale_, &v_, &v_scale_, &copies_}) written->mark();
  }

 private:
  Sequence params_;
  Py_ssize_t count_;
  Beside grads_, m_, m_scale_, v_, v_scale_, copies_;
  at::Tensor squared_norm_;
  odc_adamw_numbers numbers_ = {};
  std::vector<odc_adamw_item> items_;
};

// adamw(AdamwCall's arguments)
PyObject* adamw(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, AdamwCall::kArguments);
    expect_no_tracing("adamw_step");
    AdamwCall(args).launch();
    Py_RETURN_NONE;
  });
}

constexpr const char* kPrepared = "odc_ops_torch.adamw_prepare";

// adamw_prepare(AdamwCall's arguments) -> a call that nothing is wrong with, for adamw_launch
PyObject* adamw_prepare(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, AdamwCall::kArguments);
    expect_no_tracing("adamw_step");
    auto call = std::make_unique<AdamwCall>(args);
    call->check();
    PyObject* capsule = PyCapsule_New(call.get(), kPrepared, [](PyObject* c) { delete static_cast<AdamwCall*>(PyCapsule_GetPointer(c, kPrepared)); });
    if (capsule) (void)call.release();
    return capsule;
  });
}

// adamw_launch(what adamw_prepare returned)
PyObject* adamw_launch(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 1);
    const auto* call = static_cast<const AdamwCall*>(PyCapsule_GetPointer(args[0], kPrepared));
    if (!call) throw Failed();
    call->launch();
    Py_RETURN_NONE;
  });
}

// dequantize_blocks(codes, scales, dtype) -> values
PyObject* dequantize_blocks(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 3);
    expect_no_tracing("dequantize_blocks");
    const at::Tensor &codes = as_tensor(args[0], "codes"), &scales = as_tensor(args[1], "scales");
    if (!THPDtype_Check(args[2])) raise(PyExc_TypeError, "expected a torch.dtype, got %s", Py_TYPE(args[2])->tp_name);
    const at::ScalarType type = reinterpret_cast<THPDtype*>(args[2])->scalar_type;
    if (dtype_code(type) == ODC_OPS_NONE) raise(PyExc_TypeError, "dtype: bf16, fp16 or fp32 is supported, not %s", at::toString(type));
    expect_gpu("codes", codes);
    expect_device("scales", scales, codes.device());
    if (codes.scalar_type() != at::kFloat8_e4m3fn || scales.scalar_type() != at::kFloat8_e8m0fnu)
      raise(PyExc_TypeError, "codes are float8_e4m3fn, scales float8_e8m0fnu");
    if (!codes.is_contiguous() || !scales.is_contiguous() || scales.numel() != (codes.numel() + kBlock - 1) / kBlock)
      raise(PyExc_ValueError, "codes and scales are contiguous, with a scale for every 32 codes");
    at::Tensor values;
    {
      WithoutGil nobody;
      const c10::DeviceGuard guard(codes.device());
      values = at::empty(codes.sizes(), codes.options().dtype(type));
      check_status(p_dequantize_blocks(codes.data_ptr(), scales.data_ptr(), values.data_ptr(), (uint64_t)codes.numel(), dtype_code(type),
                                       current_stream(codes.device())));
    }
    return THPVariable_Wrap(std::move(values));
  });
}

PyMethodDef module_methods[] = {
#define ODC_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
    ODC_METHOD(bind),
    ODC_METHOD(layer_norm),
    ODC_METHOD(squared_norm),
    ODC_METHOD(adamw),
    ODC_METHOD(adamw_prepare),
    ODC_METHOD(adamw_launch),
    ODC_METHOD(dequantize_blocks),
#undef ODC_METHOD
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "odc_ops_torch", nullptr, -1, module_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_odc_ops_torch(void) {
  PyObject* module = PyModule_Create(&module_def);
#define ODC_TEXT_(x) #x
#define ODC_TEXT(x) ODC_TEXT_(x)
  if (module && PyModule_AddStringConstant(module, "built_for",
                                           "ABI " ODC_TEXT(ODC_OPS_ABI_VERSION) ", torch " ODC_TORCH_VERSION
                                           ", CPython " ODC_TEXT(PY_MAJOR_VERSION) "." ODC_TEXT(PY_MINOR_VERSION)) < 0) {
    Py_DECREF(module);
    return nullptr;
  }
  return module;
}
