// torch binding of the 8-bit operators (include/rns8/rns8_quant.h): takes and
// returns torch tensors, checks them, allocates results and scratch from
// torch's caching allocator and calls the library on the current stream.
// rns8_b200/quant.py documents the functions and holds what is not on the way
// of a call (autograd, result types). In Python the same steps cost about 8 us
// a call on the host, more than the smallest operators take on the GPU.
//
// The library's entry points are handed in by address (bind), so that this
// module uses the library that rns8_b200.abi loaded. Nothing throws past an
// entry point: every exception becomes a Python one.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "rns8/rns8_quant.h"

namespace {

struct Library {
  rns8_status (*quantize_rows)(const rns8_cuda_quantize_desc*);
  uint64_t (*linear_scratch)(const rns8_cuda_linear_desc*);
  rns8_status (*linear)(const rns8_cuda_linear_desc*);
  rns8_status (*norm)(const rns8_cuda_residual_norm_desc*);
  uint64_t (*norm_backward_scratch)(const rns8_cuda_residual_norm_backward_desc*);
  rns8_status (*norm_backward)(const rns8_cuda_residual_norm_backward_desc*);
} lib;
PyObject* check_status = nullptr;   // (status, where) -> raises
PyObject* status_address = nullptr;  // (device) -> address of its status word
PyObject* out_of_memory = nullptr;   // torch's exception for it

// A Python exception on its way out.
struct Refused {
  PyObject* type;
  std::string what;
};
struct AlreadySet {};
[[noreturn]] void value_error(std::string what) { throw Refused{PyExc_ValueError, std::move(what)}; }
[[noreturn]] void type_error(std::string what) { throw Refused{PyExc_TypeError, std::move(what)}; }

template <typename F>
PyObject* guarded(F&& f) noexcept {
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.what.c_str());
  } catch (const AlreadySet&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(out_of_memory ? out_of_memory : PyExc_MemoryError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

void expect(rns8_status status, const char* where) {
  if (status == RNS8_SUCCESS) return;
  PyObject* r = PyObject_CallFunction(check_status, "Is", static_cast<unsigned>(status), where);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s: status %u", where, static_cast<unsigned>(status));
  throw AlreadySet{};
}

uint32_t* status_word(int device) {
  // The words live as long as the process, one a device (device_status sees to
  // that). The GIL guards the table: only the call below lets other threads run.
  static std::vector<uint32_t*> known;
  if (device < static_cast<int>(known.size()) && known[device]) return known[device];
  PyObject* r = PyObject_CallFunction(status_address, "i", device);
  if (!r) throw AlreadySet{};
  uint32_t* word = static_cast<uint32_t*>(PyLong_AsVoidPtr(r));
  Py_DECREF(r);
  if (PyErr_Occurred()) throw AlreadySet{};
  if (device >= static_cast<int>(known.size())) known.resize(device + 1, nullptr);
  return known[device] = word;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) type_error(std::string(name) + ": expected a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor* optional_tensor(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

uint32_t float_type(at::ScalarType t, const char* name) {
  if (t == at::kBFloat16) return RNS8_CUDA_TYPE_BF16;
  if (t == at::kHalf) return RNS8_CUDA_TYPE_F16;
  if (t == at::kFloat) return RNS8_CUDA_TYPE_F32;
  type_error(std::string(name) + ": expected bfloat16, float16 or float32, got " + c10::toString(t));
}

int cuda_device(const at::Tensor& t, const char* name) {
  if (!t.is_cuda()) value_error(std::string(name) + ": expected a CUDA tensor");
  return t.get_device();
}
void expect_device(const at::Tensor& t, int device, const char* name) {
  if (!t.is_cuda() || t.get_device() != device)
    value_error(std::string(name) + ": expected a tensor on cuda:" + std::to_string(device));
}

// A tensor as rows of its last dimension. `held` keeps the copy alive that a
// tensor without such a view, or whose rows share memory, needs.
struct Rows {
  void* data;
  int64_t rows, cols, ld;
  at::Tensor held;
};
Rows rows_of(const at::Tensor& t, const char* name) {
  Rows r{};
  if (t.dim() == 0) value_error(std::string(name) + ": expected at least one dimension");
  const at::Tensor* two = &t;
  r.cols = t.size(-1);
  if (t.dim() != 2) {
    if (t.is_contiguous()) {
      r.rows = 1;
      for (int64_t d = 0; d + 1 < t.dim(); ++d) r.rows *= t.size(d);
      r.ld = std::max<int64_t>(r.cols, 1);
      r.data = t.data_ptr();
      return r;
    }
    int64_t rows = 1;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) rows *= t.size(d);
    r.held = t.reshape({rows, r.cols});
    two = &r.held;
  }
  r.rows = two->size(0);
  if (r.cols > 1 && two->stride(1) != 1) value_error(std::string(name) + ": elements of a row must be contiguous");
  r.ld = r.rows > 1 ? two->stride(0) : std::max<int64_t>(r.cols, 1);
  if (r.ld < r.cols) {  // rows that share memory, as of expand()
    r.held = two->contiguous();
    two = &r.held;
    r.ld = r.cols;
  }
  r.data = two->data_ptr();
  return r;
}

const float* f32_vector(const at::Tensor& t, int64_t size, int device, const char* name) {
  if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != size || !t.is_contiguous())
    type_error(std::string(name) + ": expected a contiguous float32 vector of " + std::to_string(size));
  expect_device(t, device, name);
  return static_cast<const float*>(t.data_ptr());
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int device) {
  return at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)), std::nullopt);
}
// Shape of t with its last dimension replaced.
std::vector<int64_t> with_last(const at::Tensor& t, int64_t last) {
  std::vector<int64_t> s(t.sizes().begin(), t.sizes().end());
  s.back() = last;
  return s;
}
// int8 rows in the shape of t with `cols` columns, each on a 16-byte boundary.
at::Tensor empty_q(const at::Tensor& t, int64_t cols, int device) {
  const int64_t ld = (cols + 15) / 16 * 16;
  at::Tensor q = empty(with_last(t, ld), at::kChar, device);
  return ld == cols ? q : q.narrow(-1, 0, cols);
}
void* stream_of(int device) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}

template <typename D>
D header(int device) {
  D d{};
  d.struct_size = sizeof(D);
  d.abi_version = RNS8_ABI_VERSION;
  d.device_id = device;
  return d;
}

PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
  PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (!t) throw AlreadySet{};
  Py_ssize_t i = 0;
  for (const at::Tensor& x : tensors) {
    PyObject* o = x.defined() ? THPVariable_Wrap(x) : Py_NewRef(Py_None);
    if (!o) {
      Py_DECREF(t);
      throw AlreadySet{};
    }
    PyTuple_SET_ITEM(t, i++, o);
  }
  return t;
}

void expect_args(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) type_error("expected " + std::to_string(want) + " arguments");
}

bool wants_gradient(PyObject* o) { return o != Py_None && THPVariable_Check(o) && THPVariable_Unpack(o).requires_grad(); }
// A dual tensor of forward-mode differentiation, which is independent of the
// recording of gradients.
bool has_tangent(PyObject* o) {
  return o != Py_None && THPVariable_Check(o) && c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
         THPVariable_Unpack(o)._fw_grad(/*level=*/0).defined();
}

// Operators without a derivative. Forward mode has none to give: refused before
// the call. A gradient is refused where it is asked for, as by torch's own: the
// results carry a function that raises, so that inference with parameters needs
// no torch.no_grad().
void expect_no_tangents(const char* name, std::initializer_list<PyObject*> inputs) {
  for (PyObject* o : inputs)
    if (has_tangent(o)) throw Refused{PyExc_NotImplementedError, std::string(name) + " has no forward-mode derivative"};
}
void mark_underivable(const char* name, std::initializer_list<PyObject*> inputs, std::initializer_list<at::Tensor> results) {
  if (!at::GradMode::is_enabled()) return;
  std::vector<at::Tensor> from;
  for (PyObject* o : inputs)
    if (wants_gradient(o)) from.push_back(THPVariable_Unpack(o));
  if (from.empty()) return;
  auto node = std::shared_ptr<torch::autograd::NotImplemented>(
      new torch::autograd::NotImplemented(name, torch::autograd::collect_next_edges(from)), torch::autograd::deleteNode);
  for (const at::Tensor& r : results)
    if (r.defined() && r.is_floating_point()) torch::autograd::set_history(r, node);
}

// ---- bind(quantize, linear_scratch, linear, norm, backward_scratch, backward, check, status, oom) ----
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 9);
    void* p[6];
    for (int i = 0; i < 6; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) throw AlreadySet{};
    lib.quantize_rows = reinterpret_cast<decltype(lib.quantize_rows)>(p[0]);
    lib.linear_scratch = reinterpret_cast<decltype(lib.linear_scratch)>(p[1]);
    lib.linear = reinterpret_cast<decltype(lib.linear)>(p[2]);
    lib.norm = reinterpret_cast<decltype(lib.norm)>(p[3]);
    lib.norm_backward_scratch = reinterpret_cast<decltype(lib.norm_backward_scratch)>(p[4]);
    lib.norm_backward = reinterpret_cast<decltype(lib.norm_backward)>(p[5]);
    Py_XSETREF(check_status, Py_NewRef(a[6]));
    Py_XSETREF(status_address, Py_NewRef(a[7]));
    Py_XSETREF(out_of_memory, Py_NewRef(a[8]));
    Py_RETURN_NONE;
  });
}

// ---- quantize_rows(x) -> (q, scale) ----
PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 1);
    const at::Tensor& x = tensor(a[0], "x");
    expect_no_tangents("quantize_rows", {a[0]});
    auto d = header<rns8_cuda_quantize_desc>(0);
    d.x_type = float_type(x.scalar_type(), "x");
    d.device_id = cuda_device(x, "x");
    const Rows r = rows_of(x, "x");
    if (r.cols == 0) value_error("x: rows are empty");
    at::Tensor q = empty_q(x, r.cols, d.device_id);
    at::Tensor scale = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, d.device_id);
    d.rows = r.rows, d.cols = r.cols, d.ld_x = r.ld, d.ld_q = (r.cols + 15) / 16 * 16;
    d.x = r.data, d.q = static_cast<int8_t*>(q.data_ptr()), d.scale = static_cast<float*>(scale.data_ptr());
    d.stream = stream_of(d.device_id);
    expect(lib.quantize_rows(&d), "rns8_cuda_quantize_rows_device");
    mark_underivable("quantize_rows", {a[0]}, {scale});
    return tuple_of({q, scale});
  });
}

// ---- linear(x, x_scale or None, w, w_scale, bias or None, gated, out_dtype or None, quantize) ----
// x int8 with x_scale, else floating. -> tensor, or (q, scale) with quantize.
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 8);
    const at::Tensor& x = tensor(a[0], "activations");
    const at::Tensor* x_scale = optional_tensor(a[1], "a_scale");
    const at::Tensor& w = tensor(a[2], "w");
    expect_no_tangents("the int8 product", {a[0], a[1], a[3], a[4]});
    const bool gated = a[5] == Py_True, quantize = a[7] == Py_True;
    const int device = cuda_device(x, "activations");
    auto d = header<rns8_cuda_linear_desc>(device);
    if (x_scale) {
      if (x.scalar_type() != at::kChar) type_error(std::string("a: expected int8, got ") + c10::toString(x.scalar_type()));
      if (x_scale->scalar_type() != at::kFloat || x_scale->sizes() != x.sizes().slice(0, std::max<int64_t>(x.dim(), 1) - 1) ||
          !x_scale->is_contiguous())
        type_error("a_scale: expected a contiguous float32 tensor with one value per row of a");
      expect_device(*x_scale, device, "a_scale");
      d.a_type = RNS8_CUDA_TYPE_I8;
      d.a_scale = static_cast<const float*>(x_scale->data_ptr());
    } else {
      d.a_type = float_type(x.scalar_type(), "x");
    }
    const Rows r = rows_of(x, "activations");
    if (w.scalar_type() != at::kChar || w.dim() != 2) type_error("w: expected a 2-D int8 tensor (output channels x inputs)");
    const int64_t w_rows = w.size(0);
    if (w.size(1) != r.cols)
      value_error("w: expected rows of " + std::to_string(r.cols) + ", got " + std::to_string(w.size(1)));
    if (gated && w_rows % 2) value_error("w: a gated product needs an even number of rows (gate rows, then up rows)");
    d.m = r.rows, d.n = gated ? w_rows / 2 : w_rows, d.k = r.cols;
    if (d.n == 0 || d.k == 0) value_error("w: empty");
    expect_device(w, device, "w");
    const Rows wr = rows_of(w, "w");
    d.w_scale = f32_vector(tensor(a[3], "w_scale"), w_rows, device, "w_scale");
    if (const at::Tensor* bias = optional_tensor(a[4], "bias")) d.bias = f32_vector(*bias, w_rows, device, "bias");
    at::ScalarType type = x.scalar_type();
    if (a[6] != Py_None) {
      if (!THPDtype_Check(a[6])) type_error("out_dtype: expected a torch.dtype");
      type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
    }
    d.out_type = float_type(type, "out_dtype");
    d.flags = gated ? RNS8_CUDA_LINEAR_GATED : 0;
    at::Tensor out, out_scale;
    if (quantize) {
      d.out_type = RNS8_CUDA_TYPE_I8;
      out = empty_q(x, d.n, device);
      out_scale = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, device);
      d.out_scale = static_cast<float*>(out_scale.data_ptr());
      d.ld_out = (d.n + 15) / 16 * 16;
    } else {
      out = empty(with_last(x, d.n), type, device);
      d.ld_out = d.n;
    }
    if (d.m) {
      d.ld_a = r.ld, d.ld_w = wr.ld;
      d.a = r.data, d.w = static_cast<const int8_t*>(wr.data), d.out = out.data_ptr();
      d.scratch_bytes = lib.linear_scratch(&d);
      at::Tensor scratch;
      if (d.scratch_bytes) {
        scratch = empty({static_cast<int64_t>(d.scratch_bytes)}, at::kByte, device);
        d.scratch = scratch.data_ptr();
      }
      d.status = status_word(device);
      d.stream = stream_of(device);
      expect(lib.linear(&d), "rns8_cuda_linear_device");
    }
    mark_underivable("the int8 product", {a[0], a[1], a[3], a[4]}, {quantize ? out_scale : out});
    return quantize ? tuple_of({out, out_scale}) : THPVariable_Wrap(out);
  });
}

// ---- norms ----
constexpr int64_t kMaxDim = 32768;

// x, y and the parameters of a norm, checked; D is either descriptor.
struct NormArgs {
  Rows x, y, gate;
  const at::Tensor* gate_tensor;
  int64_t groups;
};
template <typename D>
NormArgs norm_args(D& d, const at::Tensor& x, const char* x_name, const at::Tensor& y, PyObject* post_o, PyObject* pre_o,
                   PyObject* gate_o, PyObject* scale, PyObject* eps, PyObject* offset) {
  NormArgs n{};
  d.type = float_type(x.scalar_type(), x_name);
  d.device_id = cuda_device(x, x_name);
  if (y.sizes() != x.sizes() || y.scalar_type() != x.scalar_type())
    value_error(std::string("y: expected ") + x_name + "'s type and shape");
  expect_device(y, d.device_id, "y");
  n.x = rows_of(x, x_name);
  n.y = rows_of(y, "y");
  d.tokens = n.x.rows, d.dim = n.x.cols;
  if (d.dim < 1 || d.dim > kMaxDim)
    value_error(std::string(x_name) + ": rows must have 1 to " + std::to_string(kMaxDim) + " elements");
  at::ScalarType type = x.scalar_type();
  bool typed = false;
  auto join_type = [&](const at::Tensor& t, const char* name) {
    if (typed && t.scalar_type() != type) type_error(std::string(name) + ": the weights and the gate share one type");
    type = t.scalar_type();
    typed = true;
  };
  auto vector = [&](PyObject* o, const char* name) -> const void* {
    const at::Tensor* t = optional_tensor(o, name);
    if (!t) return nullptr;
    if (t->dim() != 1 || t->size(0) != d.dim || !t->is_contiguous())
      value_error(std::string(name) + ": expected a contiguous vector of " + std::to_string(d.dim));
    expect_device(*t, d.device_id, name);
    join_type(*t, name);
    return t->data_ptr();
  };
  d.post_weight = vector(post_o, "post_weight");
  d.pre_weight = vector(pre_o, "pre_weight");
  n.gate_tensor = optional_tensor(gate_o, "gate");
  d.groups = 1, d.ld_gate = d.dim;
  if (n.gate_tensor) {
    n.gate = rows_of(*n.gate_tensor, "gate");
    if (n.gate.cols != d.dim) value_error("gate: expected rows of " + std::to_string(d.dim));
    expect_device(*n.gate_tensor, d.device_id, "gate");
    join_type(*n.gate_tensor, "gate");
    d.groups = n.gate.rows, d.ld_gate = n.gate.ld, d.gate = n.gate.data;
    if (d.tokens && (d.groups == 0 || d.tokens % d.groups))
      value_error("gate: " + std::to_string(d.groups) + " rows do not divide " + std::to_string(d.tokens) + " tokens");
  }
  if (type != x.scalar_type() && type != at::kFloat)
    type_error(std::string("weights: expected ") + c10::toString(x.scalar_type()) + " or float32, got " + c10::toString(type));
  d.weight_type = float_type(type, "weights");
  d.scale = static_cast<float>(PyFloat_AsDouble(scale));
  d.eps = static_cast<float>(PyFloat_AsDouble(eps));
  d.weight_offset = static_cast<float>(PyFloat_AsDouble(offset));
  if (PyErr_Occurred()) throw AlreadySet{};
  d.ld_y = n.y.ld, d.y = n.y.data;
  d.stream = stream_of(d.device_id);
  return n;
}


// ---- residual_norm(x, y, post, pre, gate, scale, eps, offset, form) ----
// form 0: (x_out, h), or None where a derivative is wanted (the caller records
// it, or refuses); 1: (x_out, h) whatever is wanted; 2: (x_out, q, q_scale).
PyObject* residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 9);
    const long form = PyLong_AsLong(a[8]);
    if (PyErr_Occurred()) throw AlreadySet{};
    const at::Tensor& x = tensor(a[0], "x");
    const at::Tensor& y = tensor(a[1], "y");
    if (form == 0)
      for (int i = 0; i < 5; ++i)
        if ((at::GradMode::is_enabled() && wants_gradient(a[i])) || has_tangent(a[i])) Py_RETURN_NONE;
    if (form == 2) expect_no_tangents("residual_norm_quantized", {a[0], a[1], a[2], a[3], a[4]});
    auto d = header<rns8_cuda_residual_norm_desc>(0);
    const NormArgs r = norm_args(d, x, "x", y, a[2], a[3], a[4], a[5], a[6], a[7]);
    if (form == 2 && !d.pre_weight) type_error("pre_weight: needed for int8 rows");
    at::Tensor x_out = empty(x.sizes(), x.scalar_type(), d.device_id), h, q, s;
    d.ld_x_out = d.ld_h = d.dim, d.ld_q = (d.dim + 15) / 16 * 16;
    if (form == 2) {
      q = empty_q(x, d.dim, d.device_id);
      s = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, d.device_id);
      d.q = static_cast<int8_t*>(q.data_ptr()), d.q_scale = static_cast<float*>(s.data_ptr());
    } else if (d.pre_weight) {
      h = empty(x.sizes(), x.scalar_type(), d.device_id);
      d.h = h.data_ptr();
    }
    d.ld_x = r.x.ld, d.x = r.x.data, d.x_out = x_out.data_ptr();
    if (d.tokens) expect(lib.norm(&d), "rns8_cuda_residual_norm_device");
    if (form != 2) return tuple_of({x_out, h});
    mark_underivable("residual_norm_quantized", {a[0], a[1], a[2], a[3], a[4]}, {x_out, s});
    return tuple_of({x_out, q, s});
  });
}

// ---- residual_norm_backward(d_x_out, d_h, x_out, y, post, pre, gate, scale, eps, offset) ----
PyObject* residual_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    expect_args(n, 10);
    const at::Tensor& x = tensor(a[2], "x_out");
    const at::Tensor& y = tensor(a[3], "y");
    expect_no_tangents("residual_norm_backward", {a[0], a[1], a[2], a[3], a[4], a[5], a[6]});
    auto d = header<rns8_cuda_residual_norm_backward_desc>(0);
    const NormArgs r = norm_args(d, x, "x_out", y, a[4], a[5], a[6], a[7], a[8], a[9]);
    d.ld_x_out = r.x.ld, d.x_out = r.x.data;
    Rows held[2];
    auto incoming = [&](PyObject* o, const char* name, Rows& rows, int64_t& ld) -> const void* {
      ld = d.dim;
      const at::Tensor* t = optional_tensor(o, name);
      if (!t) return nullptr;
      if (t->sizes() != x.sizes() || t->scalar_type() != x.scalar_type())
        value_error(std::string(name) + ": expected x_out's type and shape");
      expect_device(*t, d.device_id, name);
      rows = rows_of(*t, name);
      ld = rows.ld;
      return rows.data;
    };
    d.d_x_out = incoming(a[0], "d_x_out", held[0], d.ld_d_x_out);
    d.d_h = incoming(a[1], "d_h", held[1], d.ld_d_h);
    const int device = d.device_id;
    at::Tensor d_x = empty(x.sizes(), x.scalar_type(), device), d_y = empty(x.sizes(), x.scalar_type(), device);
    at::Tensor d_post, d_pre, d_gate, scratch;
    d.ld_d_x = d.ld_d_y = d.ld_d_gate = d.dim;
    d.d_x = d_x.data_ptr(), d.d_y = d_y.data_ptr();
    if (d.post_weight) {
      d_post = empty({d.dim}, at::kFloat, device);
      d.d_post = static_cast<float*>(d_post.data_ptr());
    }
    if (d.pre_weight) {
      d_pre = empty({d.dim}, at::kFloat, device);
      d.d_pre = static_cast<float*>(d_pre.data_ptr());
    }
    if (r.gate_tensor) {
      const bool per_token = d.groups == d.tokens;
      if (per_token && d.weight_type == RNS8_CUDA_TYPE_F32 && d.type != RNS8_CUDA_TYPE_F32)
        d.flags |= RNS8_CUDA_NORM_D_GATE_F32;
      d_gate = empty(r.gate_tensor->sizes(), per_token && !d.flags ? x.scalar_type() : at::kFloat, device);
      d.d_gate = d_gate.data_ptr();
    }
    d.scratch_bytes = lib.norm_backward_scratch(&d);
    if (d.scratch_bytes) {
      scratch = empty({static_cast<int64_t>(d.scratch_bytes)}, at::kByte, device);
      d.scratch = scratch.data_ptr();
    }
    expect(lib.norm_backward(&d), "rns8_cuda_residual_norm_backward_device");
    mark_underivable("residual_norm_backward", {a[0], a[1], a[2], a[3], a[4], a[5], a[6]}, {d_x, d_y, d_post, d_pre, d_gate});
    return tuple_of({d_x, d_y, d_post, d_pre, d_gate});
  });
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {"quantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(quantize_rows)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(linear)), METH_FASTCALL, nullptr},
    {"residual_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(residual_norm)), METH_FASTCALL, nullptr},
    {"residual_norm_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(residual_norm_backward)),
     METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_quant_torch", "torch binding of rns8_quant.h", -1, methods,
                      nullptr,               nullptr,        nullptr,                         nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__quant_torch() { return PyModule_Create(&module); }
