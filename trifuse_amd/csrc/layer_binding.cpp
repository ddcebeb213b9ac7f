// Host side of trifuse_amd/layer.py: argument checks, output allocation and the
// C-ABI call of each operator around the block, in one native call from Python.
// A call on a few rows is bound by its host time, most of which was these checks
// in Python. The entry points' addresses come from the loaded library (bind);
// nothing is linked against it. Every function takes the stream first; the
// caller has made the tensors' device the current one.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <string>

#include "../../include/trifuse_moe.h"

namespace {

decltype(&tfm_norm_residual) p_norm_residual;
decltype(&tfm_quantize_rows) p_quantize_rows;
decltype(&tfm_int8_qmm) p_int8_qmm;
decltype(&tfm_int8_linear_workspace_bytes) p_int8_linear_workspace_bytes;
decltype(&tfm_int8_linear) p_int8_linear;
decltype(&tfm_token_logprobs) p_token_logprobs;
PyObject* raise_status;  // trifuse_amd._lib.raise_status

struct Raised {};  // a Python error is set

[[noreturn]] void fail(PyObject* type, const std::string& message) {
  PyErr_SetString(type, message.c_str());
  throw Raised{};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

void need_dev(const at::Tensor& t, const char* name) {
  if (!t.is_cuda())
    fail(PyExc_ValueError, std::string(name) + " must be a GPU tensor (the MoE path has no CPU fallback)");
  if (!t.is_contiguous()) fail(PyExc_ValueError, std::string(name) + " must be contiguous");
}

// t stands beside x: contiguous and on its device.
void need_beside(const at::Tensor& t, const char* name, const at::Tensor& x) {
  need_dev(t, name);
  if (t.device() != x.device())
    fail(PyExc_ValueError, std::string(name) + " is on " + t.device().str() + ", not on " + x.device().str());
}

int32_t storage_code(const at::Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return TFM_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return TFM_DTYPE_F16;
  fail(PyExc_NotImplementedError,
       std::string(name) + ": only bf16 and f16 storage are built (got " + c10::toString(t.scalar_type()) + ")");
}

struct Rows {
  int64_t rows;
  int32_t width;
};
Rows rows_of(const at::Tensor& t, const char* name) {
  const int64_t width = t.dim() > 0 ? t.size(-1) : 0;
  if (width <= 0) fail(PyExc_ValueError, std::string(name) + " must be [..., width] with a positive width");
  if (width > INT32_MAX) fail(PyExc_ValueError, std::string(name) + " is too wide");
  return Rows{t.numel() / width, (int32_t)width};
}

const void* vector_of(PyObject* o, const char* name, int64_t n, at::ScalarType type, const at::Tensor& x) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, name);
  need_beside(t, name, x);
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n)
    fail(PyExc_ValueError, std::string(name) + " must be " + c10::toString(type) + " [" + std::to_string(n) + "]");
  return t.data_ptr();
}

void* like(PyObject* o, const char* name, const at::Tensor& y) {
  const at::Tensor& t = tensor(o, name);
  need_beside(t, name, y);
  if (t.scalar_type() != y.scalar_type() || t.sizes() != y.sizes())
    fail(PyExc_ValueError, std::string(name) + " geometry/dtype differs");
  return t.data_ptr();
}

float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return (float)v;
}

void* stream_of(PyObject* o) {
  void* s = PyLong_AsVoidPtr(o);
  if (!s && PyErr_Occurred()) throw Raised{};
  return s;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& beside) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(beside.device()));
}
at::IntArrayRef lead(const at::Tensor& t) { return t.sizes().slice(0, t.dim() - 1); }

void need_ok(int status) {
  if (status == TFM_OK) return;
  PyObject* r = PyObject_CallFunction(raise_status, "i", status);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "trifuse_moe call failed");
  throw Raised{};
}

template <typename F>
void enqueue(F&& f) {
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = f();
  Py_END_ALLOW_THREADS;
  need_ok(status);
}

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Raised&) {
  } catch (const std::exception&) {  // torch's own types: OutOfMemoryError among them
    torch::translate_exception_to_python(std::current_exception());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "internal error");
  }
  return nullptr;
}

void need_args(Py_ssize_t have, Py_ssize_t want) {
  if (have != want) fail(PyExc_TypeError, "wrong number of arguments");
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
template <typename... T>
PyObject* pack(T... items) {  // new references
  return Py_BuildValue(std::string(sizeof...(T), 'N').insert(0, "(").append(")").c_str(), items...);
}

// norm_residual(stream, y, residual, post_weight, gate, residual_multiplier, pre_weight, eps, post_eps, quantize, out)
PyObject* norm_residual(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_args(n, 11);
    const at::Tensor& y = tensor(v[1], "y");
    const int32_t dt = storage_code(y, "y");
    need_dev(y, "y");
    const Rows r = rows_of(y, "y");
    tfm_norm_step s{};
    s.y = y.data_ptr();
    if (v[2] != Py_None) s.residual = like(v[2], "residual", y);
    s.post_weight = vector_of(v[3], "post_weight", r.width, y.scalar_type(), y);
    if (v[4] != Py_None) {
      const at::Tensor& g = tensor(v[4], "gate");
      need_beside(g, "gate", y);
      s.gate = g.data_ptr();
      if (g.scalar_type() == y.scalar_type() && g.sizes() == y.sizes())
        s.gate_kind = TFM_GATE_FULL;
      else if (g.scalar_type() == y.scalar_type() && g.dim() == 1 && g.size(0) == r.width)
        s.gate_kind = TFM_GATE_CHANNEL;
      else if (g.scalar_type() == at::kFloat &&
               (g.sizes() == lead(y) || (g.dim() == y.dim() && g.size(-1) == 1 && lead(g) == lead(y))))
        s.gate_kind = TFM_GATE_TOKEN;
      else
        fail(PyExc_ValueError, "gate must be [H] or y's shape in y's dtype, or fp32 with one value a row");
    }
    s.residual_multiplier = real(v[5]);
    s.pre_weight = vector_of(v[6], "pre_weight", r.width, y.scalar_type(), y);
    s.pre_eps = real(v[7]);
    s.post_eps = v[8] == Py_None ? s.pre_eps : real(v[8]);
    const int quantize = PyObject_IsTrue(v[9]);
    if (quantize < 0) throw Raised{};
    if (quantize && v[6] == Py_None) fail(PyExc_ValueError, "quantize needs pre_weight");
    at::Tensor h, x, codes, scales;
    if (v[10] == Py_None) {
      h = empty(y.sizes(), y.scalar_type(), y);
      s.h = h.data_ptr();
    } else {
      s.h = like(v[10], "out", y);
    }
    if (quantize) {
      codes = empty(y.sizes(), at::kChar, y);
      scales = empty(lead(y), at::kFloat, y);
      s.codes = static_cast<int8_t*>(codes.data_ptr());
      s.scales = static_cast<float*>(scales.data_ptr());
    } else if (v[6] != Py_None) {
      x = empty(y.sizes(), y.scalar_type(), y);
      s.x = x.data_ptr();
    }
    void* stream = stream_of(v[0]);
    enqueue([&] { return p_norm_residual(&s, r.rows, r.width, dt, stream); });
    PyObject* ho = v[10] == Py_None ? wrap(h) : Py_NewRef(v[10]);
    if (quantize) return pack(ho, wrap(codes), wrap(scales));
    return x.defined() ? pack(ho, wrap(x)) : ho;
  });
}

// rms_norm(stream, x, weight, eps, quantize)
PyObject* rms_norm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_args(n, 5);
    const at::Tensor& x = tensor(v[1], "x");
    const int32_t dt = storage_code(x, "x");
    need_dev(x, "x");
    const Rows r = rows_of(x, "x");
    const at::Tensor& w = tensor(v[2], "weight");
    (void)w;
    tfm_norm_step s{};
    s.y = x.data_ptr();
    s.pre_weight = vector_of(v[2], "weight", r.width, x.scalar_type(), x);
    s.residual_multiplier = 1.0f;
    s.pre_eps = real(v[3]);
    const int quantize = PyObject_IsTrue(v[4]);
    if (quantize < 0) throw Raised{};
    at::Tensor y, codes, scales;
    if (quantize) {
      codes = empty(x.sizes(), at::kChar, x);
      scales = empty(lead(x), at::kFloat, x);
      s.codes = static_cast<int8_t*>(codes.data_ptr());
      s.scales = static_cast<float*>(scales.data_ptr());
    } else {
      y = empty(x.sizes(), x.scalar_type(), x);
      s.x = y.data_ptr();
    }
    void* stream = stream_of(v[0]);
    enqueue([&] { return p_norm_residual(&s, r.rows, r.width, dt, stream); });
    return quantize ? pack(wrap(codes), wrap(scales)) : wrap(y);
  });
}

// quantize_rows(stream, x)
PyObject* quantize_rows(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_args(n, 2);
    const at::Tensor& x = tensor(v[1], "x");
    const int32_t dt = storage_code(x, "x");
    need_dev(x, "x");
    const Rows r = rows_of(x, "x");
    at::Tensor codes = empty(x.sizes(), at::kChar, x), scales = empty(lead(x), at::kFloat, x);
    void* stream = stream_of(v[0]);
    enqueue([&] {
      return p_quantize_rows(x.data_ptr(), r.rows, r.width, dt, static_cast<int8_t*>(codes.data_ptr()),
                             static_cast<float*>(scales.data_ptr()), stream);
    });
    return pack(wrap(codes), wrap(scales));
  });
}

const at::Tensor& weight_of(PyObject* o, int32_t width, const at::Tensor& x) {
  const at::Tensor& w = tensor(o, "w");
  need_beside(w, "w", x);
  if (w.scalar_type() != at::kChar || w.dim() != 2 || w.size(1) != width || w.size(0) <= 0 || w.size(0) > INT32_MAX)
    fail(PyExc_ValueError, "w must be int8 [n_out, " + std::to_string(width) + "]");
  return w;
}

at::Tensor product_out(const at::Tensor& x, int64_t n_out, at::ScalarType type) {
  c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n_out;
  return empty(shape, type, x);
}

// The library's limits on a product's sizes, before its output is allocated, which may be far larger than the
// inputs: a call without rows (or with too many) checks them and does nothing.
void need_product(const Rows& r, const at::Tensor& w, int32_t dt) {
  constexpr int64_t kTooMany = 1 << 22;
  need_ok(p_int8_qmm(nullptr, nullptr, r.rows < kTooMany ? 0 : r.rows, nullptr, nullptr, nullptr, (int32_t)w.size(0),
                     r.width, dt, nullptr, nullptr));
}

const float* floats(const void* p) { return static_cast<const float*>(p); }

// int8_qmm(stream, codes, scales, w, w_scales, bias, dtype)
PyObject* int8_qmm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_args(n, 7);
    if (!THPDtype_Check(v[6])) fail(PyExc_ValueError, "dtype must be a torch.dtype");
    const at::ScalarType type = reinterpret_cast<THPDtype*>(v[6])->scalar_type;
    if (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat)
      fail(PyExc_ValueError, std::string("unknown output dtype ") + c10::toString(type));
    const int32_t dt = type == at::kBFloat16 ? TFM_DTYPE_BF16 : type == at::kHalf ? TFM_DTYPE_F16 : TFM_DTYPE_F32;
    const at::Tensor& codes = tensor(v[1], "codes");
    need_dev(codes, "codes");
    if (codes.scalar_type() != at::kChar) fail(PyExc_ValueError, "codes must be int8");
    const Rows r = rows_of(codes, "codes");
    const at::Tensor& scales = tensor(v[2], "scales");
    need_beside(scales, "scales", codes);
    if (scales.scalar_type() != at::kFloat || scales.sizes() != lead(codes))
      fail(PyExc_ValueError, "scales must be fp32 with one value a row of codes");
    const at::Tensor& w = weight_of(v[3], r.width, codes);
    tensor(v[4], "w_scales");
    const void* ws = vector_of(v[4], "w_scales", w.size(0), at::kFloat, codes);
    const void* bias = vector_of(v[5], "bias", w.size(0), type, codes);
    need_product(r, w, dt);
    at::Tensor out = product_out(codes, w.size(0), type);
    void* stream = stream_of(v[0]);
    enqueue([&] {
      return p_int8_qmm(static_cast<const int8_t*>(codes.data_ptr()), floats(scales.data_ptr()), r.rows,
                        static_cast<const int8_t*>(w.data_ptr()), floats(ws), bias, (int32_t)w.size(0), r.width, dt,
                        out.data_ptr(), stream);
    });
    return wrap(out);
  });
}

// int8_linear(stream, x, w, w_scales, bias)
PyObject* int8_linear(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_args(n, 5);
    const at::Tensor& x = tensor(v[1], "x");
    const int32_t dt = storage_code(x, "x");
    need_dev(x, "x");
    const Rows r = rows_of(x, "x");
    const at::Tensor& w = weight_of(v[2], r.width, x);
    tensor(v[3], "w_scales");
    const void* ws = vector_of(v[3], "w_scales", w.size(0), at::kFloat, x);
    const void* bias = vector_of(v[4], "bias", w.size(0), x.scalar_type(), x);
    need_product(r, w, dt);
    at::Tensor out = product_out(x, w.size(0), x.scalar_type()), space;
    const size_t need = p_int8_linear_workspace_bytes(r.rows, r.width);
    if (need) space = empty({(int64_t)need}, at::kByte, x);
    void* stream = stream_of(v[0]);
    enqueue([&] {
      return p_int8_linear(x.data_ptr(), r.rows, static_cast<const int8_t*>(w.data_ptr()), floats(ws), bias,
                           (int32_t)w.size(0), r.width, dt, out.data_ptr(), need ? space.data_ptr() : nullptr, need,
                           stream);
    });
    return wrap(out);
  });
}

// token_logprobs(stream, logits, tokens, top, scale)
PyObject* token_logprobs(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_args(n, 5);
    const at::Tensor& x = tensor(v[1], "logits");
    const at::ScalarType type = x.scalar_type();
    if (type != at::kBFloat16 && type != at::kHalf && type != at::kFloat)
      fail(PyExc_NotImplementedError,
           std::string("logits: only bf16, f16 and fp32 are built (got ") + c10::toString(type) + ")");
    const int32_t dt = type == at::kBFloat16 ? TFM_DTYPE_BF16 : type == at::kHalf ? TFM_DTYPE_F16 : TFM_DTYPE_F32;
    if (!x.is_cuda()) need_dev(x, "logits");
    const Rows r = rows_of(x, "logits");
    int64_t stride = r.width;
    if (!x.is_contiguous()) {
      if (x.dim() != 2 || (x.stride(1) != 1 && r.width > 1))
        fail(PyExc_ValueError, "logits must be contiguous, or 2-D with contiguous rows");
      if (r.rows > 1) stride = x.stride(0);
    }
    const long top = PyLong_CheckExact(v[3]) ? PyLong_AsLong(v[3]) : -1;
    if (PyErr_Occurred()) PyErr_Clear();
    if (top < 0 || top > r.width) fail(PyExc_ValueError, "Invalid top-k");
    const float scale = real(v[4]);
    c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = top;
    at::Tensor logp, entropy = empty(lead(x), at::kFloat, x), ids = empty(shape, at::kInt, x),
                     best = empty(shape, at::kFloat, x);
    const void* tokens = nullptr;
    int32_t bits = 64;
    if (v[2] != Py_None) {
      const at::Tensor& k = tensor(v[2], "tokens");
      need_beside(k, "tokens", x);
      if ((k.scalar_type() != at::kLong && k.scalar_type() != at::kInt) || k.sizes() != lead(x))
        fail(PyExc_ValueError, "tokens must be int32 or int64 with one value a row of logits");
      bits = k.scalar_type() == at::kLong ? 64 : 32;
      tokens = k.data_ptr();
      logp = empty(lead(x), at::kFloat, x);
    }
    void* stream = stream_of(v[0]);
    enqueue([&] {
      return p_token_logprobs(x.data_ptr(), r.rows, r.width, stride, dt, tokens, bits, (int32_t)top, scale,
                              logp.defined() ? static_cast<float*>(logp.data_ptr()) : nullptr,
                              static_cast<float*>(entropy.data_ptr()), static_cast<int32_t*>(ids.data_ptr()),
                              static_cast<float*>(best.data_ptr()), stream);
    });
    return pack(logp.defined() ? wrap(logp) : Py_NewRef(Py_None), wrap(entropy), wrap(ids), wrap(best));
  });
}

// bind({name: address}, raise_status)
PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need_args(n, 2);
    auto take = [&](auto& p, const char* name) {
      PyObject* o = PyDict_GetItemString(v[0], name);
      if (!o) fail(PyExc_KeyError, name);
      p = reinterpret_cast<std::decay_t<decltype(p)>>(stream_of(o));
    };
    take(p_norm_residual, "tfm_norm_residual");
    take(p_quantize_rows, "tfm_quantize_rows");
    take(p_int8_qmm, "tfm_int8_qmm");
    take(p_int8_linear_workspace_bytes, "tfm_int8_linear_workspace_bytes");
    take(p_int8_linear, "tfm_int8_linear");
    take(p_token_logprobs, "tfm_token_logprobs");
    Py_XDECREF(raise_status);
    raise_status = Py_NewRef(v[1]);
    return Py_NewRef(Py_None);
  });
}

#define TFM_FUNC(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TFM_FUNC(bind),         TFM_FUNC(norm_residual), TFM_FUNC(rms_norm),
                         TFM_FUNC(quantize_rows), TFM_FUNC(int8_qmm),      TFM_FUNC(int8_linear),
                         TFM_FUNC(token_logprobs), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_layer", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layer() { return PyModule_Create(&module); }
