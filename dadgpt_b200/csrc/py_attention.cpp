// CPython module behind dadgpt_b200/attention.py: argument checks, the current stream and the C
// call of include/dadattn.h, for torch tensors.
//
// Why native: the smallest calls (a tiny fp32 step, a short prompt, one decoded token) are bound by
// the host. Checked in Python and called through ctypes, a call cost 10-13 us of host time, of
// which the launches themselves are 2-3 us each; here the checks and argument conversion are
// about 0.3 us. Tensors are unpacked with torch's own C++ accessor, never through attribute
// look-ups; the GIL is released around the C call (a launch can block on a full queue).
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <functional>
#include <initializer_list>
#include <string>
#include <utility>

#include "dadattn.h"

namespace {

PyObject* g_error_class = nullptr;   // DadAttnError(code, message), set by set_error_class

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kByte: return "torch.uint8";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    case at::kFloat8_e4m3fn: return "torch.float8_e4m3fn";
    default: return c10::toString(t);
  }
}

struct Bad {};   // a Python exception is set

// Positional arguments of a METH_FASTCALL function, converted in order.
class Args {
 public:
  Args(PyObject* const* a, Py_ssize_t n, Py_ssize_t want, const char* fn) : a_(a) {
    if (n != want) {
      PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", fn, want, n);
      throw Bad{};
    }
  }
  const at::Tensor& tensor(const char* name) {
    PyObject* o = a_[i_++];
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_ValueError, "%s must be a torch tensor, got %s", name, Py_TYPE(o)->tp_name);
      throw Bad{};
    }
    return THPVariable_Unpack(o);
  }
  // a contiguous CUDA tensor of the given type
  const at::Tensor& need(const char* name, at::ScalarType type) {
    const at::Tensor& t = tensor(name);
    if (!t.is_cuda()) {
      PyErr_Format(PyExc_ValueError, "%s must be a CUDA tensor (there is no CPU path)", name);
      throw Bad{};
    }
    if (t.scalar_type() != type || !t.is_contiguous()) {
      PyErr_Format(PyExc_ValueError, "%s must be contiguous %s, got %s contiguous=%s", name, type_name(type),
                   type_name(t.scalar_type()), t.is_contiguous() ? "True" : "False");
      throw Bad{};
    }
    return t;
  }
  // a CUDA tensor of the given type and shape on the current device, its elements next to each other, its other strides into
  // `strides` (those of dimensions of extent 1 as 0 where they do not matter)
  const at::Tensor& strided(const char* name, at::ScalarType type, std::initializer_list<int64_t> shape, int64_t* strides);
  // the same, on the current device and of the given shape
  const at::Tensor& here(const char* name, at::ScalarType type, std::initializer_list<int64_t> shape);
  const at::Tensor& workspace() {
    const at::Tensor& t = tensor("workspace");
    if (!t.is_cuda() || !t.is_contiguous()) {
      PyErr_SetString(PyExc_ValueError, "workspace must be a contiguous CUDA tensor");
      throw Bad{};
    }
    need_current("workspace", t);
    return t;
  }
  static void need_current(const char* name, const at::Tensor& t) {
    const int current = c10::cuda::current_device();
    if (t.get_device() == current) return;
    PyErr_Format(PyExc_ValueError, "%s is on cuda:%d, the current device is cuda:%d", name, static_cast<int>(t.get_device()), current);
    throw Bad{};
  }
  // size `dim` of the `ahead`-th argument from the next, a tensor of `dims` dimensions (`layout` says which)
  int size_of(int ahead, const char* name, int dims, int dim, const char* layout) {
    i_ += ahead;
    const at::Tensor& t = tensor(name);
    i_ -= ahead + 1;
    if (t.dim() != dims) {
      PyErr_Format(PyExc_ValueError, "%s must be %s, got %d dimensions", name, layout, static_cast<int>(t.dim()));
      throw Bad{};
    }
    const int64_t n = t.size(dim);
    if (n != static_cast<int>(n)) {
      PyErr_Format(PyExc_ValueError, "size %lld out of range", static_cast<long long>(n));
      throw Bad{};
    }
    return static_cast<int>(n);
  }
  bool none_at(int ahead) const { return a_[i_ + ahead] == Py_None; }
  // the type of the next argument, a tensor
  at::ScalarType peek_type(const char* name) {
    const at::ScalarType type = tensor(name).scalar_type();
    --i_;
    return type;
  }
  bool none() {
    if (a_[i_] != Py_None) return false;
    ++i_;
    return true;
  }
  int integer() {   // a size: larger ones than an int fit no tensor
    const int64_t v = integer64();
    if (v != static_cast<int>(v)) {
      PyErr_Format(PyExc_ValueError, "size %lld out of range", static_cast<long long>(v));
      throw Bad{};
    }
    return static_cast<int>(v);
  }
  int64_t integer64() {
    const long long v = PyLong_AsLongLong(a_[i_++]);
    if (v == -1 && PyErr_Occurred()) throw Bad{};
    return v;
  }
  uint64_t bits64() {
    const unsigned long long v = PyLong_AsUnsignedLongLongMask(a_[i_++]);
    if (v == static_cast<unsigned long long>(-1) && PyErr_Occurred()) throw Bad{};
    return v;
  }
  float real() {
    const double v = PyFloat_AsDouble(a_[i_++]);
    if (v == -1.0 && PyErr_Occurred()) throw Bad{};
    return static_cast<float>(v);
  }

 private:
  PyObject* const* a_;
  Py_ssize_t i_ = 0;
};

void need_shape(const char* name, const at::Tensor& t, std::initializer_list<int64_t> shape) {
  if (t.sizes() == at::IntArrayRef(shape.begin(), shape.size())) return;
  auto text = [](at::IntArrayRef s) {
    std::string r = "(";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + (s.size() == 1 ? ",)" : ")");
  };
  PyErr_Format(PyExc_ValueError, "%s has shape %s, expected %s", name, text(t.sizes()).c_str(),
               text(at::IntArrayRef(shape.begin(), shape.size())).c_str());
  throw Bad{};
}

const at::Tensor& Args::here(const char* name, at::ScalarType type, std::initializer_list<int64_t> shape) {
  const at::Tensor& t = need(name, type);
  need_current(name, t);
  need_shape(name, t, shape);
  return t;
}

const at::Tensor& Args::strided(const char* name, at::ScalarType type, std::initializer_list<int64_t> shape, int64_t* strides) {
  const at::Tensor& t = tensor(name);
  if (!t.is_cuda()) {
    PyErr_Format(PyExc_ValueError, "%s must be a CUDA tensor (there is no CPU path)", name);
    throw Bad{};
  }
  need_current(name, t);
  need_shape(name, t, shape);
  const int64_t last = t.dim() - 1;
  if (t.scalar_type() != type || (t.size(last) > 1 && t.stride(last) != 1)) {
    PyErr_Format(PyExc_ValueError, "%s must be %s with rows of neighbouring elements, got %s, last stride %lld", name,
                 type_name(type), type_name(t.scalar_type()), static_cast<long long>(t.stride(last)));
    throw Bad{};
  }
  for (int64_t i = 0; i < last; ++i) strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
  return t;
}

void need_shapes(std::initializer_list<std::pair<const char*, std::reference_wrapper<const at::Tensor>>> tensors,
                 std::initializer_list<int64_t> shape) {
  for (const auto& [name, t] : tensors) need_shape(name, t.get(), shape);
}

void* ptr(const at::Tensor& t) { return t.data_ptr(); }
float* f32(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }
uint8_t* b8(const at::Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }
uint16_t* b16(const at::Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); }
dadattn_stream_t stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

PyObject* done(int rc) {
  if (rc == 0) Py_RETURN_NONE;
  PyObject* e = PyObject_CallFunction(g_error_class ? g_error_class : PyExc_RuntimeError, "is", rc,
                                      dadattn_last_error());
  if (e) {
    PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(e)), e);
    Py_DECREF(e);
  }
  return nullptr;
}

template <typename F>
int without_gil(F&& f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  return rc;
}

// Runs a body that may throw Bad (exception already set) or a c10 error.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Bad&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

constexpr at::ScalarType kF = at::kFloat, kB = at::kBFloat16, k8 = at::kFloat8_e4m3fn;

// out, lse, q, k, v, BH, S, D, scale, rate, seed, offset, unit0
PyObject* fwd_f32(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 13, "fwd_f32");
    const at::Tensor &out = p.need("out", kF), &lse = p.need("lse", kF), &q = p.need("q", kF), &k = p.need("k", kF),
                     &v = p.need("v", kF);
    const int BH = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real(), rate = p.real();
    const uint64_t seed = p.bits64(), offset = p.bits64();
    const int64_t unit0 = p.integer64();
    need_shapes({{"out", out}, {"q", q}, {"k", k}, {"v", v}}, {BH, S, D});
    need_shape("lse", lse, {BH, S});
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_flash_fwd_f32_dropout(f32(out), f32(lse), f32(q), f32(k), f32(v), BH, S, D, scale, rate, seed,
                                           offset, unit0, st);
    }));
  });
}

// dq, dk, dv, delta, dout, out, lse, q, k, v, BH, S, D, scale, rate, seed, offset, unit0
PyObject* bwd_f32(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 18, "bwd_f32");
    const at::Tensor &dq = p.need("dq", kF), &dk = p.need("dk", kF), &dv = p.need("dv", kF),
                     &delta = p.need("delta", kF), &dout = p.need("dout", kF), &out = p.need("out", kF),
                     &lse = p.need("lse", kF), &q = p.need("q", kF), &k = p.need("k", kF), &v = p.need("v", kF);
    const int BH = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real(), rate = p.real();
    const uint64_t seed = p.bits64(), offset = p.bits64();
    const int64_t unit0 = p.integer64();
    need_shapes({{"dq", dq}, {"dk", dk}, {"dv", dv}, {"dout", dout}, {"out", out}, {"q", q}, {"k", k}, {"v", v}},
                {BH, S, D});
    need_shape("lse", lse, {BH, S});
    if (delta.numel() < static_cast<int64_t>(BH) * S) {
      PyErr_SetString(PyExc_ValueError, "delta scratch smaller than BH*S");
      return nullptr;
    }
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_flash_bwd_f32_dropout(f32(dq), f32(dk), f32(dv), f32(delta), f32(dout), f32(out), f32(lse),
                                           f32(q), f32(k), f32(v), BH, S, D, scale, rate, seed, offset, unit0, st);
    }));
  });
}

// out, lse, q, k, v, BH, S, D, scale, rate, seed, offset, unit0, mask_bits or None
PyObject* fwd_bf16(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 14, "fwd_bf16");
    const at::Tensor &out = p.need("out", kB), &lse = p.need("lse", kF), &q = p.need("q", kB), &k = p.need("k", kB),
                     &v = p.need("v", kB);
    const int BH = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real(), rate = p.real();
    const uint64_t seed = p.bits64(), offset = p.bits64();
    const int64_t unit0 = p.integer64();
    need_shapes({{"out", out}, {"q", q}, {"k", k}, {"v", v}}, {BH, S, D});
    need_shape("lse", lse, {BH, S});
    const bool masked = !p.none();   // (an empty tensor's pointer is null: the library refuses it)
    const uint32_t* bits = masked ? static_cast<const uint32_t*>(ptr(p.tensor("mask_bits"))) : nullptr;
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return masked ? dadattn_flash_fwd_bf16_masked(b16(out), f32(lse), b16(q), b16(k), b16(v), BH, S, D, scale, rate,
                                                    bits, st)
                    : dadattn_flash_fwd_bf16(b16(out), f32(lse), b16(q), b16(k), b16(v), BH, S, D, scale, rate, seed,
                                             offset, unit0, st);
    }));
  });
}

// dq, dk, dv, workspace, dout, out, lse, q, k, v, BH, S, D, scale, rate, seed, offset, unit0, mask_bits or None
PyObject* bwd_bf16(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 19, "bwd_bf16");
    const at::Tensor &dq = p.need("dq", kB), &dk = p.need("dk", kB), &dv = p.need("dv", kB),
                     &ws = p.tensor("workspace"), &dout = p.need("dout", kB), &out = p.need("out", kB),
                     &lse = p.need("lse", kF), &q = p.need("q", kB), &k = p.need("k", kB), &v = p.need("v", kB);
    const int BH = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real(), rate = p.real();
    const uint64_t seed = p.bits64(), offset = p.bits64();
    const int64_t unit0 = p.integer64();
    need_shapes({{"dq", dq}, {"dk", dk}, {"dv", dv}, {"dout", dout}, {"out", out}, {"q", q}, {"k", k}, {"v", v}},
                {BH, S, D});
    need_shape("lse", lse, {BH, S});
    const bool masked = !p.none();   // (an empty tensor's pointer is null: the library refuses it)
    const uint32_t* bits = masked ? static_cast<const uint32_t*>(ptr(p.tensor("mask_bits"))) : nullptr;
    void* const w = ptr(ws);
    const size_t bytes = ws.nbytes();
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return masked ? dadattn_flash_bwd_bf16_masked(b16(dq), b16(dk), b16(dv), w, bytes, b16(dout), b16(out), f32(lse),
                                                    b16(q), b16(k), b16(v), BH, S, D, scale, rate, bits, st)
                    : dadattn_flash_bwd_bf16(b16(dq), b16(dk), b16(dv), w, bytes, b16(dout), b16(out), f32(lse),
                                             b16(q), b16(k), b16(v), BH, S, D, scale, rate, seed, offset, unit0, st);
    }));
  });
}

// out, lse, q, k, v, B, H, S, D, scale, rate, seed, offset, unit0
PyObject* fwd_bf16_strided(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 14, "fwd_bf16_strided");
    const at::Tensor &out = p.need("out", kB), &lse = p.need("lse", kF), &q = p.need("q", kB), &k = p.need("k", kB),
                     &v = p.need("v", kB);
    const int B = p.integer(), H = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real(), rate = p.real();
    const uint64_t seed = p.bits64(), offset = p.bits64();
    const int64_t unit0 = p.integer64();
    need_shapes({{"out", out}, {"q", q}, {"k", k}, {"v", v}}, {int64_t(B) * S, int64_t(H) * D});
    need_shape("lse", lse, {int64_t(B) * H, S});
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_flash_fwd_bf16_strided(b16(out), f32(lse), b16(q), b16(k), b16(v), B, H, S, D, scale, rate, seed,
                                            offset, unit0, st);
    }));
  });
}

// dq, dk, dv, workspace, dout, out, lse, q, k, v, B, H, S, D, scale, rate, seed, offset, unit0
PyObject* bwd_bf16_strided(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 19, "bwd_bf16_strided");
    const at::Tensor &dq = p.need("dq", kB), &dk = p.need("dk", kB), &dv = p.need("dv", kB),
                     &ws = p.tensor("workspace"), &dout = p.need("dout", kB), &out = p.need("out", kB),
                     &lse = p.need("lse", kF), &q = p.need("q", kB), &k = p.need("k", kB), &v = p.need("v", kB);
    const int B = p.integer(), H = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real(), rate = p.real();
    const uint64_t seed = p.bits64(), offset = p.bits64();
    const int64_t unit0 = p.integer64();
    need_shapes({{"dq", dq}, {"dk", dk}, {"dv", dv}, {"dout", dout}, {"out", out}, {"q", q}, {"k", k}, {"v", v}},
                {int64_t(B) * S, int64_t(H) * D});
    need_shape("lse", lse, {int64_t(B) * H, S});
    void* const w = ptr(ws);
    const size_t bytes = ws.nbytes();
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_flash_bwd_bf16_strided(b16(dq), b16(dk), b16(dv), w, bytes, b16(dout), b16(out), f32(lse),
                                            b16(q), b16(k), b16(v), B, H, S, D, scale, rate, seed, offset, unit0, st);
    }));
  });
}

// BH, S, D, scale, window, sinks, out, lse, q, k, v
PyObject* fwd_bf16_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 11, "fwd_bf16_window");
    const int BH = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real();
    const int window = p.integer(), sinks = p.integer();
    const at::Tensor &out = p.here("out", kB, {BH, S, D}), &lse = p.here("lse", kF, {BH, S}), &q = p.here("q", kB, {BH, S, D}),
                     &k = p.here("k", kB, {BH, S, D}), &v = p.here("v", kB, {BH, S, D});
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_flash_fwd_bf16_window(b16(out), f32(lse), b16(q), b16(k), b16(v), BH, S, D, scale, window, sinks, st);
    }));
  });
}

// BH, S, D, scale, window, sinks, dq, dk, dv, workspace, dout, out, lse, q, k, v
PyObject* bwd_bf16_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 16, "bwd_bf16_window");
    const int BH = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real();
    const int window = p.integer(), sinks = p.integer();
    const at::Tensor &dq = p.here("dq", kB, {BH, S, D}), &dk = p.here("dk", kB, {BH, S, D}), &dv = p.here("dv", kB, {BH, S, D}),
                     &ws = p.workspace(), &dout = p.here("dout", kB, {BH, S, D}), &out = p.here("out", kB, {BH, S, D}),
                     &lse = p.here("lse", kF, {BH, S}), &q = p.here("q", kB, {BH, S, D}), &k = p.here("k", kB, {BH, S, D}),
                     &v = p.here("v", kB, {BH, S, D});
    void* const w = ptr(ws);
    const size_t bytes = ws.nbytes();
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_flash_bwd_bf16_window(b16(dq), b16(dk), b16(dv), w, bytes, b16(dout), b16(out), f32(lse), b16(q), b16(k),
                                           b16(v), BH, S, D, scale, window, sinks, st);
    }));
  });
}

// out, lse, q, k, v, BH, S, D, scale, workspace
PyObject* fwd_via_bf16(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 10, "fwd_via_bf16");
    const at::Tensor &out = p.need("out", kF), &lse = p.need("lse", kF), &q = p.need("q", kF), &k = p.need("k", kF),
                     &v = p.need("v", kF);
    const int BH = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real();
    const at::Tensor& ws = p.tensor("workspace");
    need_shapes({{"out", out}, {"q", q}, {"k", k}, {"v", v}}, {BH, S, D});
    need_shape("lse", lse, {BH, S});
    void* const w = ptr(ws);
    const size_t bytes = ws.nbytes();
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_flash_fwd_f32_via_bf16(f32(out), f32(lse), f32(q), f32(k), f32(v), BH, S, D, scale, w, bytes, st);
    }));
  });
}

// dq, dk, dv, dout, out, lse, q, k, v, BH, S, D, scale, workspace
PyObject* bwd_via_bf16(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 14, "bwd_via_bf16");
    const at::Tensor &dq = p.need("dq", kF), &dk = p.need("dk", kF), &dv = p.need("dv", kF),
                     &dout = p.need("dout", kF), &out = p.need("out", kF), &lse = p.need("lse", kF),
                     &q = p.need("q", kF), &k = p.need("k", kF), &v = p.need("v", kF);
    const int BH = p.integer(), S = p.integer(), D = p.integer();
    const float scale = p.real();
    const at::Tensor& ws = p.tensor("workspace");
    need_shapes({{"dq", dq}, {"dk", dk}, {"dv", dv}, {"dout", dout}, {"out", out}, {"q", q}, {"k", k}, {"v", v}},
                {BH, S, D});
    need_shape("lse", lse, {BH, S});
    void* const w = ptr(ws);
    const size_t bytes = ws.nbytes();
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_flash_bwd_f32_via_bf16(f32(dq), f32(dk), f32(dv), f32(dout), f32(out), f32(lse), f32(q), f32(k),
                                            f32(v), BH, S, D, scale, w, bytes, st);
    }));
  });
}

// bits, BH, S, rate, seed, offset, unit0
PyObject* mask_bits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 7, "mask_bits");
    const at::Tensor& bits = p.need("mask bits", at::kInt);
    const int BH = p.integer(), S = p.integer();
    const float rate = p.real();
    const uint64_t seed = p.bits64(), offset = p.bits64();
    const int64_t unit0 = p.integer64();
    uint32_t* const dst = static_cast<uint32_t*>(ptr(bits));
    const size_t bytes = bits.nbytes();
    const dadattn_stream_t st = stream();
    return done(without_gil([&] { return dadattn_dropout_mask_bits(dst, bytes, BH, S, rate, seed, offset, unit0, st); }));
  });
}

// out, q, k_new, v_new, k_cache, v_cache, pos, scale
PyObject* decode_f32(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 8, "decode_f32");
    const at::Tensor &out = p.need("out", kF), &q = p.need("q", kF), &kn = p.need("k_new", kF),
                     &vn = p.need("v_new", kF), &k = p.need("k_cache", kF), &v = p.need("v_cache", kF);
    const int64_t pos = p.integer64();
    const float scale = p.real();
    if (k.dim() != 3) {
      PyErr_SetString(PyExc_ValueError, "k_cache must be [H, max_len, D]");
      return nullptr;
    }
    const int H = static_cast<int>(k.size(0)), max_len = static_cast<int>(k.size(1)), D = static_cast<int>(k.size(2));
    if (pos < 0 || pos >= max_len) {
      PyErr_Format(PyExc_IndexError, "model_forward_cached: pos %lld outside context length %d",
                   static_cast<long long>(pos), max_len);
      return nullptr;
    }
    need_shape("v_cache", v, {H, max_len, D});
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_decode_f32(f32(out), f32(q), f32(kn), f32(vn), f32(k), f32(v), H, max_len, D,
                                static_cast<int>(pos), scale, st);
    }));
  });
}

// out, q, k_new, v_new, k_cache, v_cache, lengths, B, H, D, max_len, scale, workspace
PyObject* decode_bf16(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 13, "decode_bf16");
    const at::Tensor &out = p.need("out", kB), &q = p.need("q", kB), &kn = p.need("k_new", kB),
                     &vn = p.need("v_new", kB), &k = p.tensor("k_cache"), &v = p.tensor("v_cache"),
                     &len = p.tensor("lengths");
    const int B = p.integer(), H = p.integer(), D = p.integer(), max_len = p.integer();
    const float scale = p.real();
    const at::Tensor& ws = p.tensor("workspace");
    need_shapes({{"out", out}, {"q", q}, {"k_new", kn}, {"v_new", vn}}, {B, H, D});
    int32_t* const lengths = static_cast<int32_t*>(ptr(len));
    void* const w = ptr(ws);
    const size_t bytes = ws.numel();
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_decode_bf16(b16(out), b16(q), b16(kn), b16(vn), b16(k), b16(v), lengths, B, H, D, max_len, scale,
                                 w, bytes, st);
    }));
  });
}

// B, H, D, max_len, scale, window, sinks, out, q, k_new, v_new, k_cache, v_cache, lengths, weights or None, workspace
PyObject* decode_bf16_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 16, "decode_bf16_window");
    const int B = p.integer(), H = p.integer(), D = p.integer(), L = p.integer();
    const float scale = p.real();
    const int window = p.integer(), sinks = p.integer();
    const at::Tensor &out = p.here("out", kB, {B, H, D}), &q = p.here("q", kB, {B, H, D}),
                     &kn = p.here("k_new", kB, {B, H, D}), &vn = p.here("v_new", kB, {B, H, D}),
                     &k = p.here("k_cache", kB, {B, H, L, D}), &v = p.here("v_cache", kB, {B, H, L, D}),
                     &len = p.here("lengths", at::kInt, {B});
    float* const weights = p.none() ? nullptr : f32(p.here("weights", kF, {B, H, L}));
    const at::Tensor& ws = p.workspace();
    int32_t* const lengths = static_cast<int32_t*>(ptr(len));
    void* const w = ptr(ws);
    const size_t bytes = ws.nbytes();
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_decode_bf16_window(b16(out), b16(q), b16(kn), b16(vn), b16(k), b16(v), lengths, weights, B, H, D, L,
                                        scale, window, sinks, w, bytes, st);
    }));
  });
}

// B, H, D, max_len, scale, window, sinks, out, q, k_new, v_new, k_cache, v_cache, k_scale, v_scale, k_tail, v_tail,
// lengths, workspace
PyObject* decode_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 19, "decode_fp8");
    const int B = p.integer(), H = p.integer(), D = p.integer(), L = p.integer();
    const float scale = p.real();
    const int window = p.integer(), sinks = p.integer(), blocks = dadattn_fp8_scale_blocks(L);
    const at::Tensor &out = p.here("out", kB, {B, H, D}), &q = p.here("q", kB, {B, H, D}),
                     &kn = p.here("k_new", kB, {B, H, D}), &vn = p.here("v_new", kB, {B, H, D}),
                     &k = p.here("k_cache", k8, {B, H, L, D}), &v = p.here("v_cache", k8, {B, H, L, D}),
                     &ks = p.here("k_scale", kF, {B, H, blocks}), &vs = p.here("v_scale", kF, {B, H, blocks}),
                     &kt = p.here("k_tail", kB, {B, H, DADATTN_FP8_BLOCK, D}),
                     &vt = p.here("v_tail", kB, {B, H, DADATTN_FP8_BLOCK, D}), &len = p.here("lengths", at::kInt, {B});
    const at::Tensor& ws = p.workspace();
    int32_t* const lengths = static_cast<int32_t*>(ptr(len));
    void* const w = ptr(ws);
    const size_t bytes = ws.nbytes();
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_decode_fp8(b16(out), b16(q), b16(kn), b16(vn), b8(k), b8(v), f32(ks), f32(vs), b16(kt), b16(vt),
                                lengths, B, H, D, L, scale, window, sinks, w, bytes, st);
    }));
  });
}

// B, H, S, max_len, D, k_cache, v_cache, k_scale, v_scale, k_tail, v_tail, lengths, k_heads, v_heads, counts or None
PyObject* fill_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 15, "fill_fp8");
    const int B = p.integer(), H = p.integer(), S = p.integer(), L = p.integer(), D = p.integer();
    const int blocks = dadattn_fp8_scale_blocks(L);
    const at::Tensor &k = p.here("k_cache", k8, {B, H, L, D}), &v = p.here("v_cache", k8, {B, H, L, D}),
                     &ks = p.here("k_scale", kF, {B, H, blocks}), &vs = p.here("v_scale", kF, {B, H, blocks}),
                     &kt = p.here("k_tail", kB, {B, H, DADATTN_FP8_BLOCK, D}),
                     &vt = p.here("v_tail", kB, {B, H, DADATTN_FP8_BLOCK, D}), &len = p.here("lengths", at::kInt, {B});
    const at::ScalarType type = p.peek_type("k_heads") == kB ? kB : kF;
    const at::Tensor &kh = p.here("k_heads", type, {B, H, S, D}), &vh = p.here("v_heads", type, {B, H, S, D});
    const int32_t* const counts = p.none() ? nullptr : static_cast<const int32_t*>(ptr(p.here("counts", at::kInt, {B})));
    int32_t* const lengths = static_cast<int32_t*>(ptr(len));
    const void *const kp = ptr(kh), *const vp = ptr(vh);
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_kv_cache_fill_fp8(b8(k), b8(v), f32(ks), f32(vs), b16(kt), b16(vt), lengths, kp, vp, counts, B, H, S, L,
                                       D, type == kB, st);
    }));
  });
}

// B, H, D, max_len of the destination and of the source, budget, recent, (k, v, weights, lengths) of both
PyObject* evict_bf16(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 15, "evict_bf16");
    const int B = p.integer(), H = p.integer(), D = p.integer(), Ld = p.integer(), Ls = p.integer(), budget = p.integer(),
              recent = p.integer();
    const at::Tensor &kd = p.here("k of the destination", kB, {B, H, Ld, D}), &vd = p.here("v of the destination", kB, {B, H, Ld, D}),
                     &wd = p.here("weights of the destination", kF, {B, H, Ld}),
                     &ld = p.here("lengths of the destination", at::kInt, {B}),
                     &ks = p.here("k of the source", kB, {B, H, Ls, D}), &vs = p.here("v of the source", kB, {B, H, Ls, D}),
                     &ws = p.here("weights of the source", kF, {B, H, Ls}), &ls = p.here("lengths of the source", at::kInt, {B});
    int32_t *const to = static_cast<int32_t*>(ptr(ld)), *const from = static_cast<int32_t*>(ptr(ls));
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_kv_cache_evict_bf16(b16(kd), b16(vd), f32(wd), to, b16(ks), b16(vs), f32(ws), from, B, H, D, Ld, Ls,
                                         budget, recent, st);
    }));
  });
}

// turns, factor, rot_dim, interleaved of a RotaryPositions; turns None: no rotation
struct Rotary {
  const uint64_t* turns = nullptr;
  float factor = 1.f;
  int rot = 0, interleaved = 0;
  explicit Rotary(Args& p) {
    if (!p.none()) {
      const at::Tensor& f = p.need("turns", at::kLong);
      Args::need_current("turns", f);
      turns = static_cast<const uint64_t*>(f.data_ptr());
      n = f.numel();
    }
    factor = p.real();
    rot = p.integer();
    interleaved = p.integer();
    if (turns && n != rot / 2) {
      PyErr_Format(PyExc_ValueError, "turns has %lld elements, expected %d", static_cast<long long>(n), rot / 2);
      throw Bad{};
    }
  }
  int64_t n = 0;
};
constexpr const char* kPacked = "[tokens, heads, D]";
const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }

// backward, first, turns, factor, rot_dim, interleaved, q_out, k_out or None, q, k or None, positions or None
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 11, "rotary");
    const int back = p.integer();
    const int64_t first = p.integer64();
    const char* const layout = "[B, S, heads, D]";   // (q and k are behind the rotation's four arguments, q_out and k_out)
    const int B = p.size_of(6, "q", 4, 0, layout), S = p.size_of(6, "q", 4, 1, layout), Hq = p.size_of(6, "q", 4, 2, layout),
              D = p.size_of(6, "q", 4, 3, layout), Hk = p.none_at(7) ? 0 : p.size_of(7, "k", 4, 2, layout);
    const Rotary r(p);
    const at::ScalarType type = p.peek_type("q_out") == kB ? kB : kF;
    int64_t s[4][3] = {};   // q_out, k_out, q, k
    void *qo = ptr(p.strided("q_out", type, {B, S, Hq, D}, s[0])), *ko = nullptr;
    if (!p.none()) ko = ptr(p.strided("k_out", type, {B, S, Hk, D}, s[1]));
    const void *q = ptr(p.strided("q", type, {B, S, Hq, D}, s[2])), *k = nullptr;
    if (!p.none()) k = ptr(p.strided("k", type, {B, S, Hk, D}, s[3]));
    const int32_t* const positions = p.none() ? nullptr : ints(p.here("positions", at::kInt, {B, S}));
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_rotary(qo, ko, q, k, s[0], s[1], s[2], s[3], positions, first, B, S, Hq, Hk, D, r.turns, r.factor, r.rot,
                            r.interleaved, back, type == kB, st);
    }));
  });
}

// The paged cache's arguments: B, Hkv, D, pages, page_size, max_pages, k_pages, v_pages, page_table, lengths
struct Paged {
  int B, H, D, pages, page_size, max_pages;
  uint16_t *k, *v;
  const int32_t *table, *lengths;
  explicit Paged(Args& p)
      : B(p.integer()), H(p.integer()), D(p.integer()), pages(p.integer()), page_size(p.integer()), max_pages(p.integer()),
        k(b16(p.here("k_pages", kB, {pages, H, page_size, D}))), v(b16(p.here("v_pages", kB, {pages, H, page_size, D}))),
        table(ints(p.here("page_table", at::kInt, {B, max_pages}))), lengths(ints(p.here("lengths", at::kInt, {B}))) {}
};

// paged cache, rotary, starts or None, q_out or None, q or None, k_new, v_new
PyObject* append_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 19, "append_paged");
    const int T = p.size_of(17, "k_new", 3, 0, kPacked), Hq = p.none_at(16) ? 0 : p.size_of(16, "q", 3, 1, kPacked);
    const Paged c(p);
    const Rotary r(p);
    const int32_t* const starts = p.none() ? nullptr : ints(p.here("starts", at::kInt, {int64_t(c.B) + 1}));
    int64_t s[4][2] = {};
    uint16_t* const qo = p.none() ? nullptr : b16(p.strided("q_out", kB, {T, Hq, c.D}, s[0]));
    at::ScalarType type = kF;
    const void* q = nullptr;
    if (!p.none()) {
      type = p.peek_type("q") == kB ? kB : kF;
      q = ptr(p.strided("q", type, {T, Hq, c.D}, s[1]));
    }
    if (!q) type = p.peek_type("k_new") == kB ? kB : kF;
    const void *kn = ptr(p.strided("k_new", type, {T, c.H, c.D}, s[2])), *vn = ptr(p.strided("v_new", type, {T, c.H, c.D}, s[3]));
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_paged_append_bf16(c.k, c.v, c.table, c.lengths, starts, qo, q, kn, vn, s[0], s[1], s[2], s[3], c.B, T, Hq, c.H,
                                       c.D, c.pages, c.page_size, c.max_pages, r.turns, r.factor, r.rot, r.interleaved, type == kB, st);
    }));
  });
}

// paged cache, max_new, scale, starts or None, out, lse or None, q
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 16, "paged_attention");
    const int T = p.size_of(15, "q", 3, 0, kPacked), Hq = p.size_of(15, "q", 3, 1, kPacked);
    const Paged c(p);
    const int max_new = p.integer();
    const float scale = p.real();
    const int32_t* const starts = p.none() ? nullptr : ints(p.here("starts", at::kInt, {int64_t(c.B) + 1}));
    int64_t s[2][2] = {};
    uint16_t* const out = b16(p.strided("out", kB, {T, Hq, c.D}, s[0]));
    float* const lse = p.none() ? nullptr : f32(p.here("lse", kF, {T, Hq}));
    const uint16_t* const q = b16(p.strided("q", kB, {T, Hq, c.D}, s[1]));
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_paged_attention_bf16(out, lse, q, s[0], s[1], c.k, c.v, c.table, c.lengths, starts, c.B, T, max_new, Hq, c.H,
                                          c.D, c.pages, c.page_size, c.max_pages, scale, st);
    }));
  });
}

// paged cache, rotary, scale, out, lse or None, q, k_new, v_new
PyObject* decode_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 20, "decode_paged");
    const int Hq = p.size_of(17, "q", 3, 1, kPacked);
    const Paged c(p);
    const Rotary r(p);
    const float scale = p.real();
    int64_t s[4][2] = {};
    uint16_t* const out = b16(p.strided("out", kB, {c.B, Hq, c.D}, s[0]));
    float* const lse = p.none() ? nullptr : f32(p.here("lse", kF, {c.B, Hq}));
    const uint16_t *q = b16(p.strided("q", kB, {c.B, Hq, c.D}, s[1])), *kn = b16(p.strided("k_new", kB, {c.B, c.H, c.D}, s[2])),
                   *vn = b16(p.strided("v_new", kB, {c.B, c.H, c.D}, s[3]));
    const dadattn_stream_t st = stream();
    return done(without_gil([&] {
      return dadattn_decode_paged_bf16(out, lse, q, kn, vn, s[0], s[1], s[2], s[3], c.k, c.v, c.table, c.lengths, c.B, Hq, c.H, c.D,
                                       c.pages, c.page_size, c.max_pages, scale, r.turns, r.factor, r.rot, r.interleaved, st);
    }));
  });
}

// B, T, page_size, max_pages, lengths, starts or None
PyObject* advance_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Args p(a, n, 6, "advance_paged");
    const int B = p.integer(), T = p.integer(), page_size = p.integer(), max_pages = p.integer();
    int32_t* const lengths = static_cast<int32_t*>(ptr(p.here("lengths", at::kInt, {B})));
    const int32_t* const starts = p.none() ? nullptr : ints(p.here("starts", at::kInt, {int64_t(B) + 1}));
    const dadattn_stream_t st = stream();
    return done(without_gil([&] { return dadattn_paged_advance(lengths, starts, B, T, page_size, max_pages, st); }));
  });
}

PyObject* set_error_class(PyObject*, PyObject* cls) {
  Py_XINCREF(cls);
  Py_XDECREF(g_error_class);
  g_error_class = cls;
  Py_RETURN_NONE;
}

#define FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FAST(fwd_f32), FAST(bwd_f32), FAST(fwd_bf16), FAST(bwd_bf16), FAST(fwd_bf16_strided),
                           FAST(bwd_bf16_strided), FAST(fwd_bf16_window), FAST(bwd_bf16_window), FAST(fwd_via_bf16), FAST(bwd_via_bf16), FAST(mask_bits),
                           FAST(decode_f32), FAST(decode_bf16), FAST(decode_bf16_window), FAST(decode_fp8), FAST(fill_fp8),
                           FAST(evict_bf16), FAST(rotary), FAST(append_paged), FAST(paged_attention), FAST(decode_paged),
                           FAST(advance_paged),
                           {"set_error_class", set_error_class, METH_O, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&g_module); }
