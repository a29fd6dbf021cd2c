// The attention block's entry points for Python: argument checks, outputs from
// torch's allocator and the C-ABI call, in one native call each.  A decode step's
// kernels run for a few microseconds, and checking and allocating from Python took
// twice that (norm of one row 11.6 us a call, append 16.8).  The C-ABI's
// addresses come from the loaded library (bind), so there is one library and one
// way to it.  A C-ABI status other than SG_OK is returned as an int.
#include <Python.h>

#include <algorithm>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "sg_abi.h"

namespace {

decltype(&sg_add_rms_norm) p_add_rms_norm;
decltype(&sg_quantize_fp8) p_quantize_fp8;
decltype(&sg_fp8_linear) p_fp8_linear;
decltype(&sg_append_kv) p_append_kv;
decltype(&sg_paged_attention_work_bytes) p_work_bytes;
decltype(&sg_paged_attention_rows) p_paged_attention;

constexpr int64_t BLOCK = 128;  // values that share an 8-bit row's scale

// A Python exception is already set.
struct Raised {};

[[noreturn]] void type_error(const char* format, const char* name, int64_t a = 0, int64_t b = 0) {
  PyErr_Format(PyExc_TypeError, format, name, static_cast<long long>(a), static_cast<long long>(b));
  throw Raised();
}
[[noreturn]] void value_error(const char* text) {
  PyErr_SetString(PyExc_ValueError, text);
  throw Raised();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) type_error("%s must be a tensor", name);
  return THPVariable_Unpack(o);
}
bool is_none(PyObject* o) { return o == Py_None; }
bool on(const at::Tensor& t, int64_t device) { return t.is_cuda() && t.get_device() == device; }
bool misaligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0; }
// contiguous and 16-byte aligned: t itself, or a copy
at::Tensor packed(const at::Tensor& t) {
  at::Tensor c = t.contiguous();
  return misaligned(c) ? c.clone() : c;
}
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T>
T* at_ptr(const at::Tensor& t) {
  return static_cast<T*>(ptr(t));
}
void* stream(int64_t device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// a 2-D bf16 CUDA tensor, packed
at::Tensor rows(PyObject* o, const char* name) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kBFloat16 || !t.is_cuda() || t.dim() != 2) type_error("%s must be a 2-D bf16 CUDA tensor", name);
  return packed(t);
}
at::Tensor vector_bf16(PyObject* o, const char* name, int64_t n, int64_t device) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kBFloat16 || t.dim() != 1 || t.size(0) != n || !on(t, device))
    type_error("%s must be a bf16 [%lld] tensor on the rows' device", name, n);
  return packed(t);
}
at::Tensor matrix(PyObject* o, const char* name, at::ScalarType type, const char* type_name, int64_t a, int64_t b,
                  int64_t device) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type || t.dim() != 2 || t.size(0) != a || t.size(1) != b || !on(t, device)) {
    PyErr_Format(PyExc_TypeError, "%s must be an %s [%lld, %lld] tensor on the same device", name, type_name,
                 static_cast<long long>(a), static_cast<long long>(b));
    throw Raised();
  }
  return t.contiguous();
}
at::Tensor vector_int32(PyObject* o, const char* name, int64_t n, int64_t device) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !on(t, device))
    type_error("%s must be an int32 [%lld] tensor on the cache's device", name, n);
  return t.contiguous();
}
int checked_int(int64_t v) {
  if (v > INT32_MAX) value_error("a dimension is too large");
  return static_cast<int>(v);
}

PyObject* wrap(at::Tensor t) {
  PyObject* o = THPVariable_Wrap(std::move(t));
  if (!o) throw Raised();
  return o;
}
PyObject* tuple2(at::Tensor a, PyObject* b) {
  PyObject* t = PyTuple_New(2);
  if (!t) throw Raised();
  PyTuple_SET_ITEM(t, 0, wrap(std::move(a)));
  PyTuple_SET_ITEM(t, 1, b);
  return t;
}
PyObject* status(int st) { return PyLong_FromLong(st); }

template <typename F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Raised&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

bool want(Py_ssize_t n, Py_ssize_t expected, const char* name) {
  if (n == expected) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, expected);
  return false;
}

// add_rms_norm(x, weight, residual or None, eps, fp8): (y, h) or (y8, scales, h)
PyObject* add_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 5, "add_rms_norm")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor x = rows(a[0], "x");
    const int64_t T = x.size(0), H = x.size(1), device = x.get_device();
    const at::Tensor weight = vector_bf16(a[1], "weight", H, device);
    const double eps = PyFloat_AsDouble(a[3]);
    if (eps == -1.0 && PyErr_Occurred()) throw Raised();
    const bool fp8 = a[4] == Py_True;
    at::Tensor residual, h, y, scales;
    if (!is_none(a[2])) {
      residual = rows(a[2], "residual");
      if (residual.size(0) != T || residual.size(1) != H || residual.get_device() != device)
        value_error("residual must have x's shape and device");
      h = at::empty({T, H}, x.options());
    }
    y = at::empty({T, H}, fp8 ? x.options().dtype(at::kFloat8_e4m3fn) : x.options());
    if (fp8) scales = at::empty({(H + BLOCK - 1) / BLOCK, T}, x.options().dtype(at::kFloat));
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    const int st = p_add_rms_norm(at_ptr<uint16_t>(x), at_ptr<uint16_t>(residual), at_ptr<uint16_t>(weight), checked_int(T),
                                  checked_int(H), static_cast<float>(eps), at_ptr<uint16_t>(h),
                                  fp8 ? nullptr : at_ptr<uint16_t>(y), fp8 ? at_ptr<uint8_t>(y) : nullptr,
                                  at_ptr<float>(scales), stream(device));
    if (st != SG_OK) return status(st);
    PyObject* h_out = h.defined() ? wrap(h) : Py_NewRef(a[0]);  // without a residual the stream is x itself
    if (!fp8) return tuple2(y, h_out);
    PyObject* t = PyTuple_New(3);
    if (!t) throw Raised();
    PyTuple_SET_ITEM(t, 0, wrap(y));
    PyTuple_SET_ITEM(t, 1, wrap(scales));
    PyTuple_SET_ITEM(t, 2, h_out);
    return t;
  });
}

// quantize_fp8(x): (x8, scales)
PyObject* quantize_fp8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 1, "quantize_fp8")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor x = rows(a[0], "x");
    const int64_t T = x.size(0), K = x.size(1);
    at::Tensor x8 = at::empty({T, K}, x.options().dtype(at::kFloat8_e4m3fn));
    at::Tensor scales = at::empty({(K + BLOCK - 1) / BLOCK, T}, x.options().dtype(at::kFloat));
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(x.get_device()));
    const int st = p_quantize_fp8(at_ptr<uint16_t>(x), checked_int(T), checked_int(K), at_ptr<uint8_t>(x8),
                                  at_ptr<float>(scales), stream(x.get_device()));
    return st != SG_OK ? status(st) : tuple2(x8, wrap(scales));
  });
}

at::Tensor rows_fp8(PyObject* o, const char* name, int64_t device) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kFloat8_e4m3fn || t.dim() != 2 || !on(t, device))
    type_error("%s must be a 2-D float8_e4m3fn CUDA tensor", name);
  return packed(t);
}

// fp8_linear(x8, x_scales, w8, w_scales): out
PyObject* fp8_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 4, "fp8_linear")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& first = tensor(a[0], "x8");
    const int64_t device = first.is_cuda() ? first.get_device() : -1;
    const at::Tensor x8 = rows_fp8(a[0], "x8", device), w8 = rows_fp8(a[2], "w8", device);
    const int64_t T = x8.size(0), K = x8.size(1), N = w8.size(0), blocks = (K + BLOCK - 1) / BLOCK;
    if (w8.size(1) != K) value_error("x8 and w8 must have rows of one length");
    const at::Tensor xs = matrix(a[1], "x_scales", at::kFloat, "fp32", blocks, T, device);
    const at::Tensor ws = matrix(a[3], "w_scales", at::kFloat, "fp32", (N + BLOCK - 1) / BLOCK, blocks, device);
    at::Tensor out = at::empty({T, N}, x8.options().dtype(at::kBFloat16));
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    const int st = p_fp8_linear(at_ptr<uint8_t>(x8), at_ptr<float>(xs), at_ptr<uint8_t>(w8), at_ptr<float>(ws),
                                checked_int(T), checked_int(K), checked_int(N), at_ptr<uint16_t>(out), stream(device));
    return st != SG_OK ? status(st) : wrap(out);
  });
}

// Elements between tokens; a single token's stride says nothing (and contiguous()
// leaves it as it is).
int64_t token_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2); }

// [T, heads, D] bf16 whose heads are contiguous and whose tokens lie a multiple of
// 16 bytes apart (a view of a wider row as it is), else a copy
at::Tensor heads(PyObject* o, const char* name, int64_t D, int64_t device) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kBFloat16 || t.dim() != 3 || t.size(2) != D || !on(t, device))
    type_error("%s must be a bf16 [T, heads, %lld] tensor on the cache's device", name, D);
  if (t.stride(2) != 1 || (t.size(1) > 1 && t.stride(1) != D) || token_stride(t) % 8 || token_stride(t) < 0 || misaligned(t))
    return packed(t);
  return t;
}

const sg_kv_cache* cache_at(PyObject* address) {
  const void* p = PyLong_AsVoidPtr(address);
  if (!p) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null cache descriptor");
    throw Raised();
  }
  return static_cast<const sg_kv_cache*>(p);
}
int64_t device_of(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
at::Tensor page_table(PyObject* o, int64_t rows_needed, int64_t device) {
  const at::Tensor& t = tensor(o, "page_table");
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) < rows_needed || !on(t, device))
    type_error("%s must be an int32 [rows, pages] tensor on the cache's device", "page_table");
  return t.contiguous();
}

// append_kv(cache address, device, q, k, v, page_table, positions, rope, rows, q_weight, k_weight, eps): q_out
PyObject* append_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 12, "append_kv")) return nullptr;
  return guarded([&]() -> PyObject* {
    const sg_kv_cache* c = cache_at(a[0]);
    const int64_t device = device_of(a[1]), D = c->head_dim;
    const at::Tensor q = heads(a[2], "q", D, device), k = heads(a[3], "k", D, device), v = heads(a[4], "v", D, device);
    const int64_t T = q.size(0);
    if (k.size(0) != T || v.size(0) != T || k.size(1) != c->kv_heads || v.size(1) != c->kv_heads)
      value_error("k and v must have q's tokens and the cache's heads");
    const at::Tensor table = page_table(a[5], 0, device), positions = vector_int32(a[6], "positions", T, device);
    at::Tensor rope, row_of, q_weight, k_weight;
    if (!is_none(a[8])) row_of = vector_int32(a[8], "rows", T, device);
    else if (table.size(0) < T) value_error("without rows, page_table needs a row for every token");
    if (!is_none(a[7])) {
      const at::Tensor& t = tensor(a[7], "rope");
      if (t.scalar_type() != at::kFloat || t.dim() != 2 || !on(t, device))
        type_error("%s must be an fp32 [max_pos, rot] tensor on the cache's device", "rope");
      rope = packed(t);
    }
    if (!is_none(a[9])) q_weight = vector_bf16(a[9], "q_weight", D, device);
    if (!is_none(a[10])) k_weight = vector_bf16(a[10], "k_weight", D, device);
    const double eps = PyFloat_AsDouble(a[11]);
    if (eps == -1.0 && PyErr_Occurred()) throw Raised();
    at::Tensor out = at::empty({T, q.size(1), D}, q.options());
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    const int st = p_append_kv(
        c, at_ptr<uint16_t>(q), token_stride(q), at_ptr<uint16_t>(k), token_stride(k), at_ptr<uint16_t>(v), token_stride(v),
        checked_int(T), checked_int(q.size(1)), at_ptr<int32_t>(table), checked_int(table.size(0)),
        checked_int(table.size(1)), at_ptr<int32_t>(row_of), at_ptr<int32_t>(positions), at_ptr<float>(rope),
        rope.defined() ? checked_int(rope.size(1)) : 0, rope.defined() ? checked_int(rope.size(0)) : 0,
        at_ptr<uint16_t>(q_weight), at_ptr<uint16_t>(k_weight), static_cast<float>(eps), at_ptr<uint16_t>(out),
        stream(device));
    return st != SG_OK ? status(st) : wrap(out);
  });
}

// paged_attention(cache address, device, q, page_table, lengths, scale, rows, max_length): out
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!want(n, 8, "paged_attention")) return nullptr;
  return guarded([&]() -> PyObject* {
    const sg_kv_cache* c = cache_at(a[0]);
    const int64_t device = device_of(a[1]), D = c->head_dim;
    const at::Tensor q = heads(a[2], "q", D, device);
    const int64_t B = q.size(0), Hq = q.size(1);
    const at::Tensor table = page_table(a[3], is_none(a[6]) ? B : 0, device), lengths = vector_int32(a[4], "lengths", B, device);
    const double scale = PyFloat_AsDouble(a[5]);
    if (scale == -1.0 && PyErr_Occurred()) throw Raised();
    at::Tensor row_of;
    if (!is_none(a[6])) row_of = vector_int32(a[6], "rows", B, device);
    int64_t max_length = INT32_MAX;
    if (!is_none(a[7])) {
      max_length = PyLong_AsLongLong(a[7]);
      if (max_length == -1 && PyErr_Occurred()) throw Raised();
      if (max_length < 0) value_error("max_length must not be negative");
    }
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(device));
    const long long bytes = p_work_bytes(c, checked_int(B), checked_int(Hq));
    if (bytes < 0) return status(static_cast<int>(bytes));
    at::Tensor out = at::empty({B, Hq, D}, q.options());
    at::Tensor work = at::empty({bytes}, q.options().dtype(at::kByte));
    const int st = p_paged_attention(c, at_ptr<uint16_t>(q), token_stride(q), checked_int(B), checked_int(Hq),
                                     at_ptr<int32_t>(table), checked_int(table.size(0)), checked_int(table.size(1)),
                                     at_ptr<int32_t>(row_of), at_ptr<int32_t>(lengths),
                                     static_cast<int>(std::min<int64_t>(max_length, INT32_MAX)),
                                     static_cast<float>(scale), at_ptr<uint16_t>(out), work.data_ptr(), bytes, stream(device));
    return st != SG_OK ? status(st) : wrap(out);
  });
}

// bind({name: address}): the C-ABI functions of the loaded library
PyObject* bind(PyObject*, PyObject* names) {
  struct Entry {
    const char* name;
    void** to;
  } entries[] = {{"sg_add_rms_norm", reinterpret_cast<void**>(&p_add_rms_norm)},
                 {"sg_quantize_fp8", reinterpret_cast<void**>(&p_quantize_fp8)},
                 {"sg_fp8_linear", reinterpret_cast<void**>(&p_fp8_linear)},
                 {"sg_append_kv", reinterpret_cast<void**>(&p_append_kv)},
                 {"sg_paged_attention_work_bytes", reinterpret_cast<void**>(&p_work_bytes)},
                 {"sg_paged_attention_rows", reinterpret_cast<void**>(&p_paged_attention)}};
  if (!PyDict_Check(names)) {
    PyErr_SetString(PyExc_TypeError, "bind takes a dict of addresses");
    return nullptr;
  }
  void* found[6];
  for (int i = 0; i < 6; ++i) {
    PyObject* v = PyDict_GetItemString(names, entries[i].name);
    found[i] = v ? PyLong_AsVoidPtr(v) : nullptr;
    if (!found[i]) {
      if (!PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%s", entries[i].name);
      return nullptr;
    }
  }
  for (int i = 0; i < 6; ++i) *entries[i].to = found[i];
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {{"bind", bind, METH_O, nullptr},
                         {"add_rms_norm", FAST(add_rms_norm), METH_FASTCALL, nullptr},
                         {"quantize_fp8", FAST(quantize_fp8), METH_FASTCALL, nullptr},
                         {"fp8_linear", FAST(fp8_linear), METH_FASTCALL, nullptr},
                         {"append_kv", FAST(append_kv), METH_FASTCALL, nullptr},
                         {"paged_attention", FAST(paged_attention), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }
