// Python's way to the 8-bit layer's entry points (include/cake_abi.h): checks torch tensors, makes the
// outputs that are not given, and enqueues on the device's current stream. A decode step makes several such
// calls of a few microseconds of GPU work each, and the same checks and allocations in Python took about
// 7 us a call beside 3 us for the launch; here they take 2.
//
// Built by build_native.py against the torch headers; the entry points' addresses come from the loaded
// libcake_b200.so (init), so this module links against no kernel.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/cake_abi.h"

namespace {

decltype(&cake_quantize_rows_enqueue) g_quantize = nullptr;
decltype(&cake_rms_norm_quantize_enqueue) g_norm = nullptr;
decltype(&cake_scaled_matmul_enqueue) g_matmul = nullptr;

constexpr int64_t kGroup = 128;
constexpr int64_t kLine = 128;  // codes get row pitches of whole lines
constexpr int kCodes = 3, kScales = 4;  // dtype numbers beyond CAKE_DTYPE_*

at::ScalarType scalar_type(long dtype) {
  switch (dtype) {
    case CAKE_DTYPE_F32: return at::kFloat;
    case CAKE_DTYPE_BF16: return at::kBFloat16;
    case CAKE_DTYPE_F16: return at::kHalf;
    case kCodes: return at::kFloat8_e4m3fn;
    default: return at::kFloat8_e8m0fnu;
  }
}

std::string describe(PyObject* obj) {
  if (!THPVariable_Check(obj)) return Py_TYPE(obj)->tp_name;
  const at::Tensor& t = THPVariable_Unpack(obj);
  std::string s = std::string(c10::toString(t.scalar_type())) + " (";
  for (int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.size(d));
  return s + ") with strides (" + [&] {
    std::string u;
    for (int64_t d = 0; d < t.dim(); ++d) u += (d ? ", " : "") + std::to_string(t.stride(d));
    return u;
  }() + ") on " + t.device().str();
}

bool refuse(PyObject* obj, const char* name, const std::string& wanted) {
  PyErr_SetString(PyExc_ValueError, (std::string(name) + " must " + wanted + ", got " + describe(obj)).c_str());
  return false;
}

struct Rows {
  void* data = nullptr;
  int64_t count = 0, stride = 0;
};

// A row operand: [rows, cols] (any number of rows if `rows` is negative), contiguous rows that do not overlap.
bool rows_of(PyObject* obj, int64_t cols, at::ScalarType dtype, const char* name, c10::Device device, int64_t rows, Rows* out) {
  const bool tensor = THPVariable_Check(obj);
  if (!tensor || THPVariable_Unpack(obj).scalar_type() != dtype || THPVariable_Unpack(obj).layout() != at::kStrided || THPVariable_Unpack(obj).dim() != 2 ||
      THPVariable_Unpack(obj).size(1) != cols || (rows >= 0 && THPVariable_Unpack(obj).size(0) != rows))
    return refuse(obj, name, std::string("be a ") + c10::toString(dtype) + " tensor of shape (" + (rows < 0 ? "rows" : std::to_string(rows)) + ", " + std::to_string(cols) + ")");
  const at::Tensor& t = THPVariable_Unpack(obj);
  if (t.device() != device) return refuse(obj, name, "be on " + device.str());
  out->count = t.size(0);
  out->stride = t.stride(0);
  if ((cols > 1 && t.stride(1) != 1) || (out->count > 1 && out->stride < cols)) return refuse(obj, name, "have contiguous rows that do not overlap");
  out->data = t.data_ptr();
  return true;
}

// The caller's output, checked, or a new one; a new reference, or null with an error set.
PyObject* output(PyObject* given, int64_t rows, int64_t cols, int64_t pitch, at::ScalarType dtype, const char* name, c10::Device device, Rows* out) {
  if (given != Py_None) {
    if (!rows_of(given, cols, dtype, name, device, rows, out)) return nullptr;
    Py_INCREF(given);
    return given;
  }
  at::Tensor t = at::detail::empty_strided_cuda({rows, cols}, {pitch, 1}, dtype, device);  // what torch.empty_strided comes to, without its dispatch
  out->data = t.data_ptr();
  out->count = rows;
  out->stride = pitch;
  return THPVariable_Wrap(std::move(t));
}

// References that are dropped when a call fails.
struct Held {
  PyObject* o[3] = {nullptr, nullptr, nullptr};
  ~Held() {
    for (PyObject* p : o) Py_XDECREF(p);
  }
  PyObject* give(int i) {
    PyObject* p = o[i];
    o[i] = nullptr;
    return p;
  }
};

int64_t line_pitch(int64_t cols) { return (cols + kLine - 1) / kLine * kLine; }
int64_t groups_of(int64_t cols) { return (cols + kGroup - 1) / kGroup; }

c10::Device cuda(PyObject* index) { return c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(PyLong_AsLong(index))); }

// Calls an entry point on the device's current stream, without the interpreter's lock.
template <typename F>
int32_t enqueue(c10::Device device, F&& call) {
  const c10::cuda::CUDAGuard guard(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  int32_t code;
  Py_BEGIN_ALLOW_THREADS
  code = call(stream);
  Py_END_ALLOW_THREADS
  return code;
}

bool arguments(const char* who, Py_ssize_t got, Py_ssize_t wanted) {
  if (got == wanted) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", who, wanted, got);
  return false;
}

// Each returns its outputs, or the library's error code as an int.

// (device index, x, columns, dtype, gate, codes or None, scales or None) -> (codes, scales)
PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments("quantize_rows", n, 7)) return nullptr;
  const c10::Device device = cuda(a[0]);
  const int64_t cols = PyLong_AsLongLong(a[2]);
  const long dtype = PyLong_AsLong(a[3]), gate = PyLong_AsLong(a[4]);
  if (PyErr_Occurred()) return nullptr;
  Rows x, q, s;
  if (!rows_of(a[1], gate ? 2 * cols : cols, scalar_type(dtype), "x", device, -1, &x)) return nullptr;
  Held held;
  if (!(held.o[0] = output(a[5], x.count, cols, line_pitch(cols), at::kFloat8_e4m3fn, "codes", device, &q))) return nullptr;
  if (!(held.o[1] = output(a[6], x.count, groups_of(cols), groups_of(cols), at::kFloat8_e8m0fnu, "scales", device, &s))) return nullptr;
  const int32_t code = enqueue(device, [&](void* stream) {
    return g_quantize(x.data, static_cast<int32_t>(dtype), x.stride, static_cast<int32_t>(gate), x.count, cols, q.data, q.stride, s.data, s.stride, stream);
  });
  if (code) return PyLong_FromLong(code);
  PyObject* result = PyTuple_New(2);
  if (!result) return nullptr;
  for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(result, i, held.give(i));
  return result;
  END_HANDLE_TH_ERRORS
}

// (device index, x, columns, dtype, weight, weight dtype, epsilon, residual or None, codes, scales and residual_out or None)
// -> (codes, scales, residual_out or None)
PyObject* rms_norm_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments("rms_norm_quantize", n, 11)) return nullptr;
  const c10::Device device = cuda(a[0]);
  const int64_t cols = PyLong_AsLongLong(a[2]);
  const long dtype = PyLong_AsLong(a[3]), weight_dtype = PyLong_AsLong(a[5]);
  const double epsilon = PyFloat_AsDouble(a[6]);
  if (PyErr_Occurred()) return nullptr;
  Rows x, r, ro, q, s;
  if (!rows_of(a[1], cols, scalar_type(dtype), "x", device, -1, &x)) return nullptr;
  const bool vector = THPVariable_Check(a[4]);
  if (!vector || THPVariable_Unpack(a[4]).scalar_type() != scalar_type(weight_dtype) || THPVariable_Unpack(a[4]).dim() != 1 ||
      THPVariable_Unpack(a[4]).size(0) != cols || THPVariable_Unpack(a[4]).device() != device || (cols > 1 && THPVariable_Unpack(a[4]).stride(0) != 1)) {
    refuse(a[4], "weight", std::string("be a contiguous ") + c10::toString(scalar_type(weight_dtype)) + " vector of " + std::to_string(cols) + " on " + device.str());
    return nullptr;
  }
  const void* weight = THPVariable_Unpack(a[4]).data_ptr();
  Held held;
  if (a[7] != Py_None) {
    if (!rows_of(a[7], cols, scalar_type(dtype), "residual", device, x.count, &r)) return nullptr;
    if (!(held.o[2] = output(a[10], x.count, cols, (cols + 7) / 8 * 8, scalar_type(dtype), "residual_out", device, &ro))) return nullptr;
  } else {
    Py_INCREF(Py_None);
    held.o[2] = Py_None;
  }
  if (!(held.o[0] = output(a[8], x.count, cols, line_pitch(cols), at::kFloat8_e4m3fn, "codes", device, &q))) return nullptr;
  if (!(held.o[1] = output(a[9], x.count, groups_of(cols), groups_of(cols), at::kFloat8_e8m0fnu, "scales", device, &s))) return nullptr;
  const int32_t code = enqueue(device, [&](void* stream) {
    return g_norm(x.data, static_cast<int32_t>(dtype), x.stride, r.data, r.stride, ro.data, ro.stride, weight, static_cast<int32_t>(weight_dtype),
                  static_cast<float>(epsilon), x.count, cols, q.data, q.stride, s.data, s.stride, stream);
  });
  if (code) return PyLong_FromLong(code);
  PyObject* result = PyTuple_New(3);
  if (!result) return nullptr;
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(result, i, held.give(i));
  return result;
  END_HANDLE_TH_ERRORS
}

// (device index, address of the descriptor, address of the status word, lhs, lhs_scales, rhs, rhs_scales, out or None) -> out
PyObject* scaled_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments("scaled_matmul", n, 8)) return nullptr;
  const c10::Device device = cuda(a[0]);
  const auto* desc = static_cast<const cake_scaled_matmul_desc*>(PyLong_AsVoidPtr(a[1]));
  auto* status = static_cast<int32_t*>(PyLong_AsVoidPtr(a[2]));
  if (PyErr_Occurred()) return nullptr;
  const int64_t groups = groups_of(desc->k);
  Rows lhs, lhs_scales, rhs, rhs_scales, out;
  if (!rows_of(a[3], desc->k, at::kFloat8_e4m3fn, "lhs", device, -1, &lhs) ||
      !rows_of(a[4], groups, at::kFloat8_e8m0fnu, "lhs_scales", device, lhs.count, &lhs_scales) ||
      !rows_of(a[5], desc->k, at::kFloat8_e4m3fn, "rhs", device, desc->n, &rhs) ||
      !rows_of(a[6], groups, at::kFloat8_e8m0fnu, "rhs_scales", device, desc->n, &rhs_scales))
    return nullptr;
  Held held;
  if (!(held.o[0] = output(a[7], lhs.count, desc->n, desc->n, scalar_type(desc->out_dtype), "out", device, &out))) return nullptr;
  const int32_t code = enqueue(device, [&](void* stream) {
    return g_matmul(desc, lhs.count, lhs.data, lhs.stride, lhs_scales.data, lhs_scales.stride, rhs.data, rhs.stride, rhs_scales.data, rhs_scales.stride,
                    out.data, out.stride, status, stream);
  });
  if (code) return PyLong_FromLong(code);
  return held.give(0);
  END_HANDLE_TH_ERRORS
}

// (tensor, columns, dtype, name, device index or -1 for the CPU, rows or -1) -> (rows, row stride): the check that the
// calls above make of every row operand.
PyObject* check_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arguments("check_rows", n, 6)) return nullptr;
  const int64_t cols = PyLong_AsLongLong(a[1]), rows = PyLong_AsLongLong(a[5]);
  const long dtype = PyLong_AsLong(a[2]), index = PyLong_AsLong(a[4]);
  const char* name = PyUnicode_AsUTF8(a[3]);
  if (PyErr_Occurred()) return nullptr;
  Rows r;
  const c10::Device device = index < 0 ? c10::Device(c10::kCPU) : c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(index));
  if (!rows_of(a[0], cols, scalar_type(dtype), name, device, rows, &r)) return nullptr;
  return Py_BuildValue("LL", static_cast<long long>(r.count), static_cast<long long>(r.stride));
  END_HANDLE_TH_ERRORS
}

// (addresses of cake_quantize_rows_enqueue, cake_rms_norm_quantize_enqueue, cake_scaled_matmul_enqueue)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments("init", n, 3)) return nullptr;
  g_quantize = reinterpret_cast<decltype(g_quantize)>(PyLong_AsVoidPtr(a[0]));
  g_norm = reinterpret_cast<decltype(g_norm)>(PyLong_AsVoidPtr(a[1]));
  g_matmul = reinterpret_cast<decltype(g_matmul)>(PyLong_AsVoidPtr(a[2]));
  if (PyErr_Occurred()) return nullptr;
  if (!g_quantize || !g_norm || !g_matmul) {
    PyErr_SetString(PyExc_ValueError, "init needs three entry points");
    return nullptr;
  }
  Py_RETURN_NONE;
}

#define FASTCALL(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FASTCALL(init), FASTCALL(check_rows), FASTCALL(quantize_rows), FASTCALL(rms_norm_quantize), FASTCALL(scaled_matmul), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "cake_torch_binding", "The 8-bit layer's entry points on torch tensors.", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_cake_torch_binding() { return PyModule_Create(&g_module); }
