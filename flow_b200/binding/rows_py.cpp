// rows_py.cpp — the row-wise operators called with torch tensors, without
// ctypes. A call's host time is what bounds small batches outside a CUDA graph:
// checking six tensors from Python takes 1.9 us and ctypes another, of 6 in all
// (2.2 of them the launch).
//
// Every function takes (handle, device, record, tensors...) in the order of the
// method of flow_b200.Context, makes that method's checks of each tensor (type,
// device, contiguous or a matrix at the record's stride, with all of the
// record's elements its own) and calls the C entry with the GIL released. It
// answers the status, or None where an argument is anything but a tensor that
// passes: the method then goes its own way, through other views, addresses and
// the errors' texts. kShort stands for a matrix at the record's stride with
// fewer rows or columns than the record, whose storage goes on: nothing is
// called, and the method refuses it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include "mapal_gpu.h"

namespace {

struct Library {
  decltype(&mapal_gpu_layer_norm) layer_norm;
  decltype(&mapal_gpu_layer_norm_grad) layer_norm_grad;
  decltype(&mapal_gpu_expert_sort) expert_sort;
  decltype(&mapal_gpu_expert_dispatch) expert_dispatch;
  decltype(&mapal_gpu_expert_combine) expert_combine;
  decltype(&mapal_gpu_expert_dispatch_grad) expert_dispatch_grad;
  decltype(&mapal_gpu_expert_combine_grad) expert_combine_grad;
  decltype(&mapal_gpu_quantize_rows_i8) quantize_rows_i8;
  decltype(&mapal_gpu_matmul_i8) matmul_i8;
} lib;
enum { kHandle, kNorm, kExpert, kQuant, kI8, kTypes };
PyObject* types[kTypes];  // the ctypes classes, kept for good

constexpr int kI32 = 4;          // beside MAPAL_DTYPE_*
constexpr int kShort = 1 << 16;  // beside the statuses; flow_b200._SHORT

uint64_t span(uint64_t rows, uint64_t cols, uint64_t ld) { return rows && cols ? (rows - 1) * ld + cols : 0; }

// The bytes of a ctypes instance of exactly this class.
template <typename R>
bool record(PyObject* o, int type, R* out) {
  if ((PyObject*)Py_TYPE(o) != types[type]) return false;
  Py_buffer view;
  if (PyObject_GetBuffer(o, &view, PyBUF_SIMPLE) != 0) {
    PyErr_Clear();
    return false;
  }
  const bool ok = view.len == (Py_ssize_t)sizeof(R);
  if (ok) memcpy(out, view.buf, sizeof(R));
  PyBuffer_Release(&view);
  return ok;
}

struct Call {
  PyObject* const* args;
  MapalGpuCtx* ctx = nullptr;
  long device = -1;
  bool ok, cut = false;

  template <typename R>
  Call(PyObject* const* a, Py_ssize_t n, Py_ssize_t tensors, int type, R* site) : args(a) {
    ok = n == 3 + tensors && record(a[0], kHandle, &ctx) && PyLong_CheckExact(a[1]) && record(a[2], type, site);
    if (ok) device = PyLong_AsLong(a[1]);
  }
  // Tensor i's address: `n` contiguous elements of type `code`; null for None.
  template <typename T = void>
  T* at(int i, int code, uint64_t n) {
    return static_cast<T*>(address(i, code, n, 0, 0, 0));
  }
  // rows x cols of them at row stride ld, contiguous or of a matrix at that stride.
  template <typename T = void>
  T* at(int i, int code, uint64_t rows, uint64_t cols, uint64_t ld) {
    return static_cast<T*>(address(i, code, span(rows, cols, ld), rows, cols, ld));
  }
  void* address(int i, int code, uint64_t need, uint64_t rows, uint64_t cols, uint64_t ld) {
    PyObject* o = args[3 + i];
    if (!ok || o == Py_None) return nullptr;
    static constexpr at::ScalarType kOf[] = {at::kFloat, at::kHalf, at::kBFloat16, at::kChar, at::kInt};
    if (!THPVariable_Check(o) || code < 0 || code > kI32) {
      ok = false;
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    ok = t.scalar_type() == kOf[code] && t.layout() == at::kStrided && t.get_device() == device;
    if (!ok) return nullptr;
    if (t.is_contiguous()) {
      ok = (uint64_t)t.numel() >= need;
    } else {
      ok = ld && t.dim() == 2 && t.size(0) > 1 && t.size(1) > 0 && t.stride(1) == 1 && (uint64_t)t.stride(0) == ld &&
           t.storage().nbytes() / t.itemsize() - (size_t)t.storage_offset() >= need;
      cut |= need && ((uint64_t)t.size(0) < rows || (uint64_t)t.size(1) < cols);
    }
    return ok ? t.data_ptr() : nullptr;
  }
  // Scratch of any type.
  void* bytes(int i, uint64_t* n) {
    PyObject* o = args[3 + i];
    *n = 0;
    if (!ok || o == Py_None) return nullptr;
    ok = THPVariable_Check(o);
    if (!ok) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    ok = t.layout() == at::kStrided && t.get_device() == device && t.is_contiguous();
    if (!ok) return nullptr;
    *n = t.nbytes();
    return t.data_ptr();
  }
  template <typename F>
  PyObject* run(F&& f) {
    if (!ok) Py_RETURN_NONE;
    if (cut) return PyLong_FromLong(kShort);
    int rc;
    Py_BEGIN_ALLOW_THREADS rc = f();
    Py_END_ALLOW_THREADS return PyLong_FromLong(rc);
  }
};

// No C++ exception leaves (a tensor without storage throws when asked for its address).
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    MapalNormSite s{};
    Call c(a, n, 6, kNorm, &s);
    const void* x = c.at(0, s.dtype, s.rows, s.d, s.ldx);
    const void *w = c.at(1, s.wtype, s.d), *b = c.at(2, s.wtype, s.d);
    void* y = c.at(3, s.dtype, s.rows, s.d, s.ldy);
    float *mean = c.at<float>(4, 0, s.rows), *rstd = c.at<float>(5, 0, s.rows);
    return c.run([&] { return lib.layer_norm(c.ctx, &s, x, w, b, y, mean, rstd); });
  });
}

PyObject* layer_norm_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    MapalNormSite s{};
    Call c(a, n, 9, kNorm, &s);
    const void *x = c.at(0, s.dtype, s.rows, s.d, s.ldx), *w = c.at(1, s.wtype, s.d);
    const float *mean = c.at<float>(2, 0, s.rows), *rstd = c.at<float>(3, 0, s.rows);
    const void* dy = c.at(4, s.dtype, s.rows, s.d, s.lddy);
    void* dx = c.at(5, s.dtype, s.rows, s.d, s.lddx);
    float *dw = c.at<float>(6, 0, s.d), *db = c.at<float>(7, 0, s.d);
    uint64_t bytes;
    void* work = c.bytes(8, &bytes);
    return c.run([&] { return lib.layer_norm_grad(c.ctx, &s, x, w, mean, rstd, dy, dx, dw, db, work, bytes); });
  });
}

PyObject* expert_sort(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    MapalExpertSite s{};
    Call c(a, n, 4, kExpert, &s);
    const uint64_t slots = s.tokens * s.k;
    const int32_t* ids = c.at<int32_t>(0, kI32, slots);
    int32_t *offsets = c.at<int32_t>(1, kI32, (uint64_t)s.experts + 1), *order = c.at<int32_t>(2, kI32, slots),
            *pos = c.at<int32_t>(3, kI32, slots);
    return c.run([&] { return lib.expert_sort(c.ctx, &s, ids, offsets, order, pos); });
  });
}

PyObject* expert_dispatch(PyObject*, PyObject* const* a, Py_ssize_t n) {  // x, pos, xs, scale, scale_out
  return guarded([&] {
    MapalExpertSite s{};
    Call c(a, n, 5, kExpert, &s);
    const void* x = c.at(0, s.dtype, s.tokens, s.d, s.ldt);
    const int32_t* pos = c.at<int32_t>(1, kI32, s.tokens * s.k);
    void* xs = c.at(2, s.dtype, s.rows, s.d, s.ldr);
    const float* scale = c.at<float>(3, 0, s.tokens);
    float* scale_out = c.at<float>(4, 0, s.rows);
    return c.run([&] { return lib.expert_dispatch(c.ctx, &s, x, scale, pos, xs, scale_out); });
  });
}

PyObject* expert_combine(PyObject*, PyObject* const* a, Py_ssize_t n) {  // h, w, pos, y
  return guarded([&] {
    MapalExpertSite s{};
    Call c(a, n, 4, kExpert, &s);
    const void* h = c.at(0, s.dtype, s.rows, s.d, s.ldr);
    const float* w = c.at<float>(1, 0, s.tokens * s.k);
    const int32_t* pos = c.at<int32_t>(2, kI32, s.tokens * s.k);
    void* y = c.at(3, s.dtype, s.tokens, s.d, s.ldt);
    return c.run([&] { return lib.expert_combine(c.ctx, &s, h, w, pos, y); });
  });
}

PyObject* expert_dispatch_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {  // dxs, pos, dx
  return guarded([&] {
    MapalExpertSite s{};
    Call c(a, n, 3, kExpert, &s);
    const void* dxs = c.at(0, s.dtype, s.rows, s.d, s.ldr);
    const int32_t* pos = c.at<int32_t>(1, kI32, s.tokens * s.k);
    void* dx = c.at(2, s.dtype, s.tokens, s.d, s.ldt);
    return c.run([&] { return lib.expert_dispatch_grad(c.ctx, &s, dxs, pos, dx); });
  });
}

PyObject* expert_combine_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {  // h, w, pos, dy, dh, dw
  return guarded([&] {
    MapalExpertSite s{};
    Call c(a, n, 6, kExpert, &s);
    const void* h = c.at(0, s.dtype, s.rows, s.d, s.ldr);
    const float* w = c.at<float>(1, 0, s.tokens * s.k);
    const int32_t* pos = c.at<int32_t>(2, kI32, s.tokens * s.k);
    const void* dy = c.at(3, s.dtype, s.tokens, s.d, s.ldt);
    void* dh = c.at(4, s.dtype, s.rows, s.d, s.ldr);
    float* dw = c.at<float>(5, 0, s.tokens * s.k);
    return c.run([&] { return lib.expert_combine_grad(c.ctx, &s, h, w, pos, dy, dh, dw); });
  });
}

PyObject* quantize_rows_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&] {
    MapalQuantSite s{};
    Call c(a, n, 3, kQuant, &s);
    const void* x = c.at(0, s.dtype, s.rows, s.d, s.ldx);
    int8_t* q = c.at<int8_t>(1, MAPAL_DTYPE_I8, s.rows, s.d, s.ldq);
    float* scale = c.at<float>(2, 0, s.rows);
    return c.run([&] { return lib.quantize_rows_i8(c.ctx, &s, x, q, scale); });
  });
}

PyObject* matmul_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {  // A, scale_a, B, scale_b, C, offsets
  return guarded([&] {
    MapalI8Site s{};
    Call c(a, n, 6, kI8, &s);
    const int8_t* A = c.at<int8_t>(0, MAPAL_DTYPE_I8, s.m, s.k, s.lda);
    const float* sa = c.at<float>(1, 0, s.m);
    const int8_t* B = c.at<int8_t>(2, MAPAL_DTYPE_I8, span(s.groups, span(s.n, s.k, s.ldb), s.ldg));
    const float* sb = c.at<float>(3, 0, (uint64_t)s.groups * s.n);
    void* C = c.at(4, s.dtype, s.m, s.n, s.ldc);
    const int32_t* offsets = c.at<int32_t>(5, kI32, (uint64_t)s.groups + 1);
    return c.run([&] { return lib.matmul_i8(c.ctx, &s, A, sa, B, sb, offsets, C); });
  });
}

// bind(addresses of the nine entries in Library's order, the five classes in order)
PyObject* bind(PyObject*, PyObject* args) {
  PyObject *entries, *classes;
  if (!PyArg_ParseTuple(args, "O!O!", &PyTuple_Type, &entries, &PyTuple_Type, &classes)) return nullptr;
  void* f[sizeof(Library) / sizeof(void*)];
  if (PyTuple_GET_SIZE(entries) != (Py_ssize_t)(sizeof(f) / sizeof(f[0])) || PyTuple_GET_SIZE(classes) != kTypes) {
    PyErr_SetString(PyExc_ValueError, "nine entries and five classes");
    return nullptr;
  }
  for (size_t i = 0; i < sizeof(f) / sizeof(f[0]); ++i) {
    f[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(entries, i));
    if (!f[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null entry");
      return nullptr;
    }
  }
  memcpy(&lib, f, sizeof(f));
  for (int i = 0; i < kTypes; ++i) {
    Py_INCREF(PyTuple_GET_ITEM(classes, i));
    Py_XSETREF(types[i], PyTuple_GET_ITEM(classes, i));
  }
  Py_RETURN_NONE;
}

#define FAST(name) \
  { #name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr }
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         FAST(layer_norm),
                         FAST(layer_norm_grad),
                         FAST(expert_sort),
                         FAST(expert_dispatch),
                         FAST(expert_combine),
                         FAST(expert_dispatch_grad),
                         FAST(expert_combine_grad),
                         FAST(quantize_rows_i8),
                         FAST(matmul_i8),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rows", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__rows() { return PyModule_Create(&module); }
