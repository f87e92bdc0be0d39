// CPython entry to the GEMM calls of the library (cumpsgemm_amd/_call.<suffix>.so).
//
// A small product is bound by what one call costs on the host.  Through ctypes the
// conversion of its 17 arguments takes 1.8 us of the 5.3 us of a 128^3 product in a
// loop of calls; here 0.4 of 4.2.  The functions are called at the
// addresses that `bind` is given (the library that ctypes has loaded).  An argument
// of a type that is not the usual one -- anything but int sizes, float / complex
// scalars, and ints, None or objects with data_ptr() as pointers -- makes a call
// return None with nothing done: ctypes then converts it, or refuses it.  What an
// object's data_ptr() raises is raised by the call.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <cstring>
#include <cumpsgemm/cumpsgemm.h>
#include <cumpsgemm/cumpsgemm_ext.h>

namespace {
struct Functions {
  decltype(&cuMpSGEMM_sgemm) sgemm;
  decltype(&cuMpSGEMM_cgemm) cgemm;
  decltype(&cuMpSGEMM_sgemm_strided_batch) sgemm_strided_batch;
  decltype(&cuMpSGEMM_cgemm_strided_batch) cgemm_strided_batch;
  decltype(&cuMpSGEMM_sgemm_pipeline) sgemm_pipeline;
  decltype(&cuMpSGEMM_cgemm_pipeline) cgemm_pipeline;
  decltype(&cuMpSGEMM_sgemm_Mx2x2) sgemm_Mx2x2;
  decltype(&cuMpSGEMM_cgemm_Mx2x2) cgemm_Mx2x2;
  decltype(&cuMpSGEMM_sgemm_2xNx2) sgemm_2xNx2;
  decltype(&cuMpSGEMM_cgemm_2xNx2) cgemm_2xNx2;
} f;
constexpr Py_ssize_t kFunctions = sizeof(Functions) / sizeof(void *);
struct GroupedFunctions { // products of experts' layers
  decltype(&cuMpSGEMM_gemm_grouped) grouped;
  decltype(&cuMpSGEMM_gemm_grouped_k) grouped_k;
  decltype(&cuMpSGEMM_gemm_i8) i8;
  decltype(&cuMpSGEMM_quantize_i8) quantize;
} fg;
constexpr Py_ssize_t kGroupedFunctions = sizeof(GroupedFunctions) / sizeof(void *);
struct GatedFunctions { // gated feed-forward blocks and 8-bit floating point
  decltype(&cuMpSGEMM_gemm_gated) gated;
  decltype(&cuMpSGEMM_gemm_gated_backward) backward;
  decltype(&cuMpSGEMM_gemm_f8) f8;
  decltype(&cuMpSGEMM_gemm_gated_f8) gated_f8;
  decltype(&cuMpSGEMM_quantize_f8) quantize_f8;
} fb;
constexpr Py_ssize_t kGatedFunctions = sizeof(GatedFunctions) / sizeof(void *);
PyObject *data_ptr_name;

// The arguments of a call, taken one after the other; `ok` goes false at the first
// one that is not of the usual type, or whose data_ptr() raised (the exception is set).
struct Args {
  PyObject *const *arg;
  bool ok = true;
  uint64_t integer(PyObject *o) {
    if (!PyLong_Check(o)) {
      ok = false;
      return 0;
    }
    const uint64_t v = PyLong_AsUnsignedLongLongMask(o); // (as ctypes: no check of the range)
    if (v == (uint64_t)-1 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
  uint64_t u64() { return ok ? integer(*arg++) : 0; }
  hipblasOperation_t op() { return (hipblasOperation_t)(int)u64(); }
  template <class T> T *ptr() {
    if (!ok) return nullptr;
    PyObject *const o = *arg++;
    if (o == Py_None) return nullptr;
    if (PyLong_Check(o)) return reinterpret_cast<T *>(integer(o));
    PyObject *const p = PyObject_CallMethodNoArgs(o, data_ptr_name);
    if (p == nullptr) {
      if (PyErr_ExceptionMatches(PyExc_AttributeError)) PyErr_Clear(); // (no data_ptr)
      ok = false;
      return nullptr;
    }
    const uint64_t v = integer(p);
    Py_DECREF(p);
    return reinterpret_cast<T *>(v);
  }
  void scalar(float &v) {
    if (!ok) return;
    PyObject *const o = *arg++;
    if (PyFloat_CheckExact(o)) v = (float)PyFloat_AS_DOUBLE(o);
    else ok = false;
  }
  void scalar(hipComplex &v) {
    if (!ok) return;
    PyObject *const o = *arg++;
    if (PyComplex_CheckExact(o)) v = {(float)PyComplex_RealAsDouble(o), (float)PyComplex_ImagAsDouble(o)};
    else if (PyFloat_CheckExact(o)) v = {(float)PyFloat_AS_DOUBLE(o), 0.0f};
    else ok = false;
  }
};

template <class Call> PyObject *status(const Args &a, Call &&call) {
  if (!a.ok) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
  hipblasStatus_t st;
  Py_BEGIN_ALLOW_THREADS
  st = call();
  Py_END_ALLOW_THREADS
  return PyLong_FromLong((long)st);
}
bool count_is(const Py_ssize_t n, const Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
  return false;
}

// handle, op_a, op_b, m, n, k, alpha, a, lda, b, ldb, beta, c, ldc, mode
template <class T, class Fn> PyObject *gemm_of(PyObject *const *args, const Fn fn) {
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const auto op_a = x.op(), op_b = x.op();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  T alpha{}, beta{};
  x.scalar(alpha);
  T *const a = x.ptr<T>();
  const uint64_t lda = x.u64();
  T *const b = x.ptr<T>();
  const uint64_t ldb = x.u64();
  x.scalar(beta);
  T *const c = x.ptr<T>();
  const uint64_t ldc = x.u64();
  const auto mode = (cuMpSGEMM_compute_mode_t)(int)x.u64();
  return status(x, [&] { return fn(h, op_a, op_b, m, n, k, &alpha, a, lda, b, ldb, &beta, c, ldc, mode); });
}
// ..., a, lda, stride_a, b, ldb, stride_b, beta, c, ldc, stride_c, batch, mode
template <class T, class Fn> PyObject *strided_batch_of(PyObject *const *args, const Fn fn) {
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const auto op_a = x.op(), op_b = x.op();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  T alpha{}, beta{};
  x.scalar(alpha);
  T *const a = x.ptr<T>();
  const uint64_t lda = x.u64(), stride_a = x.u64();
  T *const b = x.ptr<T>();
  const uint64_t ldb = x.u64(), stride_b = x.u64();
  x.scalar(beta);
  T *const c = x.ptr<T>();
  const uint64_t ldc = x.u64(), stride_c = x.u64(), batch = x.u64();
  const auto mode = (cuMpSGEMM_compute_mode_t)(int)x.u64();
  return status(x, [&] {
    return fn(h, op_a, op_b, m, n, k, &alpha, a, lda, stride_a, b, ldb, stride_b, &beta, c, ldc, stride_c, batch, mode);
  });
}
// ... and restore_ab; returns (status, (three ids))
template <class T, class Fn> PyObject *pipeline_of(PyObject *const *args, const Fn fn) {
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const auto op_a = x.op(), op_b = x.op();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  T alpha{}, beta{};
  x.scalar(alpha);
  T *const a = x.ptr<T>();
  const uint64_t lda = x.u64(), stride_a = x.u64();
  T *const b = x.ptr<T>();
  const uint64_t ldb = x.u64(), stride_b = x.u64();
  x.scalar(beta);
  T *const c = x.ptr<T>();
  const uint64_t ldc = x.u64(), stride_c = x.u64(), batch = x.u64();
  const auto mode = (cuMpSGEMM_compute_mode_t)(int)x.u64();
  const int restore = (int)x.u64();
  unsigned ids[3] = {};
  PyObject *const st = status(x, [&] {
    return fn(h, op_a, op_b, m, n, k, &alpha, a, lda, stride_a, b, ldb, stride_b, &beta, c, ldc, stride_c, batch, mode,
              restore, ids);
  });
  if (st == nullptr || st == Py_None) return st;
  return Py_BuildValue("N(III)", st, ids[0], ids[1], ids[2]);
}
// handle, op_a, op_b, size, alpha, a, lda, stride_a, b, ldb, stride_b, beta, c, ldc, stride_c, batch
template <class T, class Fn> PyObject *by2x2_of(PyObject *const *args, const Fn fn) {
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const auto op_a = x.op(), op_b = x.op();
  const uint64_t size = x.u64();
  T alpha{}, beta{};
  x.scalar(alpha);
  T *const a = x.ptr<T>();
  const uint64_t lda = x.u64(), stride_a = x.u64();
  T *const b = x.ptr<T>();
  const uint64_t ldb = x.u64(), stride_b = x.u64();
  x.scalar(beta);
  T *const c = x.ptr<T>();
  const uint64_t ldc = x.u64(), stride_c = x.u64(), batch = x.u64();
  return status(x, [&] {
    return fn(h, op_a, op_b, size, &alpha, a, lda, stride_a, b, ldb, stride_b, &beta, c, ldc, stride_c, batch);
  });
}

// every function takes `cplx` first
bool is_complex(PyObject *o, bool &cplx) {
  const int r = PyObject_IsTrue(o);
  cplx = r > 0;
  return r >= 0;
}
PyObject *gemm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  bool cplx;
  if (!count_is(n, 16) || !is_complex(args[0], cplx)) return nullptr;
  return cplx ? gemm_of<hipComplex>(args + 1, f.cgemm) : gemm_of<float>(args + 1, f.sgemm);
}
PyObject *strided_batch(PyObject *, PyObject *const *args, Py_ssize_t n) {
  bool cplx;
  if (!count_is(n, 20) || !is_complex(args[0], cplx)) return nullptr;
  return cplx ? strided_batch_of<hipComplex>(args + 1, f.cgemm_strided_batch)
              : strided_batch_of<float>(args + 1, f.sgemm_strided_batch);
}
PyObject *pipeline(PyObject *, PyObject *const *args, Py_ssize_t n) {
  bool cplx;
  if (!count_is(n, 21) || !is_complex(args[0], cplx)) return nullptr;
  return cplx ? pipeline_of<hipComplex>(args + 1, f.cgemm_pipeline) : pipeline_of<float>(args + 1, f.sgemm_pipeline);
}
PyObject *mx2x2(PyObject *, PyObject *const *args, Py_ssize_t n) {
  bool cplx;
  if (!count_is(n, 17) || !is_complex(args[0], cplx)) return nullptr;
  return cplx ? by2x2_of<hipComplex>(args + 1, f.cgemm_Mx2x2) : by2x2_of<float>(args + 1, f.sgemm_Mx2x2);
}
PyObject *twoxnx2(PyObject *, PyObject *const *args, Py_ssize_t n) {
  bool cplx;
  if (!count_is(n, 17) || !is_complex(args[0], cplx)) return nullptr;
  return cplx ? by2x2_of<hipComplex>(args + 1, f.cgemm_2xNx2) : by2x2_of<float>(args + 1, f.sgemm_2xNx2);
}
// handle, op_a, m, n, k, alpha, a, lda, stride_a, b, ldb, beta, c, ldc, offsets, groups, mode, type_ab, type_c
PyObject *gemm_grouped(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  if (!count_is(n_args, 19)) return nullptr;
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const auto op_a = x.op();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  float alpha{}, beta{};
  x.scalar(alpha);
  void *const a = x.ptr<void>();
  const uint64_t lda = x.u64(), stride_a = x.u64();
  void *const b = x.ptr<void>();
  const uint64_t ldb = x.u64();
  x.scalar(beta);
  void *const c = x.ptr<void>();
  const uint64_t ldc = x.u64();
  const int *const offsets = x.ptr<int>();
  const uint64_t groups = x.u64();
  const auto mode = (cuMpSGEMM_compute_mode_t)(int)x.u64();
  const auto type_ab = (hipDataType)(int)x.u64(), type_c = (hipDataType)(int)x.u64();
  return status(x, [&] {
    return fg.grouped(h, op_a, m, n, k, &alpha, a, lda, stride_a, b, ldb, &beta, c, ldc, offsets, groups, mode, type_ab, type_c);
  });
}
// handle, m, n, k, alpha, a, lda, b, ldb, beta, c, ldc, stride_c, offsets, groups, mode, type_ab, type_c
PyObject *gemm_grouped_k(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  if (!count_is(n_args, 18)) return nullptr;
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  float alpha{}, beta{};
  x.scalar(alpha);
  void *const a = x.ptr<void>();
  const uint64_t lda = x.u64();
  void *const b = x.ptr<void>();
  const uint64_t ldb = x.u64();
  x.scalar(beta);
  void *const c = x.ptr<void>();
  const uint64_t ldc = x.u64(), stride_c = x.u64();
  const int *const offsets = x.ptr<int>();
  const uint64_t groups = x.u64();
  const auto mode = (cuMpSGEMM_compute_mode_t)(int)x.u64();
  const auto type_ab = (hipDataType)(int)x.u64(), type_c = (hipDataType)(int)x.u64();
  return status(x, [&] {
    return fg.grouped_k(h, m, n, k, &alpha, a, lda, b, ldb, &beta, c, ldc, stride_c, offsets, groups, mode, type_ab, type_c);
  });
}
// handle, m, n, k, a, lda, stride_a, scale_a, b, ldb, scale_b, c, ldc, type_c, offsets, groups
PyObject *gemm_i8(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  if (!count_is(n_args, 16)) return nullptr;
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  const int8_t *const a = x.ptr<int8_t>();
  const uint64_t lda = x.u64(), stride_a = x.u64();
  const float *const scale_a = x.ptr<float>();
  const int8_t *const b = x.ptr<int8_t>();
  const uint64_t ldb = x.u64();
  const float *const scale_b = x.ptr<float>();
  void *const c = x.ptr<void>();
  const uint64_t ldc = x.u64();
  const auto type_c = (hipDataType)(int)x.u64();
  const int *const offsets = x.ptr<int>();
  const uint64_t groups = x.u64();
  return status(x, [&] {
    return fg.i8(h, m, n, k, a, lda, stride_a, scale_a, b, ldb, scale_b, c, ldc, type_c, offsets, groups);
  });
}
// handle, k, n, x, ldx, type_x, q, ldq, scale
PyObject *quantize_i8(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  if (!count_is(n_args, 9)) return nullptr;
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const uint64_t k = x.u64(), n = x.u64();
  void *const values = x.ptr<void>();
  const uint64_t ldx = x.u64();
  const auto type_x = (hipDataType)(int)x.u64();
  int8_t *const q = x.ptr<int8_t>();
  const uint64_t ldq = x.u64();
  float *const scale = x.ptr<float>();
  return status(x, [&] { return fg.quantize(h, k, n, values, ldx, type_x, q, ldq, scale); });
}
// handle, op_a, activation, m, n, k, gate, up, lda, stride_a, b, ldb, c, ldc, z_gate, z_up, ldz, offsets, groups, mode, type
PyObject *gemm_gated(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  if (!count_is(n_args, 21)) return nullptr;
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const auto op_a = x.op();
  const auto act = (cuMpSGEMM_activation_t)(int)x.u64();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  void *const gate = x.ptr<void>(), *const up = x.ptr<void>();
  const uint64_t lda = x.u64(), stride_a = x.u64();
  void *const b = x.ptr<void>();
  const uint64_t ldb = x.u64();
  void *const c = x.ptr<void>();
  const uint64_t ldc = x.u64();
  void *const z_gate = x.ptr<void>(), *const z_up = x.ptr<void>();
  const uint64_t ldz = x.u64();
  const int *const offsets = x.ptr<int>();
  const uint64_t groups = x.u64();
  const auto mode = (cuMpSGEMM_compute_mode_t)(int)x.u64();
  const auto type = (hipDataType)(int)x.u64();
  return status(x, [&] {
    return fb.gated(h, op_a, act, m, n, k, gate, up, lda, stride_a, b, ldb, c, ldc, z_gate, z_up, ldz, offsets, groups, mode, type);
  });
}
// handle, op_a, activation, m, n, k, a, lda, stride_a, b, ldb, z_gate, z_up, ldz, d_gate, d_up, ldd, c, ldc, offsets, groups, mode,
// type
PyObject *gemm_gated_backward(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  if (!count_is(n_args, 23)) return nullptr;
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const auto op_a = x.op();
  const auto act = (cuMpSGEMM_activation_t)(int)x.u64();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  void *const a = x.ptr<void>();
  const uint64_t lda = x.u64(), stride_a = x.u64();
  void *const b = x.ptr<void>();
  const uint64_t ldb = x.u64();
  void *const z_gate = x.ptr<void>(), *const z_up = x.ptr<void>();
  const uint64_t ldz = x.u64();
  void *const d_gate = x.ptr<void>(), *const d_up = x.ptr<void>();
  const uint64_t ldd = x.u64();
  void *const c = x.ptr<void>();
  const uint64_t ldc = x.u64();
  const int *const offsets = x.ptr<int>();
  const uint64_t groups = x.u64();
  const auto mode = (cuMpSGEMM_compute_mode_t)(int)x.u64();
  const auto type = (hipDataType)(int)x.u64();
  return status(x, [&] {
    return fb.backward(h, op_a, act, m, n, k, a, lda, stride_a, b, ldb, z_gate, z_up, ldz, d_gate, d_up, ldd, c, ldc, offsets, groups,
                       mode, type);
  });
}
// handle, op_a, m, n, k, a, lda, stride_a, type_a, scale_a, stride_scale, b, ldb, type_b, scale_b, c, ldc, type_c, offsets, groups
PyObject *gemm_f8(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  if (!count_is(n_args, 20)) return nullptr;
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const auto op_a = x.op();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  void *const a = x.ptr<void>();
  const uint64_t lda = x.u64(), stride_a = x.u64();
  const auto type_a = (hipDataType)(int)x.u64();
  const float *const scale_a = x.ptr<float>();
  const uint64_t stride_scale = x.u64();
  void *const b = x.ptr<void>();
  const uint64_t ldb = x.u64();
  const auto type_b = (hipDataType)(int)x.u64();
  const float *const scale_b = x.ptr<float>();
  void *const c = x.ptr<void>();
  const uint64_t ldc = x.u64();
  const auto type_c = (hipDataType)(int)x.u64();
  const int *const offsets = x.ptr<int>();
  const uint64_t groups = x.u64();
  return status(x, [&] {
    return fb.f8(h, op_a, m, n, k, a, lda, stride_a, type_a, scale_a, stride_scale, b, ldb, type_b, scale_b, c, ldc, type_c, offsets, groups);
  });
}
// handle, activation, m, n, k, gate, up, lda, stride_a, type_a, scale_gate, scale_up, stride_scale, b, ldb, type_b, scale_b, c, ldc,
// type_c, offsets, groups
PyObject *gemm_gated_f8(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  if (!count_is(n_args, 22)) return nullptr;
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const auto act = (cuMpSGEMM_activation_t)(int)x.u64();
  const uint64_t m = x.u64(), n = x.u64(), k = x.u64();
  void *const gate = x.ptr<void>(), *const up = x.ptr<void>();
  const uint64_t lda = x.u64(), stride_a = x.u64();
  const auto type_a = (hipDataType)(int)x.u64();
  const float *const scale_gate = x.ptr<float>(), *const scale_up = x.ptr<float>();
  const uint64_t stride_scale = x.u64();
  void *const b = x.ptr<void>();
  const uint64_t ldb = x.u64();
  const auto type_b = (hipDataType)(int)x.u64();
  const float *const scale_b = x.ptr<float>();
  void *const c = x.ptr<void>();
  const uint64_t ldc = x.u64();
  const auto type_c = (hipDataType)(int)x.u64();
  const int *const offsets = x.ptr<int>();
  const uint64_t groups = x.u64();
  return status(x, [&] {
    return fb.gated_f8(h, act, m, n, k, gate, up, lda, stride_a, type_a, scale_gate, scale_up, stride_scale, b, ldb, type_b, scale_b, c, ldc,
                       type_c, offsets, groups);
  });
}
// handle, k, n, x, ldx, stride_x, type_x, block_n, q, ldq, stride_q, type_q, scale, batch
PyObject *quantize_f8(PyObject *, PyObject *const *args, Py_ssize_t n_args) {
  if (!count_is(n_args, 14)) return nullptr;
  Args x{args};
  auto *const h = x.ptr<cuMpSGEMM_handle>();
  const uint64_t k = x.u64(), n = x.u64();
  void *const values = x.ptr<void>();
  const uint64_t ldx = x.u64(), stride_x = x.u64();
  const auto type_x = (hipDataType)(int)x.u64();
  const uint64_t block_n = x.u64();
  void *const q = x.ptr<void>();
  const uint64_t ldq = x.u64(), stride_q = x.u64();
  const auto type_q = (hipDataType)(int)x.u64();
  float *const scale = x.ptr<float>();
  const uint64_t batch = x.u64();
  return status(x, [&] { return fb.quantize_f8(h, k, n, values, ldx, stride_x, type_x, block_n, q, ldq, stride_q, type_q, scale, batch); });
}
// the addresses of the functions, in the order of `Functions` (`GroupedFunctions`, `GatedFunctions`)
PyObject *bind_to(void *to, PyObject *const *args, Py_ssize_t n, const Py_ssize_t want) {
  if (!count_is(n, want)) return nullptr;
  void *p[kFunctions];
  static_assert(kGroupedFunctions <= kFunctions && kGatedFunctions <= kFunctions, "room for each of the three");
  for (Py_ssize_t i = 0; i < want; i++) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (p[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "no function");
      return nullptr;
    }
  }
  memcpy(to, p, want * sizeof(void *));
  Py_RETURN_NONE;
}
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) { return bind_to(&f, args, n, kFunctions); }
PyObject *bind_grouped(PyObject *, PyObject *const *args, Py_ssize_t n) { return bind_to(&fg, args, n, kGroupedFunctions); }

PyObject *bind_gated(PyObject *, PyObject *const *args, Py_ssize_t n) { return bind_to(&fb, args, n, kGatedFunctions); }

PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
                         {"gemm", (PyCFunction)(void (*)(void))gemm, METH_FASTCALL, nullptr},
                         {"strided_batch", (PyCFunction)(void (*)(void))strided_batch, METH_FASTCALL, nullptr},
                         {"pipeline", (PyCFunction)(void (*)(void))pipeline, METH_FASTCALL, nullptr},
                         {"mx2x2", (PyCFunction)(void (*)(void))mx2x2, METH_FASTCALL, nullptr},
                         {"twoxnx2", (PyCFunction)(void (*)(void))twoxnx2, METH_FASTCALL, nullptr},
                         {"bind_grouped", (PyCFunction)(void (*)(void))bind_grouped, METH_FASTCALL, nullptr},
                         {"gemm_grouped", (PyCFunction)(void (*)(void))gemm_grouped, METH_FASTCALL, nullptr},
                         {"gemm_grouped_k", (PyCFunction)(void (*)(void))gemm_grouped_k, METH_FASTCALL, nullptr},
                         {"gemm_i8", (PyCFunction)(void (*)(void))gemm_i8, METH_FASTCALL, nullptr},
                         {"quantize_i8", (PyCFunction)(void (*)(void))quantize_i8, METH_FASTCALL, nullptr},
                         {"bind_gated", (PyCFunction)(void (*)(void))bind_gated, METH_FASTCALL, nullptr},
                         {"gemm_gated", (PyCFunction)(void (*)(void))gemm_gated, METH_FASTCALL, nullptr},
                         {"gemm_gated_backward", (PyCFunction)(void (*)(void))gemm_gated_backward, METH_FASTCALL, nullptr},
                         {"gemm_f8", (PyCFunction)(void (*)(void))gemm_f8, METH_FASTCALL, nullptr},
                         {"gemm_gated_f8", (PyCFunction)(void (*)(void))gemm_gated_f8, METH_FASTCALL, nullptr},
                         {"quantize_f8", (PyCFunction)(void (*)(void))quantize_f8, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
} // namespace

PyMODINIT_FUNC PyInit__call(void) {
  data_ptr_name = PyUnicode_InternFromString("data_ptr");
  return data_ptr_name == nullptr ? nullptr : PyModule_Create(&module);
}
