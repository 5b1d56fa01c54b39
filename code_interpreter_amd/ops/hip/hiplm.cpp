// _hiplm: the language-model slice of the gfx950 kernel library as an
// extension module of its own, next to _hipgemm and for the same reason: a
// process that uses torch must load the kernels after torch, so that they
// register with the runtime whose streams and memory it hands them.
//
// Surface: stateless raw-pointer entry points only -- the caller (torch)
// owns memory and streams, and has checked shapes and types.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <string>

#include "lm.h"

namespace {

#define NOGIL_BEGIN           \
  std::string _nogil_err;     \
  Py_BEGIN_ALLOW_THREADS;     \
  try {
#define NOGIL_END                                               \
  }                                                             \
  catch (const std::exception& _e) { _nogil_err = _e.what(); }  \
  Py_END_ALLOW_THREADS;                                         \
  if (!_nogil_err.empty()) throw std::runtime_error(_nogil_err);

#define WRAP_BEGIN try {
#define WRAP_END                                   \
  }                                                \
  catch (const std::exception& e) {                \
    PyErr_SetString(PyExc_RuntimeError, e.what()); \
    return nullptr;                                \
  }

// The arguments of a call in their order; the first that is not what is asked
// for leaves an exception.
class Args {
 public:
  Args(PyObject* const* args, Py_ssize_t n, Py_ssize_t want)
      : args_(args), good_(n == want) {
    if (!good_)
      PyErr_Format(PyExc_TypeError, "%zd arguments wanted, got %zd", want, n);
  }
  int64_t integer() {
    if (!good_) return 0;
    const long long v = PyLong_AsLongLong(*args_++);
    good_ = !(v == -1 && PyErr_Occurred());
    return v;
  }
  template <class P = void>
  P* pointer() {
    if (!good_) return nullptr;
    const unsigned long long v = PyLong_AsUnsignedLongLong(*args_++);
    good_ = !(v == ~0ull && PyErr_Occurred());
    return (P*)v;
  }
  float real() {
    if (!good_) return 0;
    const double v = PyFloat_AsDouble(*args_++);
    good_ = !(v == -1 && PyErr_Occurred());
    return (float)v;
  }
  LmType type() {
    const int64_t v = integer();
    if (good_ && (v < 0 || v > 2)) {
      PyErr_SetString(PyExc_RuntimeError, "bad dtype code");
      good_ = false;
    }
    return (LmType)v;
  }
  int within(int64_t low, int64_t high, const char* what) {
    const int64_t v = integer();
    if (good_ && (v < low || v > high)) {
      PyErr_SetString(PyExc_RuntimeError, what);
      good_ = false;
    }
    return (int)v;
  }
  bool good() const { return good_; }

 private:
  PyObject* const* args_;
  bool good_;
};

PyObject* py_is_available(PyObject*, PyObject*) {
  int count = 0;
  hipError_t e = hipGetDeviceCount(&count);
  if (e != hipSuccess || count <= 0) Py_RETURN_FALSE;
  Py_RETURN_TRUE;
}

PyObject* py_mx_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Args a(args, n, 8);
  const LmType t = a.type();
  const void* x = a.pointer();
  const int64_t stride = a.integer();
  auto* codes = a.pointer<uint8_t>();
  auto* scales = a.pointer<uint8_t>();
  const int64_t rows = a.integer(), k = a.integer();
  auto stream = (hipStream_t)a.pointer();
  if (!a.good()) return nullptr;
  WRAP_BEGIN
  NOGIL_BEGIN
  launch_mx_quantize(t, x, stride, codes, scales, rows, k, stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_mx_dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Args a(args, n, 7);
  const LmType t = a.type();
  auto* codes = a.pointer<uint8_t>();
  auto* scales = a.pointer<uint8_t>();
  void* out = a.pointer();
  const int64_t rows = a.integer(), k = a.integer();
  auto stream = (hipStream_t)a.pointer();
  if (!a.good()) return nullptr;
  WRAP_BEGIN
  NOGIL_BEGIN
  launch_mx_dequantize(t, codes, scales, out, rows, k, stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_mx_linear_workspace(PyObject*, PyObject* const* args,
                                 Py_ssize_t n) {
  Args a(args, n, 4);
  const int64_t m = a.integer(), cols = a.integer(), k = a.integer();
  const bool packed = a.integer() != 0;
  if (!a.good()) return nullptr;
  return PyLong_FromLongLong(mx_linear_workspace(m, cols, k, packed));
}

PyObject* py_mx_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Args a(args, n, 14);
  const LmType t = a.type();
  const void* x = a.pointer();
  const int64_t stride = a.integer();
  auto* xc = a.pointer<uint8_t>();
  auto* xs = a.pointer<uint8_t>();
  auto* wc = a.pointer<uint8_t>();
  auto* ws = a.pointer<uint8_t>();
  const void* bias = a.pointer();
  void* y = a.pointer();
  const int64_t m = a.integer(), cols = a.integer(), k = a.integer();
  void* work = a.pointer();
  auto stream = (hipStream_t)a.pointer();
  if (!a.good()) return nullptr;
  WRAP_BEGIN
  NOGIL_BEGIN
  launch_mx_linear(t, x, stride, xc, xs, wc, ws, bias, y, m, cols, k, work,
                   stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_score_workspace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Args a(args, n, 4);
  const LmType t = a.type();
  const int64_t rows = a.integer(), v = a.integer();
  const int top = a.within(0, kMaxTop, "bad top");
  if (!a.good()) return nullptr;
  return PyLong_FromLongLong(score_workspace(t, rows, v, top));
}

PyObject* py_token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Args a(args, n, 16);
  const LmType t = a.type();
  const void* x = a.pointer();
  const int64_t stride = a.integer(), rows = a.integer(), v = a.integer();
  auto* tokens = a.pointer<int64_t>();
  const int64_t ignore = a.integer();
  const float inv_t = a.real();
  const int top = a.within(0, kMaxTop, "bad top");
  auto* logprobs = a.pointer<float>();
  auto* entropy = a.pointer<float>();
  auto* top_lp = a.pointer<float>();
  auto* top_ids = a.pointer<int64_t>();
  auto* stats = a.pointer<RowStats>();
  void* work = a.pointer();
  auto stream = (hipStream_t)a.pointer();
  if (!a.good()) return nullptr;
  WRAP_BEGIN
  NOGIL_BEGIN
  launch_token_logprobs(t, x, stride, rows, v, tokens, ignore, inv_t, top,
                        logprobs, entropy, top_lp, top_ids, stats, work,
                        stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_token_logprobs_bwd(PyObject*, PyObject* const* args,
                                Py_ssize_t n) {
  Args a(args, n, 12);
  const LmType t = a.type();
  const void* x = a.pointer();
  const int64_t stride = a.integer(), rows = a.integer(), v = a.integer();
  auto* tokens = a.pointer<int64_t>();
  const float inv_t = a.real();
  auto* stats = a.pointer<RowStats>();
  auto* g_lp = a.pointer<float>();
  auto* g_h = a.pointer<float>();
  void* dx = a.pointer();
  auto stream = (hipStream_t)a.pointer();
  if (!a.good()) return nullptr;
  WRAP_BEGIN
  NOGIL_BEGIN
  launch_token_logprobs_bwd(t, x, stride, rows, v, tokens, inv_t, stats, g_lp,
                            g_h, dx, stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_distill(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Args a(args, n, 18);
  const LmType t = a.type();
  const void* x = a.pointer();
  const int64_t stride = a.integer(), rows = a.integer(), v = a.integer();
  const LmType tt = a.type();
  const void* teacher = a.pointer();
  auto* ids = a.pointer<int64_t>();
  const int k = a.within(1, kMaxRecord, "bad record length");
  const float inv_t = a.real();
  auto* row_loss = a.pointer<float>();
  auto* q = a.pointer<float>();
  auto* stats = a.pointer<RowStats>();
  auto* total = a.pointer<float>();
  auto* count = a.pointer<float>();
  const bool mean = a.integer() != 0;
  void* work = a.pointer();
  auto stream = (hipStream_t)a.pointer();
  if (!a.good()) return nullptr;
  WRAP_BEGIN
  NOGIL_BEGIN
  launch_distill(t, x, stride, rows, v, tt, teacher, ids, k, inv_t, row_loss,
                 q, stats, total, count, mean, work, stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_distill_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Args a(args, n, 15);
  const LmType t = a.type();
  const void* x = a.pointer();
  const int64_t stride = a.integer(), rows = a.integer(), v = a.integer();
  auto* ids = a.pointer<int64_t>();
  auto* q = a.pointer<float>();
  const int k = a.within(1, kMaxRecord, "bad record length");
  const float inv_t = a.real();
  auto* stats = a.pointer<RowStats>();
  auto* grad = a.pointer<float>();
  const int64_t grad_stride = a.integer();
  auto* count = a.pointer<float>();
  void* dx = a.pointer();
  auto stream = (hipStream_t)a.pointer();
  if (!a.good()) return nullptr;
  WRAP_BEGIN
  NOGIL_BEGIN
  launch_distill_bwd(t, x, stride, rows, v, ids, q, k, inv_t, stats, grad,
                     grad_stride, count, dx, stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL

PyMethodDef methods[] = {
    {"is_available", py_is_available, METH_NOARGS, "GPU present?"},
    {"mx_quantize", FAST(py_mx_quantize),
     "mx_quantize(dtype, x, stride, codes, scales, rows, k, stream)"},
    {"mx_dequantize", FAST(py_mx_dequantize),
     "mx_dequantize(dtype, codes, scales, out, rows, k, stream)"},
    {"mx_linear_workspace", FAST(py_mx_linear_workspace),
     "mx_linear_workspace(m, n, k, packed) -> bytes"},
    {"mx_linear", FAST(py_mx_linear),
     "mx_linear(dtype, x, stride, xcodes, xscales, wcodes, wscales, bias, y, "
     "m, n, k, workspace, stream)"},
    {"score_workspace", FAST(py_score_workspace),
     "score_workspace(dtype, rows, v, top) -> bytes"},
    {"token_logprobs", FAST(py_token_logprobs),
     "token_logprobs(dtype, x, stride, rows, v, tokens, ignore, inv_t, top, "
     "logprobs, entropy, top_lp, top_ids, stats, workspace, stream)"},
    {"token_logprobs_bwd", FAST(py_token_logprobs_bwd),
     "token_logprobs_bwd(dtype, x, stride, rows, v, tokens, inv_t, stats, "
     "g_logprobs, g_entropy, dx, stream)"},
    {"distill", FAST(py_distill),
     "distill(dtype, x, stride, rows, v, teacher_dtype, teacher, ids, k, "
     "inv_t, row_loss, q, stats, total, count, mean, workspace, stream)"},
    {"distill_bwd", FAST(py_distill_bwd),
     "distill_bwd(dtype, x, stride, rows, v, ids, q, k, inv_t, stats, grad, "
     "grad_stride, count, dx, stream)"},
    {nullptr, nullptr, 0, nullptr},
};

struct PyModuleDef module_def = {
    PyModuleDef_HEAD_INIT, "_hiplm",
    "gfx950 language-model kernels (raw pointers, caller's stream)",
    -1, methods,
};

}  // namespace

PyMODINIT_FUNC PyInit__hiplm(void) { return PyModule_Create(&module_def); }
