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

using ull = unsigned long long;

LmType lm_type(int code) {
  if (code < 0 || code > 2) throw std::runtime_error("bad dtype code");
  return (LmType)code;
}

PyObject* py_is_available(PyObject*, PyObject*) {
  int count = 0;
  hipError_t e = hipGetDeviceCount(&count);
  if (e != hipSuccess || count <= 0) Py_RETURN_FALSE;
  Py_RETURN_TRUE;
}

PyObject* py_mx_quantize(PyObject*, PyObject* args) {
  int dt;
  ull x, codes, scales, stream;
  long long stride, rows, k;
  if (!PyArg_ParseTuple(args, "iKLKKLLK", &dt, &x, &stride, &codes, &scales,
                        &rows, &k, &stream))
    return nullptr;
  WRAP_BEGIN
  LmType t = lm_type(dt);
  NOGIL_BEGIN
  launch_mx_quantize(t, (const void*)x, stride, (uint8_t*)codes,
                     (uint8_t*)scales, rows, k, (hipStream_t)stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_mx_dequantize(PyObject*, PyObject* args) {
  int dt;
  ull codes, scales, out, stream;
  long long rows, k;
  if (!PyArg_ParseTuple(args, "iKKKLLK", &dt, &codes, &scales, &out, &rows,
                        &k, &stream))
    return nullptr;
  WRAP_BEGIN
  LmType t = lm_type(dt);
  NOGIL_BEGIN
  launch_mx_dequantize(t, (const uint8_t*)codes, (const uint8_t*)scales,
                       (void*)out, rows, k, (hipStream_t)stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_mx_linear_workspace(PyObject*, PyObject* args) {
  long long m, n, k;
  int packed;
  if (!PyArg_ParseTuple(args, "LLLp", &m, &n, &k, &packed)) return nullptr;
  return PyLong_FromLongLong(mx_linear_workspace(m, n, k, packed));
}

PyObject* py_mx_linear(PyObject*, PyObject* args) {
  int dt;
  ull x, xc, xs, wc, ws, bias, y, work, stream;
  long long stride, m, n, k;
  if (!PyArg_ParseTuple(args, "iKLKKKKKKLLLKK", &dt, &x, &stride, &xc, &xs,
                        &wc, &ws, &bias, &y, &m, &n, &k, &work, &stream))
    return nullptr;
  WRAP_BEGIN
  LmType t = lm_type(dt);
  NOGIL_BEGIN
  launch_mx_linear(t, (const void*)x, stride, (const uint8_t*)xc,
                   (const uint8_t*)xs, (const uint8_t*)wc,
                   (const uint8_t*)ws, (const void*)bias, (void*)y, m, n, k,
                   (void*)work, (hipStream_t)stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_score_workspace(PyObject*, PyObject* args) {
  int dt, top;
  long long rows, v;
  if (!PyArg_ParseTuple(args, "iLLi", &dt, &rows, &v, &top)) return nullptr;
  WRAP_BEGIN
  return PyLong_FromLongLong(score_workspace(lm_type(dt), rows, v, top));
  WRAP_END
}

PyObject* py_token_logprobs(PyObject*, PyObject* args) {
  int dt, top;
  ull x, tokens, lp, entropy, top_lp, top_ids, stats, work, stream;
  long long stride, rows, v, ignore;
  float inv_t;
  if (!PyArg_ParseTuple(args, "iKLLLKLfiKKKKKKK", &dt, &x, &stride, &rows, &v,
                        &tokens, &ignore, &inv_t, &top, &lp, &entropy,
                        &top_lp, &top_ids, &stats, &work, &stream))
    return nullptr;
  WRAP_BEGIN
  LmType t = lm_type(dt);
  if (top < 0 || top > kMaxTop) throw std::runtime_error("bad top");
  NOGIL_BEGIN
  launch_token_logprobs(t, (const void*)x, stride, rows, v,
                        (const int64_t*)tokens, ignore, inv_t, top,
                        (float*)lp, (float*)entropy, (float*)top_lp,
                        (int64_t*)top_ids, (RowStats*)stats, (void*)work,
                        (hipStream_t)stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_token_logprobs_bwd(PyObject*, PyObject* args) {
  int dt;
  ull x, tokens, stats, g_lp, g_h, dx, stream;
  long long stride, rows, v;
  float inv_t;
  if (!PyArg_ParseTuple(args, "iKLLLKfKKKKK", &dt, &x, &stride, &rows, &v,
                        &tokens, &inv_t, &stats, &g_lp, &g_h, &dx, &stream))
    return nullptr;
  WRAP_BEGIN
  LmType t = lm_type(dt);
  NOGIL_BEGIN
  launch_token_logprobs_bwd(t, (const void*)x, stride, rows, v,
                            (const int64_t*)tokens, inv_t,
                            (const RowStats*)stats, (const float*)g_lp,
                            (const float*)g_h, (void*)dx,
                            (hipStream_t)stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_distill(PyObject*, PyObject* args) {
  int dt, tt, k, mean;
  ull x, teacher, ids, row_loss, q, stats, total, work, stream;
  long long stride, rows, v;
  float inv_t;
  if (!PyArg_ParseTuple(args, "iKLLLiKKifKKKKpKK", &dt, &x, &stride, &rows,
                        &v, &tt, &teacher, &ids, &k, &inv_t, &row_loss, &q,
                        &stats, &total, &mean, &work, &stream))
    return nullptr;
  WRAP_BEGIN
  LmType t = lm_type(dt), u = lm_type(tt);
  if (k < 1 || k > kMaxRecord) throw std::runtime_error("bad record length");
  NOGIL_BEGIN
  launch_distill(t, (const void*)x, stride, rows, v, u, (const void*)teacher,
                 (const int64_t*)ids, k, inv_t, (float*)row_loss, (float*)q,
                 (RowStats*)stats, (float*)total, mean, (void*)work,
                 (hipStream_t)stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyObject* py_distill_bwd(PyObject*, PyObject* args) {
  int dt, k;
  ull x, ids, q, stats, grad, count, dx, stream;
  long long stride, rows, v, grad_stride;
  float inv_t;
  if (!PyArg_ParseTuple(args, "iKLLLKKifKKLKKK", &dt, &x, &stride, &rows, &v,
                        &ids, &q, &k, &inv_t, &stats, &grad, &grad_stride,
                        &count, &dx, &stream))
    return nullptr;
  WRAP_BEGIN
  LmType t = lm_type(dt);
  if (k < 1 || k > kMaxRecord) throw std::runtime_error("bad record length");
  NOGIL_BEGIN
  launch_distill_bwd(t, (const void*)x, stride, rows, v, (const int64_t*)ids,
                     (const float*)q, k, inv_t, (const RowStats*)stats,
                     (const float*)grad, grad_stride, (const float*)count,
                     (void*)dx, (hipStream_t)stream);
  NOGIL_END
  Py_RETURN_NONE;
  WRAP_END
}

PyMethodDef methods[] = {
    {"is_available", py_is_available, METH_NOARGS, "GPU present?"},
    {"mx_quantize", py_mx_quantize, METH_VARARGS,
     "mx_quantize(dtype, x, stride, codes, scales, rows, k, stream)"},
    {"mx_dequantize", py_mx_dequantize, METH_VARARGS,
     "mx_dequantize(dtype, codes, scales, out, rows, k, stream)"},
    {"mx_linear_workspace", py_mx_linear_workspace, METH_VARARGS,
     "mx_linear_workspace(m, n, k, packed) -> bytes"},
    {"mx_linear", py_mx_linear, METH_VARARGS,
     "mx_linear(dtype, x, stride, xcodes, xscales, wcodes, wscales, bias, y, "
     "m, n, k, workspace, stream)"},
    {"score_workspace", py_score_workspace, METH_VARARGS,
     "score_workspace(dtype, rows, v, top) -> bytes"},
    {"token_logprobs", py_token_logprobs, METH_VARARGS,
     "token_logprobs(dtype, x, stride, rows, v, tokens, ignore, inv_t, top, "
     "logprobs, entropy, top_lp, top_ids, stats, workspace, stream)"},
    {"token_logprobs_bwd", py_token_logprobs_bwd, METH_VARARGS,
     "token_logprobs_bwd(dtype, x, stride, rows, v, tokens, inv_t, stats, "
     "g_logprobs, g_entropy, dx, stream)"},
    {"distill", py_distill, METH_VARARGS,
     "distill(dtype, x, stride, rows, v, teacher_dtype, teacher, ids, k, "
     "inv_t, row_loss, q, stats, total, mean, workspace, stream)"},
    {"distill_bwd", py_distill_bwd, METH_VARARGS,
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
