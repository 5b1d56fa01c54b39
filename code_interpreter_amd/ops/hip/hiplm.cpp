// _hiplm: the language-model slice of the gfx950 kernel library as an
// extension module of its own, next to _hipgemm and for the same reason: a
// process that uses torch must load the kernels after torch, so that they
// register with the runtime whose streams and memory it hands them.
//
// Surface: tensors that the caller (hipmx, hiplm) has checked. Results and
// scratch come from torch's allocator, on the stream that uses them: of a
// captured graph, its own. The operators with gradients are nodes of torch's
// graph. All of that stands here and not in python because the host's part
// is the longer one where there is little work (us of host time, python and
// here: quantising 16 x 4096 8.3, 5.4; a row's log probabilities 18, 8; a
// loss with its gradient 94, 54, of which torch's own engine takes 36). It
// is host code: the only file that uses torch's headers.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/csrc/utils/pybind.h>

#include "lm.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

at::ScalarType scalar_type(int64_t code) {
  return code == 0 ? at::kFloat : code == 1 ? at::kBFloat16 : at::kHalf;
}

// t's values as they stand in memory: of a view that negates, a copy
Tensor resolved(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

Tensor plain(const Tensor& t) { return resolved(t).contiguous(); }

// x as [rows, v] with neighbouring elements in a row: a view where its
// strides allow one, else a copy
struct Rows {
  Tensor x;
  int64_t rows, v, stride;

  explicit Rows(const Tensor& t) : x(resolved(t)) {
    v = t.size(-1);
    rows = t.numel() / v;
    if (t.dim() != 2) x = x.reshape({rows, v});
    if (v > 1 && x.stride(1) != 1) x = x.contiguous();
    stride = rows > 1 ? x.stride(0) : v;
  }
};

// makes x's device the current one, and gives its current stream
struct Launch {
  c10::DeviceGuard guard;
  hipStream_t stream;

  explicit Launch(const Tensor& x)
      : guard(x.device()),
        stream(c10::hip::getCurrentHIPStream(x.device().index()).stream()) {}
};

at::IntArrayRef lead(const Tensor& t) {
  return t.sizes().slice(0, t.dim() - 1);
}

std::vector<int64_t> with_last(at::IntArrayRef lead, int64_t last) {
  std::vector<int64_t> size(lead.begin(), lead.end());
  size.push_back(last);
  return size;
}

// what at::empty comes to for a GPU tensor, without its way there
Tensor empty(const Tensor& like, at::IntArrayRef size, at::ScalarType type) {
  return Tensor(
      at::detail::empty_cuda(size, type, like.device(), std::nullopt));
}

// scratch of a call
Tensor bytes(const Tensor& like, int64_t size) {
  return size ? empty(like, {size}, at::kByte) : Tensor();
}

// A fake tensor and a subclass that wraps others have sizes and a device, but
// no memory. By the storage's address: a tensor's adds its offset.
void check_memory(const Tensor& t) {
  TORCH_CHECK_TYPE(t.has_storage() && (!t.numel() || t.storage().data()),
                   "a tensor with memory of its own is wanted, which a fake "
                   "tensor or a wrapper of others does not have");
}

template <class T = float>
T* data(const Tensor& t) {
  if (!t.defined()) return nullptr;
  check_memory(t);
  return (T*)t.data_ptr();
}

// ---------------------------------------------------------------------------
// microscaled 4-bit
// ---------------------------------------------------------------------------
std::pair<Tensor, Tensor> quantize(const Tensor& x, int64_t code) {
  Rows r(x);
  const int64_t nb = mx_blocks(r.v);
  Tensor codes = empty(x, with_last(lead(x), nb * kMxBytes), at::kByte);
  Tensor scales = empty(x, with_last(lead(x), nb), at::kByte);
  if (r.rows) {
    Launch on(x);
    launch_mx_quantize((LmType)code, data<void>(r.x), r.stride,
                       data<uint8_t>(codes), data<uint8_t>(scales), r.rows,
                       r.v, on.stream);
  }
  return {codes, scales};
}

// The parts of a quantised tensor are tensors, which a program can resize,
// transpose or point elsewhere in place after they were checked.
void check_parts(const Tensor& codes, const Tensor& scales, int64_t k) {
  auto good = [](const Tensor& t) {
    return t.is_cuda() && t.scalar_type() == at::kByte && t.dim() &&
           t.is_contiguous();
  };
  const int64_t nb = mx_blocks(k);
  TORCH_CHECK_VALUE(
      good(codes) && good(scales) && codes.device() == scales.device() &&
          scales.size(-1) == nb && codes.size(-1) == nb * kMxBytes &&
          lead(codes) == lead(scales) && (uintptr_t)codes.data_ptr() % 16 == 0,
      "codes and scales do not fit each other any more");
}

Tensor dequantize(const Tensor& codes, const Tensor& scales, int64_t k,
                  int64_t code) {
  check_parts(codes, scales, k);
  Tensor out = empty(codes, with_last(lead(scales), k), scalar_type(code));
  if (out.numel()) {
    Launch on(codes);
    launch_mx_dequantize((LmType)code, data<uint8_t>(codes),
                         data<uint8_t>(scales), data<void>(out),
                         out.numel() / k, k, on.stream);
  }
  return out;
}

// x: a tensor, or the codes of one with its scales in xs
Tensor linear(const Tensor& x, const Tensor& xs, const Tensor& wc,
              const Tensor& ws, const Tensor& bias, int64_t k, int64_t code) {
  const bool packed = xs.defined();
  check_parts(wc, ws, k);
  if (packed) check_parts(x, xs, k);
  TORCH_CHECK_VALUE(wc.dim() == 2 && x.device() == wc.device(),
                    "the weight is not what it was");
  const int64_t n = ws.size(0);
  Tensor y = empty(wc, with_last(lead(x), n), scalar_type(code));
  if (!y.numel()) return y;
  const int64_t m = y.numel() / n;
  Launch on(x);
  Tensor work = bytes(wc, mx_linear_workspace(m, n, k, packed));
  const Tensor b = bias.defined() ? plain(bias) : bias;
  if (packed) {
    launch_mx_linear((LmType)code, nullptr, 0, data<uint8_t>(x),
                     data<uint8_t>(xs), data<uint8_t>(wc), data<uint8_t>(ws),
                     data<void>(b), data<void>(y), m, n, k, data<void>(work),
                     on.stream);
  } else {
    Rows r(x);
    launch_mx_linear((LmType)code, data<void>(r.x), r.stride, nullptr, nullptr,
                     data<uint8_t>(wc), data<uint8_t>(ws), data<void>(b),
                     data<void>(y), m, n, k, data<void>(work), on.stream);
  }
  return y;
}

// ---------------------------------------------------------------------------
// rows of logits
// ---------------------------------------------------------------------------
// A gradient of a gradient is not computed. Where the backward itself is
// recorded, its result is a node's that answers with an error when it is
// differentiated: by the logits or the gradients that came in, so that it
// stands on the way to either, where torch would leave out a node beside it.
Tensor once(const Tensor& dx, const Tensor& logits,
            const variable_list& grads) {
  if (!at::GradMode::is_enabled()) return dx;
  variable_list of{dx, logits};
  of.insert(of.end(), grads.begin(), grads.end());
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "this operator has no second derivative", (int64_t)of.size());
  return (*error)(std::move(of))[0];
}

// A saved tensor comes back through hooks that a program may have set, which
// can make it anything: the kernels want what was saved.
void check_saved(const Tensor& t, const Tensor& grad, at::ScalarType type,
                 bool fits) {
  TORCH_CHECK(fits && t.device() == grad.device() && t.scalar_type() == type,
              "a saved tensor came back with another size, type or device "
              "than it was saved with");
}

struct Scores {
  Tensor logprobs, entropy, stats;
};

Scores score(const Tensor& logits, const Tensor& tokens, const Tensor& top_lp,
             const Tensor& top_ids, int64_t code, double inv_t, int64_t ignore,
             bool grad) {
  const LmType t = (LmType)code;
  Rows r(logits);
  const int top = (int)top_ids.size(-1);
  Scores s = {empty(logits, lead(logits), at::kFloat),
              empty(logits, lead(logits), at::kFloat), Tensor()};
  if (grad) s.stats = empty(logits, {r.rows, 4}, at::kFloat);
  if (r.rows) {
    Launch on(logits);
    Tensor work = bytes(logits, score_workspace(t, r.rows, r.v, top));
    launch_token_logprobs(t, data<void>(r.x), r.stride, r.rows, r.v,
                          data<int64_t>(tokens), ignore, (float)inv_t, top,
                          data(s.logprobs), data(s.entropy), data(top_lp),
                          data<int64_t>(top_ids), data<RowStats>(s.stats),
                          data<void>(work), on.stream);
  }
  return s;
}

class TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& logits,
                               const Tensor& tokens, const Tensor& top_lp,
                               const Tensor& top_ids, int64_t code,
                               double inv_t, int64_t ignore) {
    Scores s = score(logits, tokens, top_lp, top_ids, code, inv_t, ignore,
                     true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, tokens, s.stats});
    ctx->saved_data["code"] = code;
    ctx->saved_data["inv_t"] = inv_t;
    return {s.logprobs, s.entropy};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(7);
    if (!grads[0].defined() && !grads[1].defined()) return result;
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &grad = grads[grads[0].defined() ? 0 : 1];
    const int64_t code = ctx->saved_data["code"].toInt();
    check_saved(logits, grad, scalar_type(code),
                logits.dim() && logits.size(-1) &&
                    lead(logits) == grad.sizes());
    check_saved(saved[1], grad, at::kLong, saved[1].sizes() == grad.sizes());
    check_saved(saved[2], grad, at::kFloat,
                saved[2].numel() == 4 * grad.numel());
    Tensor dx;
    {
      at::NoGradGuard no_grad;
      const Tensor tokens = plain(saved[1]), stats = plain(saved[2]);
      Rows r(logits);
      dx = empty(logits, logits.sizes(), logits.scalar_type());
      if (r.rows) {
        const Tensor g_lp = grads[0].defined() ? plain(grads[0]) : Tensor();
        const Tensor g_h = grads[1].defined() ? plain(grads[1]) : Tensor();
        Launch on(logits);
        launch_token_logprobs_bwd(
            (LmType)code, data<void>(r.x), r.stride, r.rows, r.v,
            data<int64_t>(tokens),
            (float)ctx->saved_data["inv_t"].toDouble(),
            data<RowStats>(stats), data(g_lp), data(g_h),
            data<void>(dx), on.stream);
      }
    }
    result[0] = once(dx, logits, grads);
    return result;
  }
};

// how: 0 none, 1 sum, 2 mean. kept: the rows' numbers, the teacher's shares,
// what the loss was divided by and the rows' losses, one behind the other
struct Loss {
  Tensor loss, kept;
};

int64_t kept_size(int64_t rows, int64_t k, bool whole) {
  return rows * (4 + k) + (whole ? 1 + rows : 0);
}

Loss distill(const Tensor& logits, const Tensor& teacher, const Tensor& ids,
             int64_t code, int64_t teacher_code, double inv_t, int64_t how) {
  const LmType t = (LmType)code;
  Rows r(logits);
  const Tensor record = plain(teacher);
  const int64_t k = ids.size(-1);
  Loss l = {empty(logits, how ? at::IntArrayRef() : lead(logits), at::kFloat),
            empty(logits, {kept_size(r.rows, k, how != 0)}, at::kFloat)};
  if (!r.rows) {
    l.loss.zero_();
    return l;
  }
  float* stats = data(l.kept);
  float* q = stats + 4 * r.rows;
  float* count = how ? q + r.rows * k : nullptr;
  Launch on(logits);
  Tensor work = bytes(logits, score_workspace(t, r.rows, r.v, 0));
  launch_distill(t, data<void>(r.x), r.stride, r.rows, r.v,
                 (LmType)teacher_code, data<void>(record), data<int64_t>(ids),
                 (int)k, (float)inv_t, how ? count + 1 : data(l.loss), q,
                 (RowStats*)stats, how ? data(l.loss) : nullptr, count,
                 how == 2, data<void>(work), on.stream);
  return l;
}

class Distill : public torch::autograd::Function<Distill> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& logits,
                               const Tensor& teacher, const Tensor& ids,
                               int64_t code, int64_t teacher_code,
                               double inv_t, int64_t how) {
    Loss l = distill(logits, teacher, ids, code, teacher_code, inv_t, how);
    ctx->save_for_backward({logits, ids, l.kept});
    ctx->saved_data["code"] = code;
    ctx->saved_data["inv_t"] = inv_t;
    ctx->saved_data["whole"] = how != 0;
    return {l.loss};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(7);
    const auto saved = ctx->get_saved_variables();
    const Tensor& logits = saved[0];
    const int64_t code = ctx->saved_data["code"].toInt();
    const bool whole = ctx->saved_data["whole"].toBool();
    check_saved(logits, grads[0], scalar_type(code),
                logits.dim() && logits.size(-1) &&
                    (whole || lead(logits) == grads[0].sizes()));
    check_saved(saved[1], grads[0], at::kLong,
                saved[1].dim() == logits.dim() &&
                    lead(saved[1]) == lead(logits));
    const int64_t rows = logits.numel() / logits.size(-1);
    const int64_t k = saved[1].size(-1);
    check_saved(saved[2], grads[0], at::kFloat,
                k >= 1 && k <= kMaxRecord &&
                    saved[2].numel() == kept_size(rows, k, whole));
    Tensor dx;
    {
      at::NoGradGuard no_grad;
      const Tensor ids = plain(saved[1]), kept = plain(saved[2]);
      Rows r(logits);
      dx = empty(logits, logits.sizes(), logits.scalar_type());
      if (r.rows) {
        const Tensor grad = plain(grads[0]);
        const float* stats = data(kept);
        const float* q = stats + 4 * r.rows;
        Launch on(logits);
        launch_distill_bwd((LmType)code, data<void>(r.x), r.stride, r.rows,
                           r.v, data<int64_t>(ids), q, (int)k,
                           (float)ctx->saved_data["inv_t"].toDouble(),
                           (const RowStats*)stats, data(grad), whole ? 0 : 1,
                           whole ? q + r.rows * k : nullptr, data<void>(dx),
                           on.stream);
      }
    }
    result[0] = once(dx, logits, grads);
    return result;
  }
};

// ---------------------------------------------------------------------------
// the module
// ---------------------------------------------------------------------------
// The arguments of a call, in their order.
class Args {
 public:
  Args(PyObject* const* args, Py_ssize_t n, Py_ssize_t want) : args_(args) {
    TORCH_CHECK_TYPE(n == want, want, " arguments wanted, got ", n);
  }
  const Tensor& tensor() {
    TORCH_CHECK_TYPE(THPVariable_Check(*args_), "a tensor is wanted");
    const Tensor& t = THPVariable_Unpack(*args_++);
    check_memory(t);
    return t;
  }
  Tensor tensor_or_none() {
    if (*args_ != Py_None) return tensor();
    args_++;
    return Tensor();
  }
  int64_t integer(int64_t low = INT64_MIN, int64_t high = INT64_MAX) {
    const long long v = PyLong_AsLongLong(*args_++);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    TORCH_CHECK(v >= low && v <= high, "an argument is out of its range");
    return v;
  }
  int64_t type() { return integer(0, 2); }
  double real() {
    const double v = PyFloat_AsDouble(*args_++);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }

 private:
  PyObject* const* args_;
};

PyObject* tuple(std::initializer_list<Tensor> tensors) {
  THPObjectPtr out(PyTuple_New((Py_ssize_t)tensors.size()));
  if (!out) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) throw python_error();
    PyTuple_SET_ITEM(out.get(), i++, o);
  }
  return out.release();
}

bool has_tangent(const Tensor& t) {
  return t.defined() && t._fw_grad(0).defined();
}

// also with a forward-mode tangent, which torch then refuses
bool needs_grad(const Tensor& t) {
  return (at::GradMode::is_enabled() && t.requires_grad()) || has_tangent(t);
}

PyObject* py_mx_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(args, n, 2);
  const Tensor& x = a.tensor();
  const int64_t code = a.type();
  std::pair<Tensor, Tensor> q;
  {
    pybind11::gil_scoped_release no_gil;
    at::NoGradGuard no_grad;
    q = quantize(x, code);
  }
  return tuple({q.first, q.second});
  END_HANDLE_TH_ERRORS
}

PyObject* py_mx_dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(args, n, 4);
  const Tensor &codes = a.tensor(), &scales = a.tensor();
  const int64_t k = a.integer(1), code = a.type();
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    out = dequantize(codes, scales, k, code);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyObject* py_mx_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(args, n, 7);
  const Tensor& x = a.tensor();
  const Tensor xs = a.tensor_or_none();
  const Tensor &wc = a.tensor(), &ws = a.tensor();
  const Tensor bias = a.tensor_or_none();
  const int64_t k = a.integer(1), code = a.type();
  TORCH_CHECK(!has_tangent(x) && !has_tangent(bias),
              "hipmx.linear has no forward-mode derivative");
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    at::NoGradGuard no_grad;
    y = linear(x, xs, wc, ws, bias, k, code);
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* py_token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(args, n, 6);
  const Tensor &logits = a.tensor(), &ids = a.tensor();
  const int64_t code = a.type(), top = a.integer(0, kMaxTop);
  const double inv_t = a.real();
  const int64_t ignore = a.integer();
  Tensor logprobs, entropy, top_lp, top_ids;
  {
    pybind11::gil_scoped_release no_gil;
    const Tensor tokens = ids.contiguous();
    const auto size = with_last(lead(logits), top);
    top_lp = empty(logits, size, at::kFloat);
    top_ids = empty(logits, size, at::kLong);
    if (needs_grad(logits)) {
      auto out = TokenLogprobs::apply(logits, tokens, top_lp, top_ids, code,
                                      inv_t, ignore);
      logprobs = out[0];
      entropy = out[1];
    } else {
      at::NoGradGuard no_grad;
      Scores s = score(logits, tokens, top_lp, top_ids, code, inv_t, ignore,
                       false);
      logprobs = s.logprobs;
      entropy = s.entropy;
    }
  }
  return tuple({logprobs, entropy, top_lp, top_ids});
  END_HANDLE_TH_ERRORS
}

PyObject* py_distill(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a(args, n, 7);
  const Tensor &logits = a.tensor(), &teacher = a.tensor();
  const Tensor& teacher_ids = a.tensor();
  const int64_t code = a.type(), teacher_code = a.type();
  const double inv_t = a.real();
  const int64_t how = a.integer(0, 2);
  TORCH_CHECK(teacher_ids.size(-1) >= 1 && teacher_ids.size(-1) <= kMaxRecord,
              "bad record length");
  Tensor loss;
  {
    pybind11::gil_scoped_release no_gil;
    const Tensor ids = teacher_ids.contiguous();
    if (needs_grad(logits)) {
      loss = Distill::apply(logits, teacher, ids, code, teacher_code, inv_t,
                            how)[0];
    } else {
      at::NoGradGuard no_grad;
      loss = distill(logits, teacher, ids, code, teacher_code, inv_t, how)
                 .loss;
    }
  }
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL

// a dtype is 0 float32, 1 bfloat16, 2 float16
PyMethodDef methods[] = {
    {"mx_quantize", FAST(py_mx_quantize),
     "mx_quantize(x, dtype) -> (codes, scales)"},
    {"mx_dequantize", FAST(py_mx_dequantize),
     "mx_dequantize(codes, scales, k, dtype) -> values"},
    {"mx_linear", FAST(py_mx_linear),
     "mx_linear(x or its codes, its scales or None, weight codes, weight "
     "scales, bias or None, k, dtype) -> y"},
    {"token_logprobs", FAST(py_token_logprobs),
     "token_logprobs(logits, tokens, dtype, top, inv_t, ignore) -> (logprobs, "
     "entropy, top_logprobs, top_tokens)"},
    {"distill", FAST(py_distill),
     "distill(logits, teacher, ids, dtype, teacher dtype, inv_t, reduction) "
     "-> loss; reduction: 0 none, 1 sum, 2 mean"},
    {nullptr, nullptr, 0, nullptr},
};

struct PyModuleDef module_def = {
    PyModuleDef_HEAD_INIT, "_hiplm",
    "gfx950 language-model kernels for torch tensors", -1, methods,
};

}  // namespace

PyMODINIT_FUNC PyInit__hiplm(void) { return PyModule_Create(&module_def); }
