// The operators on rows of logits and at the two ends of a token table, called with tensors: what Python does for a call (checks, new tensors, the stream) in one step. A call
// through Python's checks and ctypes takes 12 to 15 us of host time, four fifths of it beside the launch; a step between a model and its next
// token calls these on a few rows, whose kernels take 3 to 9 us.
//
// A face takes the plain call: exact tensors on the current device with the types, shapes and strides that the operator asks for. Anything
// else gives None, and the caller's own checks say what is wrong (or take what is merely unusual, a subclass of a tensor say).
#include <Python.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>

namespace {

using AdjustEntry = int (*)(int, const void*, long long, void*, long long, int, int, const int32_t*, long long, int, int, const int32_t*, const int32_t*,
                            const int32_t*, const float*, const float*, const float*, const int32_t*, const int32_t*, const float*, int, const uint32_t*,
                            long long, int, const int32_t*, cudaStream_t);
using TopEntry = int (*)(int, const void*, long long, int, int, int, float, float*, int32_t*, float*, int*, cudaStream_t);
using DistillEntry = int (*)(int, const void*, long long, int, int, const int32_t*, const float*, int, const float*, const float*, float, float*, void*,
                             long long, int*, cudaStream_t);
using LossEntry = int (*)(int, const void*, long long, const void*, long long, int, int, int, const int32_t*, const float*, float, int, float*, float*, void*, int*, cudaStream_t);
using LossGradientEntry = int (*)(int, const void*, long long, const void*, long long, int, int, int, const int32_t*, const float*, const float*, float, void*, long long, void*,
                                  long long, void*, int*, cudaStream_t);
using LossSpace = long long (*)(int, const void*, long long, int, int, int, int, int);
using RowsEntry = int (*)(int, int, const int32_t*, const void*, long long, void*, long long, int, int, int, float, cudaStream_t);
using RowsGradientEntry = int (*)(int, int, const int32_t*, const void*, long long, void*, long long, int, int, int, float, int, void*, cudaStream_t);
using RowsSpace = long long (*)(int, int, int);
AdjustEntry adjust_entry = nullptr;
TopEntry top_entry = nullptr;
DistillEntry distill_entry = nullptr;
LossEntry loss_entry = nullptr;
LossGradientEntry loss_gradient_entry = nullptr;
LossSpace loss_space = nullptr;
RowsEntry rows_entry = nullptr;
RowsGradientEntry rows_gradient_entry = nullptr;
RowsSpace rows_space = nullptr;

constexpr int64_t MOST = 0x7fffffff, TOP_MOST = 256, TABLE_MOST = 1 << 30;

// An argument as a tensor: nullptr for None. False: not plain.
bool tensor_of(PyObject* o, const at::Tensor*& t) {
  t = nullptr;
  if (o == Py_None) return true;
  if (!THPVariable_CheckExact(o)) return false;
  t = &THPVariable_Unpack(o);
  return t->is_cuda() && t->layout() == at::kStrided;
}

struct Rows {
  const at::Tensor* t;
  int code;
  int64_t rows, vocab, ld, size;
  int device;

  bool of(PyObject* o) {
    if (!tensor_of(o, t) || t == nullptr || t->dim() != 2) return false;
    if (t->scalar_type() == at::kFloat) code = 0, size = 4;
    else if (t->scalar_type() == at::kBFloat16) code = 1, size = 2;
    else return false;
    rows = t->size(0), vocab = t->size(1), ld = t->stride(0), device = t->get_device();
    if (rows < 1 || vocab < 1 || rows > MOST || vocab > MOST || (vocab > 1 && t->stride(1) != 1) || (rows > 1 && ld < vocab)) return false;
    if (rows == 1) ld = std::max(ld, vocab);
    return device == c10::cuda::current_device();
  }
  at::TensorOptions like(at::ScalarType type) const { return at::TensorOptions().dtype(type).device(t->device()); }
};

// A number for each row. False: not plain; an address of nullptr for None.
template <typename N>
bool numbers(PyObject* o, const Rows& x, int64_t count, const N*& at) {
  const at::Tensor* t;
  at = nullptr;
  if (!tensor_of(o, t)) return false;
  if (t == nullptr) return true;
  if (t->scalar_type() != (std::is_same<N, float>::value ? at::kFloat : at::kInt) || t->get_device() != x.device || t->dim() != 1 ||
      t->numel() < count || !t->is_contiguous())
    return false;
  at = static_cast<const N*>(t->data_ptr());
  return true;
}

// A table of int32 whose rows are contiguous.
struct Table {
  const void* at = nullptr;
  int64_t rows = 0, columns = 0, ld = 0;
  bool of(PyObject* o, const Rows& x) {
    const at::Tensor* t;
    if (!tensor_of(o, t)) return false;
    if (t == nullptr) return true;
    if (t->scalar_type() != at::kInt || t->dim() != 2 || t->get_device() != x.device) return false;
    rows = t->size(0), columns = t->size(1), ld = t->stride(0);
    if ((columns > 1 && t->stride(1) != 1) || rows > MOST || columns > MOST || rows < 1) return false;
    at = t->data_ptr();
    return true;
  }
};

// The output beside the logits: `o`, or new rows as far apart and at the same place of 16 bytes.
bool output(PyObject* o, const Rows& x, at::Tensor& out, int64_t& out_ld) {
  const at::Tensor* given;
  if (!tensor_of(o, given)) return false;
  const uintptr_t from = reinterpret_cast<uintptr_t>(x.t->data_ptr());
  if (given == nullptr) {
    out_ld = x.ld > x.vocab + std::max<int64_t>(64, x.vocab / 16) ? x.vocab : x.ld;
    const int64_t skip = int64_t(from % 16) / x.size;
    out = skip == 0 ? at::empty_strided({x.rows, x.vocab}, {out_ld, 1}, x.like(x.t->scalar_type()))
                    : at::empty({(x.rows - 1) * out_ld + x.vocab + skip}, x.like(x.t->scalar_type())).as_strided({x.rows, x.vocab}, {out_ld, 1}, skip);
    return true;
  }
  if (given->scalar_type() != x.t->scalar_type() || given->dim() != 2 || given->size(0) != x.rows || given->size(1) != x.vocab ||
      given->get_device() != x.device || (x.vocab > 1 && given->stride(1) != 1) || (x.rows > 1 && given->stride(0) < x.vocab))
    return false;
  out_ld = x.rows > 1 ? given->stride(0) : std::max(given->stride(0), x.vocab);
  const uintptr_t to = reinterpret_cast<uintptr_t>(given->data_ptr());
  if (!(to == from && (x.rows == 1 || out_ld == x.ld)) && to < from + uintptr_t(((x.rows - 1) * x.ld + x.vocab) * x.size) &&
      from < to + uintptr_t(((x.rows - 1) * out_ld + x.vocab) * x.size))
    return false;   // (overlaps without being the same rows)
  out = *given;
  return true;
}

bool temperature_of(PyObject* o, float& tau) {
  if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  tau = float(v);
  return v >= 1e-6 && std::isfinite(v) && std::isfinite(tau);
}

// (status, tensors ...), or an error
template <typename... Tensors>
PyObject* answer(int status, const Tensors&... tensors) {
  constexpr Py_ssize_t n = 1 + sizeof...(tensors);
  PyObject* all[n] = {PyLong_FromLong(status), (tensors.defined() ? THPVariable_Wrap(tensors) : Py_NewRef(Py_None))...};
  PyObject* tuple = PyTuple_New(n);
  bool good = tuple != nullptr;
  for (PyObject* o : all) good = good && o != nullptr;
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (good) PyTuple_SET_ITEM(tuple, i, all[i]);
    else Py_XDECREF(all[i]);
  }
  if (good) return tuple;
  Py_XDECREF(tuple);
  return nullptr;
}

// (logits, history, slots, lengths, prompt_lengths, repetition, presence, frequency, bias_start, bias_ids, bias_values, mask, mask_rows, out)
PyObject* adjust(PyObject*, PyObject* const* arg, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Rows x;
  if (n_args != 14 || adjust_entry == nullptr || !x.of(arg[0])) Py_RETURN_NONE;
  Table history, mask;
  const int32_t *slots, *lengths, *prompt_lengths, *bias_start, *bias_ids, *mask_rows;
  const float *repetition, *presence, *frequency, *bias_values;
  if (!history.of(arg[1], x) || !mask.of(arg[11], x) || !numbers(arg[2], x, x.rows, slots) || !numbers(arg[3], x, x.rows, lengths) ||
      !numbers(arg[4], x, x.rows, prompt_lengths) || !numbers(arg[5], x, x.rows, repetition) || !numbers(arg[6], x, x.rows, presence) ||
      !numbers(arg[7], x, x.rows, frequency) || !numbers(arg[8], x, x.rows + 1, bias_start) || !numbers(arg[9], x, 0, bias_ids) ||
      !numbers(arg[10], x, 0, bias_values) || !numbers(arg[12], x, x.rows, mask_rows))
    Py_RETURN_NONE;
  if (history.at == nullptr ? repetition != nullptr || presence != nullptr || frequency != nullptr
                            : lengths == nullptr || (slots == nullptr && history.rows < x.rows))
    Py_RETURN_NONE;
  if (mask.at != nullptr && (mask.columns * 32 < x.vocab || (mask_rows == nullptr && mask.rows < x.rows))) Py_RETURN_NONE;
  int64_t n_biases = 0;
  if (arg[8] != Py_None) {
    if (arg[9] == Py_None || arg[10] == Py_None) Py_RETURN_NONE;
    n_biases = THPVariable_Unpack(arg[9]).numel();
    if (n_biases > MOST || THPVariable_Unpack(arg[10]).numel() < n_biases) Py_RETURN_NONE;
    if (n_biases == 0) bias_start = nullptr;
  } else if (arg[9] != Py_None || arg[10] != Py_None) {
    Py_RETURN_NONE;
  }
  at::Tensor out;
  int64_t out_ld;
  if (!output(arg[13], x, out, out_ld)) Py_RETURN_NONE;
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = adjust_entry(x.code, x.t->data_ptr(), x.ld, out.data_ptr(), out_ld, int(x.rows), int(x.vocab), static_cast<const int32_t*>(history.at),
                        history.ld, int(history.rows), int(history.columns), slots, lengths, prompt_lengths, repetition, presence, frequency,
                        bias_start, bias_ids, bias_values, int(n_biases), static_cast<const uint32_t*>(mask.at), mask.ld, int(mask.rows), mask_rows,
                        stream);
  Py_END_ALLOW_THREADS
  return answer(status, out);
  END_HANDLE_TH_ERRORS
}

// (logits, k, temperature, error word's address)
PyObject* top(PyObject*, PyObject* const* arg, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Rows x;
  float tau;
  if (n_args != 4 || top_entry == nullptr || !x.of(arg[0]) || !PyLong_CheckExact(arg[1]) || !temperature_of(arg[2], tau)) Py_RETURN_NONE;
  int over = 0;
  const long long k = PyLong_AsLongLongAndOverflow(arg[1], &over);
  if (over != 0 || k < 1 || k > std::min(x.vocab, TOP_MOST)) Py_RETURN_NONE;
  int* error = static_cast<int*>(PyLong_AsVoidPtr(arg[3]));
  at::Tensor values = at::empty_strided({x.rows, k}, {k, 1}, x.like(at::kFloat)), ids = at::empty_strided({x.rows, k}, {k, 1}, x.like(at::kInt)),
             log_sum = at::empty_strided({x.rows}, {1}, x.like(at::kFloat));
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = top_entry(x.code, x.t->data_ptr(), x.ld, int(x.rows), int(x.vocab), int(k), tau, static_cast<float*>(values.data_ptr()),
                     static_cast<int32_t*>(ids.data_ptr()), static_cast<float*>(log_sum.data_ptr()), error, stream);
  Py_END_ALLOW_THREADS
  return answer(status, values, ids, log_sum);
  END_HANDLE_TH_ERRORS
}

// (logits, ids, teacher, log_sum, temperature, weight, gradient, out, error word's address)
PyObject* distill(PyObject*, PyObject* const* arg, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Rows x;
  float tau;
  const at::Tensor *ids, *teacher;
  const float *log_sum, *weight;
  if (n_args != 9 || distill_entry == nullptr || !x.of(arg[0]) || !temperature_of(arg[4], tau) || !PyBool_Check(arg[6]) || !tensor_of(arg[1], ids) ||
      !tensor_of(arg[2], teacher) || ids == nullptr || teacher == nullptr || !numbers(arg[3], x, x.rows, log_sum) ||
      !numbers(arg[5], x, x.rows, weight))
    Py_RETURN_NONE;
  if (ids->scalar_type() != at::kInt || teacher->scalar_type() != at::kFloat || ids->dim() != 2 || ids->sizes() != teacher->sizes() ||
      ids->size(0) != x.rows || ids->size(1) < 1 || ids->size(1) > TOP_MOST || !ids->is_contiguous() || !teacher->is_contiguous() ||
      ids->get_device() != x.device || teacher->get_device() != x.device)
    Py_RETURN_NONE;
  const bool gradient = arg[6] == Py_True;
  if (!gradient && arg[7] != Py_None) Py_RETURN_NONE;
  int* error = static_cast<int*>(PyLong_AsVoidPtr(arg[8]));
  at::Tensor grad;
  int64_t grad_ld = 0;
  if (gradient && !output(arg[7], x, grad, grad_ld)) Py_RETURN_NONE;
  at::Tensor loss = at::empty_strided({x.rows}, {1}, x.like(at::kFloat));
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = distill_entry(x.code, x.t->data_ptr(), x.ld, int(x.rows), int(x.vocab), static_cast<const int32_t*>(ids->data_ptr()),
                         static_cast<const float*>(teacher->data_ptr()), int(ids->size(1)), log_sum, weight, tau, static_cast<float*>(loss.data_ptr()),
                         gradient ? grad.data_ptr() : nullptr, grad_ld, error, stream);
  Py_END_ALLOW_THREADS
  return answer(status, loss, grad);
  END_HANDLE_TH_ERRORS
}

// A factor or a limit.
bool number_of(PyObject* o, double& v) {
  if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
  v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return std::isfinite(v) && std::isfinite(float(v));
}

// Hidden rows, their table, tokens, weights and the limit of the logits.
struct Loss {
  Rows x, w;
  const int32_t* targets;
  const float* weight;
  double softcap;

  bool of(PyObject* hidden, PyObject* table, PyObject* tokens, PyObject* weights, PyObject* cap) {
    return x.of(hidden) && w.of(table) && w.code == x.code && w.vocab == x.vocab && w.device == x.device && x.rows <= TABLE_MOST && x.vocab <= TABLE_MOST &&
           w.rows <= TABLE_MOST && tokens != Py_None && numbers(tokens, x, x.rows, targets) && numbers(weights, x, x.rows, weight) && number_of(cap, softcap) &&
           (softcap == 0.0 || (softcap >= 1e-6 && softcap <= 1e30));
  }
  at::Tensor space(bool gradient, bool d_hidden) const {
    return at::empty_strided({loss_space(x.code, w.t->data_ptr(), w.ld, int(x.rows), int(x.vocab), int(w.rows), gradient, d_hidden)}, {1}, x.like(at::kByte));
  }
};

// (hidden, table, targets, weight, softcap, error word's address)
PyObject* token_loss(PyObject*, PyObject* const* arg, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Loss l;
  if (n_args != 6 || loss_entry == nullptr || loss_space == nullptr || !l.of(arg[0], arg[1], arg[2], arg[3], arg[4])) Py_RETURN_NONE;
  int* error = static_cast<int*>(PyLong_AsVoidPtr(arg[5]));
  at::Tensor loss = at::empty_strided({l.x.rows}, {1}, l.x.like(at::kFloat)), log_sum = at::empty_strided({l.x.rows}, {1}, l.x.like(at::kFloat)), space = l.space(false, false);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(l.x.device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = loss_entry(l.x.code, l.x.t->data_ptr(), l.x.ld, l.w.t->data_ptr(), l.w.ld, int(l.x.rows), int(l.x.vocab), int(l.w.rows), l.targets, l.weight, float(l.softcap), 0,
                      static_cast<float*>(loss.data_ptr()), static_cast<float*>(log_sum.data_ptr()), space.data_ptr(), error, stream);
  Py_END_ALLOW_THREADS
  return answer(status, loss, log_sum);
  END_HANDLE_TH_ERRORS
}

// (hidden, table, targets, log_sum, weight, softcap, hidden_gradient, table_gradient, error word's address)
PyObject* token_loss_gradient(PyObject*, PyObject* const* arg, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Loss l;
  const float* log_sum;
  if (n_args != 9 || loss_gradient_entry == nullptr || loss_space == nullptr || !l.of(arg[0], arg[1], arg[2], arg[4], arg[5]) || arg[3] == Py_None ||
      !numbers(arg[3], l.x, l.x.rows, log_sum) || !PyBool_Check(arg[6]) || !PyBool_Check(arg[7]) || (arg[6] == Py_False && arg[7] == Py_False))
    Py_RETURN_NONE;
  int* error = static_cast<int*>(PyLong_AsVoidPtr(arg[8]));
  const int64_t width = l.x.vocab;
  const at::TensorOptions options = l.x.like(l.x.t->scalar_type());
  at::Tensor d_hidden, d_table, space = l.space(true, arg[6] == Py_True);
  if (arg[6] == Py_True) d_hidden = at::empty_strided({l.x.rows, width}, {width, 1}, options);
  if (arg[7] == Py_True) d_table = at::empty_strided({l.w.rows, width}, {width, 1}, options);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(l.x.device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = loss_gradient_entry(l.x.code, l.x.t->data_ptr(), l.x.ld, l.w.t->data_ptr(), l.w.ld, int(l.x.rows), int(width), int(l.w.rows), l.targets, l.weight, log_sum,
                               float(l.softcap), d_hidden.defined() ? d_hidden.data_ptr() : nullptr, width, d_table.defined() ? d_table.data_ptr() : nullptr, width,
                               space.data_ptr(), error, stream);
  Py_END_ALLOW_THREADS
  return answer(status, d_hidden, d_table);
  END_HANDLE_TH_ERRORS
}

// The type of new rows: None is the other rows'.
bool type_of(PyObject* o, const Rows& x, at::ScalarType& type, int& code) {
  if (o == Py_None) type = x.t->scalar_type();
  else if (THPDtype_Check(o)) type = reinterpret_cast<THPDtype*>(o)->scalar_type;
  else return false;
  code = type == at::kFloat ? 0 : 1;
  return type == at::kFloat || type == at::kBFloat16;
}

// (ids, table, scale, out_dtype)
PyObject* token_rows(PyObject*, PyObject* const* arg, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Rows w;
  const int32_t* ids;
  double scale;
  at::ScalarType type;
  int code;
  if (n_args != 4 || rows_entry == nullptr || !w.of(arg[1]) || w.rows > TABLE_MOST || w.vocab > TABLE_MOST || arg[0] == Py_None || !numbers(arg[0], w, 1, ids) ||
      !number_of(arg[2], scale) || !type_of(arg[3], w, type, code))
    Py_RETURN_NONE;
  const int64_t tokens = THPVariable_Unpack(arg[0]).numel();
  if (tokens > TABLE_MOST) Py_RETURN_NONE;
  at::Tensor out = at::empty_strided({tokens, w.vocab}, {w.vocab, 1}, w.like(type));
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(w.device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = rows_entry(w.code, code, ids, w.t->data_ptr(), w.ld, out.data_ptr(), w.vocab, int(tokens), int(w.vocab), int(w.rows), float(scale), stream);
  Py_END_ALLOW_THREADS
  return answer(status, out);
  END_HANDLE_TH_ERRORS
}

// (ids, above, vocab, scale, out_dtype): into a new table
PyObject* token_rows_gradient(PyObject*, PyObject* const* arg, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  Rows x;
  const int32_t* ids;
  double scale;
  at::ScalarType type;
  int code, over = 0;
  if (n_args != 5 || rows_gradient_entry == nullptr || rows_space == nullptr || !x.of(arg[1]) || x.rows > TABLE_MOST || x.vocab > TABLE_MOST || arg[0] == Py_None ||
      !numbers(arg[0], x, x.rows, ids) || THPVariable_Unpack(arg[0]).numel() != x.rows || !PyLong_CheckExact(arg[2]) || !number_of(arg[3], scale) ||
      !type_of(arg[4], x, type, code))
    Py_RETURN_NONE;
  const long long vocab = PyLong_AsLongLongAndOverflow(arg[2], &over);
  if (over != 0 || vocab < 1 || vocab > TABLE_MOST) Py_RETURN_NONE;
  at::Tensor out = at::empty_strided({vocab, x.vocab}, {x.vocab, 1}, x.like(type)),
             space = at::empty_strided({rows_space(int(x.rows), int(x.vocab), int(vocab))}, {1}, x.like(at::kByte));
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = rows_gradient_entry(x.code, code, ids, x.t->data_ptr(), x.ld, out.data_ptr(), x.vocab, int(x.rows), int(x.vocab), int(vocab), float(scale), 0, space.data_ptr(), stream);
  Py_END_ALLOW_THREADS
  return answer(status, out);
  END_HANDLE_TH_ERRORS
}

// bind(name, address): the kernel library's entry that a face calls
PyObject* bind(PyObject*, PyObject* const* arg, Py_ssize_t n_args) {
  if (n_args != 2 || !PyUnicode_Check(arg[0])) {
    PyErr_SetString(PyExc_TypeError, "bind(name, address)");
    return nullptr;
  }
  void* address = PyLong_AsVoidPtr(arg[1]);
  if (address == nullptr && PyErr_Occurred()) return nullptr;
  if (PyUnicode_CompareWithASCIIString(arg[0], "adjust_logits") == 0) adjust_entry = reinterpret_cast<AdjustEntry>(address);
  else if (PyUnicode_CompareWithASCIIString(arg[0], "top_logits") == 0) top_entry = reinterpret_cast<TopEntry>(address);
  else if (PyUnicode_CompareWithASCIIString(arg[0], "distill") == 0) distill_entry = reinterpret_cast<DistillEntry>(address);
  else if (PyUnicode_CompareWithASCIIString(arg[0], "token_loss") == 0) loss_entry = reinterpret_cast<LossEntry>(address);
  else if (PyUnicode_CompareWithASCIIString(arg[0], "token_loss_gradient") == 0) loss_gradient_entry = reinterpret_cast<LossGradientEntry>(address);
  else if (PyUnicode_CompareWithASCIIString(arg[0], "token_loss_space") == 0) loss_space = reinterpret_cast<LossSpace>(address);
  else if (PyUnicode_CompareWithASCIIString(arg[0], "token_rows") == 0) rows_entry = reinterpret_cast<RowsEntry>(address);
  else if (PyUnicode_CompareWithASCIIString(arg[0], "token_rows_gradient") == 0) rows_gradient_entry = reinterpret_cast<RowsGradientEntry>(address);
  else if (PyUnicode_CompareWithASCIIString(arg[0], "token_rows_space") == 0) rows_space = reinterpret_cast<RowsSpace>(address);
  else {
    PyErr_SetString(PyExc_ValueError, "no such face");
    return nullptr;
  }
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
constexpr PyMethodDef face(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {face<adjust>("adjust_logits"), face<top>("top_logits"), face<distill>("distill"), face<token_loss>("token_loss"),
                         face<token_loss_gradient>("token_loss_gradient"), face<token_rows>("token_rows"), face<token_rows_gradient>("token_rows_gradient"), face<bind>("bind"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "r2faces", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_r2faces() { return PyModule_Create(&module); }
