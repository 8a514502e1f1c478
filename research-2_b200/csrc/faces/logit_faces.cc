// The operators on rows of logits, called with tensors: what Python does for a call (checks, new tensors, the stream) in one step. A call
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
AdjustEntry adjust_entry = nullptr;
TopEntry top_entry = nullptr;
DistillEntry distill_entry = nullptr;

constexpr int64_t MOST = 0x7fffffff, TOP_MOST = 256;

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

PyMethodDef methods[] = {face<adjust>("adjust_logits"), face<top>("top_logits"), face<distill>("distill"), face<bind>("bind"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "r2faces", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_r2faces() { return PyModule_Create(&module); }
