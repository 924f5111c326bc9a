// Tensor-level calls of the training-step operators, for training.py: checks of
// the tensors, outputs and scratch from torch's allocator, one call of the C ABI on
// the current stream of the tensors' device.
//
// In C++ because the smallest calls take less time on the device than on the host:
// a layer norm of 16 x 5120 takes 6.3 us there, 7 us of host time here, and took 14
// through ctypes, of which the library's own launch is 4.
//
// Each function takes its arguments by position and returns a tuple of tensors (or
// the table of an optimizer's tensors), or the library's status as an int when that
// is not 0.  Bad tensors raise ValueError.
#include <Python.h>

#include <algorithm>
#include <cstdint>
#include <limits>
#include <memory>
#include <utility>
#include <vector>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include "nvfp4_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

constexpr ScalarType kF32 = ScalarType::Float, kU8 = ScalarType::Byte;

const Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), name, ": expected a CUDA tensor");
  return THPVariable_Unpack(o);
}
// A CUDA tensor that settles the call's device.
const Tensor& first(PyObject* o, const char* name, int& device) {
  const Tensor& t = tensor(o, name);
  TORCH_CHECK_VALUE(t.is_cuda(), name, ": expected a CUDA tensor");
  device = (int)t.get_device();
  return t;
}
void on(const Tensor& t, int device, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.get_device() == device, name, ": not on cuda:", device);
}

int code_of(ScalarType t, const char* name) {
  switch (t) {
    case ScalarType::Float: return NVFP4_DTYPE_F32;
    case ScalarType::BFloat16: return NVFP4_DTYPE_BF16;
    case ScalarType::Half: return NVFP4_DTYPE_F16;
    default: break;
  }
  TORCH_CHECK_VALUE(false, name, ": unexpected type ", t);
}
ScalarType type_of(int code) {
  return code == NVFP4_DTYPE_F32    ? ScalarType::Float
         : code == NVFP4_DTYPE_BF16 ? ScalarType::BFloat16
                                    : ScalarType::Half;
}

// Row stride of an m x n tensor with unit inner stride.
int64_t rows(const Tensor& t, int64_t m, int64_t n, ScalarType type, int device,
             const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.dim() == 2 && t.size(0) == m && t.size(1) == n,
                    name, ": expected [", m, ", ", n, "] ", type, ", got ", t.sizes(), " ",
                    t.scalar_type());
  on(t, device, name);
  if (t.is_contiguous()) return n;
  TORCH_CHECK_VALUE(n <= 1 || t.stride(1) == 1, name, ": the inner stride must be 1");
  // A single row has no row stride to speak of.
  return m > 1 ? t.stride(0) : std::max(t.stride(0), n);
}
// Address of n contiguous values.
void* vector(const Tensor& t, int64_t n, int device, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name, ": expected ", n,
                    " contiguous values, got ", t.sizes());
  on(t, device, name);
  return t.data_ptr();
}
// Address of n float32, or null for None.
float* words(PyObject* o, int64_t n, int device, const char* name) {
  if (o == Py_None) return nullptr;
  const Tensor& t = tensor(o, name);
  TORCH_CHECK_VALUE(t.numel() == n && t.scalar_type() == kF32 && t.is_contiguous() &&
                        t.is_cuda() && t.get_device() == device,
                    name, ": expected ", n, " float32 on cuda:", device);
  return (float*)t.data_ptr();
}

Tensor empty(at::IntArrayRef size, ScalarType type, int device) {
  return Tensor(at::detail::empty_cuda(size, type, c10::Device(c10::DeviceType::CUDA, device),
                                       std::nullopt));
}

// The library's call `f(stream)` with the device current and the interpreter free.
template <typename F>
int launch(int device, const F& f) {
  const c10::cuda::CUDAGuard guard(device);
  nvfp4_stream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = f(stream);
  Py_END_ALLOW_THREADS
  return status;
}

PyObject* object(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
template <typename... T>
PyObject* result(int status, const T&... t) {
  if (status) return PyLong_FromLong(status);
  PyObject* r = PyTuple_New(sizeof...(T));
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(r, i++, object(t)), ...);
  return r;
}

void count(Py_ssize_t have, Py_ssize_t want) {
  TORCH_CHECK_TYPE(have == want, "expected ", want, " arguments, got ", have);
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

struct Operand {
  int64_t rows, k;
  const void *codes, *scales;
  const float* amax;
};
Operand operand(PyObject* const* o, int device, const char* name) {
  const Tensor &c = tensor(o[0], name), &s = tensor(o[1], name);
  TORCH_CHECK_VALUE(c.scalar_type() == kU8 && c.dim() == 2 && c.is_contiguous() && c.is_cuda() &&
                        c.get_device() == device,
                    name, ": codes are a contiguous 2-D uint8 tensor on cuda:", device);
  const int64_t half = c.size(1);
  TORCH_CHECK_VALUE(half % 16 == 0, name, ": k must be a multiple of 32, got ", 2 * half);
  TORCH_CHECK_VALUE(s.element_size() == 1 && s.dim() == 2 && s.size(0) == c.size(0) &&
                        s.size(1) == half / 8 && s.is_contiguous() && s.is_cuda() &&
                        s.get_device() == device,
                    name, ": scales are contiguous bytes of shape [", c.size(0), ", ", half / 8,
                    "] on cuda:", device);
  TORCH_CHECK_VALUE(o[2] != Py_None, name, ": amax: expected 1 float32 on cuda:", device);
  return {c.size(0), 2 * half, c.data_ptr(), s.data_ptr(), words(o[2], 1, device, name)};
}
Tensor scratch(size_t bytes, int device) {
  return bytes ? empty({(int64_t)bytes}, kU8, device) : Tensor();
}
void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// a, a_scales, a_amax, b, b_scales, b_amax, bias, residual, activation, out type, out,
// with_aux, amax_out -> (D, aux)
PyObject* matmul(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 13);
  int device;
  first(o[0], "a", device);
  const Operand a = operand(o, device, "a"), b = operand(o + 3, device, "b");
  TORCH_CHECK_VALUE(a.k == b.k, "a and b differ in k: ", a.k, " and ", b.k);
  const int64_t m = a.rows, n = b.rows;
  const int act = (int)integer(o[8]);
  int code;
  int64_t ldd = n;
  Tensor out;
  if (o[10] == Py_None) {
    code = (int)integer(o[9]);
    out = empty({m, n}, type_of(code), device);
  } else {
    out = tensor(o[10], "out");
    code = code_of(out.scalar_type(), "out");
    ldd = rows(out, m, n, out.scalar_type(), device, "out");
  }
  const ScalarType type = type_of(code);
  const void *bias = nullptr, *residual = nullptr;
  int bias_code = 0;
  int64_t ldr = n;
  if (o[6] != Py_None) {
    const Tensor& t = tensor(o[6], "bias");
    bias_code = code_of(t.scalar_type(), "bias");
    bias = vector(t, n, device, "bias");
  }
  if (o[7] != Py_None) {
    const Tensor& t = tensor(o[7], "residual");
    ldr = rows(t, m, n, type, device, "residual");
    residual = t.data_ptr();
  }
  float* amax = words(o[12], 1, device, "amax_out");
  const Tensor aux = PyObject_IsTrue(o[11]) ? empty({m, n}, type, device) : Tensor();
  const size_t bytes = nvfp4_gemm_workspace_bytes(m, n, a.k);
  const Tensor ws = scratch(bytes, device);
  const int status = launch(device, [&](nvfp4_stream_t stream) {
    return nvfp4_gemm(m, n, a.k, a.codes, a.scales, a.amax, b.codes, b.scales, b.amax,
                      out.data_ptr(), ldd, code, bias, bias_code, residual, ldr, act, address(aux),
                      n, amax, address(ws), bytes, 0, stream);
  });
  return result(status, out, aux);
  END_HANDLE_TH_ERRORS
}

// a, a_scales, a_amax, b, b_scales, b_amax, aux, activation, with_dbias, amax_out
// -> (D, dbias)
PyObject* matmul_dact(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 10);
  int device;
  first(o[0], "a", device);
  const Operand a = operand(o, device, "a"), b = operand(o + 3, device, "b");
  TORCH_CHECK_VALUE(a.k == b.k, "a and b differ in k: ", a.k, " and ", b.k);
  const int64_t m = a.rows, n = b.rows;
  const Tensor& aux = tensor(o[6], "aux");
  const ScalarType type = aux.scalar_type();
  const int code = code_of(type, "aux"), act = (int)integer(o[7]);
  const int64_t ldaux = rows(aux, m, n, type, device, "aux");
  float* amax = words(o[9], 1, device, "amax_out");
  const Tensor d = empty({m, n}, type, device);
  const bool with_dbias = PyObject_IsTrue(o[8]);
  const Tensor dbias = with_dbias ? empty({n}, kF32, device) : Tensor();
  const size_t bytes = with_dbias ? nvfp4_gemm_dact_workspace_bytes(m, n, a.k)
                                  : nvfp4_gemm_workspace_bytes(m, n, a.k);
  const Tensor ws = scratch(bytes, device);
  const int status = launch(device, [&](nvfp4_stream_t stream) {
    return nvfp4_gemm_dact(m, n, a.k, a.codes, a.scales, a.amax, b.codes, b.scales, b.amax,
                           aux.data_ptr(), ldaux, act, d.data_ptr(), n, code,
                           (float*)address(dbias), amax, address(ws), bytes, 0, stream);
  });
  return result(status, d, dbias);
  END_HANDLE_TH_ERRORS
}

struct Norm {
  int64_t rows, cols, ldx;
  int code, weight;
  ScalarType type;
  const void *x, *gamma;
};
Norm norm(const Tensor& x, const Tensor& gamma, int device) {
  Norm r;
  TORCH_CHECK_VALUE(x.dim() == 2, "x: expected a 2-D float32, bfloat16 or float16 tensor");
  r.type = x.scalar_type();
  r.code = code_of(r.type, "x");
  r.weight = code_of(gamma.scalar_type(), "gamma");
  TORCH_CHECK_VALUE(r.weight == 0 || r.weight == r.code, "gamma: expected ", r.type,
                    " or float32, got ", gamma.scalar_type());
  r.rows = x.size(0);
  r.cols = x.size(1);
  r.ldx = rows(x, r.rows, r.cols, r.type, device, "x");
  r.x = x.data_ptr();
  r.gamma = vector(gamma, r.cols, device, "gamma");
  return r;
}

// x, gamma, beta, eps, amax_out -> (y, mean, rstd)
PyObject* layernorm(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 5);
  int device;
  const Tensor &x = first(o[0], "x", device), &gamma = tensor(o[1], "gamma");
  const Norm a = norm(x, gamma, device);
  const void* beta = nullptr;
  if (o[2] != Py_None) {
    const Tensor& t = tensor(o[2], "beta");
    TORCH_CHECK_VALUE(t.scalar_type() == gamma.scalar_type(), "beta: expected ",
                      gamma.scalar_type(), ", got ", t.scalar_type());
    beta = vector(t, a.cols, device, "beta");
  }
  const float eps = (float)real(o[3]);
  float* amax = words(o[4], 1, device, "amax_out");
  const Tensor y = empty({a.rows, a.cols}, a.type, device);
  const Tensor mean = empty({a.rows}, kF32, device), rstd = empty({a.rows}, kF32, device);
  if (a.cols == 0) {
    // Statistics of nothing, which the library leaves as they are.
    const c10::cuda::CUDAGuard guard(device);
    for (const Tensor& t : {mean, rstd}) t.fill_(std::numeric_limits<float>::quiet_NaN());
  }
  const int status = launch(device, [&](nvfp4_stream_t stream) {
    return nvfp4_layernorm_fwd(a.rows, a.cols, a.x, a.ldx, a.gamma, beta, a.code, a.weight, eps,
                               y.data_ptr(), a.cols, (float*)mean.data_ptr(),
                               (float*)rstd.data_ptr(), amax, stream);
  });
  return result(status, y, mean, rstd);
  END_HANDLE_TH_ERRORS
}

// dy, x, mean, rstd, gamma, residual -> (dx, dgamma, dbeta)
PyObject* layernorm_backward(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 6);
  int device;
  const Tensor &x = first(o[1], "x", device), &gamma = tensor(o[4], "gamma");
  const Norm a = norm(x, gamma, device);
  const Tensor& dy = tensor(o[0], "dy");
  const int64_t lddy = rows(dy, a.rows, a.cols, a.type, device, "dy");
  const void* residual = nullptr;
  int64_t ldr = a.cols;
  if (o[5] != Py_None) {
    const Tensor& t = tensor(o[5], "residual");
    ldr = rows(t, a.rows, a.cols, a.type, device, "residual");
    residual = t.data_ptr();
  }
  TORCH_CHECK_VALUE(o[2] != Py_None && o[3] != Py_None, "mean, rstd: expected float32 tensors");
  const float *mean = words(o[2], a.rows, device, "mean"),
              *rstd = words(o[3], a.rows, device, "rstd");
  const Tensor dx = empty({a.rows, a.cols}, a.type, device);
  const Tensor dgamma = empty({a.cols}, gamma.scalar_type(), device),
               dbeta = empty({a.cols}, gamma.scalar_type(), device);
  const size_t bytes = nvfp4_layernorm_bwd_workspace_bytes(a.rows, a.cols);
  const Tensor ws = scratch(bytes, device);
  const int status = launch(device, [&](nvfp4_stream_t stream) {
    return nvfp4_layernorm_bwd(a.rows, a.cols, dy.data_ptr(), lddy, a.x, a.ldx, mean, rstd,
                               a.gamma, residual, ldr, a.code, a.weight, dx.data_ptr(), a.cols,
                               dgamma.data_ptr(), dbeta.data_ptr(), address(ws), bytes, stream);
  });
  return result(status, dx, dgamma, dbeta);
  END_HANDLE_TH_ERRORS
}

// The lists of tensors of an AdamW step.
enum List { kParams, kGrads, kAvgs, kAvgSqs, kAvgScales, kAvgSqScales, kCopies, kLists };
constexpr const char* kListName[kLists] = {"params",         "grads",
                                           "exp_avgs",       "exp_avg_sqs",
                                           "exp_avg_scales", "exp_avg_sq_scales",
                                           "copies"};

// A tensor whose address a table holds.  Holding the tensor does not hold its memory:
// `p.data = ...`, set_ and resize_ give a tensor other memory and free the old, so
// that every step looks whether the tensor is still what it was.
struct Held {
  Tensor tensor;
  const void* data;
  int64_t n;
  caffe2::TypeMeta dtype;
  explicit Held(const Tensor& t)
      : tensor(t), data(t.data_ptr()), n(t.numel()), dtype(t.dtype()) {}
  // (By the fields: the accessors' own checks are most of the time of a step of many
  // short tensors.)
  bool same() const {
    const c10::TensorImpl& t = *tensor.unsafeGetTensorImpl();
    const char* p = static_cast<const char*>(t.unsafe_storage().data());
    return t.numel() == n && t.dtype() == dtype && t.is_contiguous() &&
           (n == 0 || p + t.storage_offset() * (int64_t)dtype.itemsize() == data);
  }
};

// Memory that a step writes.
struct Range {
  uintptr_t begin, end;
  const char* name;
};
Range range_of(const Held& h, const char* name) {
  const uintptr_t p = (uintptr_t)h.data;
  return {p, p + (uintptr_t)h.n * h.dtype.itemsize(), name};
}

// The gradients, and the library's descriptors of all tensors with them.  Replaced as a
// whole: another thread may pass new ones while a step's call runs.
struct Rows {
  std::vector<nvfp4_adamw_tensor> rows;
  std::vector<Held> grads;
};

struct AdamWTable {
  int device = 0, param = 0, grad = 0, state = 0;
  size_t count = 0;
  std::shared_ptr<const Rows> now;
  std::vector<Held> lists[kLists];     // (kGrads: in `now`)
  std::vector<Held> words;             // amax_out, rng_state
  std::vector<Range> written;          // sorted; none overlaps the next
  std::vector<char> follows;           // grads[i] is params[i].grad
  float* amax = nullptr;
  const size_t* rng = nullptr;
};
constexpr const char* kTableName = "fp4_sm120a_b200.AdamWTable";
constexpr int64_t kStateBlock = 128;

AdamWTable& table_of(PyObject* o) {
  void* p = PyCapsule_GetPointer(o, kTableName);
  if (!p) throw python_error();
  return *static_cast<AdamWTable*>(p);
}

// A list's tensors: contiguous, of one type, n(i) elements each.
template <typename N>
std::vector<Held> held(PyObject* seq, size_t count, ScalarType type, List list, const N& n) {
  THPObjectPtr fast(PySequence_Fast(seq, kListName[list]));
  if (!fast) throw python_error();
  TORCH_CHECK_VALUE((size_t)PySequence_Fast_GET_SIZE(fast.get()) == count, kListName[list], ": ",
                    PySequence_Fast_GET_SIZE(fast.get()), " entries for ", count, " parameters");
  std::vector<Held> r;
  r.reserve(count);
  for (size_t i = 0; i < count; ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(fast.get(), i);
    TORCH_CHECK_VALUE(THPVariable_Check(o), kListName[list], "[", i, "]: expected a tensor");
    const Tensor& t = THPVariable_Unpack(o);
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.numel() == n(i) && t.is_contiguous(),
                      kListName[list], "[", i, "]: expected ", n(i), " contiguous ", type,
                      ", got ", t.sizes(), " ", t.scalar_type());
    r.emplace_back(t);
  }
  return r;
}
void on_device(const std::vector<Held>& list, int device, const char* name) {
  for (size_t i = 0; i < list.size(); ++i)
    TORCH_CHECK_VALUE(list[i].tensor.is_cuda() && list[i].tensor.get_device() == device, name, "[",
                      i, "]: not on the parameters' device");
}
// Sorts what a step writes: two blocks would write an overlap at once.
void sort_written(std::vector<Range>& w) {
  std::sort(w.begin(), w.end(),
            [](const Range& a, const Range& b) { return a.begin < b.begin; });
  for (size_t i = 1; i < w.size(); ++i)
    TORCH_CHECK_VALUE(w[i - 1].end <= w[i].begin, w[i - 1].name, " and ", w[i].name,
                      ": tensors that the step writes overlap (the same tensor twice?)");
}
// Refuses memory to be read that the step writes.
void apart(const std::vector<Range>& written, const Range& r) {
  const auto next = std::lower_bound(
      written.begin(), written.end(), r.end,
      [](const Range& a, uintptr_t end) { return a.begin < end; });
  TORCH_CHECK_VALUE(r.begin == r.end || next == written.begin() || (next - 1)->end <= r.begin,
                    r.name, " and ", (next - 1)->name,
                    ": a tensor that the step reads overlaps one that it writes");
}
// Takes the gradients (looked at by held), and sees which are their parameters' own
// .grad.
void put_grads(AdamWTable& t, std::vector<nvfp4_adamw_tensor> rows, std::vector<Held>&& grads) {
  for (const Held& g : grads) apart(t.written, range_of(g, kListName[kGrads]));
  on_device(grads, t.device, kListName[kGrads]);
  for (size_t i = 0; i < t.count; ++i) {
    rows[i].grad = grads[i].data;
    const Tensor& own = t.lists[kParams][i].tensor.unsafeGetTensorImpl()->grad();
    t.follows[i] = own.defined() && own.is_same(grads[i].tensor);
  }
  t.now = std::make_shared<const Rows>(Rows{std::move(rows), std::move(grads)});
}

// params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, copies,
// weight_decays, offsets, amax_out, rng_state (None where there is none; the types of
// the first tensors, and what belongs together, have been looked at) -> table
PyObject* adamw_table(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 11);
  auto t = std::make_unique<AdamWTable>();
  const Py_ssize_t tensors = PySequence_Size(o[kParams]);
  if (tensors < 0) throw python_error();
  TORCH_CHECK_VALUE(tensors > 0, "no parameters");
  TORCH_CHECK_VALUE(tensors <= INT32_MAX, "params: too many");
  auto type_of_first = [&](List list) {
    THPObjectPtr first(PySequence_GetItem(o[list], 0));
    if (!first) throw python_error();
    return tensor(first.get(), kListName[list]).scalar_type();
  };
  const ScalarType param = type_of_first(kParams), grad = type_of_first(kGrads),
                   state = type_of_first(kAvgs) == kU8 ? kU8 : kF32;
  t->param = code_of(param, "params");
  t->grad = code_of(grad, "grads");
  t->state = state == kU8 ? NVFP4_STATE_8BIT : NVFP4_STATE_F32;
  t->count = (size_t)tensors;
  t->follows.resize(t->count);
  std::vector<nvfp4_adamw_tensor> rows(t->count);
  {
    THPObjectPtr fast(PySequence_Fast(o[kParams], "params"));
    if (!fast) throw python_error();
    for (Py_ssize_t i = 0; i < tensors; ++i)
      rows[i].n = (uint64_t)tensor(PySequence_Fast_GET_ITEM(fast.get(), i), "params").numel();
  }
  auto size = [&](size_t i) { return (int64_t)rows[i].n; };
  auto blocks = [&](size_t i) { return (size(i) + kStateBlock - 1) / kStateBlock; };
  t->lists[kParams] = held(o[kParams], tensors, param, kParams, size);
  std::vector<Held> grads = held(o[kGrads], tensors, grad, kGrads, size);
  for (List list : {kAvgs, kAvgSqs}) t->lists[list] = held(o[list], tensors, state, list, size);
  if (state == kU8)
    for (List list : {kAvgScales, kAvgSqScales})
      t->lists[list] = held(o[list], tensors, kU8, list, blocks);
  if (o[kCopies] != Py_None)
    t->lists[kCopies] = held(o[kCopies], tensors, ScalarType::BFloat16, kCopies, size);

  if (o[9] != Py_None) t->words.emplace_back(tensor(o[9], "amax_out"));
  for (int list = 0; list < kLists; ++list)
    for (const Held& h : t->lists[list])
      if (h.n) t->written.push_back(range_of(h, kListName[list]));
  for (const Held& h : t->words) t->written.push_back(range_of(h, "amax_out"));
  sort_written(t->written);
  if (o[10] != Py_None) {
    t->words.emplace_back(tensor(o[10], "rng_state"));
    apart(t->written, range_of(t->words.back(), "rng_state"));
    t->rng = (const size_t*)t->words.back().data;
  }
  for (const Held& g : grads) apart(t->written, range_of(g, kListName[kGrads]));

  const Tensor& first_param = t->lists[kParams][0].tensor;
  TORCH_CHECK_VALUE(first_param.is_cuda(), "params: expected CUDA tensors");
  t->device = (int)first_param.get_device();
  for (int list = 0; list < kLists; ++list)
    on_device(t->lists[list], t->device, kListName[list]);
  t->amax = words(o[9], tensors, t->device, "amax_out");

  THPObjectPtr decays(o[7] == Py_None ? nullptr : PySequence_Fast(o[7], "weight_decays"));
  THPObjectPtr offsets(o[8] == Py_None ? nullptr : PySequence_Fast(o[8], "offsets"));
  if ((o[7] != Py_None && !decays) || (o[8] != Py_None && !offsets)) throw python_error();
  uint64_t next = 0;
  for (size_t i = 0; i < t->count; ++i) {
    nvfp4_adamw_tensor& r = rows[i];
    auto at = [&](List list) -> void* {
      return t->lists[list].empty() ? nullptr : const_cast<void*>(t->lists[list][i].data);
    };
    r.param = at(kParams);
    r.exp_avg = at(kAvgs);
    r.exp_avg_sq = at(kAvgSqs);
    r.exp_avg_scale = (uint8_t*)at(kAvgScales);
    r.exp_avg_sq_scale = (uint8_t*)at(kAvgSqScales);
    r.copy = at(kCopies);
    r.weight_decay = decays ? real(PySequence_Fast_GET_ITEM(decays.get(), i)) : 0.0;
    r.offset = offsets ? (uint64_t)integer(PySequence_Fast_GET_ITEM(offsets.get(), i)) : next;
    next += (uint64_t)(blocks(i) * kStateBlock);
  }
  put_grads(*t, std::move(rows), std::move(grads));
  PyObject* capsule = PyCapsule_New(t.get(), kTableName, [](PyObject* c) {
    delete static_cast<AdamWTable*>(PyCapsule_GetPointer(c, kTableName));
  });
  if (!capsule) throw python_error();
  t.release();
  return capsule;
  END_HANDLE_TH_ERRORS
}

// table, lr, beta1, beta2, eps, step, grad_scale, scalars, new gradients or None -> ()
PyObject* adamw_step(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 9);
  AdamWTable& t = table_of(o[0]);
  const double lr = real(o[1]), beta1 = real(o[2]), beta2 = real(o[3]), eps = real(o[4]);
  const int64_t step = integer(o[5]);
  const float *scale = words(o[6], 1, t.device, "grad_scale"),
              *scalars = words(o[7], 3, t.device, "scalars");
  if (scale) apart(t.written, {(uintptr_t)scale, (uintptr_t)(scale + 1), "grad_scale"});
  if (scalars) apart(t.written, {(uintptr_t)scalars, (uintptr_t)(scalars + 3), "scalars"});
  for (const Held& w : t.words)
    TORCH_CHECK_VALUE(w.same(), "amax_out, rng_state: the tensor has other memory now");
  auto look = [](const std::vector<Held>& list, const char* name) {
    for (size_t i = 0; i < list.size(); ++i)
      TORCH_CHECK_VALUE(list[i].same(), name, "[", i,
                        "]: the tensor has other memory, size or type than when it was listed");
  };
  for (int list = 0; list < kLists; ++list) look(t.lists[list], kListName[list]);
  if (o[8] != Py_None) {
    const std::vector<nvfp4_adamw_tensor>& rows = t.now->rows;
    put_grads(t, rows, held(o[8], t.count, type_of(t.grad), kGrads,
                            [&](size_t i) { return (int64_t)rows[i].n; }));
  } else {
    look(t.now->grads, kListName[kGrads]);
    for (size_t i = 0; i < t.count; ++i)
      TORCH_CHECK_VALUE(!t.follows[i] || t.lists[kParams][i].tensor.unsafeGetTensorImpl()
                                             ->grad().is_same(t.now->grads[i].tensor),
                        "grads[", i, "]: params[", i,
                        "].grad is another tensor now; pass the new gradients (grads=)");
  }
  const std::shared_ptr<const Rows> now = t.now;
  return result(launch(t.device, [&](nvfp4_stream_t stream) {
    return nvfp4_adamw_step(now->rows.data(), (int)t.count, t.param, t.grad, t.state, lr, beta1,
                            beta2, eps, step, scale, scalars, t.amax, t.rng, stream);
  }));
  END_HANDLE_TH_ERRORS
}

// codes, scales, moment, out type -> (values,)
PyObject* adamw_unpack_state(PyObject*, PyObject* const* o, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 4);
  int device;
  const Tensor &codes = first(o[0], "codes", device), &scales = tensor(o[1], "scales");
  TORCH_CHECK_VALUE(codes.scalar_type() == kU8 && codes.is_contiguous(),
                    "codes: expected contiguous uint8");
  const int64_t n = codes.numel(), blocks = (n + 127) / 128;
  TORCH_CHECK_VALUE(scales.scalar_type() == kU8 && scales.is_contiguous() &&
                        scales.numel() == blocks && scales.is_cuda() &&
                        scales.get_device() == device,
                    "scales: expected ", blocks, " contiguous uint8 on cuda:", device);
  const int moment = (int)integer(o[2]), code = (int)integer(o[3]);
  const Tensor out = empty(codes.sizes(), type_of(code), device);
  const int status = launch(device, [&](nvfp4_stream_t stream) {
    return nvfp4_adamw_unpack_state(codes.data_ptr(), (const uint8_t*)scales.data_ptr(),
                                    (size_t)n, moment, out.data_ptr(), code, stream);
  });
  return result(status, out);
  END_HANDLE_TH_ERRORS
}

#define NVFP4_METHOD(name) {#name, (PyCFunction)(void (*)())name, METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {NVFP4_METHOD(matmul),    NVFP4_METHOD(matmul_dact),
                          NVFP4_METHOD(layernorm), NVFP4_METHOD(layernorm_backward),
                          NVFP4_METHOD(adamw_table), NVFP4_METHOD(adamw_step),
                          NVFP4_METHOD(adamw_unpack_state),
                          {nullptr, nullptr, 0, nullptr}};
#undef NVFP4_METHOD
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_binding",
                       "Tensor-level calls of the training-step operators.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding() { return PyModule_Create(&kModule); }
