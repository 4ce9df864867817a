// Operators that take and give torch tensors in one call: their checks, the output's allocation and the call of libspd.so without the
// interpreter in between.  In Python the same takes longer than the kernels of few tokens: a product 8.2 us of host time (its kernel 7.2),
// here 4.2; a norm with its quantisation 10.3 and 5.0.
//
// What comes back is what the Python form of the operator (ops.py) gives for the same arguments, or None: for anything unusual here
// (another type, shape, stride, device, a subclass, a failing call) the Python form runs, which refuses what it refuses.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/spd.h"
#include "tensorcalls.h"

namespace {

decltype(&spd_quant_int8) quant_fn;
decltype(&spd_int8_scaled_mm) product_fn;
decltype(&spd_linear_logprobs) logprobs_fn;
decltype(&spd_linear_logprobs_workspace_bytes) logprobs_room_fn;

// a tensor of the current device; null: something else (None is no tensor: see `given`)
const at::Tensor* tensor(PyObject* o, c10::DeviceIndex device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided && !t.is_neg() ? &t : nullptr;
}

int code(at::ScalarType t) { return t == at::kBFloat16 ? SPD_BF16 : t == at::kHalf ? SPD_F16 : t == at::kChar ? SPD_I8 : -1; }

// two dimensions, the last one contiguous
bool rows(const at::Tensor& t) { return t.dim() == 2 && t.stride(1) == 1; }

bool scales(const at::Tensor& t, int64_t n) { return t.scalar_type() == at::kFloat && t.numel() == n && t.is_contiguous(); }

// (past the dispatcher: 0.25 us a tensor)
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, c10::DeviceIndex device) {
  return at::Tensor(at::detail::empty_cuda(size, type, c10::Device(at::kCUDA, device), std::nullopt));
}

struct Here {
  c10::DeviceIndex device;
  spd_stream_t stream;
  Here() {
    const auto s = c10::cuda::getCurrentCUDAStream();
    device = s.device_index();
    stream = reinterpret_cast<spd_stream_t>(s.stream());
  }
};

template <typename F>
int run(F&& f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = f();
  Py_END_ALLOW_THREADS return rc;
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject* x = THPVariable_Wrap(a);
  PyObject* y = x ? THPVariable_Wrap(b) : nullptr;
  PyObject* out = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return out;
}

// (x, residual | None, weight | None, eps, silu_mul, sm_budget)
PyObject* quant_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !quant_fn || !PyFloat_CheckExact(a[3]) || !PyLong_CheckExact(a[4]) || !PyLong_CheckExact(a[5])) Py_RETURN_NONE;
  const Here here;
  const at::Tensor *x = tensor(a[0], here.device), *residual = nullptr, *weight = nullptr;
  if (!x || !rows(*x) || x->scalar_type() == at::kChar || code(x->scalar_type()) < 0) Py_RETURN_NONE;
  const long silu = PyLong_AsLong(a[4]);
  const int budget = static_cast<int>(PyLong_AsLong(a[5]));
  const int64_t count = x->size(0), cols = x->size(1), dim = silu ? cols / 2 : cols;
  if (silu && cols % 2) Py_RETURN_NONE;
  if (a[1] != Py_None) {
    residual = tensor(a[1], here.device);
    if (!residual || residual->scalar_type() != x->scalar_type() || residual->sizes() != x->sizes() || !residual->is_contiguous() ||
        !x->is_contiguous())
      Py_RETURN_NONE;
  }
  if (a[2] != Py_None) {
    weight = tensor(a[2], here.device);
    if (!weight || weight->scalar_type() != x->scalar_type() || weight->dim() != 1 || weight->size(0) != dim || weight->stride(0) != 1)
      Py_RETURN_NONE;
  }
  const at::Tensor q = empty({count, dim}, at::kChar, here.device), s = empty({count, 1}, at::kFloat, here.device);
  const int rc = run([&] {
    return quant_fn(static_cast<int8_t*>(q.data_ptr()), static_cast<float*>(s.data_ptr()), x->data_ptr(),
                    residual ? residual->data_ptr() : nullptr, weight ? weight->data_ptr() : nullptr, count, dim,
                    count > 1 ? x->stride(0) : cols, static_cast<float>(PyFloat_AS_DOUBLE(a[3])), static_cast<int>(silu),
                    code(x->scalar_type()), budget, here.stream);
  });
  if (rc) Py_RETURN_NONE;
  return pair(q, s);
  END_HANDLE_TH_ERRORS
}

// (mat_a, mat_b, scales_a, scales_b, out_dtype, bias | None, older_weight, sm_budget)
PyObject* int8_scaled_mm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !product_fn || !THPDtype_Check(a[4]) || !PyBool_Check(a[6]) || !PyLong_CheckExact(a[7])) Py_RETURN_NONE;
  const Here here;
  const at::Tensor *x = tensor(a[0], here.device), *w = tensor(a[1], here.device), *sa = tensor(a[2], here.device),
                   *sb = tensor(a[3], here.device), *bias = nullptr;
  if (!x || !w || !sa || !sb || !rows(*x) || w->dim() != 2 || w->stride(0) != 1) Py_RETURN_NONE;
  const int64_t M = x->size(0), K = x->size(1), N = w->size(1);
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
  if (x->scalar_type() != at::kChar || w->scalar_type() != at::kChar || w->size(0) != K || !scales(*sa, M) || !scales(*sb, N) ||
      (type != at::kBFloat16 && type != at::kHalf))
    Py_RETURN_NONE;
  if (a[5] != Py_None) {
    bias = tensor(a[5], here.device);
    if (!bias || bias->scalar_type() != type || bias->numel() != N || !bias->is_contiguous()) Py_RETURN_NONE;
  }
  const int budget = static_cast<int>(PyLong_AsLong(a[7])), older = a[6] == Py_True;
  const at::Tensor out = empty({M, N}, type, here.device);
  const int rc = run([&] {
    return product_fn(out.data_ptr(), static_cast<const int8_t*>(x->data_ptr()), static_cast<const int8_t*>(w->data_ptr()),
                      static_cast<const float*>(sa->data_ptr()), static_cast<const float*>(sb->data_ptr()),
                      bias ? bias->data_ptr() : nullptr, M, N, K, M > 1 ? x->stride(0) : K, N > 1 ? w->stride(1) : K, N, code(type), older,
                      budget, here.stream);
  });
  if (rc) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// (x, weight, targets, x_scales | None, weight_scales | None, older_weight, sm_budget)
PyObject* linear_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !logprobs_fn || !logprobs_room_fn || !PyBool_Check(a[5]) || !PyLong_CheckExact(a[6])) Py_RETURN_NONE;
  const Here here;
  const at::Tensor *x = tensor(a[0], here.device), *w = tensor(a[1], here.device), *targets = tensor(a[2], here.device), *xs = nullptr,
                   *ws = nullptr;
  if (!x || !w || !targets || !rows(*x) || !rows(*w) || x->size(1) != w->size(1) || x->scalar_type() != w->scalar_type()) Py_RETURN_NONE;
  const int64_t M = x->size(0), K = x->size(1), V = w->size(0);
  const int type = code(x->scalar_type());
  if (M == 0 || type < 0 || targets->scalar_type() != at::kLong || targets->dim() != 1 || targets->size(0) != M || !targets->is_contiguous() ||
      (type == SPD_I8) != (a[3] != Py_None) || (type == SPD_I8) != (a[4] != Py_None))
    Py_RETURN_NONE;
  if (type == SPD_I8) {
    xs = tensor(a[3], here.device);
    ws = tensor(a[4], here.device);
    if (!xs || !ws || !scales(*xs, M) || !scales(*ws, V)) Py_RETURN_NONE;
  }
  const int64_t room = logprobs_room_fn(M, V);
  if (room < 0) Py_RETURN_NONE;
  const int budget = static_cast<int>(PyLong_AsLong(a[6])), older = a[5] == Py_True;
  const at::Tensor lp = empty({M}, at::kFloat, here.device), lse = empty({M}, at::kFloat, here.device),
                   work = empty({room}, at::kByte, here.device);
  const int rc = run([&] {
    return logprobs_fn(static_cast<float*>(lp.data_ptr()), static_cast<float*>(lse.data_ptr()), x->data_ptr(), w->data_ptr(),
                       xs ? static_cast<const float*>(xs->data_ptr()) : nullptr, ws ? static_cast<const float*>(ws->data_ptr()) : nullptr,
                       static_cast<const int64_t*>(targets->data_ptr()), M, V, K, M > 1 ? x->stride(0) : K, V > 1 ? w->stride(0) : K, type,
                       older, work.data_ptr(), room, budget, here.stream);
  });
  if (rc) Py_RETURN_NONE;
  return pair(lp, lse);
  END_HANDLE_TH_ERRORS
}

template <typename F>
void take(PyObject* functions, const char* name, F* out) {
  PyObject* entry = PyDict_GetItemString(functions, name);  // borrowed: (address, ctypes function)
  PyObject* address = entry && PyTuple_Check(entry) ? PyTuple_GetItem(entry, 0) : nullptr;
  void* p = address ? PyLong_AsVoidPtr(address) : nullptr;
  if (PyErr_Occurred()) PyErr_Clear();
  *out = reinterpret_cast<F>(p);
}

}  // namespace

PyMethodDef spd_tensor_methods[] = {
    {"quant_int8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&quant_int8)), METH_FASTCALL, nullptr},
    {"int8_scaled_mm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&int8_scaled_mm)), METH_FASTCALL, nullptr},
    {"linear_logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&linear_logprobs)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

void spd_tensor_bind(PyObject* functions) {
  take(functions, "spd_quant_int8", &quant_fn);
  take(functions, "spd_int8_scaled_mm", &product_fn);
  take(functions, "spd_linear_logprobs", &logprobs_fn);
  take(functions, "spd_linear_logprobs_workspace_bytes", &logprobs_room_fn);
}
