// qlin._native: the call path of the small operators from torch tensors to the C ABI (include/qlin.h).
//
// A call of a few microseconds on the GPU is dominated by what the host does for it, so the checks, the
// allocation of the outputs and the launch of such operators run here instead of in Python (measured: 4 to 8 us a
// call against 17 to 52 through ctypes).  These functions take the calls that need nothing else (tensors on
// the current device, whose layout the library reads as it is) and return None for every other one; the Python
// functions of the same names then copy, convert, switch devices or refuse.  The library's functions are given by
// address, so that the build that QLIN_LIB selects is the one that runs.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/qlin.h"

namespace {

decltype(&qlin_fp8_linear) fp8_linear_fn = nullptr;
decltype(&qlin_fp8_linear_workspace) fp8_linear_ws = nullptr;
decltype(&qlin_fp8_linear_grad_input) fp8_grad_fn = nullptr;
decltype(&qlin_fp8_linear_grad_input_workspace) fp8_grad_ws = nullptr;
decltype(&qlin_rotary_table) table_fn = nullptr;
decltype(&qlin_qk_norm_rotary) qk_fn = nullptr;
decltype(&qlin_qk_norm_rotary_backward) qk_grad_fn = nullptr;
decltype(&qlin_qk_norm_rotary_backward_workspace) qk_grad_ws = nullptr;
PyObject* check_fn = nullptr;  // qlin._lib.check: raises for a status that is not QLIN_OK

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return QLIN_F32;
    case at::kHalf: return QLIN_F16;
    case at::kBFloat16: return QLIN_BF16;
    default: return -1;
  }
}

// The tensor behind an argument; null for None and for what is not a plain tensor or parameter.
const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on_device(const at::Tensor* t, c10::DeviceIndex dev) {
  return t != nullptr && t->is_cuda() && t->get_device() == dev && t->layout() == at::kStrided;
}

// The tensor itself where nothing failed, else what qlin._lib.check raises for the status.
PyObject* answer(int rc, const char* what, PyObject* result) {
  if (rc == QLIN_OK) return result;
  Py_XDECREF(result);
  PyObject* r = PyObject_CallFunction(check_fn, "is", rc, what);
  Py_XDECREF(r);
  if (r != nullptr) PyErr_SetString(PyExc_RuntimeError, what);
  return nullptr;
}

// The tensors as a tuple; None for one that is undefined.
PyObject* tuple_of(std::initializer_list<at::Tensor> items) {
  PyObject* r = PyTuple_New((Py_ssize_t)items.size());
  Py_ssize_t i = 0;
  for (const at::Tensor& t : items) {
    if (r == nullptr) break;
    PyObject* o = THPVariable_Wrap(t);  // None where t is undefined
    if (o == nullptr) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

void* workspace(size_t bytes, const at::Tensor& like, at::Tensor& keep) {
  if (bytes == 0) return nullptr;
  keep = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
  return keep.data_ptr();
}

// Rows [m, features] with a unit inner stride, as the library reads them without a copy.
bool rows_of(const at::Tensor& x, int64_t features, int64_t& m, int64_t& ld) {
  if (x.dim() < 1 || x.size(-1) != features || x.numel() == 0) return false;
  m = x.numel() / features;
  if (x.dim() == 2) {
    ld = x.stride(0);
    return x.stride(1) == 1 && (ld >= features || m == 1);
  }
  ld = features;
  return x.is_contiguous();
}

PyObject* fp8_product(PyObject* const* args, Py_ssize_t nargs, bool grad) {
  HANDLE_TH_ERRORS
  const at::Tensor *x = tensor(args[0]), *q = tensor(args[1]), *s = tensor(args[2]);
  if (x == nullptr || !x->is_cuda()) Py_RETURN_NONE;
  const c10::DeviceIndex dev = c10::cuda::current_device();
  if (!on_device(x, dev) || !on_device(q, dev) || !on_device(s, dev)) Py_RETURN_NONE;
  const at::Tensor* bias = nargs > 3 ? tensor(args[3]) : nullptr;
  if (nargs > 3 && args[3] != Py_None && !on_device(bias, dev)) Py_RETURN_NONE;
  const int dt = code_of(x->scalar_type());
  if (dt < 0 || q->scalar_type() != at::kFloat8_e4m3fn || q->dim() != 2 || s->scalar_type() != at::kFloat || s->dim() != 2)
    Py_RETURN_NONE;
  const int64_t n = q->size(0), k = q->size(1), in = grad ? n : k, out = grad ? k : n;
  int64_t m = 0, ld = 0;
  if (n == 0 || k == 0 || k % 16 != 0 || q->stride(1) != 1 || q->stride(0) % 16 != 0 || q->stride(0) < k ||
      reinterpret_cast<uintptr_t>(q->data_ptr()) % 16 != 0 || s->size(0) != (n + 127) / 128 ||
      s->size(1) != (k + 127) / 128 || s->stride(1) != 1 || s->stride(0) < s->size(1) || !rows_of(*x, in, m, ld))
    Py_RETURN_NONE;
  int bias_dt = 0;
  if (bias != nullptr) {
    bias_dt = code_of(bias->scalar_type());
    if (bias_dt < 0 || bias->numel() != n || !bias->is_contiguous()) Py_RETURN_NONE;
  }
  at::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = out;
  at::Tensor y = at::empty(shape, x->options().requires_grad(false)), keep;
  const size_t bytes = grad ? fp8_grad_ws(m, n, k) : fp8_linear_ws(m, n, k);
  void* ws = workspace(bytes, *x, keep);
  void* stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  const void *xp = x->data_ptr(), *qp = q->data_ptr();
  const float* sp = reinterpret_cast<const float*>(s->data_ptr());
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = grad ? fp8_grad_fn(xp, dt, m, n, ld, qp, q->stride(0), k, sp, s->stride(0), y.data_ptr(), dt, k, ws, bytes, stream)
            : fp8_linear_fn(xp, dt, m, k, ld, qp, q->stride(0), n, sp, s->stride(0), bias ? bias->data_ptr() : nullptr,
                            bias_dt, y.data_ptr(), dt, n, ws, bytes, stream);
  Py_END_ALLOW_THREADS
  return answer(rc, grad ? "qlin_fp8_linear_grad_input" : "qlin_fp8_linear", THPVariable_Wrap(std::move(y)));
  END_HANDLE_TH_ERRORS
}

// fp8_linear(x, qdata, scale, bias)
PyObject* fp8_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4) Py_RETURN_NONE;
  return fp8_product(args, nargs, false);
}

// fp8_linear_grad_input(dy, qdata, scale)
PyObject* fp8_linear_grad_input(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 3) Py_RETURN_NONE;
  return fp8_product(args, nargs, true);
}

// rotary_table(positions, axes_dim, theta)
PyObject* rotary_table(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 3 || (!PyList_CheckExact(args[1]) && !PyTuple_CheckExact(args[1])) || !PyFloat_CheckExact(args[2]))
    Py_RETURN_NONE;
  const at::Tensor* pos = tensor(args[0]);
  if (pos == nullptr || !pos->is_cuda()) Py_RETURN_NONE;
  const c10::DeviceIndex dev = c10::cuda::current_device();
  if (!on_device(pos, dev) || pos->dim() < 1 || pos->numel() == 0 || !pos->is_contiguous()) Py_RETURN_NONE;
  const at::ScalarType t = pos->scalar_type();
  const int dt = t == at::kFloat ? QLIN_F32 : t == at::kInt ? QLIN_I32 : t == at::kLong ? QLIN_I64 : -1;
  const Py_ssize_t axes = PySequence_Fast_GET_SIZE(args[1]);
  int32_t dims[16];
  if (dt < 0 || axes < 1 || axes > 16 || pos->size(-1) != axes) Py_RETURN_NONE;
  int64_t sum = 0;
  for (Py_ssize_t a = 0; a < axes; ++a) {
    PyObject* item = PySequence_Fast_GET_ITEM(args[1], a);
    const long d = PyLong_CheckExact(item) ? PyLong_AsLong(item) : -1;
    if (d < 0 || d > 512 || d % 2 != 0) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    dims[a] = (int32_t)d;
    sum += d;
  }
  if (sum == 0) Py_RETURN_NONE;
  at::DimVector shape(pos->sizes().begin(), pos->sizes().end() - 1);
  shape.push_back(sum / 2);
  shape.push_back(2);
  at::Tensor out = at::empty(shape, pos->options().dtype(at::kFloat).requires_grad(false));
  const double theta = PyFloat_AS_DOUBLE(args[2]);
  void* stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = table_fn(pos->data_ptr(), dt, pos->numel() / axes, (int)axes, dims, theta, reinterpret_cast<float*>(out.data_ptr()),
                stream);
  Py_END_ALLOW_THREADS
  return answer(rc, "qlin_rotary_table", THPVariable_Wrap(std::move(out)));
  END_HANDLE_TH_ERRORS
}

// q, k, their weights and the table, as both directions of the head norm read them.
struct Heads {
  const at::Tensor *q, *k, *qw, *kw, *table;
  int dt, wdt;
  int64_t b, l, hq, hk, d, pairs, table_b;
};

bool like(const at::Tensor* t, const at::Tensor& q, int64_t heads, c10::DeviceIndex dev) {
  return on_device(t, dev) && t->dim() == 4 && t->scalar_type() == q.scalar_type() && t->size(0) == q.size(0) &&
         t->size(1) == q.size(1) && t->size(2) == heads && t->size(3) == q.size(3) && t->stride(3) == 1;
}

bool heads_of(PyObject* const* a, Heads& h) {
  h.q = tensor(a[0]);
  if (h.q == nullptr || !h.q->is_cuda()) return false;
  const c10::DeviceIndex dev = c10::cuda::current_device();
  h.k = tensor(a[1]);
  h.qw = tensor(a[2]);
  h.kw = tensor(a[3]);
  h.table = tensor(a[4]);
  if (!on_device(h.q, dev) || h.q->dim() != 4 || h.q->stride(3) != 1 || !on_device(h.k, dev) || h.k->dim() != 4 ||
      !like(h.k, *h.q, h.k->size(2), dev) || !on_device(h.table, dev))
    return false;
  h.b = h.q->size(0);
  h.l = h.q->size(1);
  h.hq = h.q->size(2);
  h.hk = h.k->size(2);
  h.d = h.q->size(3);
  h.dt = code_of(h.q->scalar_type());
  if (h.dt < 0 || h.q->numel() == 0 || h.k->numel() == 0) return false;
  if ((h.qw == nullptr && a[2] != Py_None) || (h.kw == nullptr && a[3] != Py_None)) return false;
  h.wdt = -1;
  for (const at::Tensor* w : {h.qw, h.kw}) {
    if (w == nullptr) continue;
    const int c = code_of(w->scalar_type());
    if (!on_device(w, dev) || c < 0 || w->dim() != 1 || w->size(0) != h.d || (h.d > 1 && w->stride(0) != 1) ||
        (h.wdt >= 0 && h.wdt != c))
      return false;
    h.wdt = c;
  }
  if (h.wdt < 0) h.wdt = QLIN_F32;
  const at::Tensor& t = *h.table;
  if (t.scalar_type() != at::kFloat || t.dim() != 3 || t.size(0) != h.l || t.size(2) != 2 || 2 * t.size(1) > h.d ||
      !t.is_contiguous())
    return false;
  h.pairs = t.size(1);
  return true;
}

// qk_norm_rotary(q, k, q_weight, k_weight, table, eps, interleaved)
PyObject* qk_norm_rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Heads h;
  if (nargs != 7 || !PyFloat_CheckExact(args[5]) || !PyBool_Check(args[6]) || !heads_of(args, h)) Py_RETURN_NONE;
  const auto opts = h.q->options().requires_grad(false);
  at::Tensor qo = at::empty(h.q->sizes(), opts), ko = at::empty(h.k->sizes(), opts);
  const float eps = (float)PyFloat_AS_DOUBLE(args[5]);
  void* stream = c10::cuda::getCurrentCUDAStream(h.q->get_device()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = qk_fn(h.q->data_ptr(), h.q->strides().data(), h.k->data_ptr(), h.k->strides().data(), h.dt, h.b, h.l, (int)h.hq,
             (int)h.hk, (int)h.d, h.qw ? h.qw->data_ptr() : nullptr, h.kw ? h.kw->data_ptr() : nullptr, h.wdt,
             reinterpret_cast<const float*>(h.table->data_ptr()), 0, (int)h.pairs, eps, args[6] == Py_True,
             qo.data_ptr(), qo.strides().data(), ko.data_ptr(), ko.strides().data(), stream);
  Py_END_ALLOW_THREADS
  return answer(rc, "qlin_qk_norm_rotary", tuple_of({qo, ko}));
  END_HANDLE_TH_ERRORS
}

// qk_norm_rotary_backward(dq, dk, q, k, q_weight, k_weight, table, eps, interleaved)
PyObject* qk_norm_rotary_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Heads h;
  if (nargs != 9 || !PyFloat_CheckExact(args[7]) || !PyBool_Check(args[8]) || !heads_of(args + 2, h)) Py_RETURN_NONE;
  const at::Tensor *dq = tensor(args[0]), *dk = tensor(args[1]);
  const c10::DeviceIndex dev = h.q->get_device();
  if (!like(dq, *h.q, h.hq, dev) || !like(dk, *h.q, h.hk, dev)) Py_RETURN_NONE;
  const auto opts = h.q->options().requires_grad(false);
  at::Tensor gq = at::empty(h.q->sizes(), opts), gk = at::empty(h.k->sizes(), opts), gqw, gkw, keep;
  if (h.qw) gqw = at::empty({h.d}, h.qw->options().requires_grad(false));
  if (h.kw) gkw = at::empty({h.d}, h.kw->options().requires_grad(false));
  const size_t bytes = qk_grad_ws(h.b, h.l, (int)h.hq, (int)h.hk, (int)h.d);
  void* ws = workspace(bytes, *h.q, keep);
  const float eps = (float)PyFloat_AS_DOUBLE(args[7]);
  void* stream = c10::cuda::getCurrentCUDAStream(dev).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = qk_grad_fn(dq->data_ptr(), dq->strides().data(), dk->data_ptr(), dk->strides().data(), h.q->data_ptr(),
                  h.q->strides().data(), h.k->data_ptr(), h.k->strides().data(), h.dt, h.b, h.l, (int)h.hq, (int)h.hk,
                  (int)h.d, h.qw ? h.qw->data_ptr() : nullptr, h.kw ? h.kw->data_ptr() : nullptr, h.wdt,
                  reinterpret_cast<const float*>(h.table->data_ptr()), 0, (int)h.pairs, eps, args[8] == Py_True,
                  gq.data_ptr(), gq.strides().data(), gk.data_ptr(), gk.strides().data(),
                  h.qw ? gqw.data_ptr() : nullptr, h.kw ? gkw.data_ptr() : nullptr, ws, bytes, stream);
  Py_END_ALLOW_THREADS
  return answer(rc, "qlin_qk_norm_rotary_backward", tuple_of({gq, gk, gqw, gkw}));
  END_HANDLE_TH_ERRORS
}

// bind(check, address of each library function in the order below)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 9) {
    PyErr_SetString(PyExc_TypeError, "bind takes the check function and eight addresses");
    return nullptr;
  }
  void* at[8];
  for (int i = 0; i < 8; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i + 1]);
    if (at[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  Py_INCREF(args[0]);
  Py_XSETREF(check_fn, args[0]);
  fp8_linear_fn = reinterpret_cast<decltype(fp8_linear_fn)>(at[0]);
  fp8_linear_ws = reinterpret_cast<decltype(fp8_linear_ws)>(at[1]);
  fp8_grad_fn = reinterpret_cast<decltype(fp8_grad_fn)>(at[2]);
  fp8_grad_ws = reinterpret_cast<decltype(fp8_grad_ws)>(at[3]);
  table_fn = reinterpret_cast<decltype(table_fn)>(at[4]);
  qk_fn = reinterpret_cast<decltype(qk_fn)>(at[5]);
  qk_grad_fn = reinterpret_cast<decltype(qk_grad_fn)>(at[6]);
  qk_grad_ws = reinterpret_cast<decltype(qk_grad_ws)>(at[7]);
  Py_RETURN_NONE;
}

#define QLIN_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {QLIN_METHOD(bind),
                         QLIN_METHOD(fp8_linear),
                         QLIN_METHOD(fp8_linear_grad_input),
                         QLIN_METHOD(rotary_table),
                         QLIN_METHOD(qk_norm_rotary),
                         QLIN_METHOD(qk_norm_rotary_backward),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// The torch and Python that it was compiled against, for the importer to compare with its own.
PyMODINIT_FUNC PyInit__native() {
  PyObject* m = PyModule_Create(&module_def);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", QLIN_BUILT_FOR) != 0) Py_CLEAR(m);
  return m;
}
