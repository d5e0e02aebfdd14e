// The straight way from Python into the 8-bit linear path: one C++ call that reads the tensors' pointers, strides and types and
// launches on torch's current stream. A single token's norm or product takes 2 to 7 us on the GPU, less than reading a
// dozen tensor attributes from Python (about 7 us a call beside 3 us for the launch; here under 1 us).
//
// Each function takes the arguments of its namesake in lowbit.py, in order, and returns the output(s), or a negative
// B200_E* status, or None: "not an ordinary call". Ordinary are CUDA tensors on the current device with the right types and
// shapes whose rows are evenly spaced; everything else (copies to make, errors to report) is lowbit.py's, which checks
// all over again.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "b200_ops.h"

namespace {

PyObject *not_ordinary() { Py_RETURN_NONE; }

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return B200_TYPE_F32;
    case at::kHalf: return B200_TYPE_F16;
    case at::kBFloat16: return B200_TYPE_BF16;
    case at::kFloat8_e4m3fn: return B200_TYPE_E4M3;
    default: return -1;
  }
}
bool float_code(int c) { return c == B200_TYPE_F32 || c == B200_TYPE_F16 || c == B200_TYPE_BF16; }

// A CUDA tensor on device `device` (any when -1), or null.
const at::Tensor *tensor(PyObject *o, int device) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.unsafeGetTensorImpl()->is_python_dispatch() || t.is_neg()) return nullptr;
  if (device >= 0 && t.get_device() != device) return nullptr;
  return &t;
}

// Elements between rows (last axis), or -1 when they are not evenly spaced in an obvious way.
int64_t row_stride(const at::Tensor &t) {
  const int64_t n = t.dim();
  if (n == 0) return -1;
  if (t.is_contiguous()) return t.size(n - 1);
  if (n == 2 && t.stride(1) == 1 && t.size(0) > 1) return t.stride(0);
  return -1;
}

bool leading_is(const at::Tensor &t, const at::Tensor &like, int64_t extra) {
  const int64_t n = like.dim() - 1;
  if (t.dim() != n + (extra >= 0 ? 1 : 0)) return false;
  for (int64_t i = 0; i < n; ++i)
    if (t.size(i) != like.size(i)) return false;
  return extra < 0 || t.size(n) == extra;
}

bool absent(PyObject *o) { return o == Py_None; }

// e4m3 rows that start at multiples of 16 bytes
at::Tensor empty_codes(const at::Tensor &like) {
  auto sizes = like.sizes().vec();
  const int64_t len = sizes.back(), pitch = (len + 15) / 16 * 16;
  sizes.back() = pitch;
  at::Tensor t = at::empty(sizes, like.options().dtype(at::kFloat8_e4m3fn));
  return pitch == len ? t : t.narrow(-1, 0, len);
}

PyObject *wrap(PyObject *given, const at::Tensor &t) {
  if (!absent(given)) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(t);
}

// rmsnorm(x, gamma, residual, eps, out, scale, residual_out, codes) -> (out, scale, residual_out)
PyObject *rmsnorm_impl(PyObject *const *a) {
  const at::Tensor *x = tensor(a[0], -1);
  if (!x || x->dim() == 0 || x->numel() == 0) return not_ordinary();
  const int device = x->get_device(), type = type_code(x->scalar_type());
  if (device != c10::cuda::current_device() || !float_code(type)) return not_ordinary();
  const int64_t len = x->size(-1);
  const bool codes = a[7] == Py_True;
  b200_rmsnorm_desc d = {};
  d.rows = x->numel() / len;
  d.len = len;
  d.type = d.gamma_type = type;
  d.y_type = codes ? B200_TYPE_E4M3 : type;
  d.eps = (float)PyFloat_AsDouble(a[3]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return not_ordinary();
  }
  if ((d.x_stride = row_stride(*x)) < 0) return not_ordinary();
  const at::Tensor *gamma = nullptr, *residual = nullptr;
  if (!absent(a[1])) {
    gamma = tensor(a[1], device);
    if (!gamma || gamma->dim() != 1 || gamma->size(0) != len || !gamma->is_contiguous()) return not_ordinary();
    d.gamma_type = type_code(gamma->scalar_type());
    if (d.gamma_type != type && d.gamma_type != B200_TYPE_F32) return not_ordinary();
  }
  if (!absent(a[2])) {
    residual = tensor(a[2], device);
    if (!residual || residual->scalar_type() != x->scalar_type() || !leading_is(*residual, *x, len)) return not_ordinary();
    if ((d.residual_stride = row_stride(*residual)) < 0) return not_ordinary();
  } else if (!absent(a[6])) {
    return not_ordinary();
  }
  at::Tensor made_out, made_scale, made_h;
  const at::Tensor *out = &made_out, *scale = &made_scale, *h = &made_h;
  if (!absent(a[4]) && !(out = tensor(a[4], device))) return not_ordinary();
  if (!absent(a[5]) && !(scale = tensor(a[5], device))) return not_ordinary();
  if (!absent(a[6]) && !(h = tensor(a[6], device))) return not_ordinary();
  if (!codes && !absent(a[5])) return not_ordinary();
  if (out->defined()) {
    if (type_code(out->scalar_type()) != d.y_type || !leading_is(*out, *x, len)) return not_ordinary();
  } else {
    made_out = codes ? empty_codes(*x) : at::empty(x->sizes(), x->options());
  }
  if (codes) {
    if (!scale->defined()) made_scale = at::empty(x->sizes().slice(0, x->dim() - 1), x->options().dtype(at::kFloat));
    if (scale->scalar_type() != at::kFloat || !leading_is(*scale, *x, -1) || !scale->is_contiguous()) return not_ordinary();
  }
  if (residual) {
    if (!h->defined()) made_h = at::empty(x->sizes(), x->options());
    if (h->scalar_type() != x->scalar_type() || !leading_is(*h, *x, len)) return not_ordinary();
    if ((d.h_stride = row_stride(*h)) < len) return not_ordinary();
  }
  if ((d.y_stride = row_stride(*out)) < len) {
    // new codes with padded rows of a tensor of more axes: their rows are evenly spaced by construction
    if (!absent(a[4])) return not_ordinary();
    d.y_stride = (len + 15) / 16 * 16;
  }
  const int rc = b200_rmsnorm(c10::cuda::getCurrentCUDAStream(device).stream(), &d, x->data_ptr(),
                              residual ? residual->data_ptr() : nullptr, gamma ? gamma->data_ptr() : nullptr,
                              residual ? h->data_ptr() : nullptr, out->data_ptr(),
                              codes ? static_cast<float *>(scale->data_ptr()) : nullptr);
  if (rc != B200_OK) return PyLong_FromLong(rc);
  PyObject *r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, wrap(a[4], *out));
  PyTuple_SET_ITEM(r, 1, codes ? wrap(a[5], *scale) : (Py_INCREF(Py_None), Py_None));
  PyTuple_SET_ITEM(r, 2, residual ? wrap(a[6], *h) : (Py_INCREF(Py_None), Py_None));
  return r;
}

// quantize_rows(x, gate, activation code, out, scale) -> (out, scale)
PyObject *quantize_rows_impl(PyObject *const *a) {
  const at::Tensor *x = tensor(a[0], -1);
  if (!x || x->dim() == 0 || x->numel() == 0) return not_ordinary();
  const int device = x->get_device(), type = type_code(x->scalar_type());
  if (device != c10::cuda::current_device() || !float_code(type)) return not_ordinary();
  const int64_t len = x->size(-1);
  b200_quantize_desc d = {};
  d.rows = x->numel() / len;
  d.len = len;
  d.type = type;
  d.activation = (int32_t)PyLong_AsLong(a[2]);
  if ((d.x_stride = row_stride(*x)) < 0) return not_ordinary();
  const at::Tensor *gate = nullptr;
  if (!absent(a[1])) {
    gate = tensor(a[1], device);
    if (!gate || gate->scalar_type() != x->scalar_type() || !leading_is(*gate, *x, len)) return not_ordinary();
    if ((d.gate_stride = row_stride(*gate)) < 0) return not_ordinary();
  } else if (d.activation != B200_ACT_NONE) {
    return not_ordinary();
  }
  at::Tensor made_out, made_scale;
  const at::Tensor *out = &made_out, *scale = &made_scale;
  if (!absent(a[3]) && !(out = tensor(a[3], device))) return not_ordinary();
  if (!absent(a[4]) && !(scale = tensor(a[4], device))) return not_ordinary();
  if (!out->defined()) made_out = empty_codes(*x);
  if (!scale->defined()) made_scale = at::empty(x->sizes().slice(0, x->dim() - 1), x->options().dtype(at::kFloat));
  if (out->scalar_type() != at::kFloat8_e4m3fn || !leading_is(*out, *x, len) || scale->scalar_type() != at::kFloat ||
      !leading_is(*scale, *x, -1) || !scale->is_contiguous())
    return not_ordinary();
  if ((d.q_stride = row_stride(*out)) < len) {
    if (!absent(a[3])) return not_ordinary();
    d.q_stride = (len + 15) / 16 * 16;
  }
  const int rc = b200_quantize_rows(c10::cuda::getCurrentCUDAStream(device).stream(), &d, x->data_ptr(),
                                    gate ? gate->data_ptr() : nullptr, out->data_ptr(),
                                    static_cast<float *>(scale->data_ptr()));
  if (rc != B200_OK) return PyLong_FromLong(rc);
  PyObject *r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, wrap(a[3], *out));
  PyTuple_SET_ITEM(r, 1, wrap(a[4], *scale));
  return r;
}

// The axes that are not 1 agree with the first `axes` ones of `like`, or there is at most one (all rows in order).
bool scale_shape(const at::Tensor &t, const at::Tensor &like, int64_t axes) {
  int64_t i = 0, longer = 0;
  bool agree = true;
  for (int64_t j = 0; j < t.dim(); ++j) {
    if (t.size(j) == 1) continue;
    ++longer;
    while (i < axes && like.size(i) == 1) ++i;
    agree = agree && i < axes && like.size(i++) == t.size(j);
  }
  return agree || longer <= 1;
}
// A scale operand: one entry for all rows, or one for each row of `like` (whose rows lie along its first `axes` axes).
bool scale_operand(PyObject *o, int device, const at::Tensor &like, int64_t axes, int64_t rows, const float **p, int32_t *step) {
  if (absent(o)) return true;
  const at::Tensor *t = tensor(o, device);
  if (!t || t->scalar_type() != at::kFloat || !t->is_contiguous()) return false;
  const int64_t n = t->numel();
  if (n != 1 && (n != rows || !scale_shape(*t, like, axes))) return false;
  *step = n == rows;
  *p = static_cast<const float *>(t->data_ptr());
  return true;
}
bool rows_for_tma(const at::Tensor &t, int64_t stride, int64_t rows, int64_t size) {
  return stride >= t.size(-1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (rows <= 1 || stride * size % 16 == 0);
}

// matmul_scaled(A, W, a_scale, w_scale, bias, activation code, residual, out, output type code or -1) -> out
PyObject *matmul_scaled_impl(PyObject *const *a) {
  const at::Tensor *A = tensor(a[0], -1);
  if (!A || A->dim() == 0 || A->numel() == 0) return not_ordinary();
  const int device = A->get_device();
  const at::Tensor *W = tensor(a[1], device);
  b200_gemm_scaled_desc d = {};
  d.type = type_code(A->scalar_type());
  if (device != c10::cuda::current_device() || !W || W->dim() != 2 || W->scalar_type() != A->scalar_type() ||
      W->size(1) != A->size(-1) || W->size(0) == 0 ||
      (d.type != B200_TYPE_E4M3 && d.type != B200_TYPE_F16 && d.type != B200_TYPE_BF16))
    return not_ordinary();
  d.K = A->size(-1);
  d.M = A->numel() / d.K;
  d.N = W->size(0);
  const int64_t size = d.type == B200_TYPE_E4M3 ? 1 : 2;
  d.lda = row_stride(*A);
  d.ldw = row_stride(*W);
  if (!rows_for_tma(*A, d.lda, d.M, size) || !rows_for_tma(*W, d.ldw, d.N, size)) return not_ordinary();
  const float *a_scale = nullptr, *w_scale = nullptr;
  if (!scale_operand(a[2], device, *A, A->dim() - 1, d.M, &a_scale, &d.a_scale_step) ||
      !scale_operand(a[3], device, *W, 1, d.N, &w_scale, &d.w_scale_step))
    return not_ordinary();
  const at::Tensor *bias = nullptr, *residual = nullptr;
  if (!absent(a[4])) {
    bias = tensor(a[4], device);
    if (!bias || bias->dim() != 1 || bias->size(0) != d.N || !bias->is_contiguous()) return not_ordinary();
    d.bias_type = type_code(bias->scalar_type());
    if (!float_code(d.bias_type)) return not_ordinary();
  }
  d.activation = (int32_t)PyLong_AsLong(a[5]);
  if (!absent(a[6])) {
    residual = tensor(a[6], device);
    if (!residual || !leading_is(*residual, *A, d.N)) return not_ordinary();
    d.ldr = row_stride(*residual);
    if (d.ldr < d.N) return not_ordinary();
  }
  const long asked = PyLong_AsLong(a[8]);
  if (asked >= 0 && !float_code((int)asked)) return not_ordinary();
  at::Tensor made;
  const at::Tensor *out = &made;
  if (!absent(a[7])) {
    out = tensor(a[7], device);
    if (!out || !leading_is(*out, *A, d.N)) return not_ordinary();
    d.y_type = type_code(out->scalar_type());
    if (asked >= 0 && asked != d.y_type) return not_ordinary();
  } else {
    const at::ScalarType t = asked == B200_TYPE_F32    ? at::kFloat
                             : asked == B200_TYPE_F16  ? at::kHalf
                             : asked == B200_TYPE_BF16 ? at::kBFloat16
                             : residual                ? residual->scalar_type()
                             : size == 1               ? at::kBFloat16
                                                       : A->scalar_type();
    d.y_type = type_code(t);
    if (!float_code(d.y_type)) return not_ordinary();
    auto sizes = A->sizes().vec();
    sizes.back() = d.N;
    made = at::empty(sizes, A->options().dtype(t));
  }
  if (!float_code(d.y_type) || (residual && residual->scalar_type() != out->scalar_type())) return not_ordinary();
  d.ldy = row_stride(*out);
  if (d.ldy < d.N) return not_ordinary();
  const int rc = b200_gemm_scaled(c10::cuda::getCurrentCUDAStream(device).stream(), &d, A->data_ptr(), W->data_ptr(), a_scale,
                                  w_scale, bias ? bias->data_ptr() : nullptr, residual ? residual->data_ptr() : nullptr,
                                  out->data_ptr());
  if (rc != B200_OK) return PyLong_FromLong(rc);
  return wrap(a[7], *out);
}

// What torch throws (no memory for an output) becomes torch's own Python exception.
template <PyObject *(*F)(PyObject *const *), int N>
PyObject *guarded(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  HANDLE_TH_ERRORS
  return F(args);
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"rmsnorm", (PyCFunction)(void (*)(void))guarded<rmsnorm_impl, 8>, METH_FASTCALL, nullptr},
    {"quantize_rows", (PyCFunction)(void (*)(void))guarded<quantize_rows_impl, 5>, METH_FASTCALL, nullptr},
    {"matmul_scaled", (PyCFunction)(void (*)(void))guarded<matmul_scaled_impl, 9>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "torch_calls", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_torch_calls(void) { return PyModule_Create(&kModule); }
