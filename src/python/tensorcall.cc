// The 8-bit layers (piccl_b200/ops/fp8.py) as native functions that take tensors.
//
// A layer is one or two launches of a few microseconds; checked and issued from Python through ctypes it took 23 us of host time, most of it the checks, the allocation of
// scratch and the conversion of arguments.  Each function here returns the number of launches, or 0 if anything about its arguments is not as it has to be (or nothing is to be launched): the
// Python function then looks at them itself and says what is wrong.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/python_variable.h>
#include "../ops/piccl_ops.h"

namespace {

struct Eight { const at::Tensor *v = nullptr, *s = nullptr; };

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
bool of_values(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }

// A pair of values and scales of a matrix whose device is `d`
bool eight(PyObject* o, const c10::Device& d, Eight& e) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) return false;
  e.v = tensor(PyTuple_GET_ITEM(o, 0)); e.s = tensor(PyTuple_GET_ITEM(o, 1));
  if (!e.v || !e.s || e.v->dim() != 2 || e.v->scalar_type() != at::kFloat8_e4m3fn || !e.v->is_contiguous() || e.v->size(1) % 128 || e.v->device() != d) return false;
  const int64_t want[5] = {(e.v->size(0) + 127) / 128, (e.v->size(1) + 511) / 512, 32, 4, 4};
  return e.s->scalar_type() == at::kByte && e.s->is_contiguous() && e.s->device() == d && e.s->sizes() == at::IntArrayRef(want, 5);
}
bool has_room(const Eight& e, int64_t rows, int64_t cols) { return e.v->size(0) == rows && e.v->size(1) == (cols + 127) / 128 * 128; }
// A matrix that is not empty, its rows of values next to each other
bool matrix(const at::Tensor* t, bool contiguous) {
  if (!t || t->dim() != 2 || !of_values(*t) || !t->is_cuda() || t->numel() == 0 || t->size(0) > 0x7fffff00 || t->size(1) > 0x7fffff00) return false;
  if (contiguous) return t->is_contiguous();
  return (t->size(1) == 1 || t->stride(1) == 1) && (t->size(0) == 1 || t->stride(0) >= t->size(1));
}
long long row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
bool bias_fits(PyObject* o, const at::Tensor& out, const at::Tensor*& bias) {
  bias = nullptr;
  if (o == Py_None) return true;
  bias = tensor(o);
  return bias && bias->scalar_type() == at::kBFloat16 && bias->dim() == 1 && bias->size(0) == out.size(1) && bias->is_contiguous() && bias->device() == out.device();
}
void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
void* stream() { return at::cuda::getCurrentCUDAStream().stream(); }

// Room for a matrix in 8 bits, until the end of the call (the allocator hands it on in the order of the stream)
struct Scratch {
  c10::DataPtr p; char* v; char* s;
  Scratch(int64_t rows, int64_t cols) {
    const int64_t n = rows * ((cols + 127) / 128 * 128), at = (n + 511) / 512 * 512;
    p = c10::cuda::CUDACachingAllocator::get()->allocate(at + (rows + 127) / 128 * ((cols + 511) / 512) * 512);
    v = static_cast<char*>(p.get()); s = v + at;
  }
};
PyObject* answer(int rc, int launches, const char* what) {
  if (rc == 0) return PyLong_FromLong(launches);
  PyErr_Format(PyExc_RuntimeError, "%s failed (code %d)", what, rc);
  return nullptr;
}
template <class F> PyObject* guarded(F f) {
  try { return f(); } catch (const std::exception& e) { PyErr_SetString(PyExc_RuntimeError, e.what()); return nullptr; }
}
PyObject* no() { return PyLong_FromLong(0); }

// quantize(x, out, transposed, square)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* const x = n == 4 ? tensor(a[0]) : nullptr;
    Eight q, t;
    if (!matrix(x, false) || (a[1] == Py_None && a[2] == Py_None)) return no();
    if (a[1] != Py_None && !(eight(a[1], x->device(), q) && has_room(q, x->size(0), x->size(1)))) return no();
    if (a[2] != Py_None && !(eight(a[2], x->device(), t) && has_room(t, x->size(1), x->size(0)))) return no();
    const int square = PyObject_IsTrue(a[3]);
    if (square < 0) return nullptr;
    const c10::cuda::CUDAGuard guard(x->device());
    return answer(piccl_ops_fp8_quantize(x->data_ptr(), x->scalar_type() == at::kFloat, x->size(0), x->size(1), row_stride(*x), ptr(q.v), ptr(q.s), ptr(t.v), ptr(t.s), square, stream()), 1, "fp8 quantize");
  });
}

// product(a, b, out, bias)
PyObject* product(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *const out = n == 4 ? tensor(a[2]) : nullptr, *bias;
    Eight x, w;
    if (!matrix(out, true) || !eight(a[0], out->device(), x) || !eight(a[1], out->device(), w) || !bias_fits(a[3], *out, bias)) return no();
    if (x.v->size(1) != w.v->size(1) || x.v->size(1) == 0 || x.v->size(0) != out->size(0) || w.v->size(0) != out->size(1)) return no();
    const c10::cuda::CUDAGuard guard(out->device());
    return answer(piccl_ops_fp8_gemm(ptr(x.v), ptr(x.s), ptr(w.v), ptr(w.s), ptr(bias), out->data_ptr(), out->scalar_type() == at::kFloat, (int)out->size(0), (int)out->size(1), x.v->size(1), 0, stream()), 1,
                  "fp8 product");
  });
}

// linear(x, w, out, bias, keep)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor *const x = n == 5 ? tensor(a[0]) : nullptr, *const out = n == 5 ? tensor(a[2]) : nullptr, *bias;
    Eight w, keep;
    if (!matrix(x, false) || !matrix(out, true) || out->device() != x->device() || !eight(a[1], x->device(), w) || !has_room(w, out->size(1), x->size(1)) || out->size(0) != x->size(0)) return no();
    if (!bias_fits(a[3], *out, bias) || (a[4] != Py_None && !(eight(a[4], x->device(), keep) && has_room(keep, x->size(1), x->size(0))))) return no();
    const c10::cuda::CUDAGuard guard(x->device());
    const int M = (int)x->size(0), fp32 = x->scalar_type() == at::kFloat, f32 = out->scalar_type() == at::kFloat;
    const long long K = x->size(1), stride = row_stride(*x);
    int rc;
    if (piccl_ops_fp8_linear_scratch(x->data_ptr(), fp32, stride, M, (int)out->size(1), K, keep.v != nullptr)) {
      const Scratch q(M, K);
      rc = piccl_ops_fp8_linear(x->data_ptr(), fp32, stride, ptr(w.v), ptr(w.s), ptr(bias), out->data_ptr(), f32, q.v, q.s, ptr(keep.v), ptr(keep.s), M, (int)out->size(1), K, stream());
    } else
      rc = piccl_ops_fp8_linear(x->data_ptr(), fp32, stride, ptr(w.v), ptr(w.s), ptr(bias), out->data_ptr(), f32, nullptr, nullptr, nullptr, nullptr, M, (int)out->size(1), K, stream());
    return answer(rc < 0 ? rc : 0, rc, "fp8 linear");
  });
}

// linear_bwd(dy, xt, wt, dx, dw)
PyObject* linear_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const at::Tensor* const dy = n == 5 ? tensor(a[0]) : nullptr;
    if (!matrix(dy, false) || (a[3] == Py_None && a[4] == Py_None)) return no();
    const at::Tensor *dx = nullptr, *dw = nullptr;
    Eight xt, wt;
    const int64_t M = dy->size(0), N = dy->size(1);
    if (a[3] != Py_None) {
      dx = tensor(a[3]);
      if (!matrix(dx, true) || dx->device() != dy->device() || !eight(a[2], dy->device(), wt) || !has_room(wt, dx->size(1), N) || dx->size(0) != M) return no();
    }
    if (a[4] != Py_None) {
      dw = tensor(a[4]);
      if (!matrix(dw, true) || dw->device() != dy->device() || !eight(a[1], dy->device(), xt) || !has_room(xt, dw->size(1), M) || dw->size(0) != N) return no();
    }
    const c10::cuda::CUDAGuard guard(dy->device());
    const Scratch q(dx ? M : 0, N), t(dw ? N : 0, M);
    int rc = piccl_ops_fp8_quantize(dy->data_ptr(), dy->scalar_type() == at::kFloat, M, N, row_stride(*dy), dx ? q.v : nullptr, dx ? q.s : nullptr, dw ? t.v : nullptr, dw ? t.s : nullptr, 0, stream());
    if (!rc && dx) rc = piccl_ops_fp8_gemm(q.v, q.s, ptr(wt.v), ptr(wt.s), nullptr, dx->data_ptr(), dx->scalar_type() == at::kFloat, (int)M, (int)dx->size(1), (N + 127) / 128 * 128, 0, stream());
    if (!rc && dw) rc = piccl_ops_fp8_gemm(t.v, t.s, ptr(xt.v), ptr(xt.s), nullptr, dw->data_ptr(), dw->scalar_type() == at::kFloat, (int)N, (int)dw->size(1), (M + 127) / 128 * 128, 0, stream());
    return answer(rc, 1 + (dx != nullptr) + (dw != nullptr), "fp8 linear_bwd");
  });
}

#define M_(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {M_(quantize), M_(product), M_(linear), M_(linear_bwd), {nullptr, nullptr, 0, nullptr}};
#undef M_
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensorcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensorcall(void) { return PyModule_Create(&module); }
