// The 8-bit layers (piccl_b200/ops/fp8.py) and the step of the optimiser over many tensors (optimizer.py) as native functions that take tensors.
//
// A layer is one or two launches of a few microseconds; checked and issued from Python through ctypes it took 23 us of host time, most of it the checks, the allocation of
// scratch and the conversion of arguments.  Each function here returns the number of launches, or 0 if anything about its arguments is not as it has to be (or nothing is to be launched): the
// Python function then looks at them itself and says what is wrong.
#include <Python.h>
#include <initializer_list>
#include <memory>
#include <vector>
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Exceptions.h>
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
// What is written shares no bytes with what is read, nor with what else is written (the first `written` of them); null pointers are passed over
bool apart(std::initializer_list<const at::Tensor*> all, size_t written) {
  struct Range { uintptr_t lo, hi; } r[10];
  size_t n = 0;
  for (const at::Tensor* t : all) {
    Range& q = r[n++];
    q = {0, 0};
    if (!t || t->numel() == 0) continue;
    long long last = 0;
    for (int64_t d = 0; d < t->dim(); d++) last += (t->size(d) - 1) * t->stride(d);
    q.lo = reinterpret_cast<uintptr_t>(t->data_ptr()); q.hi = q.lo + (last + 1) * t->element_size();
  }
  for (size_t i = 0; i < written; i++)
    for (size_t j = i + 1; j < n; j++)
      if (r[i].lo < r[j].hi && r[j].lo < r[i].hi) return false;
  return true;
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
  try { return f(); } catch (...) { torch::translate_exception_to_python(std::current_exception()); return nullptr; }      // out of memory stays torch.OutOfMemoryError
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
    if (!apart({q.v, q.s, t.v, t.s, x}, 4)) return no();
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
    if (!apart({out, x.v, x.s, w.v, w.s, bias}, 1)) return no();
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
    if (!apart({out, keep.v, keep.s, x, w.v, w.s, bias}, 3)) return no();
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
    if (!apart({dx, dw, dy, xt.v, xt.s, wt.v, wt.s}, 2)) return no();
    const c10::cuda::CUDAGuard guard(dy->device());
    const Scratch q(dx ? M : 0, N), t(dw ? N : 0, M);
    int rc = piccl_ops_fp8_quantize(dy->data_ptr(), dy->scalar_type() == at::kFloat, M, N, row_stride(*dy), dx ? q.v : nullptr, dx ? q.s : nullptr, dw ? t.v : nullptr, dw ? t.s : nullptr, 0, stream());
    if (!rc && dx) rc = piccl_ops_fp8_gemm(q.v, q.s, ptr(wt.v), ptr(wt.s), nullptr, dx->data_ptr(), dx->scalar_type() == at::kFloat, (int)M, (int)dx->size(1), (N + 127) / 128 * 128, 0, stream());
    if (!rc && dw) rc = piccl_ops_fp8_gemm(t.v, t.s, ptr(xt.v), ptr(xt.s), nullptr, dw->data_ptr(), dw->scalar_type() == at::kFloat, (int)N, (int)dw->size(1), (M + 127) / 128 * 128, 0, stream());
    return answer(rc, 1 + (dx != nullptr) + (dw != nullptr), "fp8 linear_bwd");
  });
}

// empty(rows, cols, device): values and scales; None if they cannot be made here
PyObject* empty(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 3 || !THPDevice_Check(a[2])) Py_RETURN_NONE;
    const int64_t rows = PyLong_AsLongLong(a[0]), cols = PyLong_AsLongLong(a[1]);
    if (PyErr_Occurred()) return nullptr;
    if (rows < 0 || cols < 0) Py_RETURN_NONE;
    const auto opt = at::TensorOptions().device(reinterpret_cast<THPDevice*>(a[2])->device);
    const int64_t blocks = (cols + 127) / 128;
    PyObject* const v = THPVariable_Wrap(at::empty({rows, blocks * 128}, opt.dtype(at::kFloat8_e4m3fn)));
    PyObject* const s = v ? THPVariable_Wrap(at::empty({(rows + 127) / 128, (blocks + 3) / 4, 32, 4, 4}, opt.dtype(at::kByte))) : nullptr;
    PyObject* const t = s ? PyTuple_Pack(2, v, s) : nullptr;
    Py_XDECREF(v); Py_XDECREF(s);
    return t;
  });
}

// What stays the same from step to step of an optimiser, and the tensors whose addresses stand in its table
struct Adam {
  int device, bits8; long long blocks; void *table, *owner, *m, *v, *ms, *vs, *step, *ticket; unsigned seed;
  std::vector<at::Tensor> tensors; std::vector<const void*> places;
};
// adamw(device, table, owner, blocks, bits8, m, v, ms, vs, step, ticket, seed: all numbers, tuple of tensors) -> handle
PyObject* adamw(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    long long x[12];
    if (n != 13 || !PyTuple_Check(a[12])) { PyErr_SetString(PyExc_TypeError, "adamw: 12 numbers and a tuple"); return nullptr; }
    for (int i = 0; i < 12; i++) { x[i] = (long long)PyLong_AsUnsignedLongLongMask(a[i]); if (PyErr_Occurred()) return nullptr; }
    auto p = [&](int i) { return reinterpret_cast<void*>(x[i]); };
    std::unique_ptr<Adam> h(new Adam{(int)x[0], (int)x[4], x[3], p(1), p(2), p(5), p(6), p(7), p(8), p(9), p(10), (unsigned)x[11], {}, {}});
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[12]); i++) {
      const at::Tensor* const t = tensor(PyTuple_GET_ITEM(a[12], i));
      if (!t) { PyErr_SetString(PyExc_TypeError, "adamw: tensors wanted"); return nullptr; }
      h->tensors.push_back(*t); h->places.push_back(t->data_ptr());
    }
    PyObject* const c = PyCapsule_New(h.get(), "adamw", [](PyObject* c) { delete static_cast<Adam*>(PyCapsule_GetPointer(c, "adamw")); });
    if (c) h.release();
    return c;
  });
}
// adamw_step(handle, lr, b1, b2, eps, wd, gscale): gscale a number or a tensor; 0 if that tensor is not one fp32 value on the device, or a tensor of the table has moved
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7) return no();
    const Adam* const h = static_cast<const Adam*>(PyCapsule_GetPointer(a[0], "adamw"));
    if (!h) return nullptr;
    double x[5], g = 1.0;
    for (int i = 0; i < 5; i++) { x[i] = PyFloat_AsDouble(a[1 + i]); if (PyErr_Occurred()) return nullptr; }
    const at::Tensor* const t = tensor(a[6]);
    if (!t) { g = PyFloat_AsDouble(a[6]); if (PyErr_Occurred()) return nullptr; }
    else if (t->scalar_type() != at::kFloat || t->numel() != 1 || !t->is_cuda() || t->device().index() != h->device) return no();
    if (!(x[1] >= 0 && x[1] < 1 && x[2] >= 0 && x[2] < 1)) return no();
    for (size_t i = 0; i < h->tensors.size(); i++) if (h->tensors[i].data_ptr() != h->places[i]) return no();
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)h->device);
    return answer(piccl_ops_adamw_many(h->table, static_cast<const int*>(h->owner), h->blocks, h->bits8, h->m, h->v, h->ms, h->vs, (float)x[0], x[1], x[2], (float)x[3], (float)x[4], (float)g,
                                       t ? t->data_ptr<float>() : nullptr, static_cast<int*>(h->step), static_cast<unsigned*>(h->ticket), h->seed, stream()), 1, "adamw_many");
  });
}

#define M_(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {M_(quantize), M_(product), M_(linear), M_(linear_bwd), M_(empty), M_(adamw), M_(adamw_step), {nullptr, nullptr, 0, nullptr}};
#undef M_
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensorcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensorcall(void) { return PyModule_Create(&module); }
