// The short way from Python to the key/value cache's entry points (include/uwc.h): a decode step's calls take
// 5 to 10 us on the GPU, and checking some ten tensors, allocating and converting 28 arguments in Python took 12 to 16.
// Each function here takes the arguments of its namesake in uwc_amd/kv.py, checks that they are of the usual
// form (dense, aligned, of the right types on one GPU), allocates and calls. For anything else it returns None and has
// done nothing: kv.py then looks at the arguments itself, and copies, converts or refuses. A call that the
// library refuses or fails to launch returns its status.
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>

#include "uwc.h"

namespace {

decltype(&uwc_kv_append) lib_append;
decltype(&uwc_kv_attend_scratch_bytes) lib_bytes;
decltype(&uwc_kv_attend) lib_attend;
decltype(&uwc_kv_read) lib_read;

// One call's tensors: `ok` turns false with the first that is not of the usual form.
struct Look {
  bool ok = true;
  c10::Device dev = c10::Device(c10::kCPU);
  const at::Tensor* get(PyObject* o) {
    if (!THPVariable_Check(o)) {
      ok = false;
      return nullptr;
    }
    return &THPVariable_Unpack(o);
  }
  const at::Tensor* any(PyObject* o, at::ScalarType type, int dims) {
    const at::Tensor* t = ok ? get(o) : nullptr;
    if (t && (t->scalar_type() != type || t->dim() != dims || t->device() != dev)) ok = false;
    return ok ? t : nullptr;
  }
  const at::Tensor* dense(PyObject* o, at::ScalarType type, int dims) {
    const at::Tensor* t = any(o, type, dims);
    if (t && !t->is_contiguous()) ok = false;
    return ok ? t : nullptr;
  }
  const at::Tensor* ints(PyObject* o, int64_t n) {
    const at::Tensor* t = dense(o, at::kInt, 1);
    if (t && t->size(0) != n) ok = false;
    return ok ? t : nullptr;
  }
  const at::Tensor* table(PyObject* o) {
    const at::Tensor* t = any(o, at::kInt, 2);
    if (t && (t->stride(1) != 1 || t->stride(0) < 0)) ok = false;
    return ok ? t : nullptr;
  }
  // 16-bit rows, dense and aligned
  const at::Tensor* rows16(PyObject* o, int dims, int* dtype) {
    const at::Tensor* t = ok ? get(o) : nullptr;
    if (!t) return nullptr;
    *dtype = t->scalar_type() == at::kBFloat16 ? UWC_KV_BF16 : UWC_KV_FP16;
    ok = (t->scalar_type() == at::kBFloat16 || t->scalar_type() == at::kHalf) && t->dim() == dims && t->device() == dev;
    ok = ok && t->stride(dims - 1) == 1 && (dims == 2 || t->stride(1) == t->size(2)) && t->stride(0) >= 0 && t->stride(0) % 8 == 0 &&
         ((uintptr_t)t->const_data_ptr() & 15) == 0;
    return ok ? t : nullptr;
  }
};

struct Cache {
  int8_t *k, *v;
  float *ks, *vs;
  int64_t pages;
  int page, Hkv, hd;
};

bool cache_of(Look& L, PyObject* const* a, Cache& c) {
  const at::Tensor* k = L.get(a[0]);
  if (!k || !k->is_cuda()) return L.ok = false;
  L.dev = k->device();
  k = L.dense(a[0], at::kChar, 4);
  const at::Tensor *v = L.dense(a[1], at::kChar, 4), *ks = L.dense(a[2], at::kFloat, 2), *vs = L.dense(a[3], at::kFloat, 2);
  if (!L.ok) return false;
  const int64_t n = k->size(0), H = k->size(1), P = k->size(2), D = k->size(3);
  if (v->size(0) != n || v->size(1) != H || v->size(2) != D || v->size(3) != P || ks->size(0) != n || ks->size(1) != H ||
      vs->size(0) != n || vs->size(1) != H || n < 1 || H < 1 || H > 65535 || P < 1 || P > 128 || D < 1 || D > 128)
    return L.ok = false;
  c = Cache{k->data_ptr<int8_t>(), v->data_ptr<int8_t>(), ks->data_ptr<float>(), vs->data_ptr<float>(), n, (int)P, (int)H, (int)D};
  return true;
}

const int* int_ptr(const at::Tensor* t) { return t ? t->const_data_ptr<int>() : nullptr; }
const float* float_ptr(const at::Tensor* t) { return t ? t->const_data_ptr<float>() : nullptr; }

PyObject* none() { Py_RETURN_NONE; }
hipStream_t stream_of(PyObject* o) { return static_cast<hipStream_t>(PyLong_AsVoidPtr(o)); }
constexpr int64_t I32MAX = 0x7fffffff;

// append(k, v, ks, vs, qkv, table, ctx, cos, sin, cu, q_norm, k_norm, eps, stream)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Look L;
  Cache c;
  if (n != 14 || !lib_append || !cache_of(L, a, c)) return none();
  int dtype = 0;
  const at::Tensor *qkv = L.rows16(a[4], 2, &dtype), *table = L.table(a[5]);
  if (!L.ok) return none();
  const int64_t T = qkv->size(0), wide = qkv->size(1), B = table->size(0), width = table->size(1);
  const int64_t H = c.hd ? wide / c.hd - 2 * c.Hkv : -1;
  const at::Tensor* ctx = L.ints(a[6], B);
  const at::Tensor *cos = L.dense(a[7], at::kFloat, 2), *sin = L.dense(a[8], at::kFloat, 2);
  const at::Tensor* cu = a[9] == Py_None ? nullptr : L.ints(a[9], B + 1);
  const at::Tensor* qn = a[10] == Py_None ? nullptr : L.dense(a[10], at::kFloat, 1);
  const at::Tensor* kn = a[11] == Py_None ? nullptr : L.dense(a[11], at::kFloat, 1);
  if (!L.ok || H < 0 || wide % c.hd || T > I32MAX || width > I32MAX || (!cu && T != B) || cos->size(1) != c.hd || sin->size(1) != c.hd ||
      cos->size(0) != sin->size(0) || cos->size(0) > I32MAX || (qn && qn->size(0) != c.hd) || (kn && kn->size(0) != c.hd))
    return none();
  const double eps = PyFloat_AsDouble(a[12]);
  const hipStream_t stream = stream_of(a[13]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor q = at::empty({T, H, c.hd}, qkv->options());
  const int st = lib_append(qkv->const_data_ptr(), qkv->stride(0), dtype, (int)T, (int)B, int_ptr(cu), int_ptr(ctx), int_ptr(table),
                               table->stride(0), (int)width, float_ptr(cos), float_ptr(sin), (int)cos->size(0), float_ptr(qn),
                               float_ptr(kn), (float)eps, (int)H, c.Hkv, c.hd, c.page, c.pages, c.k, c.v, c.ks, c.vs,
                               q.data_ptr(), stream);
  return st ? PyLong_FromLong(st) : THPVariable_Wrap(std::move(q));
}

// attend(k, v, ks, vs, q, table, lens, cu, max_new, max_len, window, sinks, scale, stream); max_new, max_len, scale or None
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Look L;
  Cache c;
  if (n != 14 || !lib_attend || !cache_of(L, a, c)) return none();
  int dtype = 0;
  const at::Tensor *q = L.rows16(a[4], 3, &dtype), *table = L.table(a[5]);
  if (!L.ok) return none();
  const int64_t T = q->size(0), H = q->size(1), B = table->size(0), width = table->size(1);
  const at::Tensor *lens = L.ints(a[6], B), *cu = a[7] == Py_None ? nullptr : L.ints(a[7], B + 1);
  for (int i = 8; i < 12; i++)
    if (!PyLong_Check(a[i]) && (i > 9 || a[i] != Py_None)) return none();
  if (!L.ok || q->size(2) != c.hd || H < 1 || H % c.Hkv || T > I32MAX || H > I32MAX || width > I32MAX || (!cu && T != B)) return none();
  const int64_t most = cu ? T : 1;
  const long long window = PyLong_AsLongLong(a[10]), sinks = PyLong_AsLongLong(a[11]);
  long long max_new = a[8] == Py_None ? most : PyLong_AsLongLong(a[8]), max_len = a[9] == Py_None ? width * c.page : PyLong_AsLongLong(a[9]);
  const double scale = a[12] == Py_None ? 1.0 / std::sqrt((double)c.hd) : PyFloat_AsDouble(a[12]);
  const hipStream_t stream = stream_of(a[13]);
  if (PyErr_Occurred()) return nullptr;
  if (window < 0 || window > I32MAX || sinks < 0 || sinks > I32MAX || (sinks && !window)) return none();
  max_new = std::max(1ll, std::min<long long>(max_new, most));
  max_len = std::max(1ll, std::min<long long>(max_len, I32MAX));
  at::Tensor o = at::empty({T, H, c.hd}, q->options()), scratch;
  const uint64_t need =
      lib_bytes((int)T, (int)B, cu != nullptr, (int)H, c.Hkv, c.hd, (int)max_new, (int)max_len, (int)window, (int)sinks);
  if (need) scratch = at::empty({(int64_t)need}, q->options().dtype(at::kByte));
  const int st = lib_attend(c.k, c.v, c.ks, c.vs, c.pages, c.page, c.Hkv, c.hd, q->const_data_ptr(), q->stride(0), dtype, (int)T,
                               (int)H, int_ptr(table), table->stride(0), (int)width, int_ptr(lens), int_ptr(cu), (int)B, (int)max_new,
                               (int)max_len, (int)window, (int)sinks, (float)scale, need ? scratch.data_ptr() : nullptr, need,
                               o.data_ptr(), stream);
  return st ? PyLong_FromLong(st) : THPVariable_Wrap(std::move(o));
}

// read(k, v, ks, vs, table, start, cu, rows, is_fp16, stream)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Look L;
  Cache c;
  if (n != 10 || !lib_read || !cache_of(L, a, c) || !PyLong_Check(a[7])) return none();
  const at::Tensor* table = L.table(a[4]);
  if (!L.ok) return none();
  const int64_t B = table->size(0), width = table->size(1), rows = PyLong_AsLongLong(a[7]);
  const at::Tensor *start = L.ints(a[5], B), *cu = L.ints(a[6], B + 1);
  const int half = PyObject_IsTrue(a[8]);
  const hipStream_t stream = stream_of(a[9]);
  if (PyErr_Occurred()) return nullptr;
  if (!L.ok || rows < 0 || rows > I32MAX || width > I32MAX) return none();
  const auto opt = at::TensorOptions().dtype(half ? at::kHalf : at::kBFloat16).device(L.dev);
  at::Tensor ko = at::empty({rows, c.Hkv, c.hd}, opt), vo = at::empty({rows, c.Hkv, c.hd}, opt);
  const int st = lib_read(c.k, c.v, c.ks, c.vs, c.pages, c.page, c.Hkv, c.hd, int_ptr(table), table->stride(0), (int)width,
                             int_ptr(start), int_ptr(cu), (int)B, (int)rows, half ? UWC_KV_FP16 : UWC_KV_BF16, ko.data_ptr(),
                             vo.data_ptr(), stream);
  if (st) return PyLong_FromLong(st);
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(ko)), THPVariable_Wrap(std::move(vo)));
}

// No C++ exception leaves a call: torch's own translation makes Python errors of them.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return F(self, a, n);
  END_HANDLE_TH_ERRORS
}

// bind(append, attend_scratch_bytes, attend, read): the addresses of the loaded library's entry points
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[4];
  if (n != 4) return PyErr_SetString(PyExc_TypeError, "bind: four addresses"), nullptr;
  for (int i = 0; i < 4; i++) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  lib_append = reinterpret_cast<decltype(lib_append)>(p[0]);
  lib_bytes = reinterpret_cast<decltype(lib_bytes)>(p[1]);
  lib_attend = reinterpret_cast<decltype(lib_attend)>(p[2]);
  lib_read = reinterpret_cast<decltype(lib_read)>(p[3]);
  return none();
}

PyObject* header_sha(PyObject*, PyObject*) { return PyUnicode_FromString(UWC_HEADER_SHA); }

#define KV_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<f>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {KV_METHOD(append), KV_METHOD(attend), KV_METHOD(read), KV_METHOD(bind),
                         {"header_sha", header_sha, METH_NOARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv(void) { return PyModule_Create(&module); }
