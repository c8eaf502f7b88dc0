// The short way from Python to the kernels of a paged cache and of drafted tokens: a call of a few microseconds on the device took fifteen to twenty
// through checks in Python, allocations and ctypes.
//
// A function here takes what the operator of its name in ops/__init__.py takes.  Where every tensor is as the kernel wants it it launches, and returns the
// results; for anything else it returns None and has done nothing, and the way through Python checks, copies or refuses.  So what a
// call may be stands there alone, and the conditions here are what implies it.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/python_headers.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <algorithm>
#include <cmath>

namespace {

using at::Tensor;

using AppendFn = int (*)(const void*, long long, const float*, const float*, int, void*, void*, int, const int*, long long, const int*, const int*, int, int, int, int,
                         int, int, void*, void*);
using AttentionFn = int (*)(const void*, const void*, const void*, int, const int*, long long, const int*, const int*, const int*, void*, int, int, int, int, int, int,
                            float, int, int, void*, long long, void*);
using RoomFn = long long (*)(int, int, int, int, int, int, int, int);
using VerifyFn = int (*)(const void*, long long, const void*, long long, int, const long long*, const int*, const float*, int, int, int, double, double*, int*,
                         long long*, void*);

AppendFn append_fn = nullptr;
AttentionFn attention_fn = nullptr;
RoomFn room_fn = nullptr;
VerifyFn verify_fn = nullptr;

PyObject* none() { Py_RETURN_NONE; }

// A plain tensor on device `dev` that nothing is recorded for: no gradient asked, no tangent, no subclass or transform
bool plain(PyObject* o, const Tensor** out) {
  if (!THPVariable_CheckExact(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_neg() || t.is_conj()) return false;
  const auto keys = t.key_set();
  if (keys.has(c10::DispatchKey::Python) || keys.has(c10::DispatchKey::FuncTorchBatched) || keys.has(c10::DispatchKey::FuncTorchGradWrapper)) return false;
  if (t.requires_grad() && at::GradMode::is_enabled()) return false;
  if (t._fw_grad(0).defined()) return false;
  *out = &t;
  return true;
}
bool on(const Tensor& t, int dev) { return t.get_device() == dev; }
bool address(const Tensor& t, uintptr_t by) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (by - 1)) == 0; }
bool ints(const Tensor& t, int64_t n, int dev) { return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && on(t, dev) && t.is_contiguous(); }

struct Pages {
  const Tensor *k, *v, *table, *starts, *pos;
  int64_t pages, h, page, d, b, m;
  int shift;
  long long ldt;
};

// A cache, table, starts and positions on the current device
bool pages_of(PyObject* cache, PyObject* table, PyObject* starts, PyObject* pos, int dev, Pages* p) {
  if (!PyTuple_Check(cache) || PyTuple_GET_SIZE(cache) != 2) return false;
  if (!plain(PyTuple_GET_ITEM(cache, 0), &p->k) || !plain(PyTuple_GET_ITEM(cache, 1), &p->v) || !plain(table, &p->table) || !plain(starts, &p->starts) || !plain(pos, &p->pos))
    return false;
  const Tensor &k = *p->k, &v = *p->v, &t = *p->table;
  if (k.dim() != 4 || t.dim() != 2 || k.scalar_type() != at::kBFloat16 || v.scalar_type() != at::kBFloat16 || v.sizes() != k.sizes() || !k.is_contiguous() ||
      !v.is_contiguous() || !on(k, dev) || !on(v, dev) || !address(k, 32) || !address(v, 32))
    return false;
  p->pages = k.size(0), p->h = k.size(1), p->page = k.size(2), p->d = k.size(3), p->b = t.size(0), p->m = t.size(1);
  p->shift = p->page == 16 ? 4 : p->page == 32 ? 5 : p->page == 64 ? 6 : p->page == 128 ? 7 : 0;
  if (!p->shift || (p->d != 64 && p->d != 128) || p->pages < 1 || p->h < 1 || p->h > 65535 || p->pages * p->h * p->page > (1ll << 31) - 256) return false;
  if (t.scalar_type() != at::kInt || !on(t, dev) || p->b < 1 || p->b > 65534 || p->m < 1 || p->m * p->page > (1ll << 31) - 128 || t.stride(1) != 1 ||
      (p->b > 1 && t.stride(0) < p->m))
    return false;
  p->ldt = p->b > 1 ? t.stride(0) : p->m;
  return ints(*p->starts, p->b + 1, dev) && ints(*p->pos, p->b, dev);
}

template <class Fn, class... Args>
void launch(const char* name, Fn fn, Args... args) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(args...);
  Py_END_ALLOW_THREADS
  if (rc != 0) throw std::runtime_error(std::string(name) + " failed with code " + std::to_string(rc));
}

void* stream(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

// (qkv, cos, sin, cache, table, starts, pos) -> q
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  const Tensor *x, *cos, *sin;
  Pages p;
  if (n_args != 7 || !append_fn || !plain(a[0], &x) || !plain(a[1], &cos) || !plain(a[2], &sin)) return none();
  const int dev = c10::cuda::current_device();
  if (!pages_of(a[3], a[4], a[5], a[6], dev, &p)) return none();
  if (x->dim() != 2 || x->scalar_type() != at::kBFloat16 || !on(*x, dev) || x->size(1) != 3 * p.h * p.d || x->size(0) < 1 || x->size(0) >= 1 << 26 || x->stride(1) != 1 ||
      !address(*x, 16) || (x->size(0) > 1 && x->stride(0) % 8))
    return none();
  if (cos->dim() != 2 || cos->size(1) != p.d / 2 || sin->sizes() != cos->sizes() || cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat || !on(*cos, dev) ||
      !on(*sin, dev) || !cos->is_contiguous() || !sin->is_contiguous() || !address(*cos, 16) || !address(*sin, 16) || cos->size(0) > (1ll << 31) - 256)
    return none();
  const int64_t n = x->size(0);
  Tensor q = at::empty({n, p.h * p.d}, x->options().requires_grad(false));
  launch("bones_paged_append", append_fn, (const void*)x->data_ptr(), (long long)x->stride(0), (const float*)cos->data_ptr(), (const float*)sin->data_ptr(),
         (int)cos->size(0), p.k->data_ptr(), p.v->data_ptr(), (int)p.pages, (const int*)p.table->data_ptr(), p.ldt, (const int*)p.starts->data_ptr(),
         (const int*)p.pos->data_ptr(), (int)p.b, (int)n, (int)p.m, (int)p.h, (int)p.d, p.shift, q.data_ptr(), stream(dev));
  return THPVariable_Wrap(std::move(q));
  END_HANDLE_TH_ERRORS
}

// (q, cache, table, starts, pos, scale, doc_start or None, window, longest or None, few tokens, largest shift) -> y
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  const Tensor *q, *doc = nullptr;
  Pages p;
  if (n_args != 11 || !attention_fn || !plain(a[0], &q) || !PyFloat_Check(a[5]) || !PyLong_CheckExact(a[7]) || (a[8] != Py_None && !PyLong_CheckExact(a[8]))) return none();
  const int dev = c10::cuda::current_device();
  if (!pages_of(a[1], a[2], a[3], a[4], dev, &p)) return none();
  const int64_t n = q->dim() == 2 ? q->size(0) : 0;
  if (n < 1 || n >= 1 << 26 || q->scalar_type() != at::kBFloat16 || !on(*q, dev) || q->size(1) != p.h * p.d || !q->is_contiguous() || !address(*q, 32)) return none();
  if (a[6] != Py_None && (!plain(a[6], &doc) || !ints(*doc, n, dev))) return none();
  const double scale = PyFloat_AS_DOUBLE(a[5]);
  int over = 0;
  const long long window = PyLong_AsLongLongAndOverflow(a[7], &over), longest = a[8] == Py_None || over ? (n + p.b - 1) / p.b : PyLong_AsLongLongAndOverflow(a[8], &over);
  if (over || window < 0 || window % 128 || longest < 0 || !(std::abs(scale) * p.d <= PyFloat_AsDouble(a[10]))) return none();
  const int tall = longest > PyLong_AsLong(a[9]), tiles = (int)std::min(window / 128, 1ll << 24);
  const long long room = room_fn((int)p.b, (int)n, (int)(p.m * p.page), (int)p.h, (int)p.d, tiles, tall, 0);
  if (room < 1) return none();
  Tensor y = at::empty({n, p.h * p.d}, q->options().requires_grad(false)), work = at::empty({room}, q->options().dtype(at::kByte).requires_grad(false));
  launch("bones_paged_attention", attention_fn, (const void*)q->data_ptr(), (const void*)p.k->data_ptr(), (const void*)p.v->data_ptr(), (int)p.pages,
         (const int*)p.table->data_ptr(), p.ldt, (const int*)p.starts->data_ptr(), (const int*)p.pos->data_ptr(), doc ? (const int*)doc->data_ptr() : nullptr, y.data_ptr(),
         (int)p.b, (int)n, (int)p.m, (int)p.h, (int)p.d, p.shift, (float)scale, tiles, tall, work.data_ptr(), room, stream(dev));
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// (logits, ids, starts, uniforms or None, draft logits or None, temperature, vocab, coldest, warmest) -> (accepted, token)
PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  const Tensor *z, *ids, *starts, *u = nullptr, *q = nullptr;
  if (n_args != 9 || !verify_fn || !plain(a[0], &z) || !plain(a[1], &ids) || !plain(a[2], &starts) || !PyFloat_Check(a[5]) || !PyLong_CheckExact(a[6])) return none();
  const int dev = c10::cuda::current_device();
  const double t = PyFloat_AS_DOUBLE(a[5]);
  if (z->dim() != 2 || !on(*z, dev) || (z->scalar_type() != at::kBFloat16 && z->scalar_type() != at::kFloat)) return none();
  const int64_t n = z->size(0), c = z->size(1);
  int over = 0;
  const long long vocab = PyLong_AsLongLongAndOverflow(a[6], &over);
  if (n < 1 || n >= 1 << 26 || over || vocab < 1 || vocab > c || vocab > 1 << 30 || z->stride(1) != 1 || (n > 1 && z->stride(0) < c)) return none();
  if (ids->dim() != 1 || ids->size(0) != n || ids->scalar_type() != at::kLong || !on(*ids, dev) || !ids->is_contiguous()) return none();
  if (starts->dim() != 1 || starts->size(0) < 2 || starts->size(0) > 65536 || !ints(*starts, starts->size(0), dev)) return none();
  if (t != 0.0) {
    if (!(t >= PyFloat_AsDouble(a[7]) && t <= PyFloat_AsDouble(a[8])) || a[3] == Py_None || !plain(a[3], &u)) return none();
    if (u->dim() != 2 || u->size(0) != n || u->size(1) != 2 || u->scalar_type() != at::kFloat || !on(*u, dev) || !u->is_contiguous()) return none();
  }
  if (a[4] != Py_None) {
    if (!plain(a[4], &q) || q->dim() != 2 || q->size(0) != n || q->size(1) < vocab || q->scalar_type() != z->scalar_type() || !on(*q, dev) || q->stride(1) != 1 ||
        (n > 1 && q->stride(0) < q->size(1)))
      return none();
    if (t == 0.0) q = nullptr;
  }
  const int64_t b = starts->size(0) - 1;
  const auto of = [&](at::ScalarType type) { return z->options().dtype(type).requires_grad(false); };
  Tensor accepted = at::empty({b}, of(at::kInt)), token = at::empty({b}, of(at::kLong)), stats = at::empty({4 * n}, of(at::kDouble));
  launch("bones_verify", verify_fn, (const void*)z->data_ptr(), (long long)z->stride(0), q ? (const void*)q->data_ptr() : nullptr, q ? (long long)q->stride(0) : 0ll,
         (int)(z->scalar_type() == at::kFloat), (const long long*)ids->data_ptr(), (const int*)starts->data_ptr(), u ? (const float*)u->data_ptr() : nullptr, (int)b, (int)n,
         (int)vocab, t, (double*)stats.data_ptr(), (int*)accepted.data_ptr(), (long long*)token.data_ptr(), stream(dev));
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(accepted)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(token)));
  return out;
  END_HANDLE_TH_ERRORS
}

// Addresses of the library's entry points, in the order of the functions above (bones_paged_room third).
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 4) {
    PyErr_SetString(PyExc_ValueError, "four addresses");
    return nullptr;
  }
  append_fn = (AppendFn)PyLong_AsVoidPtr(a[0]);
  attention_fn = (AttentionFn)PyLong_AsVoidPtr(a[1]);
  room_fn = (RoomFn)PyLong_AsVoidPtr(a[2]);
  verify_fn = (VerifyFn)PyLong_AsVoidPtr(a[3]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// What the module was compiled for (calls_for in build.py)
PyObject* built_with(PyObject*, PyObject*) { return PyUnicode_FromString(BONES_BUILT_WITH); }

PyMethodDef methods[] = {{"paged_append", (PyCFunction)(void (*)(void))paged_append, METH_FASTCALL, nullptr},
                         {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
                         {"verify_drafts", (PyCFunction)(void (*)(void))verify_drafts, METH_FASTCALL, nullptr},
                         {"built_with", built_with, METH_NOARGS, nullptr},
                         {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "bones_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_bones_calls(void) { return PyModule_Create(&module); }
