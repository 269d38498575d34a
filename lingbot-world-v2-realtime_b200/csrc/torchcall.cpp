// Calls of the paged-cache and rotary entries straight from torch tensors (CPython fastcall functions, module
// lingbot_b200._torchcall): the usual form of each call, checked, its outputs and workspace allocated and launched in one
// step. What the host spends on a call is what a small launch costs a caller who does not replay a graph: through Python
// and ctypes 19 us (rotary, two tensors) to 25 us (attention), of which the launches are 3 to 6.
//
// A function returns None for any call that is not of the usual form (other devices, types, layouts, gradients, wrong
// shapes): the Python caller then takes its own path, which handles or refuses it. So nothing here reports an argument
// error; an entry's status code other than 0 is raised as LbqError by the caller, to whom it is returned as an int.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <Python.h>
#include <cstdint>
#include <vector>

#include "../../include/lbq.h"

namespace {

// The entries, from whichever build of the library the package has loaded.
decltype(&lbq_rope) f_rope = nullptr;
decltype(&lbq_page_write) f_write = nullptr;
decltype(&lbq_page_read) f_read = nullptr;
decltype(&lbq_page_copy) f_copy = nullptr;
decltype(&lbq_paged_attn) f_attn = nullptr;
decltype(&lbq_paged_attn_splits) f_splits = nullptr;
decltype(&lbq_paged_attn_workspace) f_workspace = nullptr;

PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "init takes the addresses of 7 entries");
    return nullptr;
  }
  void* p[7];
  for (int i = 0; i < 7; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  f_rope = reinterpret_cast<decltype(f_rope)>(p[0]);
  f_write = reinterpret_cast<decltype(f_write)>(p[1]);
  f_read = reinterpret_cast<decltype(f_read)>(p[2]);
  f_attn = reinterpret_cast<decltype(f_attn)>(p[3]);
  f_splits = reinterpret_cast<decltype(f_splits)>(p[4]);
  f_workspace = reinterpret_cast<decltype(f_workspace)>(p[5]);
  f_copy = reinterpret_cast<decltype(f_copy)>(p[6]);
  Py_RETURN_NONE;
}

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
int64_t integer(PyObject* o, int i) { return PyLong_AsLongLong(PyTuple_GET_ITEM(o, i)); }
void* address(PyObject* o, int i) { return PyLong_AsVoidPtr(PyTuple_GET_ITEM(o, i)); }

constexpr int64_t kMostSize = int64_t(1) << 28;                          // of any dimension: the entries take 32-bit sizes

int dtype_code(const at::Tensor& t) {
  const auto d = t.scalar_type();
  return d == at::kBFloat16 ? 0 : d == at::kHalf ? 1 : d == at::kFloat ? 2 : -1;
}
// [B, L, heads, dim] with unit channel stride on CUDA device `dev`, no gradient wanted (nor a forward-mode tangent carried).
bool rows(const at::Tensor& t, int dev) {
  return t.dim() == 4 && t.stride(3) == 1 && t.is_cuda() && t.get_device() == dev && t.numel() > 0 &&
         t.size(0) <= kMostSize && t.size(1) <= kMostSize && t.size(2) <= kMostSize &&
         !(t.requires_grad() && c10::GradMode::is_enabled()) && !t._fw_grad(0).defined() && t.layout() == at::kStrided;
}
bool ints(const at::Tensor& t, int dev, int64_t n) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_cuda() && t.get_device() == dev &&
         (n <= 1 || t.stride(0) == 1);
}
bool table_ok(const at::Tensor& t, int dev, int64_t batch) {
  return t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == batch && t.size(1) > 0 &&
         t.size(1) <= kMostSize && t.is_cuda() && t.get_device() == dev && (t.stride(1) == 1 || t.size(1) == 1);
}
// A Python int that is not negative and below 2^62 (a count of tokens can be added to it).
bool whole(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) PyErr_Clear();
  return *v >= 0 && *v < (int64_t(1) << 62);
}
// A count of every sequence: int32 [batch] tensor or a non-negative int.
bool count(PyObject* o, int dev, int64_t batch, const int32_t** p, int64_t* v) {
  *p = nullptr;
  *v = 0;
  if (const at::Tensor* t = tensor(o)) {
    if (!ints(*t, dev, batch)) return false;
    *p = t->const_data_ptr<int32_t>();
    return true;
  }
  return whole(o, v);
}
struct Positions {
  const void* p = nullptr;
  int wide = 0;
  int64_t sb = 0, sl = 0;
};
bool positions(PyObject* o, int dev, int64_t b, int64_t l, Positions* out) {
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (t == nullptr || t->dim() != 2 || t->size(0) != b || t->size(1) != l || !t->is_cuda() || t->get_device() != dev)
    return false;
  if (t->scalar_type() != at::kInt && t->scalar_type() != at::kLong) return false;
  *out = Positions{t->const_data_ptr(), t->scalar_type() == at::kLong, t->stride(0), t->stride(1)};
  return true;
}
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

// rope_table(cos, sin, interleaved): (rotated channels, device, table args)
PyObject* rope_table(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* c = n == 3 ? tensor(args[0]) : nullptr;
  const at::Tensor* s = n == 3 ? tensor(args[1]) : nullptr;
  if (!c || !s || c->scalar_type() != at::kFloat || s->scalar_type() != at::kFloat || !c->is_cuda() ||
      c->device() != s->device() || c->dim() != 2 || c->sizes() != s->sizes() || c->strides() != s->strides() ||
      c->stride(1) != 1)
    Py_RETURN_NONE;
  const int inter = PyObject_IsTrue(args[2]);
  if (inter < 0) return nullptr;
  const long long rot = 2 * c->size(1);
  return Py_BuildValue("(Li(LLLLLi))", rot, int(c->get_device()), reinterpret_cast<long long>(c->const_data_ptr()),
                       reinterpret_cast<long long>(s->const_data_ptr()), static_cast<long long>(c->stride(0)),
                       static_cast<long long>(c->size(0)), rot, inter);
  END_HANDLE_TH_ERRORS
}

// rope(x, k or None, table args, table device, positions or None, start, inverse)
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* x = n == 7 ? tensor(args[0]) : nullptr;
  const at::Tensor* k = n == 7 && args[1] != Py_None ? tensor(args[1]) : nullptr;
  if (x == nullptr || (args[1] != Py_None && k == nullptr)) Py_RETURN_NONE;
  const int dev = static_cast<int>(PyLong_AsLong(args[3]));
  const int dt = dtype_code(*x);
  if (dt < 0 || dev != c10::cuda::current_device() || !rows(*x, dev)) Py_RETURN_NONE;
  const int64_t b = x->size(0), l = x->size(1);
  if (k != nullptr && (!rows(*k, dev) || k->scalar_type() != x->scalar_type() || k->size(0) != b || k->size(1) != l ||
                       k->size(3) != x->size(3)))
    Py_RETURN_NONE;
  Positions pos;
  int64_t start;
  if (!positions(args[4], dev, b, l, &pos) || !whole(args[5], &start)) Py_RETURN_NONE;
  const int inverse = PyObject_IsTrue(args[6]);
  if (inverse < 0) return nullptr;
  PyObject* r = args[2];
  at::Tensor y = at::empty_like(*x), z;
  if (k != nullptr) z = at::empty_like(*k);
  const int rc = f_rope(
      x->const_data_ptr(), x->stride(0), x->stride(1), x->stride(2), y.mutable_data_ptr(), y.stride(0), y.stride(1),
      y.stride(2), int(x->size(2)), k ? k->const_data_ptr() : nullptr, k ? k->stride(0) : 0, k ? k->stride(1) : 0,
      k ? k->stride(2) : 0, k ? z.mutable_data_ptr() : nullptr, k ? z.stride(0) : 0, k ? z.stride(1) : 0,
      k ? z.stride(2) : 0, k ? int(k->size(2)) : 0, int(b), int(l), int(x->size(3)),
      static_cast<const float*>(address(r, 0)), static_cast<const float*>(address(r, 1)), integer(r, 2), integer(r, 3),
      int(integer(r, 4)), int(integer(r, 5)), pos.p, pos.wide, pos.sb, pos.sl, start, inverse, dt, stream_of(dev));
  if (rc != 0) return PyLong_FromLong(rc);
  if (k == nullptr) return THPVariable_Wrap(std::move(y));
  PyObject* both = PyTuple_New(2);
  if (both == nullptr) return nullptr;
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(y)));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(z)));
  return both;
  END_HANDLE_TH_ERRORS
}

// The pool's arguments: (k_pages, k_amax, v_pages, v_amax, num_pages, heads, fmt).
struct Pool {
  void *k, *v;
  float *ka, *va;
  int64_t pages;
  int heads, fmt;
  explicit Pool(PyObject* o)
      : k(address(o, 0)), v(address(o, 2)), ka(static_cast<float*>(address(o, 1))), va(static_cast<float*>(address(o, 3))),
        pages(integer(o, 4)), heads(int(integer(o, 5))), fmt(int(integer(o, 6))) {}
};

// pool(k, v, k_amax, v_amax): (device, heads, pool args or None where it has layers, page_copy's args)
PyObject* pool(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) Py_RETURN_NONE;
  const at::Tensor *k = tensor(args[0]), *v = tensor(args[1]), *ka = tensor(args[2]), *va = tensor(args[3]);
  if (!k || !v || !ka || !va || !k->is_cuda()) Py_RETURN_NONE;
  const auto type = k->scalar_type();
  const int64_t d = k->dim();
  if ((type != at::kChar && type != at::kFloat8_e4m3fn) || v->scalar_type() != type || ka->scalar_type() != at::kFloat ||
      va->scalar_type() != at::kFloat || (d != 4 && d != 5) || k->size(d - 2) != 64 || k->size(d - 1) != 128 ||
      v->sizes() != k->sizes() || ka->sizes() != k->sizes().slice(0, d - 2) || va->sizes() != ka->sizes() ||
      !k->is_contiguous() || !v->is_contiguous() || !ka->is_contiguous() || !va->is_contiguous() ||
      v->device() != k->device() || ka->device() != k->device() || va->device() != k->device())
    Py_RETURN_NONE;
  const long long pages = k->size(d - 4), heads = k->size(d - 3), layers = d == 5 ? k->size(0) : 1;
  const auto kp = reinterpret_cast<long long>(k->const_data_ptr()), vp = reinterpret_cast<long long>(v->const_data_ptr());
  const auto kap = reinterpret_cast<long long>(ka->const_data_ptr()), vap = reinterpret_cast<long long>(va->const_data_ptr());
  const long long fmt = type == at::kChar ? 0 : 1;
  PyObject* one = d == 5 ? Py_NewRef(Py_None) : Py_BuildValue("(LLLLLLL)", kp, kap, vp, vap, pages, heads, fmt);
  if (one == nullptr) return nullptr;
  return Py_BuildValue("(iLN(LLLLLLLLL))", int(k->get_device()), heads, one, kp, kap, vp, vap, pages, heads, layers,
                       pages * heads * 64 * 128, pages * heads);
  END_HANDLE_TH_ERRORS
}

// page_write(pool, device, table, start, k, v, lens or None, rope args or None, positions or None): 0
PyObject* page_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !PyTuple_CheckExact(args[0])) Py_RETURN_NONE;
  const Pool pool(args[0]);
  const int dev = static_cast<int>(PyLong_AsLong(args[1]));
  const at::Tensor *table = tensor(args[2]), *k = tensor(args[4]), *v = tensor(args[5]);
  if (dev != c10::cuda::current_device() || !table || !k || !v || !rows(*k, dev) || !rows(*v, dev)) Py_RETURN_NONE;
  const int dt = dtype_code(*k);
  const int64_t b = k->size(0), l = k->size(1);
  if (dt < 0 || dt > 1 || v->scalar_type() != k->scalar_type() || k->sizes() != v->sizes() || k->size(2) != pool.heads ||
      k->size(3) != 128 || !table_ok(*table, dev, b))
    Py_RETURN_NONE;
  const int32_t *start, *lens = nullptr;
  int64_t start0, ignored;
  if (!count(args[3], dev, b, &start, &start0)) Py_RETURN_NONE;
  if (args[6] != Py_None && (!count(args[6], dev, b, &lens, &ignored) || lens == nullptr)) Py_RETURN_NONE;
  Positions pos;
  PyObject* r = args[7];
  const bool turn = r != Py_None;
  if (!turn && args[8] != Py_None) Py_RETURN_NONE;
  if (!positions(args[8], dev, b, l, &pos)) Py_RETURN_NONE;
  const int rc = f_write(k->const_data_ptr(), k->stride(0), k->stride(1), k->stride(2), v->const_data_ptr(), v->stride(0),
                         v->stride(1), v->stride(2), pool.k, pool.ka, pool.v, pool.va, pool.pages, pool.heads, pool.fmt,
                         table->const_data_ptr<int32_t>(), table->stride(0), int(table->size(1)), start, start0, lens,
                         int(b), int(l), turn ? static_cast<const float*>(address(r, 0)) : nullptr,
                         turn ? static_cast<const float*>(address(r, 1)) : nullptr, turn ? integer(r, 2) : 0,
                         turn ? integer(r, 3) : 0, turn ? int(integer(r, 4)) : 0, turn ? int(integer(r, 5)) : 0, pos.p,
                         pos.wide, pos.sb, pos.sl, dt, stream_of(dev));
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// page_read(pool, device, table, start, length, dtype code, lens or None): (k, v)
PyObject* page_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t length;
  if (n != 7 || !PyTuple_CheckExact(args[0]) || !whole(args[4], &length)) Py_RETURN_NONE;
  const Pool pool(args[0]);
  const int dev = static_cast<int>(PyLong_AsLong(args[1]));
  const at::Tensor* table = tensor(args[2]);
  if (dev != c10::cuda::current_device() || !table || table->dim() != 2) Py_RETURN_NONE;
  const int64_t b = table->size(0);
  const int dt = static_cast<int>(PyLong_AsLong(args[5]));
  if (b <= 0 || length <= 0 || length > kMostSize || b > kMostSize || !table_ok(*table, dev, b)) Py_RETURN_NONE;
  const int32_t *start, *lens = nullptr;
  int64_t start0, ignored;
  if (!count(args[3], dev, b, &start, &start0)) Py_RETURN_NONE;
  if (args[6] != Py_None && (!count(args[6], dev, b, &lens, &ignored) || lens == nullptr)) Py_RETURN_NONE;
  const auto opt = table->options().dtype(dt ? at::kHalf : at::kBFloat16);
  at::Tensor k = at::empty({b, length, pool.heads, 128}, opt), v = at::empty_like(k);
  const int rc = f_read(pool.k, pool.ka, pool.v, pool.va, pool.pages, pool.heads, pool.fmt, table->const_data_ptr<int32_t>(),
                        table->stride(0), int(table->size(1)), start, start0, lens, int(b), int(length),
                        k.mutable_data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.mutable_data_ptr(), v.stride(0),
                        v.stride(1), v.stride(2), dt, stream_of(dev));
  if (rc != 0) return PyLong_FromLong(rc);
  PyObject* both = PyTuple_New(2);
  if (both == nullptr) return nullptr;
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(v)));
  return both;
  END_HANDLE_TH_ERRORS
}

// paged_attn(pool, device, q, table, kv_lens, q_lens or None, causal, sm_scale, ragged or None): out
PyObject* paged_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !PyTuple_CheckExact(args[0])) Py_RETURN_NONE;
  const Pool pool(args[0]);
  const int dev = static_cast<int>(PyLong_AsLong(args[1]));
  const at::Tensor *q = tensor(args[2]), *table = tensor(args[3]);
  if (dev != c10::cuda::current_device() || !q || !table || !rows(*q, dev)) Py_RETURN_NONE;
  const int dt = dtype_code(*q);
  const int64_t b = q->size(0), lq = q->size(1), hq = q->size(2);
  if (dt < 0 || dt > 1 || q->size(3) != 128 || hq % pool.heads || !table_ok(*table, dev, b) || hq > (1 << 24))
    Py_RETURN_NONE;
  const int32_t *kv, *ql = nullptr;
  int64_t kv0, ignored;
  if (!count(args[4], dev, b, &kv, &kv0)) Py_RETURN_NONE;
  if (args[5] != Py_None && (!count(args[5], dev, b, &ql, &ignored) || ql == nullptr)) Py_RETURN_NONE;
  const int causal = PyObject_IsTrue(args[6]);
  if (causal < 0) return nullptr;
  const double scale = PyFloat_AsDouble(args[7]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  const int group = int(hq / pool.heads);
  const int64_t longest = kv ? table->size(1) * 64 : kv0;
  const int ragged = args[8] == Py_None ? kv != nullptr : PyObject_IsTrue(args[8]);
  if (ragged < 0) return nullptr;
  const int splits = f_splits(int(b), int(lq), pool.heads, group, longest, b > 1 && ragged);
  at::Tensor out = at::empty_like(*q), ws;
  const size_t need = f_workspace(int(b), int(lq), pool.heads, group, splits);
  if (need > 0) ws = at::empty({static_cast<int64_t>(need)}, q->options().dtype(at::kByte));
  const int rc = f_attn(q->const_data_ptr(), q->stride(0), q->stride(1), q->stride(2), pool.k, pool.ka, pool.v, pool.va,
                        pool.pages, pool.heads, pool.fmt, table->const_data_ptr<int32_t>(), table->stride(0),
                        int(table->size(1)), kv, kv0, ql, int(b), int(lq), group, causal, float(scale),
                        out.mutable_data_ptr(), out.stride(0), out.stride(1), out.stride(2), nullptr, splits,
                        need ? ws.mutable_data_ptr() : nullptr, need, dt, stream_of(dev));
  if (rc != 0) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// page_copy(pool with layers: (k, k_amax, v, v_amax, pages, heads, layers, bytes and floats of a layer), device, src, dst): 0
PyObject* page_copy(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !PyList_CheckExact(args[2]) || !PyList_CheckExact(args[3])) Py_RETURN_NONE;
  PyObject* o = args[0];
  const int dev = static_cast<int>(PyLong_AsLong(args[1]));
  const Py_ssize_t m = PyList_GET_SIZE(args[2]);
  const int64_t pages = integer(o, 4);
  if (dev != c10::cuda::current_device() || PyList_GET_SIZE(args[3]) != m || m == 0 || m > pages) Py_RETURN_NONE;
  std::vector<int32_t> ids(2 * m);
  std::vector<uint8_t> role(static_cast<size_t>(pages), 0);              // 1: read, 2: written
  for (Py_ssize_t i = 0; i < 2 * m; ++i) {
    PyObject* v = PyList_GET_ITEM(args[i < m ? 2 : 3], i < m ? i : i - m);
    if (!PyLong_CheckExact(v)) Py_RETURN_NONE;
    const long long id = PyLong_AsLongLong(v);
    if (id == -1 && PyErr_Occurred()) PyErr_Clear();
    if (id < 0 || id >= pages) Py_RETURN_NONE;
    uint8_t& r = role[static_cast<size_t>(id)];
    if (i < m ? false : r != 0) Py_RETURN_NONE;                          // written twice, or read as well
    r = i < m ? 1 : 2;
    ids[i] = static_cast<int32_t>(id);
  }
  const int rc = f_copy(address(o, 0), static_cast<float*>(address(o, 1)), address(o, 2), static_cast<float*>(address(o, 3)),
                        pages, int(integer(o, 5)), int(integer(o, 6)), integer(o, 7), integer(o, 8), ids.data(),
                        ids.data() + m, int(m), stream_of(dev));
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(init),      FAST(pool),      FAST(rope_table), FAST(rope),
                         FAST(page_write), FAST(page_read), FAST(page_copy),  FAST(paged_attn),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torchcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torchcall(void) { return PyModule_Create(&module); }
