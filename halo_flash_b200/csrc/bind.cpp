// The paged-cache and attention calls of ops.py on torch tensors, as a CPython extension: checks of the tensors, the
// current stream, the workspace, and the C ABI's entry point (include/halo_b200.h), nothing else.
//
// A decode step makes these calls for every layer with a few rows, where the host is what takes the time: unpacking the
// tensors here costs about a microsecond a call; in Python (some thirty attribute reads) and ctypes (some twenty
// arguments) it was eight.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <stdexcept>
#include <string>

#include "halo_b200.h"

namespace {

// What a refused call raises.
struct Refusal {
  PyObject* type;  // null: halo_flash_b200.HaloError
  std::string text;
};
[[noreturn]] void Refuse(PyObject* type, const char* fmt, ...) {
  char text[600];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(text, sizeof text, fmt, ap);
  va_end(ap);
  throw Refusal{type, text};
}

std::string Shape(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

const at::Tensor* Get(PyObject* o, const char* name, bool optional = false) {
  if (o == Py_None && optional) return nullptr;
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda())
    Refuse(PyExc_TypeError, "%s: expected a CUDA tensor (halo_flash_b200 has no CPU path)", name);
  return &THPVariable_Unpack(o);
}

enum Kinds { kAct, kHalf, kInt, kLong, kFloat, kAny };
bool Fits(at::ScalarType t, Kinds k) {
  switch (k) {
    case kAct: return t == at::kFloat || t == at::kHalf || t == at::kBFloat16;
    case kHalf: return t == at::kHalf || t == at::kBFloat16;
    case kInt: return t == at::kInt || t == at::kUInt32;
    case kLong: return t == at::kLong;
    case kFloat: return t == at::kFloat;
    case kAny: return true;
  }
  return false;
}
const char* Wanted(Kinds k) {
  switch (k) {
    case kAct: return "float32, float16 or bfloat16";
    case kHalf: return "float16 or bfloat16";
    case kInt: return "int32 or uint32";
    case kLong: return "int64";
    case kFloat: return "float32";
    case kAny: return "any";
  }
  return "";
}
void CheckType(const at::Tensor& t, const char* name, Kinds k) {
  if (!Fits(t.scalar_type(), k)) Refuse(PyExc_TypeError, "%s: dtype %s, expected %s", name, c10::toString(t.scalar_type()), Wanted(k));
}
void CheckSame(const at::Tensor& t, const char* name, const at::Tensor& as, const char* as_name) {
  if (t.scalar_type() != as.scalar_type())
    Refuse(PyExc_TypeError, "%s: dtype %s, expected %s's %s", name, c10::toString(t.scalar_type()), as_name, c10::toString(as.scalar_type()));
}
// `rank` axes, the last one contiguous.
void CheckRows(const at::Tensor& t, const char* name, int64_t rank) {
  if (t.dim() != rank) Refuse(PyExc_ValueError, "%s: expected %lld axes, got shape %s", name, static_cast<long long>(rank), Shape(t).c_str());
  if (t.size(rank - 1) > 1 && t.stride(rank - 1) != 1) Refuse(PyExc_ValueError, "%s: the last axis must be contiguous", name);
}
void* Address(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
// A contiguous tensor of n entries (n < 0: any number), or nothing.
const at::Tensor* Vector(PyObject* o, const char* name, Kinds k, int64_t n, bool optional = false) {
  const at::Tensor* t = Get(o, name, optional);
  if (!t) return t;
  CheckType(*t, name, k);
  if (!t->is_contiguous()) Refuse(PyExc_ValueError, "%s: tensor must be contiguous", name);
  if (n >= 0 && t->numel() != n)
    Refuse(PyExc_ValueError, "%s: expected %lld entries, got %lld", name, static_cast<long long>(n), static_cast<long long>(t->numel()));
  return t;
}
int Code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? HALO_B200_F32 : t.scalar_type() == at::kHalf ? HALO_B200_F16 : HALO_B200_BF16; }

// The C ABI counts in 32 bits.
uint32_t U32(int64_t v, const char* name) {
  if (v < 0 || v > 0xFFFFFFFFll) Refuse(PyExc_ValueError, "%s: %lld is out of range", name, static_cast<long long>(v));
  return static_cast<uint32_t>(v);
}

// The kernels run on the current device's current stream: every tensor must live there.
template <typename... Ts>
void* Stream(const Ts*... tensors) {
  const auto device = c10::cuda::current_device();
  for (const at::Tensor* t : {tensors...})
    if (t && t->get_device() != device)
      Refuse(PyExc_ValueError, "tensor on cuda:%d, but the current device is cuda:%d", static_cast<int>(t->get_device()), static_cast<int>(device));
  return c10::cuda::getCurrentCUDAStream(device).stream();
}

struct Caches {
  const at::Tensor *k, *v;
  uint32_t pages, page_size, heads, dim;
};
Caches GetCaches(PyObject* ko, PyObject* vo, Kinds kinds) {
  Caches c;
  c.k = Get(ko, "k_cache"), c.v = Get(vo, "v_cache");
  CheckType(*c.k, "k_cache", kinds);
  CheckSame(*c.v, "v_cache", *c.k, "k_cache");
  CheckRows(*c.k, "k_cache", 4);
  CheckRows(*c.v, "v_cache", 4);
  for (int i = 0; i < 4; ++i)  // the stride of an axis with one entry is never used
    if (c.k->size(i) != c.v->size(i) || (c.k->size(i) > 1 && c.k->stride(i) != c.v->stride(i)))
      Refuse(PyExc_ValueError, "k_cache and v_cache must have the same shape and strides");
  c.pages = U32(c.k->size(0), "pages"), c.page_size = U32(c.k->size(1), "page_size");
  c.heads = U32(c.k->size(2), "heads"), c.dim = U32(c.k->size(3), "head size");
  return c;
}

struct Table {
  const at::Tensor* t;
  uint32_t rows, cols;
  uint64_t stride;
};
Table GetTable(PyObject* o) {
  Table r;
  r.t = Get(o, "table");
  CheckType(*r.t, "table", kInt);
  CheckRows(*r.t, "table", 2);
  r.rows = U32(r.t->size(0), "table"), r.cols = U32(r.t->size(1), "table");
  if (r.rows > 1 && r.t->stride(0) < r.t->size(1)) Refuse(PyExc_ValueError, "table: rows overlap");
  r.stride = static_cast<uint64_t>(r.t->stride(0));
  return r;
}

unsigned long long g_calls = 0;  // of the C ABI's entry points, under the interpreter's lock

void Done(int rc, const char* err) {
  ++g_calls;
  if (rc != 0) Refuse(nullptr, "%s", err);
}

// Runs one call; whatever it throws becomes a Python exception.
template <typename F>
PyObject* Guard(Py_ssize_t got, Py_ssize_t want, F f) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    return nullptr;
  }
  try {
    f();
    Py_RETURN_NONE;
  } catch (const Refusal& r) {
    PyObject* type = r.type;
    if (!type) {
      PyObject* m = PyImport_ImportModule("halo_flash_b200._lib");
      type = m ? PyObject_GetAttrString(m, "HaloError") : nullptr;
      Py_XDECREF(m);
      if (!type) return nullptr;
      PyErr_SetString(type, r.text.c_str());
      Py_DECREF(type);
      return nullptr;
    }
    PyErr_SetString(type, r.text.c_str());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// table, past, fresh, free_pages, page_size, slot, pos, cu, kv_len, status
PyObject* PagedPlan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guard(n, 10, [&] {
    const Table table = GetTable(a[0]);
    const at::Tensor *past = Vector(a[1], "past", kInt, table.rows), *fresh = Vector(a[2], "fresh", kInt, table.rows);
    const at::Tensor *free_pages = Vector(a[3], "free_pages", kInt, -1), *slot = Vector(a[5], "slot", kLong, -1);
    const long long page = PyLong_AsLongLong(a[4]);
    if (page == -1 && PyErr_Occurred()) throw std::runtime_error("page_size");
    const at::Tensor *pos = Vector(a[6], "pos", kInt, slot->numel(), true), *cu = Vector(a[7], "cu", kInt, table.rows + 1ll, true);
    const at::Tensor *kv_len = Vector(a[8], "kv_len", kInt, table.rows, true), *status = Vector(a[9], "status", kInt, 3, true);
    char err[512];
    Done(halo_b200_paged_plan(Stream(table.t, past, fresh, free_pages, slot, pos, cu, kv_len, status), static_cast<int32_t*>(Address(table.t)),
                              table.stride, table.cols, static_cast<uint32_t*>(Address(past)), static_cast<uint32_t*>(Address(fresh)),
                              static_cast<int32_t*>(Address(free_pages)), U32(free_pages->numel(), "free_pages"), U32(page, "page_size"),
                              static_cast<int64_t*>(Address(slot)), static_cast<uint32_t*>(Address(pos)), static_cast<uint32_t*>(Address(cu)),
                              static_cast<uint32_t*>(Address(kv_len)), static_cast<uint32_t*>(Address(status)), table.rows,
                              U32(slot->numel(), "slot"), err, sizeof err),
         err);
  });
}

// k, v, k_cache, v_cache, slot
PyObject* PagedStore(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guard(n, 5, [&] {
    const Caches c = GetCaches(a[2], a[3], kAct);
    const at::Tensor *k = Get(a[0], "k"), *v = Get(a[1], "v");
    CheckType(*k, "k", kAct);
    CheckSame(*v, "v", *k, "k");
    CheckRows(*k, "k", 3);
    CheckRows(*v, "v", 3);
    if (k->sizes() != v->sizes() || k->size(1) != c.heads || k->size(2) != c.dim)
      Refuse(PyExc_ValueError, "k %s and v %s do not fit caches of %u heads of %u", Shape(*k).c_str(), Shape(*v).c_str(), c.heads, c.dim);
    const at::Tensor* slot = Vector(a[4], "slot", kLong, k->size(0));
    char err[512];
    Done(halo_b200_paged_store(Stream(k, v, c.k, c.v, slot), Address(k), k->stride(0), k->stride(1), Address(v), v->stride(0), v->stride(1), Code(*k),
                               Address(c.k), Address(c.v), Code(*c.k), c.k->stride(0), c.k->stride(1), c.k->stride(2), c.pages, c.page_size,
                               static_cast<int64_t*>(Address(slot)), c.heads, c.dim, U32(k->size(0), "tokens"), err, sizeof err),
         err);
  });
}

// What both forms of attention take.
struct Common {
  const at::Tensor *q, *out, *cu, *lse;
  at::Tensor own;  // a workspace of this call's
  const at::Tensor* workspace;
  uint32_t tokens, heads, dim;
  float scale;
  int causal;
  Common(PyObject* qo, PyObject* cuo, PyObject* outo, PyObject* scaleo, PyObject* causalo, PyObject* lseo, PyObject* wso) {
    q = Get(qo, "q"), out = Get(outo, "out");
    CheckType(*q, "q", kHalf);
    CheckSame(*out, "out", *q, "q");
    CheckRows(*q, "q", 3);
    CheckRows(*out, "out", 3);
    if (q->sizes() != out->sizes()) Refuse(PyExc_ValueError, "out %s must have the shape of q %s", Shape(*out).c_str(), Shape(*q).c_str());
    cu = Vector(cuo, "cu", kInt, -1);
    if (cu->numel() < 1) Refuse(PyExc_ValueError, "cu: expected batch + 1 entries");
    lse = Vector(lseo, "lse", kFloat, q->size(0) * q->size(1), true);
    tokens = U32(q->size(0), "tokens"), heads = U32(q->size(1), "heads"), dim = U32(q->size(2), "head size");
    workspace = Vector(wso, "workspace", kAny, -1, true);
    if (!workspace) {
      own = at::empty({static_cast<int64_t>(halo_b200_attention_workspace(dim))}, q->options().dtype(at::kByte));
      workspace = &own;
    }
    if (scaleo == Py_None) {
      scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(dim)));
    } else {
      const double s = PyFloat_AsDouble(scaleo);
      if (s == -1.0 && PyErr_Occurred()) throw std::runtime_error("scale");
      scale = static_cast<float>(s);
    }
    causal = PyObject_IsTrue(causalo);
    if (causal < 0) throw std::runtime_error("causal");
  }
};

// q, k, v, cu, out, scale, causal, lse, workspace
PyObject* AttentionPacked(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guard(n, 9, [&] {
    const Common c(a[0], a[3], a[4], a[5], a[6], a[7], a[8]);
    const at::Tensor *k = Get(a[1], "k"), *v = Get(a[2], "v");
    CheckSame(*k, "k", *c.q, "q");
    CheckSame(*v, "v", *c.q, "q");
    CheckRows(*k, "k", 3);
    CheckRows(*v, "v", 3);
    if (k->sizes() != v->sizes() || k->size(0) != c.q->size(0) || k->size(2) != c.q->size(2))
      Refuse(PyExc_ValueError, "k %s and v %s do not fit q %s", Shape(*k).c_str(), Shape(*v).c_str(), Shape(*c.q).c_str());
    char err[512];
    Done(halo_b200_attention_packed(Stream(c.q, k, v, c.cu, c.out, c.lse, c.workspace), Address(c.q), c.q->stride(0), c.q->stride(1), Address(k),
                                    k->stride(0), k->stride(1), Address(v), v->stride(0), v->stride(1), Address(c.out), c.out->stride(0),
                                    c.out->stride(1), Code(*c.q), static_cast<uint32_t*>(Address(c.cu)), U32(c.cu->numel() - 1, "cu"), c.tokens,
                                    c.heads, U32(k->size(1), "heads"), c.dim, c.scale, c.causal, static_cast<float*>(Address(c.lse)),
                                    Address(c.workspace), c.workspace->nbytes(), err, sizeof err),
         err);
  });
}

// q, k_cache, v_cache, table, kv_len, cu, out, scale, causal, lse, workspace
PyObject* AttentionPaged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return Guard(n, 11, [&] {
    const Common c(a[0], a[5], a[6], a[7], a[8], a[9], a[10]);
    const Caches cache = GetCaches(a[1], a[2], kHalf);
    CheckSame(*cache.k, "k_cache", *c.q, "q");
    const Table table = GetTable(a[3]);
    const int64_t batch = c.cu->numel() - 1;
    const at::Tensor* kv_len = Vector(a[4], "kv_len", kInt, batch);
    if (c.dim != cache.dim || table.rows != batch)
      Refuse(PyExc_ValueError, "q %s, table %s and cu do not fit caches %s", Shape(*c.q).c_str(), Shape(*table.t).c_str(), Shape(*cache.k).c_str());
    char err[512];
    Done(halo_b200_attention_paged(Stream(c.q, cache.k, cache.v, table.t, kv_len, c.cu, c.out, c.lse, c.workspace), Address(c.q), c.q->stride(0),
                                   c.q->stride(1), Address(cache.k), Address(cache.v), cache.k->stride(0), cache.k->stride(1), cache.k->stride(2),
                                   cache.pages, cache.page_size, static_cast<int32_t*>(Address(table.t)), table.stride, table.cols,
                                   static_cast<uint32_t*>(Address(kv_len)), Address(c.out), c.out->stride(0), c.out->stride(1), Code(*c.q),
                                   static_cast<uint32_t*>(Address(c.cu)), static_cast<uint32_t>(batch), c.tokens, c.heads, cache.heads, c.dim,
                                   c.scale, c.causal, static_cast<float*>(Address(c.lse)), Address(c.workspace), c.workspace->nbytes(), err,
                                   sizeof err),
         err);
  });
}

PyObject* Calls(PyObject*, PyObject*) { return PyLong_FromUnsignedLongLong(g_calls); }

#define HALO_METHOD(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {HALO_METHOD("paged_plan", PagedPlan), HALO_METHOD("paged_store", PagedStore), HALO_METHOD("attention_packed", AttentionPacked),
                          HALO_METHOD("attention_paged", AttentionPaged), {"calls", Calls, METH_NOARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_bind", "The paged-cache and attention calls on torch tensors; see ops.py.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&kModule); }
