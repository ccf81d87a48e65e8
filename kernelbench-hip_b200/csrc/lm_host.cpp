// lm_host.cpp — the host side of kbb200.lm's calls: checks of their arguments,
// outputs and scratch from torch's caching allocator, and the call of the C
// ABI on torch's current stream, without Python in between.
//
// Decoding makes these calls once per layer and token, and most of its kernels
// take a few microseconds: the same checks, allocations and ctypes marshalling
// in Python took 12-20 us a call, here 4-8.  Every function returns None where
// an argument is not plainly right (another type, size, layout or device than
// the one the kernels take); kbb200/lm.py then goes through its checks one by
// one, says what is wrong, or makes the call itself.  A call of the C ABI is
// made once: where it answers an error, that is raised from here, since an
// operation in several launches may have changed the cache's state before it.
//
// The C ABI is reached through the addresses that init() is given, so this
// module works with whichever libkbb200.so kbb200._lib has loaded.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/kbb200.h"

namespace {

#define KB_HOST_ENTRIES(X)                                                                                        \
  X(kb_qk_norm_rope) X(kb_qk_norm_rope_backward_workspace_size) X(kb_qk_norm_rope_backward)                        \
  X(kb_shared_prefix_attention_workspace_size) X(kb_shared_prefix_attention) X(kb_cache_reserve_workspace_size)    \
  X(kb_cache_reserve) X(kb_cache_append_granted) X(kb_cache_fork_workspace_size) X(kb_cache_fork) X(kb_cache_free)         \
  X(kb_cache_compact_workspace_size) X(kb_cache_compact) X(kb_penalize_logits)

struct Abi {
#define X(name) decltype(&::name) name = nullptr;
  KB_HOST_ENTRIES(X)
#undef X
  PyObject* check = nullptr;  // kbb200._lib.check(entry, status), which raises
} abi;

// Whether the entry answered an error, which is then raised.
bool failed(const char* entry, int status) {
  if (status == KB_OK) return false;
  PyObject* r = PyObject_CallFunction(abi.check, "si", entry, status);
  if (r) PyErr_Format(PyExc_RuntimeError, "%s failed with status %d", entry, status);
  Py_XDECREF(r);
  return true;
}

using at::Tensor;

// The tensor behind a Python object, or null.
const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int code(at::ScalarType t) {
  return t == at::kFloat ? KB_F32 : t == at::kHalf ? KB_F16 : t == at::kBFloat16 ? KB_BF16 : -1;
}

// A call's device: the first tensor's, which has to be the current one.
struct Device {
  int index = -1;
  explicit Device(const Tensor* t) {
    if (t && t->is_cuda() && t->get_device() == c10::cuda::current_device()) index = t->get_device();
  }
  bool ok() const { return index >= 0; }
  bool has(const Tensor* t, at::ScalarType type, int64_t dims) const {
    return t && t->is_cuda() && t->get_device() == index && t->scalar_type() == type && t->dim() == dims;
  }
  bool whole(const Tensor* t, at::ScalarType type, int64_t dims) const {  // and contiguous
    return has(t, type, dims) && t->is_contiguous();
  }
  bool row(const Tensor* t, at::ScalarType type, int64_t n) const { return whole(t, type, 1) && t->size(0) == n; }
  kbStream stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream(); }
};

Tensor scratch(size_t bytes, const Tensor& like) {
  return at::empty({static_cast<int64_t>(bytes > 16 ? bytes : 16)}, like.options().dtype(at::kByte));
}
Tensor like(const Tensor& x) { return at::empty(x.sizes(), x.options()); }
void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

PyObject* pair(const Tensor& a, const Tensor& b) {
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(b));
  return r;
}

// ------------------------------------------------------------ norms of queries and keys, rotation
struct Rope {
  const Tensor *q, *k, *qw, *kw, *cos, *sin, *pos;
  at::ScalarType type = at::kFloat, weights = at::kFloat;
  int64_t tokens = 0, hq = 0, hkv = 0, dim = 0, rotary = 0, rows = 0;
  int pos64 = 0;
  float eps = 0;
  int interleaved = 0;

  // args: q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved
  bool read(const Device& dev, PyObject* const* args) {
    q = tensor(args[0]), k = tensor(args[1]), cos = tensor(args[4]), sin = tensor(args[5]), pos = tensor(args[6]);
    const bool weighed = args[2] != Py_None;
    if (weighed != (args[3] != Py_None)) return false;
    qw = weighed ? tensor(args[2]) : nullptr, kw = weighed ? tensor(args[3]) : nullptr;
    if (!q || q->dim() != 3 || !pos || !cos || (weighed && (!qw || !kw))) return false;
    type = q->scalar_type();
    tokens = q->size(0), hq = q->size(1), dim = q->size(2);
    if (code(type) < 0 || !dev.has(k, type, 3) || k->size(0) != tokens || k->size(2) != dim) return false;
    hkv = k->size(1);
    if (!tokens || !hq || !hkv || dim < 2 || q->stride(2) != 1 || k->stride(2) != 1) return false;
    if (weighed) {
      weights = qw->scalar_type();
      if ((weights != type && weights != at::kFloat) || !dev.row(qw, weights, dim) || !dev.row(kw, weights, dim)) return false;
    }
    if (!dev.whole(cos, at::kFloat, 2) || !dev.whole(sin, at::kFloat, 2) || cos->sizes() != sin->sizes()) return false;
    rows = cos->size(0), rotary = 2 * cos->size(1);
    pos64 = pos->scalar_type() == at::kLong;
    if (!dev.row(pos, pos64 ? at::kLong : at::kInt, tokens)) return false;
    const double e = PyFloat_AsDouble(args[7]);
    const int i = PyObject_IsTrue(args[8]);
    if (PyErr_Occurred() || i < 0) {
      PyErr_Clear();
      return false;
    }
    eps = static_cast<float>(e), interleaved = i;
    return true;
  }
};

PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Rope r;
  if (n != 9) Py_RETURN_NONE;
  const Device dev(tensor(args[0]));
  if (!dev.ok() || !r.read(dev, args)) Py_RETURN_NONE;
  const Tensor q = like(*r.q), k = like(*r.k);
  const int status = abi.kb_qk_norm_rope(
      ptr(r.q), ptr(r.k), ptr(r.qw), ptr(r.kw), static_cast<const float*>(ptr(r.cos)), static_cast<const
      float*>(ptr(r.sin)), ptr(r.pos), q.data_ptr(), k.data_ptr(), r.tokens, r.hq, r.hkv, r.dim, r.rotary, r.rows,
      r.q->stride(0), r.q->stride(1), r.k->stride(0), r.k->stride(1), code(r.type), code(r.weights), r.pos64,
      r.interleaved, r.eps, dev.stream());
  if (failed("kb_qk_norm_rope", status)) return nullptr;
  return pair(q, k);
  END_HANDLE_TH_ERRORS
}

PyObject* rope_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Rope r;
  if (n != 11) Py_RETURN_NONE;
  const Device dev(tensor(args[2]));
  if (!dev.ok() || !r.read(dev, args + 2)) Py_RETURN_NONE;
  const Tensor *dzq = tensor(args[0]), *dzk = tensor(args[1]);
  if (!dev.whole(dzq, r.type, 3) || !dev.whole(dzk, r.type, 3) || dzq->sizes() != r.q->sizes() ||
      dzk->sizes() != r.k->sizes())
    Py_RETURN_NONE;
  const Tensor q = like(*dzq), k = like(*dzk);
  const Tensor qw = r.qw ? like(*r.qw) : Tensor(), kw = r.kw ? like(*r.kw) : Tensor();
  const size_t need = abi.kb_qk_norm_rope_backward_workspace_size(r.tokens, r.hq, r.hkv, r.dim);
  const Tensor ws = scratch(need, *r.q);
  const int status = abi.kb_qk_norm_rope_backward(
      ptr(dzq), ptr(dzk), ptr(r.q), ptr(r.k), ptr(r.qw), ptr(r.kw), static_cast<const float*>(ptr(r.cos)),
      static_cast<const float*>(ptr(r.sin)), ptr(r.pos), q.data_ptr(), k.data_ptr(), r.qw ? qw.data_ptr() : nullptr,
      r.kw ? kw.data_ptr() : nullptr, r.tokens, r.hq, r.hkv, r.dim, r.rotary, r.rows, r.q->stride(0), r.q->stride(1),
      r.k->stride(0), r.k->stride(1), code(r.type), code(r.weights), r.pos64, r.interleaved, r.eps, ws.data_ptr(), need,
      dev.stream());
  if (failed("kb_qk_norm_rope_backward", status)) return nullptr;
  PyObject* out = PyTuple_New(4);
  if (!out) return nullptr;
  const Tensor all[4] = {q, k, qw, kw};
  for (int i = 0; i < 4; ++i) {
    if (all[i].defined()) {
      PyTuple_SET_ITEM(out, i, THPVariable_Wrap(all[i]));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(out, i, Py_None);
    }
  }
  return out;
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ attention over the cache
// q, k_pages, v_pages, prefix, table, lens, scale or None
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  const Tensor *q = tensor(args[0]), *k = tensor(args[1]), *v = tensor(args[2]), *prefix = tensor(args[3]),
               *table = tensor(args[4]), *lens = tensor(args[5]);
  const Device dev(q);
  if (!dev.ok() || q->dim() != 4 || code(q->scalar_type()) < 0) Py_RETURN_NONE;
  const at::ScalarType type = q->scalar_type();
  const int64_t B = q->size(0), Q = q->size(1), hq = q->size(2), d = q->size(3);
  if (!dev.has(k, type, 4) || !dev.has(v, type, 4) || k->sizes() != v->sizes() || k->size(3) != d || d < 2 ||
      q->stride(3) != 1 || k->stride(3) != 1 || v->stride(3) != 1 || !dev.whole(prefix, at::kInt, 1) ||
      !dev.whole(table, at::kInt, 2) || table->size(0) != B || !dev.row(lens, at::kInt, B))
    Py_RETURN_NONE;
  double scale = 1.0 / std::sqrt(static_cast<double>(d));
  if (args[6] != Py_None) {
    scale = PyFloat_AsDouble(args[6]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
  }
  const int64_t pages = k->size(0), page = k->size(1), hkv = k->size(2), pre = prefix->size(0), width = table->size(1);
  const Tensor out = like(*q), lse = at::empty({B, Q, hq}, q->options().dtype(at::kFloat));
  const size_t need = abi.kb_shared_prefix_attention_workspace_size(B, Q, hq, hkv, d, pre, width, page, code(type));
  const Tensor ws = need ? scratch(need, *q) : Tensor();
  const int status = abi.kb_shared_prefix_attention(
      ptr(q), ptr(k), ptr(v), static_cast<const int32_t*>(ptr(prefix)), static_cast<const int32_t*>(ptr(table)),
      static_cast<const int32_t*>(ptr(lens)), out.data_ptr(), static_cast<float*>(lse.data_ptr()), B, Q, hq, hkv, d,
      pre, width, pages, page, q->stride(0), q->stride(1), q->stride(2), k->stride(0), k->stride(1), k->stride(2),
      v->stride(0), v->stride(1), v->stride(2), static_cast<float>(scale), code(type), need ? ws.data_ptr() : nullptr,
      need, dev.stream());
  if (failed("kb_shared_prefix_attention", status)) return nullptr;
  return pair(out, lse);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ the paged cache
struct State {
  const Tensor *table, *lens, *refs;
  // lens or refs may be left out (null)
  bool read(const Device& dev, PyObject* t, PyObject* l, PyObject* r) {
    table = tensor(t), lens = l ? tensor(l) : nullptr, refs = r ? tensor(r) : nullptr;
    return dev.ok() && dev.whole(table, at::kInt, 2) && (!l || dev.row(lens, at::kInt, table->size(0))) &&
           (!r || dev.whole(refs, at::kInt, 1));
  }
};
int32_t* ints(const Tensor* t) { return static_cast<int32_t*>(t->data_ptr()); }
// A pool [planes, pages, page_size, ...]; its pages' bytes, or -1.
int64_t page_bytes(const Device& dev, const Tensor* pool, int64_t pages) {
  if (!pool || !pool->is_cuda() || pool->get_device() != dev.index || !pool->is_contiguous() || pool->dim() < 3 ||
      pool->size(1) != pages || !pool->numel())
    return -1;
  const at::ScalarType t = pool->scalar_type();
  if (code(t) < 0 && t != at::kByte && t != at::kChar) return -1;
  return pool->stride(1) * static_cast<int64_t>(pool->element_size());
}

// table, lens, refs, seqs, tokens, page_size
PyObject* reserve(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  const Device dev(tensor(args[0]));
  State s;
  const Tensor* seqs = tensor(args[3]);
  const int64_t tokens = PyLong_Check(args[4]) ? PyLong_AsLongLong(args[4]) : -1;
  const int64_t page = PyLong_Check(args[5]) ? PyLong_AsLongLong(args[5]) : -1;
  if (PyErr_Occurred()) PyErr_Clear();
  if (tokens < 0 || page < 1 || !s.read(dev, args[0], args[1], args[2]) || !dev.whole(seqs, at::kInt, 1)) Py_RETURN_NONE;
  const int64_t m = seqs->size(0), slots = s.table->size(0), width = s.table->size(1), pages = s.refs->size(0);
  const Tensor granted = like(*seqs);
  const size_t need = abi.kb_cache_reserve_workspace_size(m, tokens, slots, width, pages, page);
  const Tensor ws = scratch(need, *s.table);
  const int status = abi.kb_cache_reserve(
      ints(s.table), ints(s.lens), ints(s.refs), ints(seqs), ints(&granted), m, tokens, slots, width, pages, page,
      ws.data_ptr(), need, dev.stream());
  if (failed("kb_cache_reserve", status)) return nullptr;
  return THPVariable_Wrap(granted);
  END_HANDLE_TH_ERRORS
}

// k, v, k_pages, v_pages, table, lens, seqs, granted or None
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) Py_RETURN_NONE;
  const Tensor *k = tensor(args[0]), *v = tensor(args[1]), *kp = tensor(args[2]), *vp = tensor(args[3]),
               *seqs = tensor(args[6]), *granted = args[7] == Py_None ? nullptr : tensor(args[7]);
  const Device dev(tensor(args[4]));
  State s;
  if (!s.read(dev, args[4], args[5], nullptr) || !kp || code(kp->scalar_type()) < 0 || !dev.whole(seqs, at::kInt, 1))
    Py_RETURN_NONE;
  const at::ScalarType type = kp->scalar_type();
  if (!dev.whole(kp, type, 4) || !dev.whole(vp, type, 4) || kp->sizes() != vp->sizes() || !dev.has(k, type, 4) ||
      !dev.has(v, type, 4) || k->sizes() != v->sizes() || k->size(0) != seqs->size(0) || k->size(2) != kp->size(2) ||
      k->size(3) != kp->size(3) || (args[7] != Py_None && !dev.row(granted, at::kInt, seqs->size(0))))
    Py_RETURN_NONE;
  const int64_t d = kp->size(3), h = kp->size(2), e = static_cast<int64_t>(kp->element_size());
  for (const Tensor* t : {k, v})
    if (t->stride(3) != 1 || t->stride(2) != d) Py_RETURN_NONE;
  const int status = abi.kb_cache_append_granted(
      ptr(k), ptr(v), ptr(kp), ptr(vp), ints(s.table), ints(s.lens), ints(seqs), granted ? ints(granted) : nullptr,
      seqs->size(0), k->size(1), s.table->size(0), s.table->size(1), kp->size(0), kp->size(1), kp->size(1) * h * d * e,
      h * d * e, k->stride(0) * e, k->stride(1) * e, v->stride(0) * e, v->stride(1) * e, dev.stream());
  if (failed("kb_cache_append", status)) return nullptr;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// pool, table, lens, refs, parents, children
PyObject* fork(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  const Tensor *pool = tensor(args[0]), *parents = tensor(args[4]), *children = tensor(args[5]);
  const Device dev(tensor(args[1]));
  State s;
  if (!s.read(dev, args[1], args[2], args[3]) || !dev.whole(parents, at::kInt, 1) ||
      !dev.row(children, at::kInt, parents->size(0)))
    Py_RETURN_NONE;
  const int64_t bytes = page_bytes(dev, pool, s.refs->size(0));
  if (bytes < 0) Py_RETURN_NONE;
  const int64_t m = parents->size(0), slots = s.table->size(0), width = s.table->size(1);
  const Tensor granted = like(*parents);
  const size_t need = abi.kb_cache_fork_workspace_size(m, slots, width);
  const Tensor ws = scratch(need, *s.table);
  const int status = abi.kb_cache_fork(
      ptr(pool), ints(s.table), ints(s.lens), ints(s.refs), ints(parents), ints(children), ints(&granted), m, slots,
      width, pool->size(0), pool->size(1), pool->size(2), bytes, ws.data_ptr(), need, dev.stream());
  if (failed("kb_cache_fork", status)) return nullptr;
  return THPVariable_Wrap(granted);
  END_HANDLE_TH_ERRORS
}

// table, lens, refs, seqs
PyObject* release(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) Py_RETURN_NONE;
  const Device dev(tensor(args[0]));
  State s;
  const Tensor* seqs = tensor(args[3]);
  if (!s.read(dev, args[0], args[1], args[2]) || !dev.whole(seqs, at::kInt, 1)) Py_RETURN_NONE;
  const int status = abi.kb_cache_free(
      ints(s.table), ints(s.lens), ints(s.refs), ints(seqs), seqs->size(0), s.table->size(0), s.table->size(1),
      s.refs->size(0), dev.stream());
  if (failed("kb_cache_free", status)) return nullptr;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// pool, table, refs
PyObject* compact(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) Py_RETURN_NONE;
  const Tensor* pool = tensor(args[0]);
  const Device dev(tensor(args[1]));
  State s;
  if (!s.read(dev, args[1], nullptr, args[2])) Py_RETURN_NONE;
  const int64_t bytes = page_bytes(dev, pool, s.refs->size(0));
  if (bytes < 0) Py_RETURN_NONE;
  const Tensor live = at::empty({1}, s.refs->options());
  const size_t need = abi.kb_cache_compact_workspace_size(s.refs->size(0));
  const Tensor ws = scratch(need, *s.table);
  const int status = abi.kb_cache_compact(
      ptr(pool), ints(s.table), ints(s.refs), ints(&live), s.table->size(0), s.table->size(1), pool->size(0),
      pool->size(1), bytes, ws.data_ptr(), need, dev.stream());
  if (failed("kb_cache_compact", status)) return nullptr;
  return THPVariable_Wrap(live);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ logits
// logits, then prompt, output, repetition, presence, frequency, bias_ids, bias_values, mask (or None)
PyObject* logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) Py_RETURN_NONE;
  const Tensor* given[9] = {};
  for (int i = 0; i < 9; ++i)
    if (args[i] != Py_None && !(given[i] = tensor(args[i]))) Py_RETURN_NONE;
  const Tensor* x = given[0];
  const Device dev(x);
  if (!dev.ok() || x->dim() != 2 || code(x->scalar_type()) < 0) Py_RETURN_NONE;
  const int64_t B = x->size(0), V = x->size(1);
  if (!B || V < 2 || x->stride(1) != 1 || !given[6] != !given[7]) Py_RETURN_NONE;
  int64_t lengths[3] = {};
  const Tensor* lists[3] = {given[1], given[2], given[6]};
  int ids64 = -1;
  for (int i = 0; i < 3; ++i) {
    if (!lists[i]) continue;
    const int is64 = lists[i]->scalar_type() == at::kLong;
    if ((ids64 >= 0 && is64 != ids64) || !dev.whole(lists[i], is64 ? at::kLong : at::kInt, 2) || lists[i]->size(0) != B)
      Py_RETURN_NONE;
    ids64 = is64;
    lengths[i] = lists[i]->size(1);
  }
  for (int i = 3; i < 6; ++i)
    if (given[i] && !dev.row(given[i], at::kFloat, B)) Py_RETURN_NONE;
  if (given[7] && (!dev.whole(given[7], at::kFloat, 2) || given[7]->sizes() != given[6]->sizes())) Py_RETURN_NONE;
  int64_t mask_stride = 0;
  if (const Tensor* m = given[8]) {
    if (!dev.whole(m, at::kInt, 2) || (m->size(0) != B && m->size(0) != 1) || m->size(1) != (V + 31) / 32) Py_RETURN_NONE;
    mask_stride = m->size(0) == B ? m->size(1) : 0;
  }
  const Tensor out = like(*x);
  auto f32 = [&](int i) { return static_cast<const float*>(ptr(given[i])); };
  const int status = abi.kb_penalize_logits(
      ptr(x), out.data_ptr(), ptr(given[1]), ptr(given[2]), f32(3), f32(4), f32(5), ptr(given[6]), f32(7),
      ptr(given[8]), B, V, x->stride(0), lengths[0], lengths[1], lengths[2], mask_stride, code(x->scalar_type()), ids64
      == 1, dev.stream());
  if (failed("kb_penalize_logits", status)) return nullptr;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------ module
// init({name: address, ..., "check": kbb200._lib.check}): the C ABI's entries
PyObject* init(PyObject*, PyObject* table) {
  PyObject* check = PyDict_Check(table) ? PyDict_GetItemString(table, "check") : nullptr;
  if (!check) {
    PyErr_SetString(PyExc_ValueError, "kbb200._lm_host: no check");
    return nullptr;
  }
#define X(name)                                                                                          \
  {                                                                                                      \
    PyObject* at = PyDict_Check(table) ? PyDict_GetItemString(table, #name) : nullptr;                   \
    void* p = at ? PyLong_AsVoidPtr(at) : nullptr;                                                       \
    if (!p) {                                                                                            \
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "kbb200._lm_host: no address of " #name); \
      return nullptr;                                                                                    \
    }                                                                                                    \
    abi.name = reinterpret_cast<decltype(&::name)>(p);                                                   \
  }
  KB_HOST_ENTRIES(X)
#undef X
  Py_INCREF(check);
  Py_XDECREF(abi.check);
  abi.check = check;
  Py_RETURN_NONE;
}

#define KB_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {KB_METHOD(rope),    KB_METHOD(rope_backward), KB_METHOD(attention), KB_METHOD(reserve),
                         KB_METHOD(append),  KB_METHOD(fork),          KB_METHOD(release),   KB_METHOD(compact),
                         KB_METHOD(logits),  {"init", init, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lm_host", "Host side of kbb200.lm's calls.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__lm_host() { return PyModule_Create(&module); }
