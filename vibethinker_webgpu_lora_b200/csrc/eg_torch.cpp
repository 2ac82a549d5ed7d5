// eg_torch.cpp -- the Python binding of the paged serving ops on torch tensors
// (module _ops): takes the sizes, strides and types from the tensors, checks
// them against each other, and calls the C ABI on the current stream.  The
// same in Python (twenty attribute reads and a ctypes call) took 13 us of a
// call whose kernel runs for 2.
//
// Each function returns the eg_status of the C call; tensors that do not fit
// raise ValueError naming the operator.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "emberglass.h"

namespace {

struct Refused {};  // the Python error is set

struct Call {
  const char* op;
  int device = -1;

  [[noreturn]] void refuse(const char* what) const {
    PyErr_Format(PyExc_ValueError, "%s: %s", op, what);
    throw Refused();
  }
  void need(bool ok, const char* what) const {
    if (!ok) refuse(what);
  }
  // a tensor argument (None only where `optional`); all lie on one CUDA device, the current one
  const at::Tensor* tensor(PyObject* o, const char* name, bool optional = false) {
    if (optional && o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_ValueError, "%s: %s must be a torch tensor", op, name);
      throw Refused();
    }
    return &THPVariable_Unpack(o);
  }
  void on_device(const at::Tensor* t) {
    if (!t) return;
    need(t->is_cuda(), "CUDA tensors required");
    if (device < 0) device = t->get_device();
    need(t->get_device() == device, "tensors are on different devices");
  }
  long integer(PyObject* o, const char* name) const {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Refused();
    if (v != (int)v) {
      PyErr_Format(PyExc_ValueError, "%s: %s is out of range", op, name);
      throw Refused();
    }
    return v;
  }
  // rows of `width` contiguous f32 values; the row stride (a single row's says
  // nothing: any multiple of 4 that spans it will do)
  int64_t rows(const at::Tensor& t, int64_t width, const char* what) const {
    need(t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(1) >= width && (t.size(1) == 1 || t.stride(1) == 1), what);
    return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 3) / 4 * 4;
  }
  void ints(const at::Tensor& t, int64_t n, const char* what) const {
    need((t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32) && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), what);
  }
  void table(const at::Tensor& t, const char* what) const {
    need((t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32) && t.dim() == 2 && t.is_contiguous(), what);
  }
  void caches(const at::Tensor& k, const at::Tensor& v) const {
    need(k.dim() == 4 && k.size(1) == 16 && k.size(3) == 128 && (k.scalar_type() == at::kHalf || k.scalar_type() == at::kFloat) &&
             k.is_contiguous(),
         "caches must be contiguous [n_pages][16][nkv][128] of f16 or f32");
    need(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.is_contiguous(),
         "k_cache and v_cache differ in shape or type");
  }
  void error_word(const at::Tensor* t) const { need(!t || (t->scalar_type() == at::kInt && t->numel() == 1), "err must be one int32"); }
  void* stream(PyObject* o) const {
    const auto cur = c10::cuda::getCurrentCUDAStream();  // of the current device
    need(device == cur.device_index(), "tensors are not on the current device");
    if (o == Py_None) return cur.stream();
    void* s = PyLong_AsVoidPtr(o);
    if (!s && PyErr_Occurred()) throw Refused();
    return s;
  }
};

template <typename T>
T* ptr(const at::Tensor* t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
int sz(int64_t v) { return v > 0x7fffffff ? -1 : (int)v; }  // what an int cannot hold is refused by the C call

template <typename F>
PyObject* guarded(PyObject* const*, Py_ssize_t n, Py_ssize_t want, const char* op, F f) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", op, want);
    return nullptr;
  }
  try {
    return PyLong_FromLong((long)f());
  } catch (const Refused&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_Format(PyExc_RuntimeError, "%s: %s", op, e.what());
    return nullptr;
  }
}

// (qkv, pos, slot, pages, k_cache, v_cache, cos_t, sin_t, nh, q_out, prefix_len, err, stream)
PyObject* kv_append_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, 13, "kv_append_paged", [&] {
    Call c{"kv_append_paged"};
    const at::Tensor &qkv = *c.tensor(a[0], "qkv"), &pos = *c.tensor(a[1], "pos"), &slot = *c.tensor(a[2], "slot"),
                     &pages = *c.tensor(a[3], "pages"), &k = *c.tensor(a[4], "k_cache"), &v = *c.tensor(a[5], "v_cache"),
                     &cs = *c.tensor(a[6], "cos_t"), &sn = *c.tensor(a[7], "sin_t");
    const at::Tensor *q = c.tensor(a[9], "q_out", true), *err = c.tensor(a[11], "err", true);
    const long nh = c.integer(a[8], "nh"), prefix = c.integer(a[10], "prefix_len");
    c.caches(k, v);
    const int64_t nkv = k.size(2), T = qkv.dim() ? qkv.size(0) : 0;
    c.need(nh >= 0, "nh must not be negative");
    const int64_t ld = c.rows(qkv, (nh + 2 * nkv) * 128, "qkv must be f32 rows of (nh + 2 nkv) * 128 contiguous values");
    c.ints(pos, T, "pos must be contiguous int32, one for each row of qkv");
    c.ints(slot, T, "slot must be contiguous int32, one for each row of qkv");
    c.table(pages, "pages must be contiguous int32 [n_slots][max_pages]");
    c.need(cs.scalar_type() == at::kFloat && cs.dim() == 2 && cs.size(1) == 128 && cs.is_contiguous() &&
               sn.scalar_type() == at::kFloat && sn.sizes() == cs.sizes() && sn.is_contiguous(),
           "cos_t and sin_t must be contiguous f32 [positions][128]");
    int64_t ldq = 0;
    if (q) {
      ldq = c.rows(*q, nh * 128, "q_out must be f32 rows of nh * 128 contiguous values");
      c.need(q->size(0) == T, "q_out must have a row for each of qkv's");
    }
    c.error_word(err);
    for (const at::Tensor* t : {&qkv, &pos, &slot, &pages, &k, &v, &cs, &sn, q, err}) c.on_device(t);
    void* st = c.stream(a[12]);
    return eg_op_kv_append_paged(ptr<const float>(&qkv), ld, sz(T), ptr<const int>(&pos), ptr<const int>(&slot),
                                 ptr<const uint32_t>(&pages), sz(pages.size(0)), sz(pages.size(1)), sz(k.size(0)),
                                 (int)prefix, ptr<void>(&k), ptr<void>(&v), ptr<const float>(&cs), ptr<const float>(&sn),
                                 sz(cs.size(0)), (int)nh, sz(nkv), k.scalar_type() == at::kHalf, ptr<float>(q), ldq,
                                 ptr<int>(err), st);
  });
}

// (q, k_cache, v_cache, prefix_pages, prefix_len, pages, lens, max_len, out, ws, err, stream)
PyObject* attn_shared_prefix(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, 12, "attn_shared_prefix", [&] {
    Call c{"attn_shared_prefix"};
    const at::Tensor &q = *c.tensor(a[0], "q"), &k = *c.tensor(a[1], "k_cache"), &v = *c.tensor(a[2], "v_cache"),
                     &pages = *c.tensor(a[5], "pages"), &lens = *c.tensor(a[6], "lens"), &out = *c.tensor(a[8], "out"),
                     &ws = *c.tensor(a[9], "ws");
    const long prefix = c.integer(a[4], "prefix_len"), max_len = c.integer(a[7], "max_len");
    const at::Tensor *pp = c.tensor(a[3], "prefix_pages", prefix <= 0), *err = c.tensor(a[10], "err", true);
    c.caches(k, v);
    c.need(q.dim() == 2 && q.size(1) % 128 == 0, "q must be [nseq][nh * 128]");
    const int64_t nseq = q.size(0), width = q.size(1);
    const int64_t ldq = c.rows(q, width, "q must be f32 rows of contiguous values");
    c.need(out.sizes() == q.sizes(), "out must have q's shape");
    const int64_t ldo = c.rows(out, width, "out must be f32 rows of contiguous values");
    c.ints(lens, nseq, "lens must be contiguous int32, one for each row of q");
    c.table(pages, "pages must be contiguous int32 [nseq][max_pages]");
    c.need(pages.size(0) == nseq, "pages must have a row for each of q's");
    if (prefix > 0) {
      c.ints(*pp, pp->numel(), "prefix_pages must be contiguous int32");
      c.need(pp->numel() * 16 >= prefix, "prefix_pages do not hold prefix_len rows");
    }
    c.need(ws.is_contiguous(), "ws must be contiguous");
    c.error_word(err);
    for (const at::Tensor* t : {&q, &k, &v, pp, &pages, &lens, &out, &ws, err}) c.on_device(t);
    void* st = c.stream(a[11]);
    return eg_op_attn_shared_prefix(ptr<const float>(&q), ldq, sz(nseq), ptr<const void>(&k), ptr<const void>(&v),
                                    sz(k.size(0)), ptr<const uint32_t>(pp), (int)prefix, ptr<const uint32_t>(&pages),
                                    sz(pages.size(1)), ptr<const int>(&lens), (int)max_len, sz(width / 128), sz(k.size(2)),
                                    k.scalar_type() == at::kHalf, ptr<float>(&out), ldo, ptr<void>(&ws),
                                    (uint64_t)(ws.numel() * ws.element_size()), ptr<int>(err), st);
  });
}

// (logits, r, ids, temp, top_k, top_p, min_p, probs, stream)
PyObject* sample_filtered(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(a, n, 9, "sample_filtered", [&] {
    Call c{"sample_filtered"};
    const at::Tensor &x = *c.tensor(a[0], "logits"), &r = *c.tensor(a[1], "r"), &ids = *c.tensor(a[2], "ids");
    const at::Tensor *temp = c.tensor(a[3], "temp", true), *k = c.tensor(a[4], "top_k", true), *p = c.tensor(a[5], "top_p", true),
                     *m = c.tensor(a[6], "min_p", true), *probs = c.tensor(a[7], "probs", true);
    c.need(x.dim() == 2 && x.size(1) >= 1, "logits must be [rows][n]");
    c.need(x.scalar_type() == at::kFloat && (x.size(1) == 1 || x.stride(1) == 1), "logits must be f32, contiguous in a row");
    const int64_t rows = x.size(0);
    for (const at::Tensor* t : {&r, temp, p, m, probs})
      c.need(!t || (t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == rows && t->is_contiguous()),
             "r, temp, top_p, min_p and probs must be contiguous f32, one for each row of logits");
    for (const at::Tensor* t : {&ids, k})
      if (t) c.ints(*t, rows, "ids and top_k must be contiguous int32, one for each row of logits");
    for (const at::Tensor* t : {&x, &r, &ids, temp, k, p, m, probs}) c.on_device(t);
    void* st = c.stream(a[8]);
    return eg_op_sample_filtered(ptr<const float>(&x), rows > 1 ? x.stride(0) : x.size(1), sz(rows), sz(x.size(1)),
                                 ptr<const float>(temp), ptr<const int>(k), ptr<const float>(p), ptr<const float>(m),
                                 ptr<const float>(&r), ptr<uint32_t>(&ids), ptr<float>(probs), st);
  });
}

PyMethodDef methods[] = {
    {"kv_append_paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv_append_paged)), METH_FASTCALL, nullptr},
    {"attn_shared_prefix", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attn_shared_prefix)), METH_FASTCALL, nullptr},
    {"sample_filtered", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(sample_filtered)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&module); }
