// The serving calls on torch tensors (module nkb_torch, used by
// nkipy_b200/runtime/serving.py): checks of types, shapes and strides, outputs
// and workspaces from torch's allocator, and the call into libnkb.so on the
// current stream.  At a few tokens these calls are bound by the host; the same
// steps in Python took 8 us of a 14 us attention call.
#include <Python.h>

#include <ATen/Functions.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "nkb.h"

namespace {

using at::Tensor;

[[noreturn]] void fail(PyObject *type, const std::string &message) {
  PyErr_SetString(type, message.c_str());
  throw python_error();
}
[[noreturn]] void invalid(const std::string &message) { fail(PyExc_ValueError, message); }
[[noreturn]] void wrong_type(const std::string &message) { fail(PyExc_TypeError, message); }

// A tensor argument, or none.
struct Arg {
  const char *name;
  const Tensor *t = nullptr;
  Arg(const char *name, PyObject *o) : name(name) {
    if (o == Py_None) return;
    if (!THPVariable_Check(o)) wrong_type(std::string(name) + ": expected a tensor, got " + Py_TYPE(o)->tp_name);
    t = &THPVariable_Unpack(o);
  }
  explicit operator bool() const { return t; }
  const Tensor &operator*() const {
    if (!t) wrong_type(std::string(name) + ": expected a tensor, got None");
    return *t;
  }
  const Tensor *operator->() const { return &**this; }
  template <class T = void>
  T *ptr() const { return t ? static_cast<T *>(t->data_ptr()) : nullptr; }
  std::string text() const { return c10::str(name, " ", (*this)->sizes(), " ", (*this)->scalar_type()); }
};

void on_device(int64_t device, std::initializer_list<const Arg *> args) {
  for (const Arg *a : args)
    if (*a && (!(*a)->is_cuda() || (*a)->get_device() != device))
      invalid(c10::str(a->name, ": expected a tensor on cuda:", device, " (this process's device), got one on ", (*a)->device()));
}

// The calls record nothing for a backward pass: tensors that want one are refused.
void without_gradient(std::initializer_list<const Arg *> args) {
  if (!c10::GradMode::is_enabled()) return;
  for (const Arg *a : args)
    if (*a && (*a)->requires_grad())
      fail(PyExc_RuntimeError, std::string(a->name) + ": requires a gradient, which this call does not have; call it under torch.no_grad(), or on detached tensors");
}
// What a call writes repeats no element, and covers no part of `others` (a given output may be its own input).
void apart(const Arg &out, std::initializer_list<const Arg *> others) {
  if (!out) return;
  if (at::has_internal_overlap(*out) == at::MemOverlap::Yes) invalid(std::string(out.name) + ": written, but some of its elements are the same memory");
  for (const Arg *a : others)
    if (*a) {
      const at::MemOverlapStatus s = at::get_overlap_status(*out, **a);
      if (s == at::MemOverlapStatus::Partial || s == at::MemOverlapStatus::Full) invalid(c10::str(out.name, ": written, but shares memory with ", a->name));
    }
}
void apart_or_same(const Arg &out, const Arg &in) {
  if (out && in && at::get_overlap_status(*out, *in) == at::MemOverlapStatus::Partial)
    invalid(c10::str(out.name, ": written, but shares a part of its memory with ", in.name));
}

// A tensor that a call has written into: autograd sees that it changed.
void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int64_t code_of(const Arg &a) {
  switch (a->scalar_type()) {
    case at::kFloat: return NKB_F32;
    case at::kBFloat16: return NKB_BF16;
    case at::kHalf: return NKB_F16;
    default: wrong_type(c10::str(a.name, ": expected float32, bfloat16 or float16, got ", a->scalar_type()));
  }
}
// type code of a float tensor with `ndim` axes, the last one contiguous
int64_t rows(const Arg &a, int64_t ndim) {
  const int64_t code = code_of(a);
  if (a->dim() != ndim) invalid(c10::str(a.name, ": expected ", ndim, " axes, got shape ", a->sizes()));
  if (a->stride(-1) != 1 && a->size(-1) > 1 && a->numel()) invalid(std::string(a.name) + ": the last axis must be contiguous");
  return code;
}
// a contiguous vector of `length` elements (-1: any number)
void vector(const Arg &a, at::ScalarType type, int64_t length) {
  if (a->scalar_type() != type) wrong_type(c10::str(a.name, ": expected ", type, ", got ", a->scalar_type()));
  if (a->dim() != 1 || (length >= 0 && a->numel() != length) || !a->is_contiguous())
    invalid(c10::str(a.name, ": expected a contiguous vector", length < 0 ? "" : c10::str(" of ", length), ", got shape ", a->sizes()));
}

// what both calls on a cache have: its layout, the page table and the lengths
template <class Args>
int64_t cache_and_batch(Args &x, const Arg &k, const Arg &v, const Arg &table, const Arg &kv_len, const Arg &q_start) {
  const int64_t code = rows(k, 4);
  if (v->scalar_type() != k->scalar_type() || v->sizes() != k->sizes()) invalid("k_cache and v_cache differ: " + k.text() + ", " + v.text());
  rows(v, 4);
  x.k_cache = k.ptr();
  x.v_cache = v.ptr();
  x.pages = k->size(0);
  x.page_size = k->size(1);
  x.k_page = k->stride(0);
  x.k_slot = k->stride(1);
  x.k_cache_head = k->stride(2);
  x.v_page = v->stride(0);
  x.v_slot = v->stride(1);
  x.v_cache_head = v->stride(2);
  if (table->scalar_type() != at::kInt) wrong_type(c10::str("page_table: expected int32, got ", table->scalar_type()));
  if (table->dim() != 2) invalid(c10::str("page_table: expected 2 axes, got shape ", table->sizes()));
  x.seqs = table->size(0);
  x.table_width = table->size(1);
  x.table_stride = table->stride(0);
  if (table->stride(1) != 1 && x.table_width > 1 && x.seqs) invalid("page_table: the last axis must be contiguous");
  vector(kv_len, at::kInt, x.seqs);
  if (q_start)
    vector(q_start, at::kInt, x.seqs + 1);
  else if (x.tokens != x.seqs)
    invalid(c10::str("without q_start there is one token per sequence: ", x.tokens, " tokens, ", x.seqs, " sequences"));
  x.page_table = table.ptr<int32_t>();
  x.kv_len = kv_len.ptr<int32_t>();
  x.q_start = q_start.ptr<int32_t>();
  return code;
}

// `out`, checked against `like`, or a new contiguous tensor
Tensor output(const Arg &out, const Arg &like, int64_t code) {
  if (!out) return at::empty(like->sizes(), like->options());
  if (rows(out, 3) != code || out->sizes() != like->sizes()) invalid(out.text() + " differs from " + like.text());
  return *out;
}

int64_t integer(PyObject *o) {
  const int64_t x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return x;
}

PyObject *check_status;  // nkipy_b200.spike._nkb.check
void check(int status) {
  if (!status) return;
  Py_XDECREF(PyObject_CallFunction(check_status, "i", status));
  throw python_error();
}

// Issues a call on the current stream of `device`.
template <class Args>
void issue(int (*call)(const Args *, void *), const Args &args, int64_t device) {
  void *stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = call(&args, stream);
  Py_END_ALLOW_THREADS;
  check(status);
}

#define EXPECT(n) \
  if (nargs != n) wrong_type(c10::str("expected ", n, " arguments, got ", nargs))

// (device, k, v, k_cache, v_cache, page_table, kv_len, q_start, q, cos, sin, pos_offset, q_out)
PyObject *paged_append(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  EXPECT(13);
  const int64_t device = integer(o[0]);
  const Arg k("k", o[1]), v("v", o[2]), kc("k_cache", o[3]), vc("v_cache", o[4]), table("page_table", o[5]), len("kv_len", o[6]),
      q_start("q_start", o[7]), q("q", o[8]), cos("cos", o[9]), sin("sin", o[10]), q_out("q_out", o[12]);
  without_gradient({&k, &v, &kc, &vc, &q, &cos, &sin, &q_out});
  on_device(device, {&k, &v, &kc, &vc, &table, &len, &q_start, &q, &cos, &sin, &q_out});
  apart(kc, {&vc, &k, &v});
  apart(vc, {&k, &v});
  apart(q_out, {&k, &v});
  apart_or_same(q_out, q);
  nkb_paged_append_args x = {};
  x.dtype = rows(k, 3);
  x.tokens = k->size(0);
  x.kv_heads = k->size(1);
  x.head_dim = k->size(2);
  if (v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type()) invalid("k and v differ: " + k.text() + ", " + v.text());
  rows(v, 3);
  x.cache_dtype = cache_and_batch(x, kc, vc, table, len, q_start);
  if (kc->size(2) != x.kv_heads || kc->size(3) != x.head_dim) invalid(kc.text() + " does not go with " + k.text());
  if (bool(cos) != bool(sin)) invalid("cos and sin go together");
  if (cos) {
    x.rope_dtype = rows(cos, 2);
    if (sin->sizes() != cos->sizes() || sin->scalar_type() != cos->scalar_type() || sin->strides() != cos->strides())
      invalid("cos and sin differ in shape, type or strides");
    x.rope_rows = cos->size(0);
    x.rot_dim = 2 * cos->size(1);
    x.rope_stride = cos->stride(0);
    if (x.rot_dim > x.head_dim) invalid(c10::str("cos and sin rotate ", x.rot_dim, " dimensions, head_dim is ", x.head_dim));
  }
  x.pos_offset = integer(o[11]);
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  Tensor out;
  if (q) {
    if (rows(q, 3) != x.dtype || q->size(0) != x.tokens || q->size(2) != x.head_dim) invalid(q.text() + " does not go with " + k.text());
    out = output(q_out, q, x.dtype);
    x.q_heads = q->size(1);
    x.q_token = q->stride(0);
    x.q_head = q->stride(1);
    x.q_out_token = out.stride(0);
    x.q_out_head = out.stride(1);
    x.q = q.ptr();
    x.q_out = out.data_ptr();
  } else if (q_out) {
    invalid("q_out without q");
  }
  x.k = k.ptr();
  x.v = v.ptr();
  x.k_token = k->stride(0);
  x.k_head = k->stride(1);
  x.v_token = v->stride(0);
  x.v_head = v->stride(1);
  x.cos = cos.ptr();
  x.sin = sin.ptr();
  issue(nkb_paged_append, x, device);
  written(*kc);
  written(*vc);
  if (!q) Py_RETURN_NONE;
  if (!q_out) return THPVariable_Wrap(std::move(out));
  written(out);
  return Py_NewRef(o[12]);
  END_HANDLE_TH_ERRORS
}

// (device, q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, out, prefix_pages, prefix_len)
PyObject *attention(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  EXPECT(13);
  const int64_t device = integer(o[0]);
  const Arg q("q", o[1]), kc("k_cache", o[2]), vc("v_cache", o[3]), table("page_table", o[4]), len("kv_len", o[5]),
      q_start("q_start", o[6]), given("out", o[10]), prefix("prefix_pages", o[11]);
  without_gradient({&q, &kc, &vc, &given});
  on_device(device, {&q, &kc, &vc, &table, &len, &q_start, &given, &prefix});
  apart(given, {&kc, &vc});
  apart_or_same(given, q);
  nkb_paged_attention_args x = {};
  x.dtype = rows(q, 3);
  x.tokens = q->size(0);
  x.q_heads = q->size(1);
  x.head_dim = q->size(2);
  x.window = integer(o[7]);
  x.sinks = integer(o[8]);
  x.prefix_len = integer(o[12]);
  if (cache_and_batch(x, kc, vc, table, len, q_start) != x.dtype) wrong_type(q.text() + " does not go with " + kc.text());
  x.kv_heads = kc->size(2);
  if (kc->size(3) != x.head_dim || x.kv_heads == 0 || x.q_heads % x.kv_heads) invalid(q.text() + " does not go with " + kc.text());
  if (prefix) {
    vector(prefix, at::kInt, -1);
    if (x.prefix_len < 0) invalid("prefix_len must not be negative");
    if (x.prefix_len > prefix->numel() * x.page_size)
      invalid(c10::str("prefix of ", x.prefix_len, " tokens needs more than ", prefix->numel(), " pages of ", x.page_size));
  }
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  Tensor out = output(given, q, x.dtype);
  x.q = q.ptr();
  x.out = out.data_ptr();
  x.q_token = q->stride(0);
  x.q_head = q->stride(1);
  x.out_token = out.stride(0);
  x.out_head = out.stride(1);
  x.prefix_pages = prefix.ptr<int32_t>();
  if (o[9] == Py_None) {
    x.scale = 1.0 / std::sqrt((double)x.head_dim);
  } else {
    x.scale = PyFloat_AsDouble(o[9]);
    if (PyErr_Occurred()) throw python_error();
  }
  size_t need = 0;
  check(nkb_paged_attention_workspace(&x, &need));
  c10::DataPtr room;
  if (need) room = c10::cuda::CUDACachingAllocator::get()->allocate(need);
  x.workspace = room.get();
  x.workspace_bytes = (int64_t)need;
  issue(nkb_paged_attention, x, device);
  if (given) written(out);
  if (given) return Py_NewRef(o[10]);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (device, logits, u, temperature, top_k, top_p, min_p, out)
PyObject *sample_tokens(PyObject *, PyObject *const *o, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  EXPECT(8);
  const int64_t device = integer(o[0]);
  const Arg logits("logits", o[1]), u("u", o[2]), temperature("temperature", o[3]), top_k("top_k", o[4]), top_p("top_p", o[5]),
      min_p("min_p", o[6]), given("out", o[7]);
  without_gradient({&logits, &u, &temperature, &top_p, &min_p});
  on_device(device, {&logits, &u, &temperature, &top_k, &top_p, &min_p, &given});
  nkb_sample_args x = {};
  x.dtype = rows(logits, 2);
  x.rows = logits->size(0);
  x.vocab = logits->size(1);
  x.row_stride = logits->stride(0);
  for (const Arg *a : {&u, &temperature, &top_p, &min_p}) {
    if (a != &u && !*a) continue;
    if ((*a)->scalar_type() != at::kFloat) invalid(c10::str(a->name, ": expected float32, got ", (*a)->scalar_type()));
    vector(*a, at::kFloat, x.rows);
  }
  if (top_k) vector(top_k, at::kInt, x.rows);
  if (given) vector(given, at::kInt, x.rows);
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  Tensor out = given ? *given : at::empty({x.rows}, logits->options().dtype(at::kInt));
  x.logits = logits.ptr();
  x.u = u.ptr<float>();
  x.temperature = temperature.ptr<float>();
  x.top_k = top_k.ptr<int32_t>();
  x.top_p = top_p.ptr<float>();
  x.min_p = min_p.ptr<float>();
  x.tokens = static_cast<int32_t *>(out.data_ptr());
  issue(nkb_sample_tokens, x, device);
  if (given) written(out);
  if (given) return Py_NewRef(o[7]);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"paged_append", (PyCFunction)(void *)paged_append, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void *)attention, METH_FASTCALL, nullptr},
    {"sample_tokens", (PyCFunction)(void *)sample_tokens, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "nkb_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_nkb_torch() {
  PyObject *nkb = PyImport_ImportModule("nkipy_b200.spike._nkb");
  if (!nkb) return nullptr;
  check_status = PyObject_GetAttrString(nkb, "check");
  Py_DECREF(nkb);
  if (!check_status) return nullptr;
  PyObject *m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", NKB_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
