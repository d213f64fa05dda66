// The ordinary case of the generation operators' host side (ops.py: pages_reserve, pages_fork,
// pages_free, pages_compact, paged_attn_fwd, path_step), for calls whose time on the GPU is a few
// microseconds: the same checks, allocations and library call as the Python functions, without their
// 10 us of interpreter.  Anything that is not ordinary - a wrong type, shape, device or stride, another
// current device - returns None before anything is allocated or launched, and the Python function takes
// the call: its errors are the ones a user sees.  A status that the library returns comes back as an int.
//
// The library's entry points are handed over by address (bind), so that this file needs no link to it
// and calls the library that _lib.py has loaded.  All functions run under the interpreter's lock.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <utility>

#include "../../include/hoa.h"

namespace {

struct Fns {
  decltype(&hoa_pages_workspace_bytes) pages_ws;
  decltype(&hoa_pages_reserve) reserve;
  decltype(&hoa_pages_fork) fork;
  decltype(&hoa_pages_free) free_;
  decltype(&hoa_pages_compact) compact;
  decltype(&hoa_paged_attn_workspace_bytes) attn_ws;
  decltype(&hoa_paged_attn_fwd) attn;
  decltype(&hoa_path_step) step;
} g_fn{};

struct Device { int sms = 0; int* status = nullptr; };
constexpr int kMaxDevices = 64;
Device g_dev[kMaxDevices];

constexpr size_t kScratchMost = 32u << 20;          // larger ones are allocated for their call alone

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// the device of a call: `t` on the current device, which has been introduced (device()); else -1
int dev_index(const at::Tensor& t) {
  if (!t.is_cuda()) return -1;
  const int i = t.get_device();
  return i >= 0 && i < kMaxDevices && g_dev[i].status != nullptr && c10::cuda::current_device() == i ? i : -1;
}

bool ints(const at::Tensor* t, int idx, at::IntArrayRef shape) {
  return t && t->scalar_type() == at::kInt && t->is_cuda() && t->get_device() == idx && t->sizes() == shape && t->is_contiguous();
}

bool code(const at::Tensor& t, int* c) {
  if (t.scalar_type() == at::kFloat) *c = HOA_F32;
  else if (t.scalar_type() == at::kBFloat16) *c = HOA_BF16;
  else return false;
  return true;
}

// Scratch of a call: one buffer a device and stream, except large ones and under graph capture.  A call enqueues all its
// launches under the interpreter's lock, so no other call's come between them on the stream.  The buffers are never destroyed: at the interpreter's exit the CUDA context may be gone first.
struct Scratch { void* p; at::Tensor keep; };
Scratch scratch(const at::Tensor& like, int idx, cudaStream_t s, size_t n) {
  static auto& held = *new std::map<std::pair<int, cudaStream_t>, at::Tensor>;
  const auto opt = at::TensorOptions().dtype(at::kByte).device(like.device());
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (n <= kScratchMost && cudaStreamIsCapturing(s, &cap) == cudaSuccess && cap == cudaStreamCaptureStatusNone) {
    at::Tensor& t = held[{idx, s}];
    if (!t.defined() || (size_t)t.numel() < n) t = at::empty({(int64_t)(n > (1u << 20) ? n : (1u << 20))}, opt);
    return {t.data_ptr(), at::Tensor()};
  }
  at::Tensor t = at::empty({(int64_t)n}, opt);
  void* p = t.data_ptr();
  return {p, t};
}

PyObject* wrap2(const at::Tensor& a, const at::Tensor& b) {
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(b));
  return r;
}
PyObject* wrap3(const at::Tensor& a, const at::Tensor& b, const at::Tensor& c) {
  PyObject* r = PyTuple_New(3);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(b));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(c));
  return r;
}

struct Books { int idx; int S, W, n_pages; cudaStream_t s; };
bool books(const at::Tensor* table, const at::Tensor* lens, const at::Tensor* refs, bool want_lens, Books* b) {
  if (!table || !refs || table->dim() != 2 || refs->dim() != 1 || table->numel() == 0 || refs->numel() == 0) return false;
  b->idx = dev_index(*table);
  if (b->idx < 0 || table->size(0) > 65536 || table->numel() > 0x7ffffffe || refs->numel() > 0x7ffffffe) return false;
  b->S = (int)table->size(0);
  b->W = (int)table->size(1);
  b->n_pages = (int)refs->size(0);
  if (!ints(table, b->idx, {b->S, b->W}) || !ints(refs, b->idx, {b->n_pages}) || (want_lens && !ints(lens, b->idx, {b->S}))) return false;
  b->s = c10::cuda::getCurrentCUDAStream(b->idx).stream();
  return true;
}

constexpr int kPools = 64;
struct Pools { void* base[kPools]; long long stride[kPools], bytes[kPools]; int n; };
bool pools(PyObject* list, const Books& b, Pools* q) {
  if (!PyList_Check(list) || PyList_GET_SIZE(list) > kPools) return false;
  q->n = (int)PyList_GET_SIZE(list);
  for (int i = 0; i < q->n; ++i) {
    const at::Tensor* t = tensor(PyList_GET_ITEM(list, i));
    if (!t || !t->is_cuda() || t->get_device() != b.idx || t->dim() < 2 || t->size(0) != b.n_pages || !t->is_contiguous()) return false;
    q->base[i] = t->data_ptr();
    q->bytes[i] = (long long)t->numel() / b.n_pages * t->element_size();   // (a pool of one page may have any stride)
    q->stride[i] = (long long)t->stride(0) * t->element_size();
  }
  return true;
}

bool integer(PyObject* o, long long* v) {
  if (!PyLong_Check(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (PyErr_Occurred()) { PyErr_Clear(); return false; }
  return *v >= 1 && *v <= 0x7fffffff;
}

PyObject* status(int st) { return PyLong_FromLong(st); }

// ---------------------------------------------------------------------------
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) { PyErr_SetString(PyExc_TypeError, "bind takes 8 addresses"); return nullptr; }
  void** f = reinterpret_cast<void**>(&g_fn);
  for (int i = 0; i < 8; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  Py_RETURN_NONE;
}

PyObject* device(PyObject*, PyObject* const* a, Py_ssize_t n) {   // index, SM count, address of the mapped status word
  const long i = n == 3 ? PyLong_AsLong(a[0]) : -1, sms = n == 3 ? PyLong_AsLong(a[1]) : 0;
  void* p = n == 3 ? PyLong_AsVoidPtr(a[2]) : nullptr;
  if (PyErr_Occurred()) return nullptr;
  if (i >= 0 && i < kMaxDevices) g_dev[i] = {(int)sms, static_cast<int*>(p)};
  Py_RETURN_NONE;
}

PyObject* pages_reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {   // table, lens, refs, counts, page
  Books b;
  long long page;
  if (n != 5) Py_RETURN_NONE;
  const at::Tensor *table = tensor(a[0]), *lens = tensor(a[1]), *refs = tensor(a[2]), *counts = tensor(a[3]);
  if (!books(table, lens, refs, true, &b) || !ints(counts, b.idx, {b.S}) || !integer(a[4], &page)) Py_RETURN_NONE;
  at::Tensor t = at::empty_like(*table), l = at::empty_like(*lens), r = at::empty_like(*refs);
  const size_t nb = g_fn.pages_ws(b.S, b.n_pages);
  const Scratch ws = scratch(*table, b.idx, b.s, nb);
  const int st = g_fn.reserve(table->data_ptr<int>(), lens->data_ptr<int>(), refs->data_ptr<int>(), counts->data_ptr<int>(),
                              t.data_ptr<int>(), l.data_ptr<int>(), r.data_ptr<int>(), b.S, b.W, b.n_pages, (int)page, ws.p, nb,
                              g_dev[b.idx].status, b.s);
  return st ? status(st) : wrap3(t, l, r);
}

PyObject* pages_fork(PyObject*, PyObject* const* a, Py_ssize_t n) {      // pools, table, lens, refs, src, dst, page
  Books b;
  Pools q;
  long long page;
  if (n != 7) Py_RETURN_NONE;
  const at::Tensor *table = tensor(a[1]), *lens = tensor(a[2]), *refs = tensor(a[3]), *src = tensor(a[4]), *dst = tensor(a[5]);
  if (!books(table, lens, refs, true, &b) || !src || src->numel() > b.S || !ints(src, b.idx, {src->numel()}) ||
      !ints(dst, b.idx, {src->numel()}) || !integer(a[6], &page) || !pools(a[0], b, &q))
    Py_RETURN_NONE;
  const int k = (int)src->numel();
  at::Tensor t = at::empty_like(*table), l = at::empty_like(*lens), r = at::empty_like(*refs);
  const size_t nb = g_fn.pages_ws(k, b.n_pages);
  const Scratch ws = scratch(*table, b.idx, b.s, nb);
  const int st = g_fn.fork(table->data_ptr<int>(), lens->data_ptr<int>(), refs->data_ptr<int>(), src->data_ptr<int>(),
                           dst->data_ptr<int>(), k, t.data_ptr<int>(), l.data_ptr<int>(), r.data_ptr<int>(), b.S, b.W, b.n_pages,
                           (int)page, q.base, q.stride, q.bytes, q.n, ws.p, nb, g_dev[b.idx].status, b.s);
  return st ? status(st) : wrap3(t, l, r);
}

PyObject* pages_free(PyObject*, PyObject* const* a, Py_ssize_t n) {      // table, lens, refs, rows, page
  Books b;
  long long page;
  if (n != 5) Py_RETURN_NONE;
  const at::Tensor *table = tensor(a[0]), *lens = tensor(a[1]), *refs = tensor(a[2]), *rows = tensor(a[3]);
  if (!books(table, lens, refs, true, &b) || !rows || rows->numel() > 0x7fffffff || !ints(rows, b.idx, {rows->numel()}) ||
      !integer(a[4], &page))
    Py_RETURN_NONE;
  at::Tensor t = at::empty_like(*table), l = at::empty_like(*lens), r = at::empty_like(*refs);
  const int st = g_fn.free_(table->data_ptr<int>(), lens->data_ptr<int>(), refs->data_ptr<int>(), rows->data_ptr<int>(),
                            (int)rows->numel(), t.data_ptr<int>(), l.data_ptr<int>(), r.data_ptr<int>(), b.S, b.W, b.n_pages,
                            (int)page, g_dev[b.idx].status, b.s);
  return st ? status(st) : wrap3(t, l, r);
}

PyObject* pages_compact(PyObject*, PyObject* const* a, Py_ssize_t n) {   // pools, table, refs
  Books b;
  Pools q;
  if (n != 3) Py_RETURN_NONE;
  const at::Tensor *table = tensor(a[1]), *refs = tensor(a[2]);
  if (!books(table, nullptr, refs, false, &b) || !pools(a[0], b, &q)) Py_RETURN_NONE;
  at::Tensor t = at::empty_like(*table), r = at::empty_like(*refs), live = at::empty({1}, refs->options());
  const size_t nb = g_fn.pages_ws(0, b.n_pages);
  const Scratch ws = scratch(*table, b.idx, b.s, nb);
  const int st = g_fn.compact(table->data_ptr<int>(), refs->data_ptr<int>(), t.data_ptr<int>(), r.data_ptr<int>(),
                              live.data_ptr<int>(), b.S, b.W, b.n_pages, q.base, q.stride, q.bytes, q.n, ws.p, nb,
                              g_dev[b.idx].status, b.s);
  return st ? status(st) : wrap3(t, r, live);
}

struct Cache { int idx, n_pages, H, page, d, code; long long st[3]; };
bool cache(const at::Tensor* k, const at::Tensor* v, Cache* c) {
  if (!k || !v || k->dim() != 4 || k->numel() == 0 || k->sizes() != v->sizes() || k->strides() != v->strides() ||
      k->scalar_type() != v->scalar_type() || (k->stride(3) != 1 && k->size(3) != 1) || !code(*k, &c->code))
    return false;
  c->idx = dev_index(*k);
  if (c->idx < 0 || !v->is_cuda() || v->get_device() != c->idx) return false;
  for (int i = 0; i < 4; ++i)
    if (k->size(i) > 0x7fffffff) return false;
  c->n_pages = (int)k->size(0); c->H = (int)k->size(1); c->page = (int)k->size(2); c->d = (int)k->size(3);
  for (int i = 0; i < 3; ++i) c->st[i] = k->stride(i);
  return true;
}
bool row_table(const at::Tensor* t, int64_t B, int idx) {
  return t && t->scalar_type() == at::kInt && t->dim() == 2 && t->size(0) == B && t->is_cuda() && t->get_device() == idx &&
         t->size(1) <= 0x7fffffff && (t->size(1) <= 1 || t->stride(1) == 1);
}
bool path(const at::Tensor* t, int idx, at::IntArrayRef shape) {
  return t && t->scalar_type() == at::kFloat && t->is_cuda() && t->get_device() == idx && t->sizes() == shape && t->is_contiguous();
}

// q, k_pages, v_pages, table, lens, scale, shared or None, paths or None (out in q's type)
PyObject* paged_attn_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Cache c;
  if (n != 8 || !PyFloat_Check(a[5])) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *table = tensor(a[3]), *lens = tensor(a[4]);
  const at::Tensor *shared = a[6] == Py_None ? nullptr : tensor(a[6]), *paths = a[7] == Py_None ? nullptr : tensor(a[7]);
  if (!q || q->dim() != 4 || q->numel() == 0 || !cache(k, v, &c) || !q->is_cuda() || q->get_device() != c.idx ||
      q->scalar_type() != k->scalar_type() || q->size(3) != c.d || (c.d > 1 && q->stride(3) != 1) || c.d > 128 ||
      q->size(2) % c.H != 0 || q->numel() > 0x7fffffffffll)
    Py_RETURN_NONE;
  const int64_t B = q->size(0), Tq = q->size(1), H = q->size(2), d = c.d;
  if (B > 0x7fffffff || Tq > 0x7fffffff || H > 0x7fffffff || !row_table(table, B, c.idx) || !ints(lens, c.idx, {B})) Py_RETURN_NONE;
  if (a[6] != Py_None && (!shared || shared->numel() > 0x7fffffff || !ints(shared, c.idx, {shared->numel()}))) Py_RETURN_NONE;
  if (a[7] != Py_None && (Tq != 1 || !path(paths, c.idx, {B, H, d, d}))) Py_RETURN_NONE;
  const cudaStream_t s = c10::cuda::getCurrentCUDAStream(c.idx).stream();
  const int ns = shared ? (int)shared->numel() : 0, W = (int)table->size(1), sms = g_dev[c.idx].sms;
  const size_t nb = g_fn.attn_ws((int)B, (int)Tq, (int)H, c.H, c.d, c.page, ns, W, sms);
  at::Tensor out = at::empty({B, Tq, H, d}, q->options()), lse = at::empty({B, Tq, H}, q->options().dtype(at::kFloat));
  const Scratch ws = scratch(*q, c.idx, s, nb);
  const long long qs[3] = {q->stride(0), q->stride(1), q->stride(2)};
  const int st = g_fn.attn(q->data_ptr(), qs, k->data_ptr(), v->data_ptr(), c.st, c.code, ns ? shared->data_ptr<int>() : nullptr, ns,
                           table->data_ptr<int>(), table->stride(0), W, lens->data_ptr<int>(),
                           paths ? paths->data_ptr<float>() : nullptr, out.data_ptr(), c.code, lse.data_ptr<float>(),
                           (float)PyFloat_AS_DOUBLE(a[5]), (int)B, (int)Tq, (int)H, c.H, c.d, c.page, c.n_pages, sms, ws.p, nb,
                           g_dev[c.idx].status, s);
  return st ? status(st) : wrap2(out, lse);
}

// a, P, qkv, n_heads, edge_scale, k_pages, v_pages, table, lens, P_out or None (packed generators, no bias)
PyObject* path_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Cache c;
  long long heads;
  if (n != 10 || !PyFloat_Check(a[4]) || !integer(a[3], &heads)) Py_RETURN_NONE;
  const at::Tensor *g = tensor(a[0]), *P = tensor(a[1]), *qkv = tensor(a[2]), *k = tensor(a[5]), *v = tensor(a[6]),
                   *table = tensor(a[7]), *lens = tensor(a[8]), *Po = a[9] == Py_None ? nullptr : tensor(a[9]);
  int qcode;
  if (!qkv || !cache(k, v, &c) || c.H != heads || c.d < 2 || c.d > 120 || qkv->dim() != 2 || qkv->size(0) == 0 ||
      qkv->size(1) != 3ll * c.H * c.d || qkv->stride(1) != 1 || !qkv->is_cuda() || qkv->get_device() != c.idx || !code(*qkv, &qcode))
    Py_RETURN_NONE;
  const int64_t B = qkv->size(0), H = c.H, d = c.d;
  if (B * H > 0x7fffffff || !path(g, c.idx, {B, H * (d * (d - 1) / 2)}) || !path(P, c.idx, {B, H, d, d}) ||
      !row_table(table, B, c.idx) || table->size(1) == 0 || !ints(lens, c.idx, {B}) ||
      (a[9] != Py_None && !path(Po, c.idx, {B, H, d, d})))
    Py_RETURN_NONE;
  const cudaStream_t s = c10::cuda::getCurrentCUDAStream(c.idx).stream();
  at::Tensor out = Po ? *Po : at::empty_like(*P), qh = at::empty({B, H, d}, k->options());
  const int st = g_fn.step(g->data_ptr<float>(), HOA_F32, nullptr, (float)PyFloat_AS_DOUBLE(a[4]), P->data_ptr<float>(),
                           out.data_ptr<float>(), qkv->data_ptr(), qcode, qkv->stride(0), qh.data_ptr(), k->data_ptr(), v->data_ptr(),
                           c.code, c.st, table->data_ptr<int>(), table->stride(0), (int)table->size(1), lens->data_ptr<int>(), (int)B,
                           c.H, c.d, c.page, c.n_pages, g_dev[c.idx].status, s);
  return st ? status(st) : wrap2(out, qh);
}

// No C++ exception leaves a function: an allocation that fails (out of memory) or any other error of the tensor
// library becomes None, and the Python function meets it again with its own message.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(self, a, n);
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<f>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(device), METHOD(pages_reserve), METHOD(pages_fork), METHOD(pages_free),
                         METHOD(pages_compact), METHOD(paged_attn_fwd), METHOD(path_step), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hoa_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hoa_torch() { return PyModule_Create(&module); }
