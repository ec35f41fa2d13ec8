// tcb_torch.cpp - the serving entry points of include/tcb.h for torch tensors
// (Python module _tcb_torch, used by tcb_b200/serve.py): the checks on the
// tensors, their addresses and strides, the current stream, and the call.  A
// dozen tensors checked in Python and a call through ctypes took 8 us, longer
// than the kernels of a decode step (4 to 9 us); this takes about 1.  Every
// function returns the library's status; tensors that are not what the entry
// wants raise ValueError before anything is called.
#include <Python.h>

#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "../../include/tcb.h"

namespace {

// the entry points, as libtcb.so was loaded by tcb_b200.lib()
struct Entries {
  decltype(&tcb_page_plan) plan;
  decltype(&tcb_kv_append) append;
  decltype(&tcb_page_attn) attn;
  decltype(&tcb_prefix_attn) prefix;
  decltype(&tcb_logits_penalize) penalize;
} g;

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct Raised {};  // a Python error is set

void need(bool ok, const char *what) {
  if (!ok) throw Refused(what);
}

long whole(PyObject *o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
int whole32(PyObject *o, const char *name) {
  const long v = whole(o);
  if (v != (int)v) throw Refused(std::string(name) + ": a 32-bit whole number is wanted");
  return (int)v;
}
double real(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}
template <class T>
T *address(PyObject *o) {
  void *p = o == Py_None ? nullptr : PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) throw Raised();
  return static_cast<T *>(p);
}

// a CUDA tensor of the context's device
const at::Tensor &tensor(PyObject *o, int device, const char *name) {
  if (!THPVariable_Check(o)) throw Refused(std::string(name) + ": a tensor is wanted");
  const at::Tensor &t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != device) throw Refused(std::string(name) + ": a tensor on the context's CUDA device is wanted");
  return t;
}
template <class T>
T *vec(PyObject *o, int64_t n, at::ScalarType type, int device, const char *name) {
  const at::Tensor &t = tensor(o, device, name);
  if (t.dim() != 1 || t.scalar_type() != type || t.numel() < n || !t.is_contiguous())
    throw Refused(std::string(name) + ": a contiguous " + c10::toString(type) + " vector of at least " + std::to_string(n) + " elements is wanted");
  return static_cast<T *>(t.data_ptr());
}
template <class T>
T *vec_or_none(PyObject *o, int64_t n, at::ScalarType type, int device, const char *name) {
  return o == Py_None ? nullptr : vec<T>(o, n, type, device, name);
}
// a 2-D tensor with dense rows
struct Rows {
  void *p = nullptr;
  int64_t n = 0, width = 0, ld = 0;
};
Rows rows_of(const at::Tensor &t, const char *name) {
  Rows r;
  if (t.dim() == 2) {
    r = {t.data_ptr(), t.size(0), t.size(1), t.size(0) > 1 ? t.stride(0) : t.size(1)};
    if (r.width <= 1 || t.stride(1) == 1) {
      if (r.width > 0x7FFFFFFF) throw Refused(std::string(name) + ": too wide");
      return r;
    }
  }
  throw Refused(std::string(name) + ": a 2-D tensor with dense rows is wanted");
}
Rows rows(PyObject *o, at::ScalarType type, int device, const char *name) {
  const at::Tensor &t = tensor(o, device, name);
  if (t.scalar_type() != type) throw Refused(std::string(name) + ": elements of type " + c10::toString(type) + " are wanted");
  return rows_of(t, name);
}
// the library's number of an activation type, -1 for others
int type_of(const at::Tensor &t) {
  switch (t.scalar_type()) {
  case at::kFloat: return TCB_F32;
  case at::kHalf: return TCB_F16;
  case at::kBFloat16: return TCB_BF16;
  default: return -1;
  }
}

void *stream_of(PyObject *o, int device) {
  if (o == Py_None) return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
  if (PyLong_Check(o)) return address<void>(o);
  PyObject *h = PyObject_GetAttrString(o, "cuda_stream");
  if (!h) throw Raised();
  void *s = PyLong_AsVoidPtr(h);
  Py_DECREF(h);
  if (!s && PyErr_Occurred()) throw Raised();
  return s;
}

template <class F>
int unlocked(F call) {  // the launch queue may be full: other Python threads go on
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = call();
  Py_END_ALLOW_THREADS
  return rc;
}

// q and out of the attention calls
struct Q {
  int T, H;
  const void *q;
  void *out;
  long ldq, ldo;
  bool typed;  // of the cache's type
};
Q queries(const tcb_kv_pages *kv, PyObject *oq, PyObject *oo, int device) {
  const at::Tensor &q = tensor(oq, device, "q"), &o = tensor(oo, device, "out");
  need(q.dim() == 3 && o.dim() == 3 && q.sizes() == o.sizes() && q.size(2) == kv->head_dim, "q and out: [T, H, head dim of the cache] is wanted");
  const int64_t T = q.size(0), H = q.size(1), hd = q.size(2);
  need(T <= 0x7FFFFFFF && H <= 0x7FFFFFFF, "q and out: too many rows or heads");
  for (const at::Tensor *t : {&q, &o}) need(t->stride(2) == 1 && (H == 1 || t->stride(1) == hd), "q and out: dense heads are wanted");
  return {(int)T, (int)H, q.data_ptr(), o.data_ptr(), T > 1 ? (long)q.stride(0) : (long)(H * hd), T > 1 ? (long)o.stride(0) : (long)(H * hd),
          type_of(q) == kv->dtype && type_of(o) == kv->dtype};
}
float scale_of(PyObject *o, int head_dim) {
  return o == Py_None ? (head_dim == 64 ? 0.125f : 0.08838834764831845f) : (float)real(o);  // 1 / sqrt(64), 1 / sqrt(128)
}

int plan(PyObject *const *a) {
  tcb_ctx *ctx = address<tcb_ctx>(a[0]);
  const int dev = whole32(a[1], "device"), page = whole32(a[2], "page");
  const at::Tensor &c = tensor(a[3], dev, "cached"), &s = tensor(a[10], dev, "slots"), &f = tensor(a[6], dev, "free");
  need(c.dim() == 1 && s.dim() == 1 && f.dim() == 1, "cached, slots and free: vectors are wanted");
  const int64_t B = c.size(0), n = s.size(0);
  need(B <= 0x7FFFFFFF && n <= 0x7FFFFFFF && f.numel() <= 0x7FFFFFFF, "cached, slots and free: too long");
  const int *cached = vec<int>(a[3], B, at::kInt, dev, "cached"), *fresh = vec<int>(a[4], B, at::kInt, dev, "fresh");
  const Rows t = rows(a[5], at::kInt, dev, "tables");
  need(t.n >= B, "tables: a row per request is wanted");
  const int *free_pages = vec<int>(a[6], 0, at::kInt, dev, "free"), *n_free = vec<int>(a[7], 1, at::kInt, dev, "n_free");
  int *row_start = vec<int>(a[8], B + 1, at::kInt, dev, "row_start"), *kv_len = vec<int>(a[9], B, at::kInt, dev, "kv_len");
  int64_t *slots = vec<int64_t>(a[10], n, at::kLong, dev, "slots");
  int *positions = vec<int>(a[11], n, at::kInt, dev, "positions"), *balance = vec<int>(a[12], 1, at::kInt, dev, "balance");
  int *taken = vec_or_none<int>(a[13], 1, at::kInt, dev, "taken");
  void *stream = stream_of(a[14], dev);
  return unlocked([&] {
    return g.plan(ctx, (int)B, page, cached, fresh, static_cast<int *>(t.p), (int)t.width, (long)t.ld, free_pages, (int)f.numel(), n_free, (int)n,
                  row_start, kv_len, slots, positions, balance, taken, stream);
  });
}

int append(PyObject *const *a) {
  tcb_ctx *ctx = address<tcb_ctx>(a[0]);
  const int dev = whole32(a[1], "device");
  const tcb_kv_pages *kv = address<const tcb_kv_pages>(a[2]);
  const at::Tensor &k = tensor(a[3], dev, "k"), &v = tensor(a[4], dev, "v");
  const Rows rk = rows_of(k, "k"), rv = rows_of(v, "v");
  need(rk.n == rv.n && rk.width == rv.width && rk.width == (int64_t)kv->n_kv_heads * kv->head_dim && rk.n <= 0x7FFFFFFF,
       "k and v: two [T, KV heads * head dim] tensors are wanted");
  if (type_of(k) < 0 || k.scalar_type() != v.scalar_type()) return TCB_ERR_DTYPE;
  const int64_t *slots = vec<int64_t>(a[5], rk.n, at::kLong, dev, "slots");
  void *stream = stream_of(a[6], dev);
  return unlocked([&] { return g.append(ctx, kv, (int)rk.n, rk.p, (long)rk.ld, rv.p, (long)rv.ld, type_of(k), slots, stream); });
}

int attend(PyObject *const *a) {
  tcb_ctx *ctx = address<tcb_ctx>(a[0]);
  const int dev = whole32(a[1], "device");
  const tcb_kv_pages *kv = address<const tcb_kv_pages>(a[2]);
  const Q q = queries(kv, a[3], a[4], dev);
  if (!q.typed) return TCB_ERR_DTYPE;
  const at::Tensor &len = tensor(a[6], dev, "kv_len");
  need(len.dim() == 1 && len.size(0) <= 0x7FFFFFFF, "kv_len: a vector is wanted");
  const int B = (int)len.size(0);
  const int *row_start = vec<int>(a[5], B + 1l, at::kInt, dev, "row_start"), *kv_len = vec<int>(a[6], B, at::kInt, dev, "kv_len");
  const Rows t = rows(a[7], at::kInt, dev, "tables");
  need(t.n >= B, "tables: a row per request is wanted");
  const int max_rows = whole32(a[8], "max_rows"), max_len = whole32(a[9], "max_len");
  const float scale = scale_of(a[10], kv->head_dim);
  const int window = a[11] == Py_None ? -1 : whole32(a[11], "window"), sinks = whole32(a[12], "sinks");
  need(a[11] == Py_None || window >= 0, "window: None or a whole number from 0 is wanted");
  void *stream = stream_of(a[13], dev);
  return unlocked([&] {
    return g.attn(ctx, kv, B, q.T, q.H, q.q, q.ldq, q.out, q.ldo, row_start, kv_len, static_cast<int *>(t.p), (int)t.width, (long)t.ld, max_rows,
                  max_len, scale, window, sinks, stream);
  });
}

int attend_prefix(PyObject *const *a) {
  tcb_ctx *ctx = address<tcb_ctx>(a[0]);
  const int dev = whole32(a[1], "device");
  const tcb_kv_pages *kv = address<const tcb_kv_pages>(a[2]);
  const Q q = queries(kv, a[3], a[4], dev);
  if (!q.typed) return TCB_ERR_DTYPE;
  const int prefix_len = whole32(a[6], "prefix_len");
  need(prefix_len >= 0, "prefix_len: a whole number from 0 is wanted");
  // pools without positions are the entry's to refuse
  const int64_t pages = kv->page > 0 ? ((int64_t)prefix_len + kv->page - 1) / kv->page : 0;
  const int *prefix = vec<int>(a[5], pages, at::kInt, dev, "prefix");
  const int *kv_len = vec<int>(a[7], q.T, at::kInt, dev, "kv_len");
  const Rows t = rows(a[8], at::kInt, dev, "tables");
  need(t.n >= q.T, "tables: a row per request is wanted");
  const int max_len = whole32(a[9], "max_len");
  const float scale = scale_of(a[10], kv->head_dim);
  void *stream = stream_of(a[11], dev);
  return unlocked([&] {
    return g.prefix(ctx, kv, q.T, q.H, q.q, q.ldq, q.out, q.ldo, prefix, prefix_len, kv_len, static_cast<int *>(t.p), (int)t.width, (long)t.ld,
                    max_len, scale, stream);
  });
}

int penalize(PyObject *const *a) {
  tcb_ctx *ctx = address<tcb_ctx>(a[0]);
  const int dev = whole32(a[1], "device");
  const at::Tensor &x = tensor(a[2], dev, "logits"), &o = tensor(a[3], dev, "out");
  const Rows rx = rows_of(x, "logits"), ro = rows_of(o, "out");
  need(rx.n == ro.n && rx.width == ro.width && rx.n <= 0x7FFFFFFF, "logits and out: two [B, V] tensors are wanted");
  if (type_of(x) < 0 || type_of(o) < 0) return TCB_ERR_DTYPE;
  tcb_logits_args p = {};
  const int64_t B = rx.n;
  p.B = (int)B, p.V = (int)rx.width;
  p.logits = rx.p, p.dtype = type_of(x), p.ld = rx.ld;
  p.out = ro.p, p.odtype = type_of(o), p.ldo = ro.ld;
  p.token = vec_or_none<int64_t>(a[4], B, at::kLong, dev, "token");
  if (a[5] != Py_None) {
    const Rows h = rows(a[5], at::kLong, dev, "history");
    need(h.n >= B && a[7] != Py_None, "history: a row per sequence and total_len are wanted");
    p.history = static_cast<const int64_t *>(h.p), p.hist_width = (int)h.width, p.ldh = h.ld;
    if (h.width == 0) p.history = nullptr;
  }
  p.prompt_len = vec_or_none<int>(a[6], B, at::kInt, dev, "prompt_len");
  p.total_len = vec_or_none<int>(a[7], B, at::kInt, dev, "total_len");
  p.repetition = vec_or_none<float>(a[8], B, at::kFloat, dev, "repetition");
  p.frequency = vec_or_none<float>(a[9], B, at::kFloat, dev, "frequency");
  p.presence = vec_or_none<float>(a[10], B, at::kFloat, dev, "presence");
  if (a[11] != Py_None) {
    const Rows i = rows(a[11], at::kInt, dev, "bias_ids"), v = rows(a[12], at::kFloat, dev, "bias");
    need(i.width == v.width && i.ld == v.ld && i.n >= B && v.n >= B, "bias_ids and bias: two tensors of one shape and stride are wanted");
    p.bias_ids = static_cast<const int *>(i.p), p.bias = static_cast<const float *>(v.p), p.n_bias = (int)i.width, p.ldb = i.ld;
  }
  if (a[13] != Py_None) {
    const Rows m = rows(a[13], at::kInt, dev, "mask");
    need(m.width >= (rx.width + 31) / 32 && m.n <= 0x7FFFFFFF && (a[14] != Py_None || m.n >= B),
         "mask: ceil(V / 32) words in a row, and a row per sequence or mask_row, are wanted");
    p.mask = static_cast<const uint32_t *>(m.p), p.n_masks = (int)m.n, p.ldm = m.ld;
  }
  p.mask_row = vec_or_none<int>(a[14], B, at::kInt, dev, "mask_row");
  void *stream = stream_of(a[15], dev);
  return unlocked([&] { return g.penalize(ctx, &p, stream); });
}

// a function of n positional arguments; C++ exceptions end here
template <int (*F)(PyObject *const *), int N>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments are wanted, got %zd", N, n);
    return nullptr;
  }
  try {
    return PyLong_FromLong(F(args));
  } catch (const Raised &) {
  } catch (const Refused &e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

int bind(PyObject *const *a) {
  g.plan = reinterpret_cast<decltype(g.plan)>(address<void>(a[0]));
  g.append = reinterpret_cast<decltype(g.append)>(address<void>(a[1]));
  g.attn = reinterpret_cast<decltype(g.attn)>(address<void>(a[2]));
  g.prefix = reinterpret_cast<decltype(g.prefix)>(address<void>(a[3]));
  g.penalize = reinterpret_cast<decltype(g.penalize)>(address<void>(a[4]));
  return TCB_OK;
}

template <int (*F)(PyObject *const *), int N>
PyCFunction as_method() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>));
}

PyMethodDef methods[] = {{"bind", as_method<bind, 5>(), METH_FASTCALL, "addresses of the library's entry points"},
                         {"plan", as_method<plan, 15>(), METH_FASTCALL, "tcb_page_plan"},
                         {"append", as_method<append, 7>(), METH_FASTCALL, "tcb_kv_append"},
                         {"attend", as_method<attend, 14>(), METH_FASTCALL, "tcb_page_attn"},
                         {"attend_prefix", as_method<attend_prefix, 12>(), METH_FASTCALL, "tcb_prefix_attn"},
                         {"penalize", as_method<penalize, 16>(), METH_FASTCALL, "tcb_logits_penalize"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tcb_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tcb_torch() { return PyModule_Create(&module); }
