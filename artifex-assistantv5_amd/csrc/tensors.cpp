// _tensors: calls of the paged and sampling entry points straight from torch tensors.
//
// Each function takes the arguments of its namesake in paged.py or sampling.py, all of them, checks
// what that one checks, and calls the entry point on the current stream.  It returns True if the call
// has been made, and False with nothing done where the arguments do not fit: the Python function then
// makes its own checks, which name what is wrong, and the calls whose device is not the current one.
// A call that failed otherwise may have launched some of its kernels, so it is not to be made again:
// it raises what `on_failure` was given for that.
//
// Checks in Python, tensor by tensor, and the arguments' packing cost 4 us a call, more than the smaller
// kernels take.  us of calls from Python, before and with these: attention over 300 slots 10.4, 8.5; 146
// rows stored and 246 read back 16.3, 9.9; a fork and room for 4 sequences 18.9, 12.9; compaction of 74
// pages 12.3, 9.4.
#include <torch/csrc/autograd/python_variable.h>

#include <cfloat>
#include <cmath>

#include "gguf_hip_paged.h"
#include "gguf_hip_sample.h"

namespace {

// The entry points, of the library that is loaded, and torch's current device and stream.
struct Entries {
  decltype(&gguf_hip_paged_append) append;
  decltype(&gguf_hip_paged_attention) attention;
  decltype(&gguf_hip_paged_load) load;
  decltype(&gguf_hip_paged_fork) fork;
  decltype(&gguf_hip_paged_grow) grow;
  decltype(&gguf_hip_paged_compact) compact;
  decltype(&gguf_hip_sample) sample;
} entry;
constexpr int kEntries = sizeof(Entries) / sizeof(void *);
PyObject *current_device, *current_stream;
PyObject *failure;  // called with an entry point's code, raises

using at::ScalarType;

// The arguments of a call.  What does not fit clears `ok`; what is read after that is zero.
struct Args {
  PyObject *const *a;
  bool ok;
  int device = -1;

  Args(PyObject *const *args, Py_ssize_t n, int want) : a(args), ok(n == want && entry.append) {}

  bool none(int i) const { return a[i] == Py_None; }
  bool is_tensor(int i) const { return THPVariable_Check(a[i]); }
  // A tensor on the call's device, which is the first one's.
  const at::Tensor *tensor(int i) {
    if (!ok || !is_tensor(i)) return ok = false, nullptr;
    const at::Tensor &t = THPVariable_Unpack(a[i]);
    if (!t.is_cuda() || t.layout() != at::kStrided) return ok = false, nullptr;
    if (device < 0) device = t.get_device();
    if (t.get_device() != device) return ok = false, nullptr;
    return &t;
  }
  // Contiguous, of that type and shape.
  void *array(int i, ScalarType type, at::IntArrayRef shape) {
    const at::Tensor *t = tensor(i);
    if (!t || t->scalar_type() != type || t->sizes() != shape || !t->is_contiguous())
      return ok = false, nullptr;
    return t->data_ptr();
  }
  void *optional(int i, ScalarType type, at::IntArrayRef shape) {
    return !ok || none(i) ? nullptr : array(i, type, shape);
  }
  template <typename T>
  T *ints(int i, at::IntArrayRef shape) {
    return (T *)array(i, sizeof(T) == 8 ? ScalarType::Long : ScalarType::Int, shape);
  }
  template <typename T>
  T *ints_or_none(int i, at::IntArrayRef shape) {
    return !ok || none(i) ? nullptr : ints<T>(i, shape);
  }
  // f32 rows of at least `width` values; `n` of them (any number: -1, which is set).
  float *rows(int i, int64_t &n, int64_t width, int64_t &ld) {
    const at::Tensor *t = tensor(i);
    if (!t || t->scalar_type() != ScalarType::Float || t->dim() != 2) return ok = false, nullptr;
    const int64_t columns = t->size(1);
    ld = t->size(0) <= 1 ? columns : t->stride(0);
    if (n < 0) n = t->size(0);
    if (t->size(0) != n || columns < width || ld < columns || t->stride(1) != 1) return ok = false, nullptr;
    return (float *)t->data_ptr();
  }
  // RoPE tables [positions, head_dim / 2]; sin comes after cos.
  const float *rope(int i, int64_t half, int64_t &positions, const float *&sin) {
    const at::Tensor *t = tensor(i);
    if (!t || t->dim() != 2) return ok = false, nullptr;
    positions = t->size(0);
    const float *cos = (const float *)array(i, ScalarType::Float, {positions, half});
    sin = (const float *)array(i + 1, ScalarType::Float, {positions, half});
    return cos;
  }
  void *work(int i, int64_t &bytes) {
    const at::Tensor *t = tensor(i);
    if (!t || !t->is_contiguous()) return ok = false, nullptr;
    bytes = (int64_t)t->nbytes();
    return t->data_ptr();
  }
  int32_t number(int i) {
    if (!ok || !PyLong_Check(a[i])) return ok = false, 0;
    const long long v = PyLong_AsLongLong(a[i]);
    if (PyErr_Occurred() || v != (int32_t)v) PyErr_Clear(), ok = false;
    return (int32_t)v;
  }
  float real(int i) {
    if (!ok || !(PyFloat_Check(a[i]) || PyLong_Check(a[i]))) return ok = false, 0.f;
    const double v = PyFloat_AsDouble(a[i]);
    if (PyErr_Occurred() || (std::isfinite(v) && std::fabs(v) > FLT_MAX)) PyErr_Clear(), ok = false;
    return (float)v;
  }
  // torch's current stream, where the tensors' device is the current one.
  void *stream() {
    if (!ok || device < 0) return ok = false, nullptr;
    void *s = nullptr;
    PyObject *d = PyObject_CallNoArgs(current_device);
    ok = d && PyLong_AsLong(d) == device;
    if (PyObject *r = ok ? PyObject_CallOneArg(current_stream, d) : nullptr) {
      s = PyLong_AsVoidPtr(r);
      Py_DECREF(r);
    } else {
      ok = false;
    }
    Py_XDECREF(d);
    if (PyErr_Occurred()) PyErr_Clear(), ok = false;
    return s;
  }
};

// A pool [n_pages, 2, n_kv_heads, page, head_dim], or [n_layers, ..].
struct Pool {
  void *kv = nullptr;
  int64_t pages = 0, page = 0, heads = 0, hd = 0, layers = 1;
  int dtype = 0;
  Pool(Args &x, int i, bool several = false) {
    const at::Tensor *t = x.tensor(i);
    const int more = t && several && t->dim() == 6;
    if (!t || t->dim() != 5 + more || !t->is_contiguous() || t->size(more + 1) != 2) {
      x.ok = false;
      return;
    }
    dtype = t->scalar_type() == ScalarType::Half       ? GGUF_HIP_PAGED_F16
            : t->scalar_type() == ScalarType::BFloat16 ? GGUF_HIP_PAGED_BF16
                                                       : 0;
    if (more) layers = t->size(0);
    pages = t->size(more), heads = t->size(more + 2), page = t->size(more + 3), hd = t->size(more + 4);
    kv = t->data_ptr();
    for (int64_t n : {layers, pages, page, heads, hd})
      if (n <= 0 || n > INT32_MAX) x.ok = false;
    if (!dtype) x.ok = false;
  }
};
struct Tables {
  int64_t n = 0, columns = 0;
  int32_t *p = nullptr;
  Tables(Args &x, int i) {
    const at::Tensor *t = x.tensor(i);
    if (!t || t->dim() != 2) {
      x.ok = false;
      return;
    }
    n = t->size(0), columns = t->size(1);
    p = x.ints<int32_t>(i, {n, columns});
    if (n > INT32_MAX) x.ok = false;
  }
};

// The call, if everything fits, without the interpreter's lock; no exception of C++ passes.
constexpr int kRefused = 1;  // no code of an entry point
template <typename F>
PyObject *guarded(F make) {
  int rc = kRefused;
  try {
    rc = make();
  } catch (...) {
  }
  if (PyErr_Occurred()) PyErr_Clear();
  if (rc == GGUF_HIP_OK || rc == kRefused) return PyBool_FromLong(rc == GGUF_HIP_OK);
  PyObject *r = failure ? PyObject_CallFunction(failure, "i", rc) : nullptr;
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "a call failed with %d", rc);
  return nullptr;
}
template <typename E, typename... T>
int launch(Args &x, E call, T... args) {
  void *stream = x.stream();
  if (!x.ok) return kRefused;
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = call(args..., stream);
  Py_END_ALLOW_THREADS;
  return rc <= GGUF_HIP_ERR_TYPE && rc >= GGUF_HIP_ERR_BYTES ? kRefused : rc;  // by its own checks
}

PyObject *append(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&] {  // qkv, lengths, tables, cos, sin, kv, n_heads, starts, room
    Args x(args, n, 9);
    const Pool c(x, 5);
    const Tables t(x, 2);
    const int32_t heads = x.number(6);
    int64_t count = -1, ld = 0, positions = 0;
    const float *qkv = x.rows(0, count, (heads + 2 * c.heads) * c.hd, ld), *sin;
    const int64_t *lengths = x.ints<int64_t>(1, {t.n}), *starts = x.ints_or_none<int64_t>(7, {t.n + 1}),
                  *room = x.ints_or_none<int64_t>(8, {t.n});
    const float *cos = x.rope(3, c.hd / 2, positions, sin);
    return launch(x, entry.append, qkv, ld, count, starts, lengths, room, t.p, cos, sin, positions, c.kv,
                  c.dtype, c.pages, (int)c.page, t.columns, (int)t.n, heads, (int)c.heads, (int)c.hd);
  });
}

PyObject *attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&] {  // qkv, lengths, tables, cos, sin, kv, out, n_heads, work, room
    Args x(args, n, 10);
    const Pool c(x, 5);
    const Tables t(x, 2);
    const int32_t heads = x.number(7);
    int64_t count = t.n, ld = 0, ldo = 0, positions = 0, bytes = 0;
    const float *qkv = x.rows(0, count, (heads + 2 * c.heads) * c.hd, ld), *sin;
    float *out = x.rows(6, count, heads * c.hd, ldo);
    const int64_t *lengths = x.ints<int64_t>(1, {t.n}), *room = x.ints_or_none<int64_t>(9, {t.n});
    const float *cos = x.rope(3, c.hd / 2, positions, sin);
    void *work = x.work(8, bytes);
    return launch(x, entry.attention, qkv, ld, lengths, room, t.p, cos, sin, positions, c.kv, c.dtype, out,
                  ldo, c.pages, (int)c.page, t.columns, (int)t.n, heads, (int)c.heads, (int)c.hd, work, bytes);
  });
}

PyObject *load(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&] {  // kv, tables, lengths, k_out, v_out
    Args x(args, n, 5);
    const Pool c(x, 0);
    const Tables t(x, 1);
    const at::Tensor *k = x.tensor(3);
    const int64_t slots = k && k->dim() == 4 ? k->size(2) : 0;
    float *ko = (float *)x.array(3, ScalarType::Float, {t.n, c.heads, slots, c.hd});
    float *vo = (float *)x.array(4, ScalarType::Float, {t.n, c.heads, slots, c.hd});
    const int64_t *lengths = x.ints<int64_t>(2, {t.n});
    return launch(x, entry.load, c.kv, c.dtype, t.p, lengths, ko, vo, slots, c.pages, (int)c.page, t.columns,
                  (int)t.n, (int)c.heads, (int)c.hd);
  });
}

PyObject *fork(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&] {  // tables, lengths, refs, parents, tables_out, lengths_out, refs_out
    Args x(args, n, 7);
    const Tables t(x, 0);
    const at::Tensor *r = x.tensor(2);
    const int64_t pages = r && r->dim() == 1 ? r->size(0) : 0;
    int64_t *lengths = x.ints<int64_t>(1, {t.n});
    int32_t *refs = x.ints<int32_t>(2, {pages});
    const int64_t *parents = x.ints<int64_t>(3, {t.n});
    int32_t *to = x.ints_or_none<int32_t>(4, {t.n, t.columns});
    int64_t *lo = x.ints_or_none<int64_t>(5, {t.n});
    int32_t *ro = x.ints_or_none<int32_t>(6, {pages});
    return launch(x, entry.fork, t.p, lengths, refs, parents, to ? to : t.p, lo ? lo : lengths,
                  ro ? ro : refs, pages, t.columns, (int)t.n);
  });
}

PyObject *grow(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&] {  // kv, tables, lengths, refs, rows, room, work
    Args x(args, n, 7);
    const Pool c(x, 0, true);
    const Tables t(x, 1);
    const int64_t *lengths = x.ints<int64_t>(2, {t.n});
    int32_t *refs = x.ints<int32_t>(3, {c.pages});
    const int64_t *rows = x.ints<int64_t>(4, {t.n});
    int64_t *room = x.ints<int64_t>(5, {t.n}), bytes = 0;
    void *work = x.work(6, bytes);
    return launch(x, entry.grow, c.kv, t.p, lengths, refs, rows, room, (int)c.layers, c.pages, (int)c.page,
                  t.columns, (int)t.n, (int)c.heads, (int)c.hd, work, bytes);
  });
}

PyObject *compact(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&] {  // kv, tables, refs, live, work, tables_out, refs_out
    Args x(args, n, 7);
    const Pool c(x, 0, true);
    const Tables t(x, 1);
    int32_t *refs = x.ints<int32_t>(2, {c.pages});
    int64_t *live = x.ints<int64_t>(3, {1}), bytes = 0;
    void *work = x.work(4, bytes);
    int32_t *to = x.ints_or_none<int32_t>(5, {t.n, t.columns}), *ro = x.ints_or_none<int32_t>(6, {c.pages});
    return launch(x, entry.compact, c.kv, t.p, refs, to ? to : t.p, ro ? ro : refs, live, (int)c.layers,
                  c.pages, (int)c.page, t.columns, (int)t.n, (int)c.heads, (int)c.hd, work, bytes);
  });
}

PyObject *sample(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return guarded([&] {  // logits, u, out, work, temperature, top_k, top_p, min_p, probs
    Args x(args, n, 9);
    int64_t count = -1, ld = 0, bytes = 0;
    const float *logits = x.rows(0, count, 1, ld);
    const int64_t vocab = x.ok ? THPVariable_Unpack(args[0]).size(1) : 0;
    const float *u = (const float *)x.array(1, ScalarType::Float, {count});
    int64_t *out = x.ints<int64_t>(2, {count});
    void *work = x.work(3, bytes);
    const float *each[3];  // a setting's array, or its value for all
    float all[3] = {};
    for (int i = 0, at = 4; i < 3; ++i, at = i + 5) {
      each[i] = x.ok && x.is_tensor(at) ? (const float *)x.array(at, ScalarType::Float, {count}) : nullptr;
      if (x.ok && !each[i]) all[i] = x.real(at);
    }
    const int32_t *top_k = x.ok && x.is_tensor(5) ? x.ints<int32_t>(5, {count}) : nullptr;
    const int32_t top_k_all = x.ok && !top_k ? x.number(5) : 0;
    float *probs = (float *)x.optional(8, ScalarType::Float, {count});
    if (!count) x.ok = false;  // its settings have no addresses
    return launch(x, entry.sample, logits, ld, count, vocab, u, each[0], all[0], top_k,
                  top_k_all > 0 ? top_k_all : 0, each[1], all[1], each[2], all[2], out, probs, work, bytes);
  });
}

// The addresses of the library's entry points, in the order of Entries.
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != kEntries) return PyErr_Format(PyExc_TypeError, "%d addresses", kEntries);
  void *p[kEntries];
  for (int i = 0; i < kEntries; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null address");
      return nullptr;
    }
  }
  memcpy(&entry, p, sizeof entry);
  Py_RETURN_NONE;
}

// What a failed call raises by: called with its code.
PyObject *on_failure(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != 1 || !PyCallable_Check(args[0])) return PyErr_Format(PyExc_TypeError, "one callable");
  Py_INCREF(args[0]);
  Py_XDECREF(failure);
  failure = args[0];
  Py_RETURN_NONE;
}

#define FUNCTION(name) {#name, (PyCFunction)(void *)name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FUNCTION(append), FUNCTION(attention), FUNCTION(load),   FUNCTION(fork),
                         FUNCTION(grow),   FUNCTION(compact),   FUNCTION(sample), FUNCTION(bind),
                         FUNCTION(on_failure), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) {
  PyObject *torch = PyImport_ImportModule("torch._C");
  if (!torch) return nullptr;
  current_device = PyObject_GetAttrString(torch, "_cuda_getDevice");
  current_stream = PyObject_GetAttrString(torch, "_cuda_getCurrentRawStream");
  Py_DECREF(torch);
  if (!current_device || !current_stream) return nullptr;
  return PyModule_Create(&module);
}
