// CPython module _gcb200_host: the call path of the small, repeated calls (one matmul, one attention, one execute of a
// partition) from Python objects to the C ABI of libGcDnnlApi.so.
//
// Through ctypes a call spends 8 us (matmul, four tensors) to 50 us (execute, a dozen tensors) on attribute look-ups,
// argument conversion and structure building in the interpreter - more than the kernels of a small problem.  Here the
// tensors' addresses and shapes go straight into C structures.  Only the C API of Python is used: no torch headers, no
// ABI beyond the methods data_ptr / shape / is_cuda / dtype / is_contiguous of the tensors.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstddef>
#include <cstdint>

#include "../../include/dnnl_graph_compiler.h"
#include "../../include/gc_b200.h"

namespace {

// interned names and cached objects of the torch module (set by setup())
PyObject *s_data_ptr, *s_shape, *s_is_cuda, *s_dtype, *s_is_contiguous, *s_stride, *s_get_device;
PyObject *t_tensor, *t_bf16, *f_get_device, *f_raw_stream, *t_ndarray;
PyObject *t_f16, *t_e4m3, *t_i32, *t_f32, *t_f64, *t_u8;

struct Ref {   // owned reference
  PyObject *p;
  explicit Ref(PyObject *o) : p(o) {}
  ~Ref() { Py_XDECREF(p); }
  Ref(const Ref &) = delete;
  operator PyObject *() const { return p; }
};

bool address(PyObject *t, void **out) {
  Ref r(PyObject_CallMethodNoArgs(t, s_data_ptr));
  if (!r.p) return false;
  *out = PyLong_AsVoidPtr(r);
  return !PyErr_Occurred();
}
// Shape of a tensor; -1 on error, -2 when it has more than `cap` dimensions.
int shape(PyObject *t, int64_t *dims, int cap) {
  Ref r(PyObject_GetAttr(t, s_shape));
  if (!r.p) return -1;
  if (!PyTuple_Check(r.p)) {
    PyErr_SetString(PyExc_TypeError, "shape is not a tuple");
    return -1;
  }
  const Py_ssize_t n = PyTuple_GET_SIZE(r.p);
  if (n > cap) return -2;
  for (Py_ssize_t i = 0; i < n; ++i) {
    dims[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(r.p, i));
    if (dims[i] == -1 && PyErr_Occurred()) return -1;
  }
  return int(n);
}
bool is_true(PyObject *t, PyObject *attr, bool call, bool *out) {
  Ref r(call ? PyObject_CallMethodNoArgs(t, attr) : PyObject_GetAttr(t, attr));
  if (!r.p) return false;
  *out = r.p == Py_True;
  return true;
}
bool require(bool ok, const char *what) {
  if (!ok) PyErr_SetString(PyExc_AssertionError, what);
  return ok;
}
// A bf16 CUDA tensor (contiguous): its address and two-dimensional or larger shape.
bool operand(PyObject *t, bool check_type, void **ptr, int64_t *dims, int *nd) {
  bool v = false;
  if (check_type) {
    if (!is_true(t, s_is_cuda, false, &v) || !require(v, "the operands must be CUDA tensors")) return false;
    Ref dt(PyObject_GetAttr(t, s_dtype));
    if (!dt.p || !require(dt.p == t_bf16, "the operands must be bfloat16")) return false;
  }
  if (!is_true(t, s_is_contiguous, true, &v) || !require(v, "the operands must be contiguous")) return false;
  *nd = shape(t, dims, DNNL_MAX_NDIMS);
  if (*nd == -2) PyErr_SetString(PyExc_ValueError, "too many dimensions");
  return *nd >= 0 && address(t, ptr);
}
bool current_stream(void **out) {
  Ref dev(PyObject_CallNoArgs(f_get_device));
  if (!dev.p) return false;
  Ref st(PyObject_CallOneArg(f_raw_stream, dev));
  if (!st.p) return false;
  *out = PyLong_AsVoidPtr(st);
  return !PyErr_Occurred();
}

// matmul_bf16(A, B, bias | None, relu, transpose_a, transpose_b, out) -> status
PyObject *matmul_bf16(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 7) return PyErr_Format(PyExc_TypeError, "matmul_bf16 takes 7 arguments"), nullptr;
  void *pa, *pb, *pbias = nullptr, *po, *stream;
  int64_t da[DNNL_MAX_NDIMS], db[DNNL_MAX_NDIMS];
  int na, nb;
  const int relu = PyObject_IsTrue(a[3]), ta = PyObject_IsTrue(a[4]), tb = PyObject_IsTrue(a[5]);
  if (relu < 0 || ta < 0 || tb < 0) return nullptr;
  if (!operand(a[0], true, &pa, da, &na) || !operand(a[1], false, &pb, db, &nb)) return nullptr;
  if (!require(na == 2 && nb == 2, "the operands must be matrices")) return nullptr;
  const int64_t M = ta ? da[1] : da[0], K = ta ? da[0] : da[1], N = tb ? db[0] : db[1];
  if (!require((tb ? db[1] : db[0]) == K, "inner dimensions differ")) return nullptr;
  if (a[2] != Py_None && !address(a[2], &pbias)) return nullptr;
  if (!address(a[6], &po) || !current_stream(&stream)) return nullptr;
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = gcb200_matmul_bf16(pa, pb, pbias, po, M, N, K, ta, tb, relu, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// attention_bf16(Q, K, V, scale, causal, out) -> status
PyObject *attention_bf16(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 6) return PyErr_Format(PyExc_TypeError, "attention_bf16 takes 6 arguments"), nullptr;
  void *q, *k, *v, *o, *stream;
  int64_t d[DNNL_MAX_NDIMS];
  int nd;
  if (!operand(a[1], false, &k, d, &nd) || !operand(a[2], false, &v, d, &nd) || !operand(a[0], true, &q, d, &nd)) return nullptr;
  if (!require(nd >= 2, "Q must have at least two dimensions")) return nullptr;
  const double scale = PyFloat_AsDouble(a[3]);
  const int causal = PyObject_IsTrue(a[4]);
  if (PyErr_Occurred() || causal < 0 || !address(a[5], &o) || !current_stream(&stream)) return nullptr;
  int64_t bh = 1;
  for (int i = 0; i + 2 < nd; ++i) bh *= d[i];
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = gcb200_attention_bf16(q, k, v, o, bh, d[nd - 2], d[nd - 1], float(scale), causal, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// ----------------------------------------------------------------------------- decode operators
// A strided tensor on the current device.
struct View {
  void *ptr = nullptr;
  int nd = 0;
  int64_t dims[4] = {}, strides[4] = {};
  PyObject *dtype = nullptr;   // one of the torch module's: it outlives the call
};
bool say(const char *name, const char *what) {
  PyErr_Format(PyExc_AssertionError, "%s %s", name, what);
  return false;
}
// `device`: the current device's number.  The tensor must have `nd` dimensions and a dense last one.
bool view(PyObject *t, const char *name, int nd, long device, View *v) {
  if (!PyObject_TypeCheck(t, reinterpret_cast<PyTypeObject *>(t_tensor))) return say(name, "must be a tensor");
  Ref dev(PyObject_CallMethodNoArgs(t, s_get_device));
  if (!dev.p) return false;
  if (PyLong_AsLong(dev) != device) return say(name, "must be on the current CUDA device");
  v->nd = shape(t, v->dims, 4);
  if (v->nd == -1) return false;
  if (v->nd != nd) return say(name, "has another number of dimensions than it should");
  Ref st(PyObject_CallMethodNoArgs(t, s_stride));
  if (!st.p || !PyTuple_Check(st.p)) return false;
  for (int i = 0; i < nd; ++i) v->strides[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(st.p, i));
  if (v->dims[nd - 1] > 1 && v->strides[nd - 1] != 1) return say(name, "must be contiguous in its last dimension");
  Ref dt(PyObject_GetAttr(t, s_dtype));
  if (!dt.p) return false;
  v->dtype = dt.p;
  return address(t, &v->ptr) && !PyErr_Occurred();
}
// The same for None or a contiguous vector of `n` elements.
bool vector(PyObject *t, const char *name, PyObject *dtype, int64_t n, long device, void **ptr) {
  *ptr = nullptr;
  if (t == Py_None) return true;
  View v;
  if (!view(t, name, 1, device, &v)) return false;
  if (v.dtype != dtype) return say(name, "has the wrong type");
  if (v.dims[0] != n) return say(name, "has the wrong length");
  *ptr = v.ptr;
  return true;
}
bool current_device(long *device) {
  if (t_f16 == nullptr) {
    PyErr_SetString(PyExc_RuntimeError, "torch is not loaded");
    return false;
  }
  Ref dev(PyObject_CallNoArgs(f_get_device));
  if (!dev.p) return false;
  *device = PyLong_AsLong(dev);
  return !PyErr_Occurred();
}
int dtype_code(PyObject *t) { return t == t_bf16 ? GCB200_BF16 : t == t_f16 ? GCB200_F16 : t == t_e4m3 ? GCB200_F8_E4M3 : 0; }
// The cache of a call whose queries, keys or values are `dtype`.
bool cache_of(PyObject *keys, PyObject *values, PyObject *table, PyObject *key_scale, PyObject *value_scale, PyObject *dtype, long device,
              gcb200_paged_cache *c) {
  View k, v, t;
  if (!view(keys, "key_cache", 4, device, &k) || !view(values, "value_cache", 4, device, &v) || !view(table, "page_table", 2, device, &t)) return false;
  c->dtype = dtype_code(dtype);
  if (c->dtype != GCB200_BF16 && c->dtype != GCB200_F16) return say("queries, keys and values", "must be bfloat16 or float16");
  c->cache_dtype = dtype_code(k.dtype);
  if (k.dtype != v.dtype) return say("key_cache and value_cache", "must have the same type");
  if (c->cache_dtype != c->dtype && c->cache_dtype != GCB200_F8_E4M3) return say("the cache", "must have the type of the new keys and values, or float8_e4m3fn");
  for (int i = 0; i < 4; ++i)
    if (k.dims[i] != v.dims[i]) return say("key_cache and value_cache", "must have the same shape");
  if (t.dtype != t_i32) return say("page_table", "must be int32");
  c->pages = k.dims[0];
  c->kv_heads = k.dims[1];
  c->page_size = k.dims[2];
  c->head_dim = k.dims[3];
  c->keys = k.ptr;
  c->values = v.ptr;
  for (int i = 0; i < 3; ++i) {
    c->key_stride[i] = k.strides[i];
    c->value_stride[i] = v.strides[i];
  }
  void *ks, *vs;
  if (!vector(key_scale, "key_scale", t_f32, c->kv_heads, device, &ks) || !vector(value_scale, "value_scale", t_f32, c->kv_heads, device, &vs)) return false;
  c->key_scale = static_cast<const float *>(ks);
  c->value_scale = static_cast<const float *>(vs);
  c->page_table = static_cast<const int32_t *>(t.ptr);
  c->sequences = t.dims[0];
  c->max_pages = t.dims[1];
  c->page_table_stride = t.strides[0];
  return true;
}
bool rows_of(PyObject *t, const char *name, PyObject *dtype, int64_t n, int64_t heads, int64_t dim, long device, View *v) {
  if (!view(t, name, 3, device, v)) return false;
  if (v->dtype != dtype) return say(name, "has another type than the other operands");
  if (v->dims[0] != n || v->dims[1] != heads || v->dims[2] != dim) return say(name, "has the wrong shape");
  return true;
}

// paged_kv_append(q | None, k, v, key_cache, value_cache, page_table, positions, sequences | None, inv_freq | None, interleaved,
//                 key_scale | None, value_scale | None, out | None) -> status
PyObject *paged_kv_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 13) return PyErr_Format(PyExc_TypeError, "paged_kv_append takes 13 arguments"), nullptr;
  long dev;
  View k, v, q, o, f;
  gcb200_paged_cache c = {};
  void *pos, *seq, *stream;
  if (!current_device(&dev) || !view(a[1], "k", 3, dev, &k)) return nullptr;
  if (!cache_of(a[3], a[4], a[5], a[10], a[11], k.dtype, dev, &c)) return nullptr;
  const int64_t tokens = k.dims[0];
  if (!rows_of(a[1], "k", k.dtype, tokens, c.kv_heads, c.head_dim, dev, &k) || !rows_of(a[2], "v", k.dtype, tokens, c.kv_heads, c.head_dim, dev, &v)) return nullptr;
  if (a[0] != Py_None) {
    if (!view(a[0], "q", 3, dev, &q) || !rows_of(a[0], "q", k.dtype, tokens, q.dims[1], c.head_dim, dev, &q) ||
        !rows_of(a[12], "out", k.dtype, tokens, q.dims[1], c.head_dim, dev, &o))
      return nullptr;
  }
  if (!require(a[6] != Py_None, "positions must be a tensor") || !vector(a[6], "positions", t_i32, tokens, dev, &pos) ||
      !vector(a[7], "sequences", t_i32, tokens, dev, &seq))
    return nullptr;
  if (a[8] != Py_None) {
    if (!view(a[8], "inv_freq", 1, dev, &f)) return nullptr;
    if (f.dtype != t_f64) return say("inv_freq", "must be float64"), nullptr;
  }
  const int interleaved = PyObject_IsTrue(a[9]);
  if (interleaved < 0 || !current_stream(&stream)) return nullptr;
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = gcb200_paged_kv_append(&c, q.ptr, q.strides, q.dims[1], k.ptr, k.strides, v.ptr, v.strides, o.ptr, o.strides, static_cast<const int32_t *>(seq),
                              static_cast<const int32_t *>(pos), tokens, static_cast<const double *>(f.ptr), 2 * f.dims[0], interleaved, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// paged_attention(q, key_cache, value_cache, page_table, lengths, scale, window, key_scale | None, value_scale | None, out,
//                 lse | None, workspace) -> status
PyObject *paged_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 12) return PyErr_Format(PyExc_TypeError, "paged_attention takes 12 arguments"), nullptr;
  long dev;
  View q, o, l, w;
  gcb200_paged_cache c = {};
  void *lengths, *stream;
  if (!current_device(&dev) || !view(a[0], "q", 3, dev, &q)) return nullptr;
  if (!cache_of(a[1], a[2], a[3], a[7], a[8], q.dtype, dev, &c)) return nullptr;
  if (!rows_of(a[0], "q", q.dtype, c.sequences, q.dims[1], c.head_dim, dev, &q) ||
      !rows_of(a[9], "out", q.dtype, c.sequences, q.dims[1], c.head_dim, dev, &o) ||
      !require(a[4] != Py_None, "lengths must be a tensor") || !vector(a[4], "lengths", t_i32, c.sequences, dev, &lengths) ||
      !view(a[11], "workspace", 1, dev, &w))
    return nullptr;
  if (w.dtype != t_u8) return say("workspace", "must be uint8"), nullptr;
  if (a[10] != Py_None) {
    if (!view(a[10], "lse", 2, dev, &l)) return nullptr;
    if (l.dtype != t_f32 || l.dims[0] != q.dims[0] || l.dims[1] != q.dims[1] || (l.dims[0] > 1 && l.strides[0] != l.dims[1]))
      return say("lse", "must be a contiguous float32 tensor [sequences, heads]"), nullptr;
  }
  const double scale = PyFloat_AsDouble(a[5]);
  const long long window = PyLong_AsLongLong(a[6]);
  if (PyErr_Occurred() || !current_stream(&stream)) return nullptr;
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = gcb200_paged_attention(&c, q.ptr, q.strides, q.dims[1], static_cast<const int32_t *>(lengths), float(scale), window, o.ptr, o.strides,
                              static_cast<float *>(l.ptr), w.ptr, size_t(w.dims[0]), stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// matmul_w4(x, packed, dtype, N, K, group, has_zeros, bias | None, relu, out) -> status
PyObject *matmul_w4(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 10) return PyErr_Format(PyExc_TypeError, "matmul_w4 takes 10 arguments"), nullptr;
  long dev;
  View x, w, o;
  void *bias, *stream;
  if (!current_device(&dev) || !view(a[0], "x", 2, dev, &x) || !view(a[1], "the packed weights", 1, dev, &w) || !view(a[9], "out", 2, dev, &o)) return nullptr;
  const int64_t N = PyLong_AsLongLong(a[3]), K = PyLong_AsLongLong(a[4]), group = PyLong_AsLongLong(a[5]);
  const int zeros = PyObject_IsTrue(a[6]), relu = PyObject_IsTrue(a[8]);
  if (PyErr_Occurred() || zeros < 0 || relu < 0) return nullptr;
  if (x.dtype != a[2]) return say("x", "must have the type of the weights' scales"), nullptr;
  if (x.dims[1] != K) return say("x", "must have as many columns as the weights have k"), nullptr;
  if (o.dtype != x.dtype || o.dims[0] != x.dims[0] || o.dims[1] != N) return say("out", "has the wrong type or shape"), nullptr;
  if (!vector(a[7], "bias", x.dtype, N, dev, &bias) || !current_stream(&stream)) return nullptr;
  size_t bytes = 0;
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = gcb200_w4_packed_bytes(N, K, group, zeros, &bytes);
  if (st == GCB200_OK && size_t(w.dims[0]) >= bytes)
    st = gcb200_matmul_w4(dtype_code(x.dtype), x.ptr, x.strides[0], w.ptr, bias, o.ptr, o.strides[0], x.dims[0], N, K, group, zeros, relu, stream);
  Py_END_ALLOW_THREADS
  if (st == GCB200_OK && size_t(w.dims[0]) < bytes) return say("the packed weights", "are too few bytes for their sizes"), nullptr;
  return PyLong_FromLong(st);
}

// types(float16, float8_e4m3fn, int32, float32, float64, uint8)
PyObject *types(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 6) return PyErr_Format(PyExc_TypeError, "types takes 6 arguments"), nullptr;
  PyObject **slots[6] = {&t_f16, &t_e4m3, &t_i32, &t_f32, &t_f64, &t_u8};
  for (int i = 0; i < 6; ++i) {
    Py_INCREF(a[i]);
    Py_XSETREF(*slots[i], a[i]);
  }
  Py_RETURN_NONE;
}

constexpr int kMaxTensors = 64;
struct Pack {
  dnnl_graph_compiler_tensor t[kMaxTensors + 1];
  int64_t dims[kMaxTensors][DNNL_MAX_NDIMS];
  Py_buffer views[kMaxTensors];
  PyObject *held[kMaxTensors];   // the call runs without the interpreter's lock: another thread may change the dictionary
  int n = 0, n_views = 0, n_held = 0;
  ~Pack() {
    for (int i = 0; i < n_views; ++i) PyBuffer_Release(&views[i]);
    for (int i = 0; i < n_held; ++i) Py_DECREF(held[i]);
  }
  // 1: packed, 0: something this path does not take (the caller packs it in Python), -1: error.  Only tensors and numpy
  // arrays are taken: other objects with a buffer (bytes, memoryview) are no arguments of a partition, and an output among
  // them could be memory that must not change.
  int add(PyObject *key, PyObject *val) {
    if (n == kMaxTensors) return 0;
    const bool tensor = PyObject_TypeCheck(val, reinterpret_cast<PyTypeObject *>(t_tensor));
    if (!tensor && !(t_ndarray && PyObject_TypeCheck(val, reinterpret_cast<PyTypeObject *>(t_ndarray)))) return 0;
    const size_t id = PyLong_AsSize_t(key);
    if (id == size_t(-1) && PyErr_Occurred()) {
      PyErr_Clear();
      return 0;
    }
    Py_INCREF(val);
    held[n_held++] = val;
    int64_t *d = dims[n];
    void *p;
    int nd;
    if (tensor) {
      nd = shape(val, d, DNNL_MAX_NDIMS);
      if (nd == -2) return 0;
      if (nd < 0 || !address(val, &p)) return -1;
    } else {
      Py_buffer *b = &views[n_views];
      if (PyObject_GetBuffer(val, b, PyBUF_STRIDED_RO) != 0) {
        PyErr_Clear();
        return 0;
      }
      ++n_views;
      nd = b->ndim;
      if (nd > DNNL_MAX_NDIMS) return 0;
      for (int i = 0; i < nd; ++i) d[i] = b->shape[i];
      p = b->buf;
    }
    t[n].id = id;
    t[n].ndims = uint8_t(nd);
    t[n].dims = d;
    t[n].data = p;
    ++n;
    return 1;
  }
  int add_all(PyObject *dict) {
    PyObject *k, *v;
    Py_ssize_t pos = 0;
    while (PyDict_Next(dict, &pos, &k, &v)) {
      const int r = add(k, v);
      if (r != 1) return r;
    }
    for (int i = n; i <= kMaxTensors; ++i) t[i].id = ~size_t(0);   // a call with too few tensors finds none of these
    return 1;
  }
};

// execute(handle, inputs, outputs, stream): stream None = the synchronous call, True = the current stream, else a raw
// handle.  Returns the status, or None when an argument is nothing this path takes.
PyObject *execute(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 4) return PyErr_Format(PyExc_TypeError, "execute takes 4 arguments"), nullptr;
  if (!PyDict_CheckExact(a[1]) || !PyDict_CheckExact(a[2])) Py_RETURN_NONE;
  auto *exe = static_cast<const dnnl_graph_compiler_executable *>(PyLong_AsVoidPtr(a[0]));
  if (PyErr_Occurred()) return nullptr;
  Pack in, out;
  for (int i = 0; i < 2; ++i) {
    const int r = i == 0 ? in.add_all(a[1]) : out.add_all(a[2]);
    if (r < 0) return nullptr;
    if (r == 0) Py_RETURN_NONE;
  }
  void *stream = nullptr;
  if (a[3] == Py_True) {
    if (!current_stream(&stream)) return nullptr;
  } else if (a[3] != Py_None) {
    stream = PyLong_AsVoidPtr(a[3]);
    if (PyErr_Occurred()) return nullptr;
  }
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = a[3] == Py_None ? int(dnnl_graph_compiler_execute(exe, in.t, out.t)) : gcb200_execute_on_stream(exe, in.t, out.t, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(st);
}

// setup(torch.Tensor, torch.bfloat16, get_device, get_raw_stream, numpy.ndarray)
PyObject *setup(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 5) return PyErr_Format(PyExc_TypeError, "setup takes 5 arguments"), nullptr;
  PyObject **slots[5] = {&t_tensor, &t_bf16, &f_get_device, &f_raw_stream, &t_ndarray};
  for (int i = 0; i < 5; ++i) {
    Py_INCREF(a[i]);
    Py_XSETREF(*slots[i], a[i]);
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"setup", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(setup)), METH_FASTCALL, nullptr},
    {"matmul_bf16", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(matmul_bf16)), METH_FASTCALL, nullptr},
    {"attention_bf16", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(attention_bf16)), METH_FASTCALL, nullptr},
    {"types", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(types)), METH_FASTCALL, nullptr},
    {"paged_kv_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(paged_kv_append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(paged_attention)), METH_FASTCALL, nullptr},
    {"matmul_w4", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(matmul_w4)), METH_FASTCALL, nullptr},
    {"execute", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(execute)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_gcb200_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit__gcb200_host() {
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_shape = PyUnicode_InternFromString("shape");
  s_is_cuda = PyUnicode_InternFromString("is_cuda");
  s_dtype = PyUnicode_InternFromString("dtype");
  s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
  s_stride = PyUnicode_InternFromString("stride");
  s_get_device = PyUnicode_InternFromString("get_device");
  return PyModule_Create(&module);
}
