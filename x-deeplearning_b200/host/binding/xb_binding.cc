// The calls of the Python binding that a serving loop makes many times a second, without ctypes: filling a structure field by
// field and converting every argument cost more than the launch behind it (gemm 4.9 us of Python, a feed 3.1 of which 1.0
// was the address of a NumPy array). No computation: the functions reach the C ABI through addresses that bind() is given, so
// that this module works on whichever libraries capi.py and blaze_api.py have loaded. Every C call runs without the
// interpreter lock, as ctypes does it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "xdlb200.h"

namespace {

struct Api {
  int (*gemm)(const xb_gemm_args*, xb_stream_t) = nullptr;
  int (*pool)(const xb_pool_group*, int32_t, void*, size_t, xb_stream_t) = nullptr;
  int (*reshape)(void*, const char*, const int*, int) = nullptr;
  int (*feed)(void*, const char*, void*, int) = nullptr;
  int (*ssm_conv)(const xb_ssm_conv_args*, xb_stream_t) = nullptr;
  size_t (*ssm_scan_bytes)(const xb_ssm_scan_args*) = nullptr;
  int (*ssm_scan)(const xb_ssm_scan_args*, void*, size_t, xb_stream_t) = nullptr;
  size_t (*lora_bytes)(const xb_lora_args*) = nullptr;
  int (*lora)(const xb_lora_args*, void*, size_t, xb_stream_t) = nullptr;
} api;

PyObject *s_data_ptr, *s_dtype, *s_stride, *s_dim, *s_shape, *s_get_device, *g_dtypes, *g_minus2, *g_scratch;

// 0 and no exception, or -1 with one
int tensor_ptr(PyObject* t, void** out) {
  PyObject* r = PyObject_CallMethodNoArgs(t, s_data_ptr);
  if (!r) return -1;
  *out = PyLong_AsVoidPtr(r);
  Py_DECREF(r);
  return *out == nullptr && PyErr_Occurred() ? -1 : 0;
}
int tensor_dtype(PyObject* t, int32_t* out) {
  PyObject* d = PyObject_GetAttr(t, s_dtype);
  if (!d) return -1;
  PyObject* code = PyDict_GetItemWithError(g_dtypes, d);
  if (!code && !PyErr_Occurred()) PyErr_SetObject(PyExc_KeyError, d);
  Py_DECREF(d);
  if (!code) return -1;
  *out = (int32_t)PyLong_AsLong(code);
  return 0;
}
int as_i64(PyObject* v, int64_t* out) {
  *out = PyLong_AsLongLong(v);
  return *out == -1 && PyErr_Occurred() ? -1 : 0;
}
int as_i32(PyObject* v, int32_t* out) {
  const long x = PyLong_AsLong(v);
  if (x == -1 && PyErr_Occurred()) return -1;
  if (x < INT32_MIN || x > INT32_MAX) { PyErr_SetString(PyExc_OverflowError, "a size does not fit 32 bits"); return -1; }
  *out = (int32_t)x;
  return 0;
}
int as_flag(PyObject* v, int32_t* out) {
  const int x = PyObject_IsTrue(v);
  *out = x;
  return x < 0 ? -1 : 0;
}
int as_f32(PyObject* v, float* out) {
  const double x = PyFloat_AsDouble(v);
  *out = (float)x;
  return x == -1.0 && PyErr_Occurred() ? -1 : 0;
}
// a leading dimension: as given, or the tensor's stride of its last but one dimension
int leading(PyObject* given, PyObject* tensor, int64_t* out) {
  if (given != Py_None) return as_i64(given, out);
  PyObject* r = PyObject_CallMethodOneArg(tensor, s_stride, g_minus2);
  if (!r) return -1;
  const int rc = as_i64(r, out);
  Py_DECREF(r);
  return rc;
}

// gemm(A, B, Y, bias, trans_a, trans_b, alpha, beta, epilogue, ep, ep_count, nosqrt, engine, batch, strides, M, N, K, lda, ldb,
//      ldy, bias_kind, stride_ep, ldbias, bias_row_group, stream) -> xb_gemm's result. ops.gemm says what they are.
PyObject* py_gemm(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 26) { PyErr_SetString(PyExc_TypeError, "gemm: 26 arguments"); return nullptr; }
  xb_gemm_args a;
  memset(&a, 0, sizeof(a));
  void* p = nullptr;
  PyObject *A = v[0], *B = v[1], *Y = v[2], *bias = v[3], *ep = v[9], *strides = v[14];
  if (!PyTuple_Check(strides) || !PyTuple_Check(ep)) { PyErr_SetString(PyExc_TypeError, "gemm: strides and ep are tuples"); return nullptr; }
  if (PyTuple_GET_SIZE(strides) < 4 || PyTuple_GET_SIZE(ep) < 3) {
    PyErr_SetString(PyExc_IndexError, "gemm: four strides and three activation parameters");
    return nullptr;
  }
  auto st = [&](int i) { return PyTuple_GET_ITEM(strides, i); };
  if (as_i32(v[15], &a.M) || as_i32(v[16], &a.N) || as_i32(v[17], &a.K) || as_flag(v[4], &a.trans_a) || as_flag(v[5], &a.trans_b) ||
      as_f32(v[6], &a.alpha) || as_f32(v[7], &a.beta))
    return nullptr;
  if (tensor_ptr(A, &p) || leading(v[18], A, &a.lda) || as_i64(st(0), &a.stride_a)) return nullptr;
  a.A = p;
  if (tensor_ptr(B, &p) || leading(v[19], B, &a.ldb) || as_i64(st(1), &a.stride_b)) return nullptr;
  a.B = p;
  if (bias != Py_None) {
    int32_t kind = 0;
    int64_t dim = 2;
    if (v[21] == Py_None || v[23] == Py_None) {
      PyObject* d = PyObject_CallMethodNoArgs(bias, s_dim);
      if (!d) return nullptr;
      const int rc = as_i64(d, &dim);
      Py_DECREF(d);
      if (rc) return nullptr;
    }
    if (v[21] == Py_None) kind = dim == 1 ? XB_BIAS_ROW : XB_BIAS_FULL;
    else if (as_i32(v[21], &kind)) return nullptr;
    if (v[23] == Py_None && dim <= 1) a.ldbias = 0;
    else if (leading(v[23], bias, &a.ldbias)) return nullptr;
    if (tensor_ptr(bias, &p) || tensor_dtype(bias, &a.bias_dtype) || as_i64(st(2), &a.stride_bias) || as_i64(v[24], &a.bias_row_group))
      return nullptr;
    a.bias = p;
    a.bias_kind = kind;
  }
  if (tensor_ptr(Y, &p) || leading(v[20], Y, &a.ldy) || as_i64(st(3), &a.stride_y)) return nullptr;
  a.Y = p;
  if (as_i32(v[13], &a.batch) || tensor_dtype(A, &a.ab_dtype) || tensor_dtype(Y, &a.y_dtype) || as_i32(v[8], &a.epilogue)) return nullptr;
  const float** slots[3] = {&a.ep_a, &a.ep_b, &a.ep_c};
  for (int i = 0; i < 3; ++i) {
    PyObject* e = PyTuple_GET_ITEM(ep, i);
    if (e == Py_None) continue;
    if (tensor_ptr(e, &p)) return nullptr;
    *slots[i] = static_cast<const float*>(p);
  }
  if (as_i32(v[10], &a.ep_count) || as_flag(v[11], &a.dice_nosqrt) || as_i64(v[22], &a.stride_ep) || as_i32(v[12], &a.engine)) return nullptr;
  void* stream = PyLong_AsVoidPtr(v[25]);
  if (!stream && PyErr_Occurred()) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.gemm(&a, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// pool(address of the groups, how many, address and bytes of the scratch, stream) -> xb_embedding_pool's result
PyObject* py_pool(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 5) { PyErr_SetString(PyExc_TypeError, "pool: 5 arguments"); return nullptr; }
  int32_t count = 0;
  int64_t bytes = 0;
  const void* groups = PyLong_AsVoidPtr(v[0]);
  void* scratch = PyLong_AsVoidPtr(v[2]);
  void* stream = PyLong_AsVoidPtr(v[4]);
  if (PyErr_Occurred() || as_i32(v[1], &count) || as_i64(v[3], &bytes)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.pool(static_cast<const xb_pool_group*>(groups), count, scratch, (size_t)bytes, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// feed(predictor handle, name, C-contiguous array) -> result of ReshapeInput to the array's shape and of Feed of its bytes
PyObject* py_feed(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 3) { PyErr_SetString(PyExc_TypeError, "feed: 3 arguments"); return nullptr; }
  void* handle = PyLong_AsVoidPtr(v[0]);
  if (!handle && PyErr_Occurred()) return nullptr;
  const char* name = PyUnicode_AsUTF8(v[1]);
  if (!name) return nullptr;
  Py_buffer b;
  if (PyObject_GetBuffer(v[2], &b, PyBUF_ND) != 0) return nullptr;
  std::vector<int> shape(b.ndim);
  for (int i = 0; i < b.ndim; ++i) shape[i] = (int)b.shape[i];
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = api.reshape(handle, name, shape.data(), b.ndim);
  if (rc == 0) rc = api.feed(handle, name, b.buf, (int)b.len);
  Py_END_ALLOW_THREADS
  PyBuffer_Release(&b);
  return PyLong_FromLong(rc);
}

// ---- calls that check their tensors here: a text for what they refuse, the C function's result otherwise ----

struct Refused {};                         // `text` of Call holds why
struct Raised {};                          // a Python exception is set

struct View {
  void* at = nullptr;
  int dim = 0;
  int64_t size[3] = {0, 0, 0}, stride[3] = {0, 0, 0};
  int32_t dtype = 0;
  explicit operator bool() const { return dim > 0; }
};

struct Call {
  const char* what;
  int64_t device;
  char text[256];
  template <typename... A>
  [[noreturn]] void refuse(const char* format, A... a) {
    const int n = snprintf(text, sizeof(text), "%s: ", what);
    if constexpr (sizeof...(a) == 0) snprintf(text + n, sizeof(text) - n, "%s", format);
    else snprintf(text + n, sizeof(text) - n, format, a...);
    throw Refused();
  }
  void ints(PyObject* tuple, const char* name, int64_t* to, int* n) {
    if (!tuple) throw Raised();
    const Py_ssize_t have = PyTuple_Check(tuple) ? PyTuple_GET_SIZE(tuple) : -1;
    if (have < 1 || have > 3) { Py_DECREF(tuple); refuse("%s has 1 to 3 dimensions", name); }
    for (Py_ssize_t i = 0; i < have; ++i) to[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
    Py_DECREF(tuple);
    if (PyErr_Occurred()) throw Raised();
    *n = (int)have;
  }
  // None: an empty view
  View view(PyObject* t, const char* name) {
    View v;
    if (t == Py_None) return v;
    ints(PyObject_GetAttr(t, s_shape), name, v.size, &v.dim);
    int n = 0;
    ints(PyObject_CallMethodNoArgs(t, s_stride), name, v.stride, &n);
    PyObject* d = PyObject_CallMethodNoArgs(t, s_get_device);
    int64_t on = 0;
    if (!d) throw Raised();
    const int rc = as_i64(d, &on);
    Py_DECREF(d);
    if (rc) throw Raised();
    if (on != device) refuse("%s is on device %lld, the call on %lld", name, (long long)on, (long long)device);
    d = PyObject_GetAttr(t, s_dtype);
    if (!d) throw Raised();
    PyObject* code = PyDict_GetItemWithError(g_dtypes, d);
    Py_DECREF(d);
    if (!code && PyErr_Occurred()) throw Raised();
    v.dtype = code ? (int32_t)PyLong_AsLong(code) : -1;
    if (tensor_ptr(t, &v.at)) throw Raised();
    return v;
  }
  // [rows, width] of a type with adjacent columns; the row stride
  int64_t rows(const View& v, const char* name, int64_t rows, int64_t width, int32_t dtype) {
    if (v.dim != 2 || v.size[0] != rows || v.size[1] != width || v.dtype != dtype || (width > 1 && v.stride[1] != 1))
      refuse("%s is [%lld, %lld] of the call's type with adjacent columns", name, (long long)rows, (long long)width);
    return rows <= 1 && v.stride[0] < width ? width : v.stride[0];
  }
  void dense(const View& v, const char* name, int dim, int64_t a, int64_t b, int64_t c, int32_t dtype) {
    const int64_t want[3] = {a, b, c};
    bool ok = v.dim == dim && v.dtype == dtype;
    int64_t step = 1;
    for (int i = dim - 1; ok && i >= 0; --i) {
      ok = (want[i] < 0 || v.size[i] == want[i]) && (v.size[i] <= 1 || v.stride[i] == step);
      step *= v.size[i];
    }
    for (int i = 0; !ok && v.dim == dim && i < dim; ++i)
      if (v.size[i] == 0 && v.dtype == dtype && (want[i] < 0 || want[i] == 0)) return;     // nothing in it: strides say nothing
    if (!ok) refuse("%s has another shape or type, or is not contiguous", name);
  }
  int32_t i32(int64_t v, const char* name) {
    if (v < 0 || v > INT32_MAX) refuse("%s does not fit 32 bits", name);
    return (int32_t)v;
  }
  int64_t number(PyObject* v) {
    int64_t n = 0;
    if (as_i64(v, &n)) throw Raised();
    return n;
  }
  int32_t flag(PyObject* v) {
    int32_t n = 0;
    if (as_flag(v, &n)) throw Raised();
    return n;
  }
  // lists, slots and kept states; first and last [slots, a, b]
  template <typename Args>
  void lists(Args& g, int64_t n_rows, const View& offsets, PyObject* T, const View& slots, const View& first, const View& last, int64_t a, int64_t b,
             int32_t dtype) {
    g.rows = n_rows;
    if (offsets) {
      dense(offsets, "offsets", 1, -1, 0, 0, XB_I32);
      if (offsets.size[0] < 1) refuse("offsets are [lists + 1]");
      g.batch = i32(offsets.size[0] - 1, "lists");
      g.offsets = static_cast<const int32_t*>(offsets.at);
    } else {
      const int64_t t = T == Py_None ? n_rows : number(T);
      if (t < 0 || (n_rows && (t < 1 || n_rows % t))) refuse("lists of %lld rows in %lld rows", (long long)t, (long long)n_rows);
      g.batch = t ? i32(n_rows / t, "lists") : 0;
    }
    if (slots) {
      dense(slots, "slots", 1, g.batch, 0, 0, XB_I32);
      g.slots = static_cast<const int32_t*>(slots.at);
    }
    if (first) dense(first, "the array of first states", 3, -1, a, b, dtype);
    if (last) dense(last, "the array of last states", 3, first ? first.size[0] : -1, a, b, dtype);
    g.n_slots = first ? i32(first.size[0], "slots") : last ? i32(last.size[0], "slots") : 0;
  }
  // the scratch that was handed in, or the call's own (a new reference that outlives the launch)
  void* scratch(PyObject* given, PyObject* like, size_t need, size_t* have, PyObject** own) {
    if (given != Py_None) {
      const View v = view(given, "workspace");
      if (v.dim != 1 || v.stride[0] > 1) refuse("the workspace is a contiguous uint8 vector");
      *have = (size_t)v.size[0];
      return v.at;
    }
    *have = need;
    if (!need) return nullptr;
    *own = PyObject_CallFunction(g_scratch, "On", like, (Py_ssize_t)need);
    void* at = nullptr;
    if (!*own || tensor_ptr(*own, &at)) throw Raised();
    return at;
  }
};

template <typename F>
PyObject* checked_call(const char* what, PyObject* device, F f) {
  Call c;
  c.what = what;
  PyObject* own = nullptr;
  PyObject* r = nullptr;
  try {
    c.device = c.number(device);
    r = PyLong_FromLong(f(c, &own));
  } catch (const Refused&) {
    r = PyUnicode_FromString(c.text);
  } catch (const Raised&) {
  }
  Py_XDECREF(own);
  return r;
}

// ssm_conv(x, w, bias, offsets, T, state_in, state_out, slots, silu, out, device, stream)
PyObject* py_ssm_conv(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 12) { PyErr_SetString(PyExc_TypeError, "ssm_conv: 12 arguments"); return nullptr; }
  return checked_call("ssm_conv", v[10], [&](Call& c, PyObject**) {
    const View x = c.view(v[0], "x"), w = c.view(v[1], "w"), bias = c.view(v[2], "bias"), offsets = c.view(v[3], "offsets"),
               first = c.view(v[5], "state_in"), last = c.view(v[6], "state_out"), slots = c.view(v[7], "slots"), out = c.view(v[9], "out");
    if (x.dim != 2 || w.dim != 2) c.refuse("x is [rows, D] and w [D, K]");
    const int64_t rows = x.size[0], D = x.size[1], K = w.size[1];
    xb_ssm_conv_args a;
    memset(&a, 0, sizeof(a));
    a.ldx = c.rows(x, "x", rows, D, x.dtype);
    a.ldy = c.rows(out, "out", rows, D, x.dtype);
    c.dense(w, "w", 2, D, K, 0, x.dtype);
    if (bias) c.dense(bias, "bias", 1, D, 0, 0, x.dtype);
    c.lists(a, rows, offsets, v[4], slots, first, last, K - 1, D, x.dtype);
    a.x = x.at; a.y = out.at; a.w = w.at; a.bias = bias.at; a.state_in = first.at; a.state_out = last.at;
    a.D = c.i32(D, "D"); a.K = c.i32(K, "K"); a.silu = c.flag(v[8]); a.dtype = x.dtype;
    void* stream = PyLong_AsVoidPtr(v[11]);
    if (!stream && PyErr_Occurred()) throw Raised();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = api.ssm_conv(&a, stream);
    Py_END_ALLOW_THREADS
    return rc;
  });
}

// ssm_scan(x, delta, A, B, C, D, z, delta_bias, groups, softplus, offsets, T, longest, h_in, h_out, slots, out, workspace, device, stream)
PyObject* py_ssm_scan(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 20) { PyErr_SetString(PyExc_TypeError, "ssm_scan: 20 arguments"); return nullptr; }
  return checked_call("ssm_scan", v[18], [&](Call& c, PyObject** own) {
    const View x = c.view(v[0], "x"), delta = c.view(v[1], "delta"), A = c.view(v[2], "A"), B = c.view(v[3], "B"), C = c.view(v[4], "C"),
               skip = c.view(v[5], "D"), z = c.view(v[6], "z"), bias = c.view(v[7], "delta_bias"), offsets = c.view(v[10], "offsets"),
               first = c.view(v[13], "h_in"), last = c.view(v[14], "h_out"), slots = c.view(v[15], "slots"), out = c.view(v[16], "out");
    if (x.dim != 2 || A.dim != 2) c.refuse("x is [rows, D] and A [D, N]");
    const int64_t rows = x.size[0], D = x.size[1], N = A.size[1], groups = c.number(v[8]);
    if (groups < 1 || groups > D) c.refuse("%lld groups of %lld channels", (long long)groups, (long long)D);
    xb_ssm_scan_args a;
    memset(&a, 0, sizeof(a));
    a.ldx = c.rows(x, "x", rows, D, x.dtype);
    a.lddelta = c.rows(delta, "delta", rows, D, x.dtype);
    if (z) a.ldz = c.rows(z, "z", rows, D, x.dtype);
    a.ldb = c.rows(B, "B", rows, groups * N, x.dtype);
    a.ldc = c.rows(C, "C", rows, groups * N, x.dtype);
    a.ldy = c.rows(out, "out", rows, D, x.dtype);
    c.dense(A, "A", 2, D, N, 0, XB_F32);
    if (skip) c.dense(skip, "D", 1, D, 0, 0, XB_F32);
    if (bias) c.dense(bias, "delta_bias", 1, D, 0, 0, XB_F32);
    c.lists(a, rows, offsets, v[11], slots, first, last, D, N, XB_F32);
    a.x = x.at; a.delta = delta.at; a.z = z.at; a.B = B.at; a.C = C.at; a.y = out.at;
    a.A = static_cast<const float*>(A.at); a.skip = static_cast<const float*>(skip.at); a.delta_bias = static_cast<const float*>(bias.at);
    a.h_in = static_cast<const float*>(first.at); a.h_out = static_cast<float*>(last.at);
    a.longest = c.number(v[12]);
    a.D = c.i32(D, "D"); a.N = c.i32(N, "N"); a.groups = c.i32(groups, "groups"); a.softplus = c.flag(v[9]); a.dtype = x.dtype;
    size_t have = 0;
    void* ws = c.scratch(v[17], v[0], api.ssm_scan_bytes(&a), &have, own);
    void* stream = PyLong_AsVoidPtr(v[19]);
    if (!stream && PyErr_Occurred()) throw Raised();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = api.ssm_scan(&a, ws, have, stream);
    Py_END_ALLOW_THREADS
    return rc;
  });
}

// lora_gemm(X, W, A, B, adapter, bias, scale, trans_b, Y, workspace, device, stream)
PyObject* py_lora(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 12) { PyErr_SetString(PyExc_TypeError, "lora_gemm: 12 arguments"); return nullptr; }
  return checked_call("lora_gemm", v[10], [&](Call& c, PyObject** own) {
    const View X = c.view(v[0], "X"), W = c.view(v[1], "W"), A = c.view(v[2], "A"), B = c.view(v[3], "B"), adapter = c.view(v[4], "adapter"),
               bias = c.view(v[5], "bias"), scale = c.view(v[6], "scale"), Y = c.view(v[8], "Y");
    const int32_t trans = c.flag(v[7]);
    if (X.dim != 2 || W.dim != 2 || A.dim != 3 || B.dim != 3) c.refuse("X and W have two dimensions, A and B three");
    const int64_t M = X.size[0], K = X.size[1], N = W.size[trans ? 0 : 1], adapters = A.size[0], r = A.size[1];
    xb_lora_args a;
    memset(&a, 0, sizeof(a));
    a.ldx = c.rows(X, "X", M, K, X.dtype);
    a.ldw = c.rows(W, "W", trans ? N : K, trans ? K : N, X.dtype);
    a.ldy = c.rows(Y, "Y", M, N, Y.dtype);
    c.dense(adapter, "adapter", 1, M, 0, 0, XB_I32);
    auto stack = [&](const View& t, const char* name, int64_t rows, int64_t cols, int64_t* ld, int64_t* step) {
      if (t.size[0] != adapters || t.size[1] != rows || t.size[2] != cols || t.dtype != X.dtype || (cols > 1 && t.stride[2] != 1))
        c.refuse("%s is [%lld, %lld, %lld] of the call's type with adjacent columns", name, (long long)adapters, (long long)rows, (long long)cols);
      *ld = rows <= 1 && t.stride[1] < cols ? cols : t.stride[1];
      *step = t.stride[0];
    };
    stack(A, "A", r, K, &a.lda, &a.stride_a);
    stack(B, "B", N, r, &a.ldb, &a.stride_b);
    if (bias) c.dense(bias, "bias", 1, N, 0, 0, XB_F32);
    if (scale) c.dense(scale, "scale", 1, adapters, 0, 0, XB_F32);
    a.M = c.i32(M, "M"); a.N = c.i32(N, "N"); a.K = c.i32(K, "K"); a.r = c.i32(r, "the rank"); a.n_adapters = c.i32(adapters, "adapters");
    a.trans_w = trans; a.X = X.at; a.W = W.at; a.A = A.at; a.B = B.at; a.Y = Y.at;
    a.scale = static_cast<const float*>(scale.at); a.bias = static_cast<const float*>(bias.at); a.adapter = static_cast<const int32_t*>(adapter.at);
    a.dtype = X.dtype; a.y_dtype = Y.dtype;
    size_t have = 0;
    void* ws = c.scratch(v[9], v[0], api.lora_bytes(&a), &have, own);
    void* stream = PyLong_AsVoidPtr(v[11]);
    if (!stream && PyErr_Occurred()) throw Raised();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = api.lora(&a, ws, have, stream);
    Py_END_ALLOW_THREADS
    return rc;
  });
}

// scratch(callable): (a tensor, bytes) -> uint8 scratch beside it
PyObject* py_scratch(PyObject*, PyObject* f) {
  Py_INCREF(f);
  Py_XSETREF(g_scratch, f);
  Py_RETURN_NONE;
}

// bind(name, address): where a C function is
PyObject* py_bind(PyObject*, PyObject* args) {
  const char* name = nullptr;
  PyObject* at = nullptr;
  if (!PyArg_ParseTuple(args, "sO", &name, &at)) return nullptr;
  void* f = PyLong_AsVoidPtr(at);
  if (!f) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
    return nullptr;
  }
  if (!strcmp(name, "xb_gemm")) api.gemm = reinterpret_cast<decltype(api.gemm)>(f);
  else if (!strcmp(name, "xb_embedding_pool")) api.pool = reinterpret_cast<decltype(api.pool)>(f);
  else if (!strcmp(name, "xb_ssm_conv")) api.ssm_conv = reinterpret_cast<decltype(api.ssm_conv)>(f);
  else if (!strcmp(name, "xb_ssm_scan_workspace_bytes")) api.ssm_scan_bytes = reinterpret_cast<decltype(api.ssm_scan_bytes)>(f);
  else if (!strcmp(name, "xb_ssm_scan")) api.ssm_scan = reinterpret_cast<decltype(api.ssm_scan)>(f);
  else if (!strcmp(name, "xb_lora_workspace_bytes")) api.lora_bytes = reinterpret_cast<decltype(api.lora_bytes)>(f);
  else if (!strcmp(name, "xb_lora_gemm")) api.lora = reinterpret_cast<decltype(api.lora)>(f);
  else if (!strcmp(name, "Blaze_PredictorReshapeInput")) api.reshape = reinterpret_cast<decltype(api.reshape)>(f);
  else if (!strcmp(name, "Blaze_PredictorFeed")) api.feed = reinterpret_cast<decltype(api.feed)>(f);
  else { PyErr_Format(PyExc_KeyError, "bind: %s", name); return nullptr; }
  Py_RETURN_NONE;
}

// dtypes({torch dtype: code})
PyObject* py_dtypes(PyObject*, PyObject* d) {
  if (!PyDict_Check(d)) { PyErr_SetString(PyExc_TypeError, "dtypes: a dict"); return nullptr; }
  Py_INCREF(d);
  Py_XSETREF(g_dtypes, d);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_gemm)), METH_FASTCALL, nullptr},
    {"pool", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_pool)), METH_FASTCALL, nullptr},
    {"feed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_feed)), METH_FASTCALL, nullptr},
    {"ssm_conv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_ssm_conv)), METH_FASTCALL, nullptr},
    {"ssm_scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_ssm_scan)), METH_FASTCALL, nullptr},
    {"lora_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_lora)), METH_FASTCALL, nullptr},
    {"scratch", py_scratch, METH_O, nullptr},
    {"bind", py_bind, METH_VARARGS, nullptr},
    {"dtypes", py_dtypes, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "xb_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_xb_binding(void) {
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_dtype = PyUnicode_InternFromString("dtype");
  s_stride = PyUnicode_InternFromString("stride");
  s_dim = PyUnicode_InternFromString("dim");
  s_shape = PyUnicode_InternFromString("shape");
  s_get_device = PyUnicode_InternFromString("get_device");
  g_minus2 = PyLong_FromLong(-2);
  g_dtypes = PyDict_New();
  if (!s_data_ptr || !s_dtype || !s_stride || !s_dim || !s_shape || !s_get_device || !g_minus2 || !g_dtypes) return nullptr;
  return PyModule_Create(&module);
}
