// The calls of the Python binding that take many tensors and check them: shapes, types, strides and devices are read off torch's own tensors
// here. The same checks by Python calls took 10 us of a call with twelve tensors, and most of the time of a small one. No computation:
// the functions reach the C ABI through addresses that bind() is given. Every C call runs without the interpreter lock.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <ATen/core/Tensor.h>

#include <cstdint>
#include <cstdio>
#include <cstring>

#include "xdlb200.h"

namespace {

struct Api {
  int (*ssm_conv)(const xb_ssm_conv_args*, xb_stream_t) = nullptr;
  size_t (*ssm_scan_bytes)(const xb_ssm_scan_args*) = nullptr;
  int (*ssm_scan)(const xb_ssm_scan_args*, void*, size_t, xb_stream_t) = nullptr;
  size_t (*lora_bytes)(const xb_lora_args*) = nullptr;
  int (*lora)(const xb_lora_args*, void*, size_t, xb_stream_t) = nullptr;
  int (*rope)(const xb_qk_norm_rope_args*, xb_stream_t) = nullptr;
  size_t (*linear_bytes)(const xb_linear_attention_args*) = nullptr;
  int (*linear)(const xb_linear_attention_args*, void*, size_t, xb_stream_t) = nullptr;
  size_t (*prefix_bytes)(const xb_prefix_attention_args*) = nullptr;
  int (*prefix)(const xb_prefix_attention_args*, void*, size_t, xb_stream_t) = nullptr;
} api;

struct Refused {};                         // `text` of Call holds why
struct Raised {};                          // a Python exception is set

struct View {
  void* at = nullptr;
  int dim = 0;
  int64_t size[4] = {0, 0, 0, 0}, stride[4] = {0, 0, 0, 0};
  int32_t dtype = 0;
  explicit operator bool() const { return dim > 0; }
};

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return XB_F32;
    case at::kHalf: return XB_F16;
    case at::kBFloat16: return XB_BF16;
    case at::kInt: return XB_I32;
    case at::kLong: return XB_I64;
    default: return -1;
  }
}

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
  const at::Tensor& tensor(PyObject* t, const char* name) {
    if (!THPVariable_Check(t)) {
      PyErr_Format(PyExc_TypeError, "%s: %s is a tensor", what, name);
      throw Raised();
    }
    return THPVariable_Unpack(t);
  }
  View view(const at::Tensor& t, const char* name, int most = 3) {
    View v;
    v.dim = (int)t.dim();
    if (v.dim < 1 || v.dim > most || t.layout() != at::kStrided) refuse("%s has 1 to %d dimensions", name, most);
    for (int i = 0; i < v.dim; ++i) {
      v.size[i] = t.sizes()[i];
      v.stride[i] = t.strides()[i];
    }
    if (t.get_device() != device) refuse("%s is on device %lld, the call on %lld", name, (long long)t.get_device(), (long long)device);
    v.dtype = dtype_code(t.scalar_type());
    v.at = t.data_ptr();
    return v;
  }
  // None: an empty view
  View view(PyObject* t, const char* name, int most = 3) { return t == Py_None ? View() : view(tensor(t, name), name, most); }
  // [rows, width] of a type with adjacent columns; the row stride
  int64_t rows(const View& v, const char* name, int64_t rows, int64_t width, int32_t dtype) {
    if (v.dim != 2 || v.size[0] != rows || v.size[1] != width || v.dtype != dtype || (width > 1 && v.stride[1] != 1))
      refuse("%s is [%lld, %lld] of the call's type with adjacent columns", name, (long long)rows, (long long)width);
    return rows <= 1 && v.stride[0] < width ? width : v.stride[0];
  }
  // [rows, heads, width] of a type whose heads have adjacent elements; the strides of rows and heads (of one row or head any do)
  template <typename Row>
  void heads(const View& v, const char* name, int64_t rows, int64_t heads, int64_t width, int32_t dtype, const void** at, Row* row, Row* head) {
    if (v.dim != 3 || v.size[0] != rows || v.size[1] != heads || v.size[2] != width || v.dtype != dtype || (width > 1 && v.stride[2] != 1))
      refuse("%s is [%lld, %lld, %lld] of the call's type with adjacent elements", name, (long long)rows, (long long)heads, (long long)width);
    *at = v.at;
    *head = heads <= 1 && v.stride[1] < width ? width : v.stride[1];
    *row = rows <= 1 ? *head * heads : v.stride[0];
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
  at::ScalarType type(PyObject* v) {
    if (!THPDtype_Check(v)) {
      PyErr_Format(PyExc_TypeError, "%s: out_dtype is a torch.dtype", what);
      throw Raised();
    }
    return reinterpret_cast<THPDtype*>(v)->scalar_type;
  }
  int64_t number(PyObject* v) {
    int64_t n = 0;
    n = PyLong_AsLongLong(v);
    if (n == -1 && PyErr_Occurred()) throw Raised();
    return n;
  }
  int32_t flag(PyObject* v) {
    const int x = PyObject_IsTrue(v);
    if (x < 0) throw Raised();
    return x;
  }
  // the tensor that was handed in for a result, or a new one of a shape
  const at::Tensor& result(PyObject* given, const char* name, const at::Tensor& like, at::IntArrayRef shape, at::Tensor& own) {
    if (given != Py_None) return tensor(given, name);
    own = like.new_empty(shape);
    return own;
  }
  void* stream(PyObject* v) {
    void* s = PyLong_AsVoidPtr(v);
    if (!s && PyErr_Occurred()) throw Raised();
    return s;
  }
  float real(PyObject* v) {
    const double x = PyFloat_AsDouble(v);
    if (x == -1.0 && PyErr_Occurred()) throw Raised();
    return (float)x;
  }
  // lists, slots and kept states; first and last [slots, a, b]
  template <typename Args>
  void lists(Args& g, int64_t n_rows, const View& offsets, PyObject* T, const View& slots, const View& first, const View& last, int64_t a, int64_t b,
             int32_t dtype) {
    batch(g, n_rows, offsets, T);
    if (slots) {
      dense(slots, "slots", 1, g.batch, 0, 0, XB_I32);
      g.slots = static_cast<const int32_t*>(slots.at);
    }
    if (first) dense(first, "the array of first states", 3, -1, a, b, dtype);
    if (last) dense(last, "the array of last states", 3, first ? first.size[0] : -1, a, b, dtype);
    g.n_slots = first ? i32(first.size[0], "slots") : last ? i32(last.size[0], "slots") : 0;
  }
  template <typename Args>
  void batch(Args& g, int64_t n_rows, const View& offsets, PyObject* T) {
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
  }
  // the scratch that was handed in, or the call's own, which outlives the launch: its memory is the stream's
  void* scratch(PyObject* given, const at::Tensor& like, size_t need, size_t* have, at::Tensor& own) {
    if (given != Py_None) {
      const View v = view(given, "workspace");
      if (v.dim != 1 || (v.size[0] > 1 && v.stride[0] != 1) || tensor(given, "workspace").element_size() != 1) refuse("the workspace is a contiguous uint8 vector");
      *have = (size_t)v.size[0];
      return v.at;
    }
    *have = need;
    if (!need) return nullptr;
    own = like.new_empty({(int64_t)need}, at::TensorOptions().dtype(at::kByte));
    return own.data_ptr();
  }
};

// The call's result tensor, or the text of a refusal. `f` gives the C function's status, and the tensor in its last argument.
template <typename F>
PyObject* checked_call(const char* what, PyObject* device, F f) {
  Call c;
  c.what = what;
  at::Tensor out;
  try {
    c.device = c.number(device);
    const int rc = f(c, out);
    if (rc != 0) return PyLong_FromLong(rc);
    return THPVariable_Wrap(out);
  } catch (const Refused&) {
    return PyUnicode_FromString(c.text);
  } catch (const Raised&) {
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {             // (torch.OutOfMemoryError, as from torch's own calls)
    if (PyObject* torch = PyImport_ImportModule("torch")) {
      if (PyObject* type = PyObject_GetAttrString(torch, "OutOfMemoryError")) {
        PyErr_SetString(type, e.what_without_backtrace());
        Py_DECREF(type);
      }
      Py_DECREF(torch);
    }
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// ssm_conv(x, w, bias, offsets, T, state_in, state_out, slots, silu, out, device, stream)
PyObject* py_ssm_conv(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 12) { PyErr_SetString(PyExc_TypeError, "ssm_conv: 12 arguments"); return nullptr; }
  return checked_call("ssm_conv", v[10], [&](Call& c, at::Tensor& result) {
    const View x = c.view(v[0], "x"), w = c.view(v[1], "w"), bias = c.view(v[2], "bias"), offsets = c.view(v[3], "offsets"),
               first = c.view(v[5], "state_in"), last = c.view(v[6], "state_out"), slots = c.view(v[7], "slots");
    if (x.dim != 2 || w.dim != 2) c.refuse("x is [rows, D] and w [D, K]");
    result = v[9] == Py_None ? c.tensor(v[0], "x").new_empty({x.size[0], x.size[1]}) : c.tensor(v[9], "out");
    const View out = c.view(result, "out");
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
  return checked_call("ssm_scan", v[18], [&](Call& c, at::Tensor& result) {
    const View x = c.view(v[0], "x"), delta = c.view(v[1], "delta"), A = c.view(v[2], "A"), B = c.view(v[3], "B"), C = c.view(v[4], "C"),
               skip = c.view(v[5], "D"), z = c.view(v[6], "z"), bias = c.view(v[7], "delta_bias"), offsets = c.view(v[10], "offsets"),
               first = c.view(v[13], "h_in"), last = c.view(v[14], "h_out"), slots = c.view(v[15], "slots");
    if (x.dim != 2 || A.dim != 2) c.refuse("x is [rows, D] and A [D, N]");
    result = v[16] == Py_None ? c.tensor(v[0], "x").new_empty({x.size[0], x.size[1]}) : c.tensor(v[16], "out");
    const View out = c.view(result, "out");
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
    at::Tensor own;
    void* ws = c.scratch(v[17], c.tensor(v[0], "x"), api.ssm_scan_bytes(&a), &have, own);
    void* stream = PyLong_AsVoidPtr(v[19]);
    if (!stream && PyErr_Occurred()) throw Raised();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = api.ssm_scan(&a, ws, have, stream);
    Py_END_ALLOW_THREADS
    return rc;
  });
}

// lora_gemm(X, W, A, B, adapter, bias, scale, trans_b, Y, out_dtype, workspace, device, stream)
PyObject* py_lora(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 13) { PyErr_SetString(PyExc_TypeError, "lora_gemm: 13 arguments"); return nullptr; }
  return checked_call("lora_gemm", v[11], [&](Call& c, at::Tensor& result) {
    const View X = c.view(v[0], "X"), W = c.view(v[1], "W"), A = c.view(v[2], "A"), B = c.view(v[3], "B"), adapter = c.view(v[4], "adapter"),
               bias = c.view(v[5], "bias"), scale = c.view(v[6], "scale");
    const int32_t trans = c.flag(v[7]);
    if (X.dim != 2 || W.dim != 2 || A.dim != 3 || B.dim != 3) c.refuse("X and W have two dimensions, A and B three");
    const int64_t M = X.size[0], K = X.size[1], N = W.size[trans ? 0 : 1], adapters = A.size[0], r = A.size[1];
    if (v[8] != Py_None) {
      result = c.tensor(v[8], "Y");
      if (v[9] != Py_None && c.type(v[9]) != result.scalar_type()) c.refuse("Y has another type than out_dtype");
    } else {
      const at::Tensor& x = c.tensor(v[0], "X");
      result = v[9] == Py_None ? x.new_empty({M, N}) : x.new_empty({M, N}, at::TensorOptions().dtype(c.type(v[9])));
    }
    const View Y = c.view(result, "Y");
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
    at::Tensor own;
    void* ws = c.scratch(v[10], c.tensor(v[0], "X"), api.lora_bytes(&a), &have, own);
    void* stream = PyLong_AsVoidPtr(v[12]);
    if (!stream && PyErr_Occurred()) throw Raised();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = api.lora(&a, ws, have, stream);
    Py_END_ALLOW_THREADS
    return rc;
  });
}

// qk_norm_rope(q, k, positions, freqs, q_weight, k_weight, eps, norm, adjacent, out_q, out_k, device, stream) -> (q', k' or None)
PyObject* py_rope(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 13) { PyErr_SetString(PyExc_TypeError, "qk_norm_rope: 13 arguments"); return nullptr; }
  at::Tensor of_k;
  PyObject* first = checked_call("qk_norm_rope", v[11], [&](Call& c, at::Tensor& result) {
    const View q = c.view(v[0], "q"), k = c.view(v[1], "k"), positions = c.view(v[2], "positions"), freqs = c.view(v[3], "freqs"),
               wq = c.view(v[4], "q_weight"), wk = c.view(v[5], "k_weight");
    if (q.dim != 3) c.refuse("q is [rows, heads, d]");
    const int64_t rows = q.size[0], d = q.size[2];
    xb_qk_norm_rope_args a;
    memset(&a, 0, sizeof(a));
    const void* at = nullptr;
    at::Tensor own;
    c.heads(q, "q", rows, q.size[1], d, q.dtype, &a.q, &a.q_row, &a.q_head);
    result = c.result(v[9], "out_q", c.tensor(v[0], "q"), {rows, q.size[1], d}, own);
    c.heads(c.view(result, "out_q"), "out_q", rows, q.size[1], d, q.dtype, &at, &a.yq_row, &a.yq_head);
    a.yq = const_cast<void*>(at);
    if (k) {
      c.heads(k, "k", rows, k.dim == 3 ? k.size[1] : 0, d, q.dtype, &a.k, &a.k_row, &a.k_head);
      a.Hk = c.i32(k.size[1], "heads");
      of_k = c.result(v[10], "out_k", c.tensor(v[1], "k"), {rows, k.size[1], d}, own);
      c.heads(c.view(of_k, "out_k"), "out_k", rows, k.size[1], d, q.dtype, &at, &a.yk_row, &a.yk_head);
      a.yk = const_cast<void*>(at);
    } else if (v[10] != Py_None || wk) {
      c.refuse("out_k and k_weight need k");
    }
    if (positions) c.dense(positions, "positions", 1, rows, 0, 0, XB_I32);
    if (freqs) c.dense(freqs, "freqs", 1, -1, 0, 0, XB_F32);
    if (freqs && !positions) c.refuse("freqs need positions");
    if (wq) c.dense(wq, "q_weight", 1, d, 0, 0, XB_F32);
    if (wk) c.dense(wk, "k_weight", 1, d, 0, 0, XB_F32);
    if (freqs && freqs.size[0] > d) c.refuse("%lld freqs for heads of %lld", (long long)freqs.size[0], (long long)d);
    a.q_weight = static_cast<const float*>(wq.at); a.k_weight = static_cast<const float*>(wk.at);
    a.positions = static_cast<const int32_t*>(positions.at); a.freqs = static_cast<const float*>(freqs.at);
    a.rows = rows; a.Hq = c.i32(q.size[1], "heads"); a.d = c.i32(d, "d"); a.rot = freqs ? (int32_t)(2 * freqs.size[0]) : 0;
    a.eps = c.real(v[6]); a.norm = c.flag(v[7]); a.adjacent = c.flag(v[8]); a.dtype = q.dtype;
    void* stream = c.stream(v[12]);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = api.rope(&a, stream);
    Py_END_ALLOW_THREADS
    return rc;
  });
  if (!first || !THPVariable_Check(first)) return first;
  PyObject* second = Py_None;
  if (of_k.defined()) second = THPVariable_Wrap(of_k);
  else Py_INCREF(second);
  if (!second) { Py_DECREF(first); return nullptr; }
  PyObject* both = PyTuple_Pack(2, first, second);
  Py_DECREF(first);
  Py_DECREF(second);
  return both;
}

// linear_attention(q, k, v, log_decay, scale, offsets, T, longest, h_in, h_out, slots, out, workspace, device, stream)
PyObject* py_linear(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 15) { PyErr_SetString(PyExc_TypeError, "linear_attention: 15 arguments"); return nullptr; }
  return checked_call("linear_attention", v[13], [&](Call& c, at::Tensor& result) {
    const View q = c.view(v[0], "q"), k = c.view(v[1], "k"), x = c.view(v[2], "v"), decay = c.view(v[3], "log_decay"), offsets = c.view(v[5], "offsets"),
               first = c.view(v[8], "h_in", 4), last = c.view(v[9], "h_out", 4), slots = c.view(v[10], "slots");
    if (q.dim != 3 || k.dim != 3 || x.dim != 3) c.refuse("q, k and v are [rows, heads, width]");
    const int64_t rows = q.size[0], H = q.size[1], Hkv = k.size[1], dk = q.size[2], dv = x.size[2];
    xb_linear_attention_args a;
    memset(&a, 0, sizeof(a));
    const void* at = nullptr;
    at::Tensor own;
    c.heads(q, "q", rows, H, dk, q.dtype, &a.q, &a.q_row, &a.q_head);
    c.heads(k, "k", rows, Hkv, dk, q.dtype, &a.k, &a.k_row, &a.k_head);
    c.heads(x, "v", rows, Hkv, dv, q.dtype, &a.v, &a.v_row, &a.v_head);
    result = c.result(v[11], "out", c.tensor(v[0], "q"), {rows, H, dv}, own);
    c.heads(c.view(result, "out"), "out", rows, H, dv, q.dtype, &at, &a.y_row, &a.y_head);
    a.y = const_cast<void*>(at);
    c.dense(decay, "log_decay", 1, H, 0, 0, XB_F32);
    c.batch(a, rows, offsets, v[6]);
    if (slots) {
      c.dense(slots, "slots", 1, a.batch, 0, 0, XB_I32);
      a.slots = static_cast<const int32_t*>(slots.at);
    }
    // (states [slots, H, dk, dv])
    auto states = [&](const View& t, const char* name) {
      const int64_t want[4] = {-1, H, dk, dv};
      bool ok = t.dim == 4 && t.dtype == XB_F32;
      int64_t step = 1;
      for (int i = 3; ok && i >= 0; --i) {
        ok = (want[i] < 0 || t.size[i] == want[i]) && (t.size[0] == 0 || t.size[i] <= 1 || t.stride[i] == step);
        step *= t.size[i];
      }
      if (!ok) c.refuse("%s is not a contiguous fp32 [slots, %lld, %lld, %lld]", name, (long long)H, (long long)dk, (long long)dv);
    };
    if (first) states(first, "h_in");
    if (last) states(last, "h_out");
    if (first && last && first.size[0] != last.size[0]) c.refuse("h_in and h_out have different numbers of slots");
    a.n_slots = first ? c.i32(first.size[0], "slots") : last ? c.i32(last.size[0], "slots") : 0;
    a.log_decay = static_cast<const float*>(decay.at); a.h_in = static_cast<const float*>(first.at); a.h_out = static_cast<float*>(last.at);
    a.longest = c.number(v[7]);
    a.H = c.i32(H, "heads"); a.Hkv = c.i32(Hkv, "heads"); a.dk = c.i32(dk, "dk"); a.dv = c.i32(dv, "dv"); a.scale = c.real(v[4]); a.dtype = q.dtype;
    size_t have = 0;
    at::Tensor scratch;
    void* ws = c.scratch(v[12], c.tensor(v[0], "q"), api.linear_bytes(&a), &have, scratch);
    void* stream = c.stream(v[14]);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = api.linear(&a, ws, have, stream);
    Py_END_ALLOW_THREADS
    return rc;
  });
}

// prefix_attention(q, k, v, offsets, T, own_offsets, prefix_k, prefix_v, prefix_offsets, members, scale, out, workspace, device, stream)
PyObject* py_prefix(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 15) { PyErr_SetString(PyExc_TypeError, "prefix_attention: 15 arguments"); return nullptr; }
  return checked_call("prefix_attention", v[13], [&](Call& c, at::Tensor& result) {
    const View q = c.view(v[0], "q"), k = c.view(v[1], "k"), x = c.view(v[2], "v"), offsets = c.view(v[3], "offsets"), own = c.view(v[5], "own_offsets"),
               pk = c.view(v[6], "prefix_k"), pv = c.view(v[7], "prefix_v"), at_prefix = c.view(v[8], "prefix_offsets"), members = c.view(v[9], "members");
    if (q.dim != 3) c.refuse("q is [rows, heads, d]");
    if (!k != !x || !pk != !pv) c.refuse("keys and values come together");
    if (own && !k) c.refuse("own_offsets need k and v");
    if ((at_prefix || members) && !pk) c.refuse("prefix_offsets and members need prefix_k and prefix_v");
    const View& keys = k ? k : pk;
    if (keys && keys.dim != 3) c.refuse("keys and values are [rows, heads, d]");
    const int64_t rows = q.size[0], H = q.size[1], d = q.size[2], Hkv = keys ? keys.size[1] : H;
    xb_prefix_attention_args a;
    memset(&a, 0, sizeof(a));
    const void* at = nullptr;
    at::Tensor fresh;
    c.heads(q, "q", rows, H, d, q.dtype, &a.q, &a.q_row, &a.q_head);
    if (k) {
      a.own_rows = k.size[0];
      c.heads(k, "k", a.own_rows, Hkv, d, q.dtype, &a.k, &a.k_row, &a.k_head);
      c.heads(x, "v", a.own_rows, Hkv, d, q.dtype, &a.v, &a.v_row, &a.v_head);
    }
    if (pk) {
      a.prefix_rows = pk.dim == 3 ? pk.size[0] : 0;
      c.heads(pk, "prefix_k", a.prefix_rows, Hkv, d, q.dtype, &a.prefix_k, &a.prefix_k_row, &a.prefix_k_head);
      c.heads(pv, "prefix_v", a.prefix_rows, Hkv, d, q.dtype, &a.prefix_v, &a.prefix_v_row, &a.prefix_v_head);
      if (at_prefix) {
        c.dense(at_prefix, "prefix_offsets", 1, -1, 0, 0, XB_I32);
        if (at_prefix.size[0] < 1) c.refuse("prefix_offsets are [prefixes + 1]");
        a.prefix_offsets = static_cast<const int32_t*>(at_prefix.at);
      }
      if (members) {
        c.dense(members, "members", 1, at_prefix ? at_prefix.size[0] : -1, 0, 0, XB_I32);
        if (members.size[0] < 1) c.refuse("members are [prefixes + 1]");
        a.members = static_cast<const int32_t*>(members.at);
      }
      a.prefixes = at_prefix ? c.i32(at_prefix.size[0] - 1, "prefixes") : members ? c.i32(members.size[0] - 1, "prefixes") : 1;
    }
    result = c.result(v[11], "out", c.tensor(v[0], "q"), {rows, H, d}, fresh);
    c.heads(c.view(result, "out"), "out", rows, H, d, q.dtype, &at, &a.y_row, &a.y_head);
    a.y = const_cast<void*>(at);
    c.batch(a, rows, offsets, v[4]);
    if (own) {
      c.dense(own, "own_offsets", 1, (int64_t)a.batch + 1, 0, 0, XB_I32);
      a.own_offsets = static_cast<const int32_t*>(own.at);
    }
    a.H = c.i32(H, "heads"); a.Hkv = c.i32(Hkv, "heads"); a.d = c.i32(d, "d"); a.scale = c.real(v[10]); a.dtype = q.dtype;
    size_t have = 0;
    at::Tensor scratch;
    void* ws = c.scratch(v[12], c.tensor(v[0], "q"), api.prefix_bytes(&a), &have, scratch);
    void* stream = c.stream(v[14]);
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = api.prefix(&a, ws, have, stream);
    Py_END_ALLOW_THREADS
    return rc;
  });
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
  if (!strcmp(name, "xb_ssm_conv")) api.ssm_conv = reinterpret_cast<decltype(api.ssm_conv)>(f);
  else if (!strcmp(name, "xb_ssm_scan_workspace_bytes")) api.ssm_scan_bytes = reinterpret_cast<decltype(api.ssm_scan_bytes)>(f);
  else if (!strcmp(name, "xb_ssm_scan")) api.ssm_scan = reinterpret_cast<decltype(api.ssm_scan)>(f);
  else if (!strcmp(name, "xb_lora_workspace_bytes")) api.lora_bytes = reinterpret_cast<decltype(api.lora_bytes)>(f);
  else if (!strcmp(name, "xb_lora_gemm")) api.lora = reinterpret_cast<decltype(api.lora)>(f);
  else if (!strcmp(name, "xb_qk_norm_rope")) api.rope = reinterpret_cast<decltype(api.rope)>(f);
  else if (!strcmp(name, "xb_linear_attention_workspace_bytes")) api.linear_bytes = reinterpret_cast<decltype(api.linear_bytes)>(f);
  else if (!strcmp(name, "xb_linear_attention")) api.linear = reinterpret_cast<decltype(api.linear)>(f);
  else if (!strcmp(name, "xb_prefix_attention_workspace_bytes")) api.prefix_bytes = reinterpret_cast<decltype(api.prefix_bytes)>(f);
  else if (!strcmp(name, "xb_prefix_attention")) api.prefix = reinterpret_cast<decltype(api.prefix)>(f);
  else { PyErr_Format(PyExc_KeyError, "bind: %s", name); return nullptr; }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"ssm_conv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_ssm_conv)), METH_FASTCALL, nullptr},
    {"ssm_scan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_ssm_scan)), METH_FASTCALL, nullptr},
    {"lora_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_lora)), METH_FASTCALL, nullptr},
    {"qk_norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_rope)), METH_FASTCALL, nullptr},
    {"linear_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_linear)), METH_FASTCALL, nullptr},
    {"prefix_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_prefix)), METH_FASTCALL, nullptr},
    {"bind", py_bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "xb_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_xb_tensors(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0) {        // (the torch whose tensors these are)
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
