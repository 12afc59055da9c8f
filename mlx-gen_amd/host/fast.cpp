// fast.cpp — native call path of the Python operators (module mlxq._fast).
//
// A decode-sized call spends more host time in Python than its kernel takes on the GPU: shape and
// dtype checks, one ctypes conversion per argument and the stream object came to ~14 us a call,
// against 5-7 us of kernel.  Each function here takes the call whose operands need no preparation
// (GPU tensors of the expected ranks, shapes and dtypes, contiguous and aligned), allocates the
// result and calls the C ABI; for anything else, and for a call that the library refuses, it returns
// None and the caller's general path prepares the operands or reports the error.  A device error is
// raised from here: the launch that failed is not made a second time.  Nothing is kept from one call to
// the next.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>

#include <math.h>
#include <string.h>

#include <vector>

#include "../../include/mlxq.h"

namespace {

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MLXQ_FLOAT32;
    case at::kBFloat16: return MLXQ_BFLOAT16;
    case at::kHalf: return MLXQ_FLOAT16;
    default: return -1;
  }
}

at::ScalarType type_of(int code) { return code == MLXQ_BFLOAT16 ? at::kBFloat16 : at::kFloat; }

// A plain GPU tensor in row-major order whose data starts at a multiple of `align` bytes (a nested tensor
// calls itself strided and contiguous too, and is for the general path to refuse).
const at::Tensor* plain(PyObject* o, size_t align) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.is_nested()) return nullptr;
  if (!t.is_contiguous() || t.is_conj() || t.is_neg()) return nullptr;
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % align != 0) return nullptr;
  return &t;
}

struct Pack {  // owns its tensors: the caller's list may change while the lock is released
  at::Tensor wq, s, b;
  int64_t N;
  int dt;
};

bool get_pack(PyObject* wq, PyObject* s, PyObject* b, int64_t K, long gs, long bits, Pack& p) {
  if ((bits != 4 && bits != 8) || (gs != 32 && gs != 64 && gs != 128) || K <= 0 || K % gs != 0) return false;
  const at::Tensor *w = plain(wq, 16), *ps = plain(s, 4), *pb = plain(b, 4);
  if (!w || !ps || !pb || w->dim() != 2 || ps->dim() != 2 || pb->dim() != 2) return false;
  if (w->scalar_type() != at::kInt && w->scalar_type() != at::kUInt32) return false;
  p.N = w->size(0);
  p.dt = code_of(ps->scalar_type());
  if ((p.dt != MLXQ_BFLOAT16 && p.dt != MLXQ_FLOAT32) || pb->scalar_type() != ps->scalar_type()) return false;
  const int64_t G = K / gs;
  if (p.N <= 0 || w->size(1) * 32 != K * bits || ps->size(0) != p.N || ps->size(1) != G || pb->size(0) != p.N ||
      pb->size(1) != G)
    return false;
  p.wq = *w;
  p.s = *ps;
  p.b = *pb;
  return true;
}

// Activations [..., K] of at least one row.
const at::Tensor* get_x(PyObject* o, int64_t& M, int64_t& K, int& dt) {
  const at::Tensor* x = plain(o, 16);
  if (!x || x->dim() < 1) return nullptr;
  K = x->size(-1);
  dt = code_of(x->scalar_type());
  if (dt < 0 || K <= 0 || x->numel() == 0) return nullptr;
  M = x->numel() / K;
  return x;
}

at::Tensor result(const at::Tensor& x, int64_t N, int dt) {
  if (x.dim() == 2) return at::empty({x.size(0), N}, x.options().dtype(type_of(dt)));
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  return at::empty(shape, x.options().dtype(type_of(dt)));
}

// torch's query of a device's raw current stream, looked up when the module is loaded: a lookup on first
// use under a static's guard could yield the interpreter lock to a thread that then waits for the guard.
PyObject* g_stream_query = nullptr;

void* stream_of(const at::Tensor& t, bool& ok) {
  ok = false;
  PyObject* index = PyLong_FromLong(t.get_device());
  PyObject* r = index ? PyObject_CallOneArg(g_stream_query, index) : nullptr;
  Py_XDECREF(index);
  if (!r) return nullptr;
  void* st = PyLong_AsVoidPtr(r);
  Py_DECREF(r);
  ok = !PyErr_Occurred();
  return st;
}

// MlxqError, given by the Python side when it loads the module.
PyObject* g_error = nullptr;

// A status that no second attempt may hide, raised as MlxqError(status, message).
struct DeviceError {
  int rc;
};

void refuse(int rc) {
  if (rc != MLXQ_OK && rc != MLXQ_EINVAL && rc != MLXQ_EUNSUPPORTED) throw DeviceError{rc};
}

// Calls the library without the interpreter lock, as ctypes does; its last error is this thread's.
template <typename F>
int unlocked(F&& call) {
  PyThreadState* save = PyEval_SaveThread();
  const int rc = call();
  PyEval_RestoreThread(save);
  refuse(rc);
  return rc;
}

// Runs f with C++ exceptions turned into "take the general path", which meets and reports them.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    if (PyObject* r = f()) return r;
  } catch (const DeviceError& e) {
    if (g_error) {
      PyErr_Clear();
      if (PyObject* v = PyObject_CallFunction(g_error, "is", e.rc, mlxq_last_error())) {
        PyErr_SetObject(g_error, v);
        Py_DECREF(v);
      }
      return nullptr;
    }
  } catch (...) {
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

bool ints(PyObject* const* a, int n, long* out) {
  for (int i = 0; i < n; ++i) {
    if (!PyLong_CheckExact(a[i])) return false;
    out[i] = PyLong_AsLong(a[i]);
  }
  return !PyErr_Occurred();
}

// quantized_matmul(x, wq, scales, biases, group_size, bits)
PyObject* quantized_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int64_t M, K;
    int dt;
    long v[2];
    Pack p;
    if (n != 6 || !ints(a + 4, 2, v)) return nullptr;
    const at::Tensor* x = get_x(a[0], M, K, dt);
    if (!x || !get_pack(a[1], a[2], a[3], K, v[0], v[1], p)) return nullptr;
    bool ok;
    void* st = stream_of(*x, ok);
    if (!ok) return nullptr;
    at::Tensor y = result(*x, p.N, dt == MLXQ_BFLOAT16 && p.dt == MLXQ_BFLOAT16 ? MLXQ_BFLOAT16 : MLXQ_FLOAT32);
    if (unlocked([&] { return mlxq_quantized_matmul(x->data_ptr(), dt, M, K, (const uint32_t*)p.wq.data_ptr(), p.s.data_ptr(),
                              p.b.data_ptr(), p.dt, p.N, 1, (int)v[0], (int)v[1], y.data_ptr(), st); }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(y));
  });
}

// linear(x, wq, scales, biases, group_size, bits, bias, lora_a, lora_b, lora_scale, activation)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int64_t M, K;
    int dt;
    long v[2], act;
    Pack p;
    if (n != 11 || !ints(a + 4, 2, v) || !ints(a + 10, 1, &act)) return nullptr;
    const at::Tensor* x = get_x(a[0], M, K, dt);
    if (!x || !get_pack(a[1], a[2], a[3], K, v[0], v[1], p)) return nullptr;
    mlxq_epilogue ep = {};
    ep.activation = (int)act;
    ep.bias_dtype = ep.lora_dtype = dt;
    ep.lora_scale = (float)PyFloat_AsDouble(a[9]);
    if (PyErr_Occurred()) return nullptr;
    if (a[6] != Py_None) {
      const at::Tensor* bias = plain(a[6], 2);
      if (!bias || bias->dim() != 1 || bias->size(0) != p.N) return nullptr;
      ep.bias = bias->data_ptr();
      ep.bias_dtype = code_of(bias->scalar_type());
      if (ep.bias_dtype < 0) return nullptr;
    }
    if ((a[7] == Py_None) != (a[8] == Py_None)) return nullptr;
    if (a[7] != Py_None) {
      const at::Tensor *la = plain(a[7], 2), *lb = plain(a[8], 2);
      if (!la || !lb || la->dim() != 2 || lb->dim() != 2 || la->size(0) != K || lb->size(1) != p.N ||
          la->size(1) != lb->size(0) || la->scalar_type() != lb->scalar_type())
        return nullptr;
      ep.lora_a = la->data_ptr();
      ep.lora_b = lb->data_ptr();
      ep.lora_rank = la->size(1);
      ep.lora_dtype = code_of(la->scalar_type());
      if (ep.lora_dtype < 0) return nullptr;
    }
    const int odt = mlxq_linear_out_dtype(dt, p.dt, &ep);
    if (odt < 0) return nullptr;
    bool ok;
    void* st = stream_of(*x, ok);
    if (!ok) return nullptr;
    const size_t need = mlxq_linear_workspace_size(dt, p.dt, M, p.N, &ep);
    at::Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, x->options().dtype(at::kByte));
    at::Tensor y = result(*x, p.N, odt);
    if (unlocked([&] { return mlxq_linear(x->data_ptr(), dt, M, K, (const uint32_t*)p.wq.data_ptr(), p.s.data_ptr(), p.b.data_ptr(), p.dt,
                    p.N, (int)v[0], (int)v[1], &ep, y.data_ptr(), need ? ws.data_ptr() : nullptr, need, st); }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(y));
  });
}

// swiglu(x, gate, up, group_size, bits) with gate and up (wq, scales, biases) tuples or lists
PyObject* swiglu(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int64_t M, K;
    int dt;
    long v[2];
    Pack p[2];
    if (n != 5 || !ints(a + 3, 2, v)) return nullptr;
    const at::Tensor* x = get_x(a[0], M, K, dt);
    if (!x) return nullptr;
    for (int i = 0; i < 2; ++i) {
      PyObject* t = a[1 + i];
      if ((!PyTuple_CheckExact(t) && !PyList_CheckExact(t)) || PySequence_Fast_GET_SIZE(t) != 3) return nullptr;
      PyObject** e = PySequence_Fast_ITEMS(t);
      if (!get_pack(e[0], e[1], e[2], K, v[0], v[1], p[i])) return nullptr;
    }
    if (p[0].N != p[1].N || p[0].dt != p[1].dt) return nullptr;
    bool ok;
    void* st = stream_of(*x, ok);
    if (!ok) return nullptr;
    at::Tensor h = result(*x, p[0].N, dt == MLXQ_BFLOAT16 && p[0].dt == MLXQ_BFLOAT16 ? MLXQ_BFLOAT16 : MLXQ_FLOAT32);
    if (unlocked([&] { return mlxq_swiglu(x->data_ptr(), dt, M, K, (const uint32_t*)p[0].wq.data_ptr(), p[0].s.data_ptr(),
                    p[0].b.data_ptr(), (const uint32_t*)p[1].wq.data_ptr(), p[1].s.data_ptr(), p[1].b.data_ptr(),
                    p[0].dt, p[0].N, (int)v[0], (int)v[1], h.data_ptr(), st); }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(h));
  });
}

// embedding(ids, wq, scales, biases, group_size, bits, bf16): int32 ids
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    long v[3];
    Pack p;
    if (n != 7 || !ints(a + 4, 3, v) || (v[1] != 4 && v[1] != 8)) return nullptr;
    const at::Tensor *ids = plain(a[0], 4), *wq = plain(a[1], 16);
    if (!ids || !wq || ids->scalar_type() != at::kInt || ids->numel() == 0 || wq->dim() != 2) return nullptr;
    const int64_t hidden = wq->size(1) * 32 / v[1];
    if (!get_pack(a[1], a[2], a[3], hidden, v[0], v[1], p)) return nullptr;
    bool ok;
    void* st = stream_of(*wq, ok);
    if (!ok) return nullptr;
    at::DimVector shape(ids->sizes().begin(), ids->sizes().end());
    shape.push_back(hidden);
    const int odt = v[2] ? MLXQ_BFLOAT16 : MLXQ_FLOAT32;
    at::Tensor out = at::empty(shape, wq->options().dtype(type_of(odt)));
    if (unlocked([&] { return mlxq_embedding(ids->data_ptr<int32_t>(), ids->numel(), (const uint32_t*)wq->data_ptr(), p.s.data_ptr(),
                       p.b.data_ptr(), p.dt, p.N, hidden, (int)v[0], (int)v[1], out.data_ptr(), odt, st); }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(out));
  });
}

// dequantize(wq, scales, biases, group_size, bits)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    long v[2];
    Pack p;
    if (n != 5 || !ints(a + 3, 2, v) || (v[1] != 4 && v[1] != 8)) return nullptr;
    const at::Tensor* wq = plain(a[0], 16);
    if (!wq || wq->dim() != 2) return nullptr;
    const int64_t K = wq->size(1) * 32 / v[1];
    if (!get_pack(a[0], a[1], a[2], K, v[0], v[1], p)) return nullptr;
    bool ok;
    void* st = stream_of(p.wq, ok);
    if (!ok) return nullptr;
    at::Tensor out = at::empty({p.N, K}, p.s.options());
    if (unlocked([&] {
          return mlxq_dequantize((const uint32_t*)p.wq.data_ptr(), p.s.data_ptr(), p.b.data_ptr(), p.dt, p.N, K,
                                 (int)v[0], (int)v[1], out.data_ptr(), st);
        }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(out));
  });
}

// quantize_batched(weights, group_size, bits): a list of equal 2-D weights -> a list of (wq, scales,
// biases), the scales and biases of each two views of one allocation, the biases 256 to 511 bytes past
// the scales' end.
PyObject* quantize_batched(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    long v[2];
    if (n != 3 || !PyList_CheckExact(a[0]) || !ints(a + 1, 2, v)) return nullptr;
    const Py_ssize_t count = PyList_GET_SIZE(a[0]);
    const long gs = v[0], bits = v[1];
    if (count < 1 || (bits != 4 && bits != 8) || (gs != 32 && gs != 64 && gs != 128)) return nullptr;
    std::vector<at::Tensor> w;
    for (Py_ssize_t i = 0; i < count; ++i) {
      const at::Tensor* t = plain(PyList_GET_ITEM(a[0], i), 16);
      if (!t || t->dim() != 2 || t->numel() == 0) return nullptr;
      if (i && (t->sizes() != w[0].sizes() || t->scalar_type() != w[0].scalar_type() || t->device() != w[0].device()))
        return nullptr;
      w.push_back(*t);
    }
    const int64_t N = w[0].size(0), K = w[0].size(1), G = K / gs;
    const int dt = code_of(w[0].scalar_type());
    if ((dt != MLXQ_BFLOAT16 && dt != MLXQ_FLOAT32) || K % gs != 0) return nullptr;
    bool ok;
    void* st = stream_of(w[0], ok);
    if (!ok) return nullptr;
    const int64_t esz = dt == MLXQ_FLOAT32 ? 4 : 2, off = (N * G * esz + 511) / 256 * 256 / esz;
    std::vector<at::Tensor> q, s, b;
    std::vector<const void*> wp;
    std::vector<uint32_t*> qp;
    std::vector<void*> sp, bp;
    for (Py_ssize_t i = 0; i < count; ++i) {
      q.push_back(at::empty({N, K * bits / 32}, w[0].options().dtype(at::kInt)));
      at::Tensor sb = at::empty({off + N * G}, w[0].options());
      s.push_back(sb.as_strided({N, G}, {G, 1}, 0));
      b.push_back(sb.as_strided({N, G}, {G, 1}, off));
      wp.push_back(w[i].data_ptr());
      qp.push_back((uint32_t*)q[i].data_ptr());
      sp.push_back(s[i].data_ptr());
      bp.push_back(b[i].data_ptr());
    }
    if (unlocked([&] {
          return mlxq_quantize_batched(wp.data(), (int)count, dt, N, K, (int)gs, (int)bits, qp.data(), sp.data(),
                                       bp.data(), st);
        }) != MLXQ_OK)
      return nullptr;
    PyObject* out = PyList_New(count);
    for (Py_ssize_t i = 0; out && i < count; ++i) {
      PyObject* t = PyTuple_New(3);
      if (!t) {
        Py_CLEAR(out);
        break;
      }
      PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(q[i]));
      PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(s[i]));
      PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(b[i]));
      PyList_SET_ITEM(out, i, t);
    }
    return out;
  });
}

// ---- the paged cache (mlxq/paged.py) ---------------------------------------------------------------

// A GPU tensor of one dtype and rank, whatever its strides.
const at::Tensor* strided(PyObject* o, int64_t dim) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.is_nested() || t.is_conj() || t.is_neg() || t.dim() != dim) return nullptr;
  return &t;
}

// [T, heads, D] with contiguous features and 16-byte heads.
const at::Tensor* get_heads(PyObject* o, mlxq_heads& h) {
  const at::Tensor* t = strided(o, 3);
  if (!t || code_of(t->scalar_type()) < 0 || t->numel() == 0) return nullptr;
  const int64_t C = 16 / t->element_size();
  if (t->stride(2) != 1 || t->stride(0) % C != 0 || t->stride(1) % C != 0 ||
      reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 != 0)
    return nullptr;
  h = {t->data_ptr(), t->size(1), t->stride(0), t->stride(1)};
  return t;
}

// A contiguous tensor of one dtype and shape on `like`'s device.
const at::Tensor* get_exact(PyObject* o, at::ScalarType type, at::IntArrayRef shape, const at::Tensor& like) {
  const at::Tensor* t = plain(o, 4);
  if (!t || t->scalar_type() != type || t->sizes() != shape || t->device() != like.device()) return nullptr;
  return t;
}

bool get_table(PyObject* o, const at::Tensor& like, const float*& p, int64_t& rows, int64_t& R, at::Tensor& keep) {
  p = nullptr;
  rows = R = 0;
  if (o == Py_None) return true;
  const at::Tensor* t = plain(o, 16);
  if (!t || t->dim() != 3 || t->size(2) != 2 || t->numel() == 0 || t->scalar_type() != at::kFloat || t->device() != like.device())
    return false;
  p = t->data_ptr<float>();
  rows = t->size(0);
  R = 2 * t->size(1);
  keep = *t;
  return true;
}

// Tensors that a call points into are held for its time: the lock is released, and the caller's tuple may
// change.
struct Cache {
  at::Tensor k, v;
  mlxq_paged_cache c;
};

bool pages_apart(const at::Tensor& t, int64_t page, int64_t& stride) {
  int64_t n = 1;
  for (int64_t d = t.dim() - 1; d >= 1; --d) {
    if (t.size(d) != 1 && t.stride(d) != n) return false;
    n *= t.size(d);
  }
  if (t.size(0) > 1 && t.stride(0) < page) return false;  // pages that share memory are refused
  stride = t.stride(0) < page ? page : t.stride(0);
  return true;
}

bool get_cache(PyObject* ko, PyObject* vo, Cache& c) {
  const at::Tensor *k = strided(ko, 6), *v = strided(vo, 5);
  if (!k || !v) return false;
  const int dt = code_of(k->scalar_type());
  if (dt < 0 || v->scalar_type() != k->scalar_type() || v->device() != k->device() || k->numel() == 0) return false;
  const int64_t C = 16 / k->element_size(), pages = k->size(0), heads = k->size(1), P = k->size(2) * 16, D = k->size(3) * C;
  if (k->size(4) != 16 || k->size(5) != C || v->size(0) != pages || v->size(1) != heads || v->size(2) * C != P ||
      v->size(3) != D || v->size(4) != C)
    return false;
  c.c = {k->data_ptr(), v->data_ptr(), 0, 0, pages, P, heads, D, dt};
  if (!pages_apart(*k, heads * P * D, c.c.k_page_stride) || !pages_apart(*v, heads * P * D, c.c.v_page_stride)) return false;
  c.k = *k;
  c.v = *v;
  return true;
}

struct Step {
  at::Tensor tables, starts, lens;
  mlxq_paged_batch b;
};

// (block_tables, q_starts, kv_lens, max_q, max_kv), a tuple or a subclass of one.
bool get_batch(PyObject* o, const at::Tensor& like, Step& s) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 5) return false;
  const at::Tensor* t = strided(PyTuple_GET_ITEM(o, 0), 2);
  if (!t || t->scalar_type() != at::kInt || t->device() != like.device() || t->numel() == 0) return false;
  const int64_t B = t->size(0);
  if (t->stride(1) != 1 || (B > 1 && t->stride(0) < t->size(1))) return false;
  const at::Tensor* q = get_exact(PyTuple_GET_ITEM(o, 1), at::kInt, {B + 1}, like);
  const at::Tensor* l = get_exact(PyTuple_GET_ITEM(o, 2), at::kInt, {B}, like);
  PyObject* n[2] = {PyTuple_GET_ITEM(o, 3), PyTuple_GET_ITEM(o, 4)};
  long v[2];
  if (!q || !l || !ints(n, 2, v)) return false;
  s.tables = *t;
  s.starts = *q;
  s.lens = *l;
  s.b = {t->data_ptr<int32_t>(), q->data_ptr<int32_t>(), l->data_ptr<int32_t>(), B, t->size(1), t->stride(0), v[0], v[1]};
  return true;
}

bool truth(PyObject* o, int& v) {
  if (!PyBool_Check(o)) return false;
  v = o == Py_True;
  return true;
}

at::Tensor like_heads(const at::Tensor& x, mlxq_heads& h) {
  at::Tensor y = at::empty(x.sizes(), x.options());
  h = {y.data_ptr(), y.size(1), y.stride(0), y.stride(1)};
  return y;
}

// rotary(x, positions, table, interleaved, inverse)
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    mlxq_heads xh, yh;
    int inter, inverse;
    const float* table;
    int64_t rows, R;
    at::Tensor keep;
    if (n != 5 || !truth(a[3], inter) || !truth(a[4], inverse)) return nullptr;
    const at::Tensor* xp = get_heads(a[0], xh);
    if (!xp) return nullptr;
    const at::Tensor x = *xp;
    const at::Tensor* pos = get_exact(a[1], at::kInt, {x.size(0)}, x);
    if (!pos || !get_table(a[2], x, table, rows, R, keep) || !table) return nullptr;
    const at::Tensor held = *pos;
    bool ok;
    void* st = stream_of(x, ok);
    if (!ok) return nullptr;
    at::Tensor y = like_heads(x, yh);
    if (unlocked([&] {
          return mlxq_rotary(&xh, code_of(x.scalar_type()), x.size(0), x.size(2), held.data_ptr<int32_t>(), table, rows, R,
                             inter, inverse, &yh, st);
        }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(y));
  });
}

// cache_append(k, v, k_cache, v_cache, batch, q, table, positions, interleaved) -> the rotated q, True without q
PyObject* cache_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    mlxq_heads h[4];
    Cache c;
    Step s;
    int inter;
    const float* table;
    int64_t rows, R;
    at::Tensor t[3], keep, pos, out;
    if (n != 9 || !truth(a[8], inter) || !get_cache(a[2], a[3], c) || !get_batch(a[4], c.k, s)) return nullptr;
    const bool has_q = a[5] != Py_None;
    PyObject* o[3] = {a[0], a[1], a[5]};
    for (int i = 0; i < (has_q ? 3 : 2); ++i) {
      const at::Tensor* p = get_heads(o[i], h[i]);
      if (!p || p->scalar_type() != c.k.scalar_type() || p->device() != c.k.device() || p->size(2) != c.c.head_dim) return nullptr;
      t[i] = *p;
      if (t[i].size(0) != t[0].size(0) || (i < 2 && h[i].heads != c.c.heads)) return nullptr;
    }
    if (!get_table(a[6], c.k, table, rows, R, keep)) return nullptr;
    if (a[7] != Py_None) {
      const at::Tensor* p = get_exact(a[7], at::kInt, {t[0].size(0)}, c.k);
      if (!p) return nullptr;
      pos = *p;
    }
    bool ok;
    void* st = stream_of(c.k, ok);
    if (!ok) return nullptr;
    if (has_q) out = like_heads(t[2], h[3]);
    if (unlocked([&] {
          return mlxq_cache_append(&h[0], &h[1], t[0].size(0), &c.c, &s.b, pos.defined() ? pos.data_ptr<int32_t>() : nullptr,
                                   table, rows, R, inter, has_q ? &h[2] : nullptr, has_q ? &h[3] : nullptr, st);
        }) != MLXQ_OK)
      return nullptr;
    if (has_q) return THPVariable_Wrap(std::move(out));
    Py_RETURN_TRUE;
  });
}

// paged_attention(q, k_cache, v_cache, batch, scale, causal, window, softcap, prefix_lens, alibi_slopes, sinks)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    mlxq_heads qh, oh;
    Cache c;
    Step s;
    long window;
    at::Tensor keep[3];
    mlxq_attention opt = {};
    if (n != 11 || !truth(a[5], opt.causal) || !ints(a + 6, 1, &window)) return nullptr;
    const at::Tensor* qp = get_heads(a[0], qh);
    if (!qp || !get_cache(a[1], a[2], c) || qp->scalar_type() != c.k.scalar_type() || qp->device() != c.k.device() ||
        qp->size(2) != c.c.head_dim || qh.heads % c.c.heads != 0)
      return nullptr;
    const at::Tensor q = *qp;
    if (!get_batch(a[3], q, s)) return nullptr;
    opt.window = window;
    opt.scale = a[4] == Py_None ? (float)(1.0 / sqrt((double)c.c.head_dim)) : (float)PyFloat_AsDouble(a[4]);
    opt.softcap = (float)PyFloat_AsDouble(a[7]);
    if (PyErr_Occurred()) return nullptr;
    const at::ScalarType types[3] = {at::kInt, at::kFloat, at::kFloat};
    const int64_t sizes[3] = {s.b.sequences, qh.heads, qh.heads};
    for (int i = 0; i < 3; ++i) {
      if (a[8 + i] == Py_None) continue;
      const at::Tensor* t = get_exact(a[8 + i], types[i], {sizes[i]}, q);
      if (!t) return nullptr;
      keep[i] = *t;
    }
    opt.prefix_lens = keep[0].defined() ? keep[0].data_ptr<int32_t>() : nullptr;
    opt.alibi_slopes = keep[1].defined() ? keep[1].data_ptr<float>() : nullptr;
    opt.sinks = keep[2].defined() ? keep[2].data_ptr<float>() : nullptr;
    bool ok;
    void* st = stream_of(q, ok);
    if (!ok) return nullptr;
    const size_t need = mlxq_paged_attention_workspace_size(q.size(0), qh.heads, &c.c, &s.b, &opt);
    at::Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
    at::Tensor out = like_heads(q, oh);
    if (unlocked([&] {
          return mlxq_paged_attention(&qh, q.size(0), &c.c, &s.b, &opt, &oh, need ? ws.data_ptr() : nullptr, need, st);
        }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(out));
  });
}

// copy_pages(cache, src, dst, block_tables, dim) -> True
PyObject* copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    long dim;
    if (n != 5 || !ints(a + 4, 1, &dim)) return nullptr;
    const at::Tensor* p = plain(a[0], 16);
    if (!p || code_of(p->scalar_type()) < 0 || p->dim() < 5 || dim < 0 || dim >= p->dim() - 1 || p->numel() == 0) return nullptr;
    const at::Tensor cache = *p;
    const at::Tensor* sp = plain(a[1], 4);
    if (!sp || sp->dim() != 1) return nullptr;
    const int64_t count = sp->size(0);
    sp = get_exact(a[1], at::kInt, {count}, cache);
    const at::Tensor* dp = get_exact(a[2], at::kInt, {count}, cache);
    if (!sp || !dp || count == 0) return nullptr;
    const at::Tensor src = *sp, dst = *dp;
    at::Tensor tables;
    if (a[3] != Py_None) {
      const at::Tensor* t = strided(a[3], 2);
      if (!t || t->scalar_type() != at::kInt || t->device() != cache.device() || t->numel() == 0 || t->stride(1) != 1 ||
          (t->size(0) > 1 && t->stride(0) < t->size(1)))
        return nullptr;
      tables = *t;
    }
    int64_t planes = 1, page = cache.element_size();
    for (int64_t i = 0; i < dim; ++i) planes *= cache.size(i);
    for (int64_t i = dim + 1; i < cache.dim(); ++i) page *= cache.size(i);
    bool ok;
    void* st = stream_of(cache, ok);
    if (!ok) return nullptr;
    if (unlocked([&] {
          return mlxq_cache_copy_pages(cache.data_ptr(), planes, cache.size(dim) * page, cache.size(dim), page, page,
                                       src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(), count,
                                       tables.defined() ? tables.data_ptr<int32_t>() : nullptr,
                                       tables.defined() ? tables.size(0) : 0, tables.defined() ? tables.size(1) : 0,
                                       tables.defined() ? tables.stride(0) : 0, st);
        }) != MLXQ_OK)
      return nullptr;
    Py_RETURN_TRUE;
  });
}

// ---- a decoder block in microscaled types (mlxq/mx.py) ---------------------------------------------

// The one stride between the rows (last dimension) of t; false where there is none.
bool row_stride(const at::Tensor& t, int64_t& stride) {
  const int64_t d = t.dim();
  if (d < 1 || (t.size(d - 1) > 1 && t.stride(d - 1) != 1)) return false;
  int64_t rows = 0;
  stride = t.size(d - 1);
  for (int64_t i = d - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (rows == 0) {
      stride = t.stride(i);
      rows = t.size(i);
    } else if (t.stride(i) != stride * rows) {
      return false;
    } else {
      rows *= t.size(i);
    }
  }
  return true;
}

const at::Tensor* any_gpu(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.is_nested() || t.is_conj() || t.is_neg() || t.dim() < 1 || t.numel() == 0)
    return nullptr;
  return &t;
}

struct MxOperand {
  at::Tensor codes, scales;
  int64_t rows, K;
  mlxq_mx m;
};

int64_t scale_pitch(int64_t K) { return (K / 32 + 3) / 4 * 4; }

// (codes, scales), a tuple or a subclass of one, as the library reads them.
bool get_mx(PyObject* o, MxOperand& x) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) return false;
  const at::Tensor *c = plain(PyTuple_GET_ITEM(o, 0), 16), *s = any_gpu(PyTuple_GET_ITEM(o, 1));
  if (!c || !s || c->dim() < 1 || c->numel() == 0 || s->scalar_type() != at::kByte || s->dim() != c->dim() || s->device() != c->device())
    return false;
  const bool four = c->scalar_type() == at::kByte;
  if (!four && c->scalar_type() != at::kFloat8_e4m3fn) return false;
  x.K = c->size(-1) * (four ? 2 : 1);
  if (x.K % 32 != 0 || s->size(-1) * 32 != x.K) return false;
  for (int64_t i = 0; i + 1 < c->dim(); ++i)
    if (c->size(i) != s->size(i)) return false;
  x.rows = c->numel() / c->size(-1);
  int64_t stride;
  if (!row_stride(*s, stride) || reinterpret_cast<uintptr_t>(s->data_ptr()) % 4 != 0) return false;
  if (x.rows == 1) stride = scale_pitch(x.K);
  if (stride % 4 != 0 || stride < x.K / 32) return false;
  x.codes = *c;
  x.scales = *s;
  x.m = {c->data_ptr(), s->data_ptr(), stride, four ? MLXQ_MX_E2M1 : MLXQ_MX_E4M3};
  return true;
}

// New codes and scales for rows of K; `lead` are the dimensions before it.
void new_mx(const at::Tensor& like, at::IntArrayRef shape, int format, MxOperand& x) {
  at::DimVector d(shape.begin(), shape.end());
  x.K = d.back();
  d.back() = format == MLXQ_MX_E2M1 ? x.K / 2 : x.K;
  x.codes = at::empty(d, like.options().dtype(format == MLXQ_MX_E2M1 ? at::kByte : at::kFloat8_e4m3fn));
  const int64_t n = x.K / 32, pitch = scale_pitch(x.K);
  d.back() = pitch;
  x.scales = at::empty(d, like.options().dtype(at::kByte));
  x.m = {x.codes.data_ptr(), x.scales.data_ptr(), pitch, format};
  if (n != pitch) x.scales = x.scales.narrow(-1, 0, n);
}

PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* v = out ? THPVariable_Wrap(t) : nullptr;
    if (!v) {
      Py_XDECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, v);
  }
  return out;
}

at::ScalarType float_type(int dt) { return dt == MLXQ_BFLOAT16 ? at::kBFloat16 : dt == MLXQ_FLOAT16 ? at::kHalf : at::kFloat; }

// A float scalar of any Python number.
bool number(PyObject* o, float& v) {
  if (!PyFloat_CheckExact(o) && !PyLong_CheckExact(o)) return false;
  v = (float)PyFloat_AsDouble(o);
  return !PyErr_Occurred();
}

// None, or a contiguous float tensor of this shape.
bool get_float(PyObject* o, at::IntArrayRef shape, const at::Tensor& like, at::Tensor& keep, int& dt) {
  dt = 0;
  if (o == Py_None) return true;
  const at::Tensor* t = plain(o, 1);
  if (!t || code_of(t->scalar_type()) < 0 || t->sizes() != shape || t->device() != like.device()) return false;
  keep = *t;
  dt = code_of(t->scalar_type());
  return true;
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

at::Tensor workspace(const at::Tensor& like, size_t need) {
  return need ? at::empty({(int64_t)need}, like.options().dtype(at::kByte)) : at::Tensor();
}

// mx_quantize(x, e4m3) -> (codes, scales)
PyObject* mx_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int e4m3;
    if (n != 2 || !truth(a[1], e4m3)) return nullptr;
    const at::Tensor* p = any_gpu(a[0]);
    if (!p || code_of(p->scalar_type()) < 0) return nullptr;
    const at::Tensor x = *p;
    int64_t stride;
    const int64_t K = x.size(-1), C = 16 / x.element_size();
    if (K % 32 != 0 || !row_stride(x, stride) || stride % C != 0 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) return nullptr;
    bool ok;
    void* st = stream_of(x, ok);
    if (!ok) return nullptr;
    MxOperand out;
    new_mx(x, x.sizes(), e4m3 ? MLXQ_MX_E4M3 : MLXQ_MX_E2M1, out);
    if (unlocked([&] { return mlxq_mx_quantize(x.data_ptr(), code_of(x.scalar_type()), x.numel() / K, K, stride, &out.m, st); }) != MLXQ_OK)
      return nullptr;
    return tuple_of({out.codes, out.scales});
  });
}

// mx_dequantize(x, dtype code)
PyObject* mx_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    MxOperand x;
    long dt;
    if (n != 2 || !get_mx(a[0], x) || !ints(a + 1, 1, &dt)) return nullptr;
    bool ok;
    void* st = stream_of(x.codes, ok);
    if (!ok) return nullptr;
    at::DimVector d(x.codes.sizes().begin(), x.codes.sizes().end());
    d.back() = x.K;
    at::Tensor out = at::empty(d, x.codes.options().dtype(float_type((int)dt)));
    if (unlocked([&] { return mlxq_mx_dequantize(&x.m, x.rows, x.K, out.data_ptr(), (int)dt, st); }) != MLXQ_OK) return nullptr;
    return THPVariable_Wrap(std::move(out));
  });
}

// mx_matmul(x, w, bias, dtype code)
PyObject* mx_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    MxOperand x, w;
    long dt;
    if (n != 4 || !get_mx(a[0], x) || !get_mx(a[1], w) || !ints(a + 3, 1, &dt)) return nullptr;
    if (w.codes.dim() != 2 || w.K != x.K || w.codes.device() != x.codes.device()) return nullptr;
    const int64_t N = w.rows;
    at::Tensor bias;
    int bias_dt;
    if (!get_float(a[2], {N}, x.codes, bias, bias_dt)) return nullptr;
    bool ok;
    void* st = stream_of(x.codes, ok);
    if (!ok) return nullptr;
    at::DimVector d(x.codes.sizes().begin(), x.codes.sizes().end());
    d.back() = N;
    at::Tensor out = at::empty(d, x.codes.options().dtype(float_type((int)dt)));
    if (unlocked([&] { return mlxq_mx_matmul(&x.m, x.rows, x.K, &w.m, N, ptr(bias), bias_dt, out.data_ptr(), (int)dt, st); }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(out));
  });
}

// [..., D] as [tokens, heads, D] with two strides.
bool get_rows(PyObject* o, at::Tensor& keep, mlxq_heads& h, int64_t& T) {
  const at::Tensor* p = any_gpu(o);
  if (!p || code_of(p->scalar_type()) < 0) return false;
  const at::Tensor& t = *p;
  const int64_t d = t.dim(), D = t.size(d - 1);
  if (D > 1 && t.stride(d - 1) != 1) return false;
  if (d == 1) {
    h = {t.data_ptr(), 1, D, 0};
    T = 1;
  } else if (d == 2) {
    h = {t.data_ptr(), 1, t.stride(0), 0};
    T = t.size(0);
  } else if (d == 3) {
    h = {t.data_ptr(), t.size(1), t.stride(0), t.stride(1)};
    T = t.size(0);
  } else {
    if (!t.is_contiguous()) return false;
    h = {t.data_ptr(), t.size(d - 2), t.size(d - 2) * D, D};
    T = t.numel() / (D * t.size(d - 2));
  }
  keep = t;
  return true;
}

bool get_rows_like(PyObject* o, const at::Tensor& like, at::Tensor& keep, mlxq_heads& h) {
  int64_t T;
  if (o == Py_None) return true;
  return get_rows(o, keep, h, T) && keep.sizes() == like.sizes() && keep.scalar_type() == like.scalar_type() && keep.device() == like.device();
}

at::Tensor new_rows(const at::Tensor& x, const mlxq_heads& like, mlxq_heads& h) {
  at::Tensor y = at::empty(x.sizes(), x.options());
  const int64_t D = x.size(-1);
  h = {y.data_ptr(), like.heads, like.heads * D, D};
  return y;
}

// rms_norm(x, weight, residual, eps, mx) -> y, (y, sum), (codes, scales) or (codes, scales, sum)
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    at::Tensor x, res, w, y, sum;
    mlxq_heads xh, rh, yh, sh;
    int64_t T;
    float eps;
    int mx, w_dt;
    if (n != 5 || !number(a[3], eps) || !truth(a[4], mx) || !get_rows(a[0], x, xh, T) || !get_rows_like(a[2], x, res, rh)) return nullptr;
    const int64_t D = x.size(-1);
    if ((mx && D % 32 != 0) || !get_float(a[1], {D}, x, w, w_dt)) return nullptr;
    bool ok;
    void* st = stream_of(x, ok);
    if (!ok) return nullptr;
    MxOperand q;
    if (mx) new_mx(x, x.sizes(), MLXQ_MX_E4M3, q);
    else y = new_rows(x, xh, yh);
    if (res.defined()) sum = new_rows(x, xh, sh);
    if (unlocked([&] {
          return mlxq_rms_norm(&xh, code_of(x.scalar_type()), T, D, res.defined() ? &rh : nullptr, sum.defined() ? &sh : nullptr, ptr(w),
                               w_dt, eps, mx ? nullptr : &yh, mx ? &q.m : nullptr, st);
        }) != MLXQ_OK)
      return nullptr;
    if (mx) return sum.defined() ? tuple_of({q.codes, q.scales, sum}) : tuple_of({q.codes, q.scales});
    return sum.defined() ? tuple_of({y, sum}) : THPVariable_Wrap(std::move(y));
  });
}

// rms_norm_backward(dy, x, weight, dsum, eps) -> (dx, dweight)
PyObject* rms_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    at::Tensor x, dy, ds, w, dw;
    mlxq_heads xh, yh, sh, oh;
    int64_t T;
    float eps;
    int w_dt;
    if (n != 5 || a[0] == Py_None || !number(a[4], eps) || !get_rows(a[1], x, xh, T) || !get_rows_like(a[0], x, dy, yh) ||
        !get_rows_like(a[3], x, ds, sh))
      return nullptr;
    const int64_t D = x.size(-1);
    if (!get_float(a[2], {D}, x, w, w_dt)) return nullptr;
    bool ok;
    void* st = stream_of(x, ok);
    if (!ok) return nullptr;
    at::Tensor dx = new_rows(x, xh, oh);
    size_t need = 0;
    if (w.defined()) {
      dw = at::empty(w.sizes(), w.options());
      need = mlxq_rms_norm_backward_workspace_size(T, xh.heads, D, code_of(x.scalar_type()));
    }
    at::Tensor ws = workspace(x, need);
    if (unlocked([&] {
          return mlxq_rms_norm_backward(&yh, &xh, code_of(x.scalar_type()), T, D, ptr(w), w_dt, ds.defined() ? &sh : nullptr, eps, &oh,
                                        ptr(dw), ptr(ws), need, st);
        }) != MLXQ_OK)
      return nullptr;
    if (dw.defined()) return tuple_of({dx, dw});
    PyObject* first = THPVariable_Wrap(std::move(dx));
    PyObject* out = first ? PyTuple_Pack(2, first, Py_None) : nullptr;
    Py_XDECREF(first);
    return out;
  });
}

bool get_scoring(PyObject* o, int& v) {
  if (!PyUnicode_CheckExact(o)) return false;
  if (PyUnicode_CompareWithASCIIString(o, "softmax") == 0) v = MLXQ_ROUTE_SOFTMAX;
  else if (PyUnicode_CompareWithASCIIString(o, "sigmoid") == 0) v = MLXQ_ROUTE_SIGMOID;
  else return false;
  return true;
}

bool get_logits(PyObject* o, at::Tensor& z) {
  const at::Tensor* p = any_gpu(o);
  if (!p || p->dim() != 2 || code_of(p->scalar_type()) < 0 || (p->stride(1) != 1 && p->size(1) > 1)) return false;
  z = *p;
  return true;
}

// route_experts(logits, top_k, scoring, bias, groups, kept_groups, group_best, normalize, scale, active)
PyObject* route_experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    at::Tensor z, bias, active;
    mlxq_router r = {};
    long k, g[3];
    if (n != 10 || !get_logits(a[0], z) || !ints(a + 1, 1, &k) || !get_scoring(a[2], r.scoring) || !ints(a + 4, 3, g) ||
        !truth(a[7], r.normalize) || !number(a[8], r.scale) || k < 1 || k > 64)
      return nullptr;
    const int64_t T = z.size(0), E = z.size(1);
    if (a[3] != Py_None) {
      const at::Tensor* t = get_exact(a[3], at::kFloat, {E}, z);
      if (!t) return nullptr;
      bias = *t;
    }
    if (a[9] != Py_None) {
      const at::Tensor* t = plain(a[9], 1);
      if (!t || t->scalar_type() != at::kBool || t->dim() != 1 || t->size(0) != T || t->device() != z.device()) return nullptr;
      active = *t;
    }
    r.top_k = k;
    r.bias = (const float*)ptr(bias);
    r.groups = g[0];
    r.kept_groups = g[1];
    r.group_best = g[2];
    bool ok;
    void* st = stream_of(z, ok);
    if (!ok) return nullptr;
    at::Tensor ids = at::empty({T, k}, z.options().dtype(at::kInt)), w = at::empty({T, k}, z.options().dtype(at::kFloat)),
               starts = at::empty({E + 1}, z.options().dtype(at::kInt)), rows = at::empty({T * k}, z.options().dtype(at::kInt));
    const mlxq_routing out = {ids.data_ptr<int32_t>(), w.data_ptr<float>(), starts.data_ptr<int32_t>(), rows.data_ptr<int32_t>(), T, k, E};
    const size_t need = mlxq_route_workspace_size(T * k, E);
    at::Tensor ws = workspace(z, need);
    if (unlocked([&] {
          return mlxq_route_experts(z.data_ptr(), code_of(z.scalar_type()), z.stride(0), &r, (const uint8_t*)ptr(active), &out, ptr(ws),
                                    need, st);
        }) != MLXQ_OK)
      return nullptr;
    return tuple_of({ids, w, starts, rows});
  });
}

// route_experts_backward(dweights, logits, ids, scoring, normalize, scale)
PyObject* route_experts_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    at::Tensor z;
    mlxq_router r = {};
    if (n != 6 || !get_logits(a[1], z) || !get_scoring(a[3], r.scoring) || !truth(a[4], r.normalize) || !number(a[5], r.scale)) return nullptr;
    const at::Tensor* ip = plain(a[2], 4);
    if (!ip || ip->scalar_type() != at::kInt || ip->dim() != 2 || ip->size(0) != z.size(0) || ip->device() != z.device()) return nullptr;
    const at::Tensor ids = *ip;
    const int64_t k = ids.size(1);
    const at::Tensor* wp = get_exact(a[0], at::kFloat, {z.size(0), k}, z);
    if (!wp || k < 1) return nullptr;
    const at::Tensor dw = *wp;
    bool ok;
    void* st = stream_of(z, ok);
    if (!ok) return nullptr;
    r.top_k = k;
    at::Tensor out = at::empty(z.sizes(), z.options());
    const mlxq_routing routing = {ids.data_ptr<int32_t>(), nullptr, nullptr, nullptr, z.size(0), k, z.size(1)};
    if (unlocked([&] {
          return mlxq_route_experts_backward(dw.data_ptr<float>(), z.data_ptr(), code_of(z.scalar_type()), z.stride(0), &r, &routing,
                                             out.data_ptr(), st);
        }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(out));
  });
}

// mx_experts(x, w, routing, bias, combine, dtype code)
PyObject* mx_experts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    MxOperand x, w;
    int combine;
    long dt;
    if (n != 6 || !get_mx(a[0], x) || !get_mx(a[1], w) || !truth(a[4], combine) || !ints(a + 5, 1, &dt)) return nullptr;
    if (w.codes.dim() != 3 || w.K != x.K || w.codes.device() != x.codes.device()) return nullptr;
    const int64_t E = w.codes.size(0), N = w.codes.size(1);
    if (!PyTuple_Check(a[2]) || PyTuple_GET_SIZE(a[2]) != 4) return nullptr;
    const at::Tensor* ip = plain(PyTuple_GET_ITEM(a[2], 0), 4);
    if (!ip || ip->scalar_type() != at::kInt || ip->dim() != 2 || ip->device() != x.codes.device()) return nullptr;
    const at::Tensor ids = *ip;
    const int64_t T = ids.size(0), k = ids.size(1), xd = x.codes.dim();
    const at::Tensor* wt = get_exact(PyTuple_GET_ITEM(a[2], 1), at::kFloat, {T, k}, ids);
    const at::Tensor* sp = get_exact(PyTuple_GET_ITEM(a[2], 2), at::kInt, {E + 1}, ids);
    const at::Tensor* rp = get_exact(PyTuple_GET_ITEM(a[2], 3), at::kInt, {T * k}, ids);
    if (!wt || !sp || !rp || (xd != 2 && xd != 3) || x.codes.size(0) != T || (xd == 3 && x.codes.size(1) != k)) return nullptr;
    const at::Tensor weights = *wt, starts = *sp, rows = *rp;
    at::Tensor bias;
    int bias_dt;
    const int64_t bias_shape[2] = {E, N};
    if (!get_float(a[3], at::IntArrayRef(bias_shape, 2), x.codes, bias, bias_dt)) return nullptr;
    bool ok;
    void* st = stream_of(x.codes, ok);
    if (!ok) return nullptr;
    const auto options = x.codes.options().dtype(float_type((int)dt));
    at::Tensor out = combine ? at::empty({T, N}, options) : at::empty({T, k, N}, options);
    const mlxq_routing routing = {ids.data_ptr<int32_t>(), weights.data_ptr<float>(), starts.data_ptr<int32_t>(), rows.data_ptr<int32_t>(),
                                  T, k, E};
    const size_t need = mlxq_mx_experts_workspace_size(T, k, N, combine, (int)dt);
    at::Tensor ws = workspace(x.codes, need);
    if (unlocked([&] {
          return mlxq_mx_experts(&x.m, xd == 3, x.K, &w.m, N, ptr(bias), bias_dt, &routing, combine, out.data_ptr(), (int)dt, ptr(ws), need,
                                 st);
        }) != MLXQ_OK)
      return nullptr;
    return THPVariable_Wrap(std::move(out));
  });
}

// set_error_type(MlxqError)
PyObject* set_error_type(PyObject*, PyObject* type) {
  Py_INCREF(type);
  Py_XSETREF(g_error, type);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"set_error_type", (PyCFunction)set_error_type, METH_O, nullptr},
    {"quantized_matmul", (PyCFunction)(void*)quantized_matmul, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void*)linear, METH_FASTCALL, nullptr},
    {"swiglu", (PyCFunction)(void*)swiglu, METH_FASTCALL, nullptr},
    {"embedding", (PyCFunction)(void*)embedding, METH_FASTCALL, nullptr},
    {"dequantize", (PyCFunction)(void*)dequantize, METH_FASTCALL, nullptr},
    {"quantize_batched", (PyCFunction)(void*)quantize_batched, METH_FASTCALL, nullptr},
    {"rotary", (PyCFunction)(void*)rotary, METH_FASTCALL, nullptr},
    {"cache_append", (PyCFunction)(void*)cache_append, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void*)paged_attention, METH_FASTCALL, nullptr},
    {"copy_pages", (PyCFunction)(void*)copy_pages, METH_FASTCALL, nullptr},
    {"mx_quantize", (PyCFunction)(void*)mx_quantize, METH_FASTCALL, nullptr},
    {"mx_dequantize", (PyCFunction)(void*)mx_dequantize, METH_FASTCALL, nullptr},
    {"mx_matmul", (PyCFunction)(void*)mx_matmul, METH_FASTCALL, nullptr},
    {"rms_norm", (PyCFunction)(void*)rms_norm, METH_FASTCALL, nullptr},
    {"rms_norm_backward", (PyCFunction)(void*)rms_norm_backward, METH_FASTCALL, nullptr},
    {"route_experts", (PyCFunction)(void*)route_experts, METH_FASTCALL, nullptr},
    {"route_experts_backward", (PyCFunction)(void*)route_experts_backward, METH_FASTCALL, nullptr},
    {"mx_experts", (PyCFunction)(void*)mx_experts, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fast", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

// Built against one torch's headers: another one's objects may be laid out differently.
bool built_for_this_torch() {
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* v = torch ? PyObject_GetAttrString(torch, "__version__") : nullptr;
  const char* text = v ? PyUnicode_AsUTF8(v) : nullptr;
  const bool same = text && strcmp(text, MLXQ_TORCH_VERSION) == 0;
  if (text && !same) PyErr_Format(PyExc_ImportError, "mlxq._fast is built for torch %s, not %s", MLXQ_TORCH_VERSION, text);
  Py_XDECREF(v);
  Py_XDECREF(torch);
  return same;
}

}  // namespace

PyMODINIT_FUNC PyInit__fast(void) {
  if (!built_for_this_torch()) return nullptr;
  PyObject* c = PyImport_ImportModule("torch._C");
  Py_XSETREF(g_stream_query, c ? PyObject_GetAttrString(c, "_cuda_getCurrentRawStream") : nullptr);
  Py_XDECREF(c);
  return g_stream_query ? PyModule_Create(&kModule) : nullptr;
}
