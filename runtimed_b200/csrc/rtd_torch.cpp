// rtd_torch.cpp -- torch tensors into the C ABI of libruntimed_b200 for the calls of a decode
// step (runtimed_b200/kv4.py, sampling.py).
//
// Their kernels take a few microseconds, so what the host does per call counts: through
// ctypes a call took 15 us (20 argument conversions and as many attribute reads), of which
// the launch is 4.  Here the checks read the tensors' fields directly; a call takes 5 us.
// Positional arguments only: kv4.py and sampling.py give them their names and defaults.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <string>
#include <vector>

#include "rtd.h"

namespace {

PyObject* g_config_error = nullptr;  // runtimed_b200.errors
PyObject* g_shape_error = nullptr;
PyObject* g_raise = nullptr;         // (status, device) -> raises
PyObject* g_context = nullptr;       // (device) -> address of its rtd_ctx
constexpr int kMaxDevices = 64;
rtd_ctx* g_ctx[kMaxDevices] = {};

struct Failed {};  // a Python error is set

[[noreturn]] void config_error(const std::string& what) {
  PyErr_SetString(g_config_error, what.c_str());
  throw Failed{};
}

[[noreturn]] void shape_error(const char* name, std::vector<int64_t> want, at::IntArrayRef got) {
  PyObject* w = PyList_New((Py_ssize_t)want.size());
  for (size_t i = 0; i < want.size(); ++i) PyList_SET_ITEM(w, (Py_ssize_t)i, PyLong_FromLongLong(want[i]));
  PyObject* g = PyList_New((Py_ssize_t)got.size());
  for (size_t i = 0; i < got.size(); ++i) PyList_SET_ITEM(g, (Py_ssize_t)i, PyLong_FromLongLong(got[i]));
  PyObject* e = PyObject_CallFunction(g_shape_error, "sNN", name, w, g);
  if (e) {
    PyErr_SetObject(g_shape_error, e);
    Py_DECREF(e);
  }
  throw Failed{};
}

const at::Tensor& tensor(const char* name, PyObject* o) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: a tensor is wanted, got %.100s", name, Py_TYPE(o)->tp_name);
    throw Failed{};
  }
  return THPVariable_Unpack(o);
}

int64_t integer(const char* name, PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Failed{};
  if (v < INT32_MIN || v > INT32_MAX) config_error(std::string(name) + ": " + std::to_string(v) + " is no 32-bit number");
  return v;
}

int dtype_code(const char* name, at::ScalarType t) {
  switch (t) {
    case at::kFloat: return RTD_DT_F32;
    case at::kHalf: return RTD_DT_F16;
    case at::kBFloat16: return RTD_DT_BF16;
    default: config_error(std::string(name) + ": " + c10::toString(t) + " (f32, f16 or bf16)");
  }
}

at::ScalarType scalar_of(int code) { return code == RTD_DT_F32 ? at::kFloat : code == RTD_DT_F16 ? at::kHalf : at::kBFloat16; }

// A dense tensor of this type and shape on `dev`.
void* dense(const char* name, const at::Tensor& t, at::ScalarType type, c10::Device dev, std::initializer_list<int64_t> shape) {
  if (t.scalar_type() != type || t.device() != dev || !t.is_contiguous())
    config_error(std::string(name) + ": a contiguous " + c10::toString(type) + " tensor on " + dev.str() + " is wanted, got " +
                 c10::toString(t.scalar_type()) + " on " + t.device().str());
  const at::IntArrayRef got = t.sizes();
  if (!got.equals(at::IntArrayRef(shape.begin(), shape.size()))) shape_error(name, std::vector<int64_t>(shape), got);
  return t.data_ptr();
}

struct Pool {
  int64_t blocks, n_kv, head_dim;
  c10::Device dev;
  void* at;
};

Pool pool(const at::Tensor& t) {
  if (t.scalar_type() != at::kByte || t.dim() != 3 || !t.is_contiguous() || !t.is_cuda())
    config_error("pages: a contiguous uint8 CUDA tensor [blocks, n_kv, page bytes] is wanted");
  const int64_t bytes = t.size(2), d = bytes / 20;
  if (bytes % 640 || d < 32 || d > 128)
    config_error("pages: " + std::to_string(bytes) + " bytes a page (20 times a head_dim of 32, 64, 96 or 128)");
  if (t.size(1) < 1 || t.size(1) > INT32_MAX) config_error("pages: " + std::to_string(t.size(1)) + " kv heads");
  if (t.size(0) > INT32_MAX / 16) config_error("pages: more than 2^27 - 1 blocks");
  return Pool{t.size(0), t.size(1), d, t.device(), t.data_ptr()};
}

// Elements between the tokens of x [T, heads, D], whose heads lie side by side.
int64_t heads(const char* name, const at::Tensor& x, const Pool& p) {
  if (x.dim() != 3 || x.size(2) != p.head_dim) shape_error(name, {-1, -1, p.head_dim}, x.sizes());
  if (x.device() != p.dev) config_error(std::string(name) + ": on " + x.device().str() + ", the pages on " + p.dev.str());
  const int64_t t = x.size(0), h = x.size(1);
  if (x.stride(2) != 1 || (h > 1 && x.stride(1) != p.head_dim) || (t > 1 && x.stride(0) < h * p.head_dim))
    config_error(std::string(name) + ": strides (" + std::to_string(x.stride(0)) + ", " + std::to_string(x.stride(1)) + ", " +
                 std::to_string(x.stride(2)) + ") (a token's heads must lie side by side, tokens apart)");
  return t > 1 ? x.stride(0) : h * p.head_dim;
}

rtd_ctx* context(c10::Device dev) {
  const int d = dev.index();
  if (d < 0 || d >= kMaxDevices) config_error("device " + dev.str());
  if (!g_ctx[d]) {
    PyObject* h = PyObject_CallFunction(g_context, "i", d);
    if (!h) throw Failed{};
    g_ctx[d] = static_cast<rtd_ctx*>(PyLong_AsVoidPtr(h));
    Py_DECREF(h);
    if (PyErr_Occurred()) throw Failed{};
  }
  return g_ctx[d];
}

void* stream(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

void check(rtd_status st, c10::Device dev) {
  if (st == RTD_OK) return;
  PyObject* r = PyObject_CallFunction(g_raise, "ii", (int)st, (int)dev.index());
  if (r) {
    Py_DECREF(r);
    PyErr_Format(PyExc_RuntimeError, "rtd status %d", (int)st);
  }
  throw Failed{};
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device dev) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(dev));
}

void arity(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments are wanted, got %zd", want, got);
    throw Failed{};
  }
}

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }

// plan(want, length, table, free_list, free_count, max_tokens or None, out or None)
PyObject* plan(PyObject* const* a, Py_ssize_t n) {
  arity(n, 7);
  const at::Tensor &want = tensor("want", a[0]), &length = tensor("length", a[1]), &table = tensor("table", a[2]);
  const at::Tensor &list = tensor("free_list", a[3]), &count = tensor("free_count", a[4]);
  const c10::Device dev = table.device();
  if (!table.is_cuda()) config_error("table: on " + dev.str() + ", a CUDA device is wanted");
  if (table.dim() != 2) shape_error("table", {-1, -1}, table.sizes());
  const int64_t s = table.size(0), most = table.size(1), blocks = list.numel();
  if (s > INT32_MAX || most > INT32_MAX || blocks > INT32_MAX) config_error("plan: sizes beyond 32 bits");
  void* lists[4] = {};
  int64_t tokens = 0;
  at::Tensor fresh[4];
  if (a[6] != Py_None) {
    if (!PyTuple_Check(a[6]) || PyTuple_GET_SIZE(a[6]) != 4) config_error("out: (q_start, tok_seq, tok_pos, tok_slot) is wanted");
    static const char* names[4] = {"q_start", "tok_seq", "tok_pos", "tok_slot"};
    for (int i = 0; i < 4; ++i) {
      const at::Tensor& t = tensor(names[i], PyTuple_GET_ITEM(a[6], i));
      if (i == 1) tokens = t.numel();
      lists[i] = dense(names[i], t, at::kInt, dev, {i ? tokens : s + 1});
    }
    if (tokens > INT32_MAX) config_error("plan: sizes beyond 32 bits");
  } else if (a[5] != Py_None) {
    tokens = integer("max_tokens", a[5]);
    if (tokens < 0) config_error("max_tokens: " + std::to_string(tokens));
    for (int i = 0; i < 4; ++i) {
      fresh[i] = empty({i ? tokens : s + 1}, at::kInt, dev);
      lists[i] = fresh[i].data_ptr();
    }
  }
  const rtd_status st = rtd_kv_plan(context(dev), static_cast<int32_t*>(dense("want", want, at::kInt, dev, {s})), (int32_t)s,
                                    static_cast<int32_t*>(dense("length", length, at::kInt, dev, {s})),
                                    static_cast<int32_t*>(dense("table", table, at::kInt, dev, {s, most})), (int32_t)most,
                                    static_cast<int32_t*>(dense("free_list", list, at::kInt, dev, {blocks})),
                                    static_cast<int32_t*>(dense("free_count", count, at::kInt, dev, {1})), (int32_t)blocks,
                                    static_cast<int32_t*>(lists[0]), static_cast<int32_t*>(lists[1]),
                                    static_cast<int32_t*>(lists[2]), static_cast<int32_t*>(lists[3]), (int32_t)tokens,
                                    stream(dev));
  check(st, dev);
  if (a[6] != Py_None) return Py_NewRef(a[6]);
  if (a[5] == Py_None) Py_RETURN_NONE;
  PyObject* result = PyTuple_New(4);
  for (int i = 0; result && i < 4; ++i) PyTuple_SET_ITEM(result, i, wrap(std::move(fresh[i])));
  return result;
}

// append(q, k, v, inv_freq, tok_pos, tok_slot, pages, q_out or None)
PyObject* append(PyObject* const* a, Py_ssize_t n) {
  arity(n, 8);
  const at::Tensor &q = tensor("q", a[0]), &k = tensor("k", a[1]), &v = tensor("v", a[2]), &inv = tensor("inv_freq", a[3]);
  const at::Tensor &pos = tensor("tok_pos", a[4]), &slot = tensor("tok_slot", a[5]);
  const Pool p = pool(tensor("pages", a[6]));
  const int64_t ldq = heads("q", q, p), ldk = heads("k", k, p), ldv = heads("v", v, p);
  const int64_t t = q.size(0), n_head = q.size(1);
  for (const at::Tensor* x : {&k, &v})
    if (x->size(0) != t || x->size(1) != p.n_kv) shape_error(x == &k ? "k" : "v", {t, p.n_kv, p.head_dim}, x->sizes());
  const int dt = dtype_code("q", q.scalar_type());
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    config_error(std::string("q, k and v of one type are wanted, got ") + c10::toString(q.scalar_type()) + ", " +
                 c10::toString(k.scalar_type()) + ", " + c10::toString(v.scalar_type()));
  const int64_t half = inv.numel();
  dense("inv_freq", inv, at::kDouble, p.dev, {half});
  if (2 * half > p.head_dim) shape_error("inv_freq", {p.head_dim / 2}, inv.sizes());
  at::Tensor out = a[7] == Py_None ? empty({t, n_head, p.head_dim}, at::kFloat, p.dev) : tensor("q_out", a[7]);
  if (a[7] != Py_None) dense("q_out", out, at::kFloat, p.dev, {t, n_head, p.head_dim});
  check(rtd_rope_kv4_append(context(p.dev), q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, (uint32_t)dt, t,
                            (int32_t)n_head, (int32_t)p.n_kv, (int32_t)p.head_dim, (int32_t)(2 * half),
                            static_cast<double*>(inv.data_ptr()),
                            static_cast<int32_t*>(dense("tok_pos", pos, at::kInt, p.dev, {t})),
                            static_cast<int32_t*>(dense("tok_slot", slot, at::kInt, p.dev, {t})), p.at, (int32_t)p.blocks,
                            static_cast<float*>(out.data_ptr()), stream(p.dev)),
        p.dev);
  return wrap(std::move(out));
}

// read(pages, slots, dtype code)
PyObject* read(PyObject* const* a, Py_ssize_t n) {
  arity(n, 3);
  const Pool p = pool(tensor("pages", a[0]));
  const at::Tensor& slots = tensor("slots", a[1]);
  const int64_t rows = slots.numel(), dt = integer("dtype", a[2]);
  void* at_slots = dense("slots", slots, at::kInt, p.dev, {rows});
  at::Tensor k = empty({rows, p.n_kv, p.head_dim}, scalar_of((int)dt), p.dev);
  at::Tensor v = empty({rows, p.n_kv, p.head_dim}, scalar_of((int)dt), p.dev);
  check(rtd_kv4_read(context(p.dev), static_cast<int32_t*>(at_slots), rows, (int32_t)p.n_kv, (int32_t)p.head_dim, p.at,
                     (int32_t)p.blocks, k.data_ptr(), v.data_ptr(), (uint32_t)dt, stream(p.dev)),
        p.dev);
  PyObject* r = PyTuple_New(2);
  if (r) {
    PyTuple_SET_ITEM(r, 0, wrap(std::move(k)));
    PyTuple_SET_ITEM(r, 1, wrap(std::move(v)));
  }
  return r;
}

// attention(q, pages, table, q_start, ctx_len, max_q, max_ctx, scale or None, dtype code, out or None)
PyObject* attention(PyObject* const* a, Py_ssize_t n) {
  arity(n, 10);
  const at::Tensor &q = tensor("q", a[0]), &table = tensor("table", a[2]), &start = tensor("q_start", a[3]);
  const at::Tensor& len = tensor("ctx_len", a[4]);
  const Pool p = pool(tensor("pages", a[1]));
  const int64_t ldq = heads("q", q, p), t = q.size(0), n_head = q.size(1);
  const int qdt = dtype_code("q", q.scalar_type());
  if (table.dim() != 2) shape_error("table", {-1, -1}, table.sizes());
  const int64_t s = table.size(0), most = table.size(1);
  if (s > INT32_MAX || most > INT32_MAX) config_error("attention: sizes beyond 32 bits");
  const int64_t max_q = integer("max_q", a[5]), max_ctx = integer("max_ctx", a[6]);
  const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)p.head_dim) : PyFloat_AsDouble(a[7]);
  if (scale == -1.0 && PyErr_Occurred()) throw Failed{};
  at::Tensor out;
  if (a[9] == Py_None) {
    out = empty(q.sizes(), scalar_of((int)integer("dtype", a[8])), p.dev);
  } else {
    out = tensor("out", a[9]);
    if (!out.sizes().equals(q.sizes())) shape_error("out", q.sizes().vec(), out.sizes());
  }
  const int64_t ldo = heads("out", out, p);
  if (n_head % p.n_kv) config_error("attention: " + std::to_string(n_head) + " query heads over " + std::to_string(p.n_kv) + " kv heads");
  if (max_q < 1 || max_ctx < 1 || (max_ctx + 15) / 16 > most)
    config_error("attention: max_q " + std::to_string(max_q) + ", max_ctx " + std::to_string(max_ctx) + " with a table of " +
                 std::to_string(most) + " blocks a sequence");
  check(rtd_attention_kv4(context(p.dev), q.data_ptr(), (uint32_t)qdt, ldq, t, (int32_t)n_head, (int32_t)p.n_kv,
                          (int32_t)p.head_dim, (float)scale,
                          static_cast<int32_t*>(dense("q_start", start, at::kInt, p.dev, {s + 1})),
                          static_cast<int32_t*>(dense("ctx_len", len, at::kInt, p.dev, {s})), (int32_t)s,
                          static_cast<int32_t*>(dense("table", table, at::kInt, p.dev, {s, most})), (int32_t)most,
                          (int32_t)max_q, (int32_t)max_ctx, p.at, (int32_t)p.blocks, out.data_ptr(),
                          (uint32_t)dtype_code("out", out.scalar_type()), ldo, stream(p.dev)),
        p.dev);
  return wrap(std::move(out));
}

// sample(logits, u, temperature, top_k, top_p, min_p, out), the last five or None
PyObject* sample(PyObject* const* a, Py_ssize_t n) {
  arity(n, 7);
  const at::Tensor& x = tensor("logits", a[0]);
  if (x.dim() != 2) shape_error("logits", {-1, -1}, x.sizes());
  const c10::Device dev = x.device();
  if (!x.is_cuda()) config_error("logits: on " + dev.str() + ", a CUDA device is wanted");
  const int dt = dtype_code("logits", x.scalar_type());
  const int64_t rows = x.size(0), vocab = x.size(1), ld = rows > 1 ? x.stride(0) : vocab;
  if ((vocab > 1 && x.stride(1) != 1) || ld < vocab)
    config_error("logits: strides (" + std::to_string(x.stride(0)) + ", " + std::to_string(x.stride(1)) + ") (rows must be dense)");
  if (vocab < 1 || vocab > (1 << 19)) config_error("logits: " + std::to_string(vocab) + " entries a row (1 to 524288)");
  static const char* names[5] = {"u", "temperature", "top_k", "top_p", "min_p"};
  void* per_row[5] = {};
  for (int i = 0; i < 5; ++i)
    if (i == 0 || a[1 + i] != Py_None)
      per_row[i] = dense(names[i], tensor(names[i], a[1 + i]), i == 2 ? at::kInt : at::kFloat, dev, {rows});
  at::Tensor out = a[6] == Py_None ? empty({rows}, at::kInt, dev) : tensor("out", a[6]);
  if (a[6] != Py_None) dense("out", out, at::kInt, dev, {rows});
  check(rtd_sample(context(dev), x.data_ptr(), (uint32_t)dt, ld, rows, vocab, static_cast<float*>(per_row[1]),
                   static_cast<int32_t*>(per_row[2]), static_cast<float*>(per_row[3]), static_cast<float*>(per_row[4]),
                   static_cast<float*>(per_row[0]), static_cast<int32_t*>(out.data_ptr()), stream(dev)),
        dev);
  return wrap(std::move(out));
}

// setup(ConfigError, ShapeError, raise, context)
PyObject* setup(PyObject* const* a, Py_ssize_t n) {
  arity(n, 4);
  g_config_error = Py_NewRef(a[0]);
  g_shape_error = Py_NewRef(a[1]);
  g_raise = Py_NewRef(a[2]);
  g_context = Py_NewRef(a[3]);
  Py_RETURN_NONE;
}

// forget(device): its context was closed
PyObject* forget(PyObject* const* a, Py_ssize_t n) {
  arity(n, 1);
  const int64_t d = integer("device", a[0]);
  if (d >= 0 && d < kMaxDevices) g_ctx[d] = nullptr;
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(args, n);
  } catch (const Failed&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

#define ENTRY(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<f>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(plan),   ENTRY(append), ENTRY(read),   ENTRY(attention),
                         ENTRY(sample), ENTRY(setup),  ENTRY(forget), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rtd_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__rtd_torch(void) { return PyModule_Create(&module); }
