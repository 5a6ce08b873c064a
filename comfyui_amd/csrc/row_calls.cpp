// The calls of functional.py's layer norm, balance loss and adapters without the interpreter's share, which on a few rows is longer than the kernels
// (a layer norm of 77 rows 8.5 us of the host from Python, a router's loss and gradients 29). As in block_calls.cpp a function here checks what its Python
// counterpart checks and makes the same library call, and answers None where anything is not as that takes it: Python then goes its own way and
// has the words. Tensors are made with torch's allocator; the stream is the caller's current one and its device the current device.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>

#include <exception>
#include <initializer_list>

#include "../../include/hdmoe.h"

namespace {

struct Otherwise : std::exception {};   // for Python to say what it is, or to do
void need(bool ok) {
  if (!ok) throw Otherwise();
}

// Other Python threads may run while this one allocates or enqueues
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

decltype(&hdmoe_layer_norm) layer_norm;
decltype(&hdmoe_layer_norm_backward_workspace_bytes) layer_norm_bytes;
decltype(&hdmoe_layer_norm_backward) layer_norm_backward;
decltype(&hdmoe_gate_balance_workspace_bytes) balance_bytes;
decltype(&hdmoe_gate_balance) balance;
decltype(&hdmoe_gate_balance_backward) balance_backward;
decltype(&hdmoe_adapters_workspace_bytes) adapters_bytes;
decltype(&hdmoe_add_adapters) add_adapters;
decltype(&hdmoe_add_adapters_backward) add_adapters_backward;

const at::Tensor& tensor(PyObject* o) {
  need(THPVariable_Check(o));
  return THPVariable_Unpack(o);
}
const at::Tensor none;
const at::Tensor& optional(PyObject* o) { return o == Py_None ? none : tensor(o); }

int code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return HDMOE_T_BF16;
    case at::kHalf: return HDMOE_T_F16;
    case at::kFloat: return HDMOE_T_F32;
    default: throw Otherwise();
  }
}
// The rows a call is about: contiguous, on a device, with values in them
const at::Tensor& rows_of(PyObject* o, bool half) {
  const at::Tensor& x = tensor(o);
  need(x.is_cuda() && x.dim() > 0 && x.is_contiguous() && x.numel() > 0 && x.size(-1) < (1ll << 30) && x.numel() / x.size(-1) < (1ll << 30));
  need(!half || code(x) != HDMOE_T_F32);
  return x;
}
void like(const at::Tensor& t, const at::Tensor& x, at::ScalarType type, at::IntArrayRef shape) {
  need(t.scalar_type() == type && t.device() == x.device() && t.sizes() == shape && t.is_contiguous());
}
template <class T>
T* data(const at::Tensor& t) {
  return t.defined() ? static_cast<T*>(const_cast<void*>(t.const_data_ptr())) : nullptr;
}
at::Tensor make(const at::Tensor& x, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, at::TensorOptions().dtype(type).device(x.device())); }
at::Tensor make_like(const at::Tensor& t) { return t.defined() ? make(t, t.sizes(), t.scalar_type()) : at::Tensor(); }
template <class Args>
at::Tensor room(Args& a, const at::Tensor& x, size_t n) {
  at::Tensor t;
  if (n > 0) {
    t = make(x, {static_cast<int64_t>(n)}, at::kByte);
    a.workspace = t.mutable_data_ptr();
    a.workspace_bytes = n;
  }
  return t;
}

PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
PyObject* tuple(std::initializer_list<at::Tensor> tensors) {
  PyObject* const r = PyTuple_New(tensors.size());
  if (r == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) PyTuple_SET_ITEM(r, i++, wrap(t));
  return r;
}
// f's answer; None where f threw
template <class F>
PyObject* answer(F&& f) {
  try {
    return f();
  } catch (const std::exception&) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}
#define HDMOE_ARGUMENTS(n) \
  if (count != (n)) { PyErr_SetString(PyExc_TypeError, "wrong number of arguments"); return nullptr; }

void* stream_of(PyObject* o) { return PyLong_AsVoidPtr(o); }
float number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  need(PyErr_Occurred() == nullptr);
  return static_cast<float>(v);
}
int64_t integer(PyObject* o) {
  need(PyLong_Check(o));
  const long long v = PyLong_AsLongLong(o);
  need(PyErr_Occurred() == nullptr);
  return v;
}

// ---- layer norm ----------------------------------------------------------------------------------------------------

struct Norm {
  const at::Tensor &x, &w, &b;
  int64_t D, rows;
  int gain;
  Norm(PyObject* px, PyObject* pw, PyObject* pb) : x(rows_of(px, false)), w(optional(pw)), b(optional(pb)) {
    D = x.size(-1);
    need(D <= HDMOE_NORM_MAX_D);
    rows = x.numel() / D;
    gain = code(x);
    for (const at::Tensor* t : {&w, &b})
      if (t->defined()) {
        need((code(*t) == code(x) || t->scalar_type() == at::kFloat) && t->device() == x.device() && t->dim() == 1 && t->size(0) == D && t->is_contiguous());
        gain = code(*t);
      }
    need(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type());
  }
};

// (x, weight, bias, eps, stream)
PyObject* do_layer_norm(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(5)
  return answer([&]() -> PyObject* {
    const Norm n(o[0], o[1], o[2]);
    const float eps = number(o[3]);
    void* const stream = stream_of(o[4]);
    at::Tensor y;
    int rc;
    {
      Unlocked u;
      y = make_like(n.x);
      rc = layer_norm(code(n.x), data<void>(n.x), n.rows, static_cast<int>(n.D), n.gain, data<void>(n.w), data<void>(n.b), eps, y.mutable_data_ptr(), stream);
    }
    return rc != 0 ? PyLong_FromLong(rc) : wrap(y);
  });
}

int norm_backward(hdmoe_norm_grad_args& a, const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w, at::Tensor& dx, at::Tensor& dw, at::Tensor& db, void* stream) {
  dx = make_like(x);
  a.dtype = code(x);
  a.dy = data<void>(dy), a.x = data<void>(x), a.weight = data<void>(w);
  a.dx = data<void>(dx), a.dweight = data<void>(dw), a.dbias = data<void>(db);
  const at::Tensor ws = room(a, x, dw.defined() || db.defined() ? layer_norm_bytes(a.rows, a.D, a.rows_per_group) : 0);
  return layer_norm_backward(&a, stream);
}

// (dy, x, weight, bias, eps, gains, stream)
PyObject* do_layer_norm_backward(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(7)
  return answer([&]() -> PyObject* {
    const Norm n(o[1], o[2], o[3]);
    const at::Tensor& dy = tensor(o[0]);
    like(dy, n.x, n.x.scalar_type(), n.x.sizes());
    hdmoe_norm_grad_args a = {};
    a.gain_dtype = n.gain, a.D = static_cast<int>(n.D), a.rows = a.rows_per_group = n.rows, a.eps = number(o[4]);
    const int gains = PyObject_IsTrue(o[5]);
    need(gains >= 0);
    void* const stream = stream_of(o[6]);
    at::Tensor dx, dw, db;
    int rc;
    {
      Unlocked u;
      if (gains) dw = make_like(n.w), db = make_like(n.b);
      rc = norm_backward(a, dy, n.x, n.w, dx, dw, db, stream);
    }
    return rc != 0 ? PyLong_FromLong(rc) : tuple({dx, dw, db});
  });
}

// (dy, x, scale, tokens_per_batch, eps, stream)
PyObject* do_ln_modulate_backward(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(6)
  return answer([&]() -> PyObject* {
    const at::Tensor &x = rows_of(o[1], false), &dy = tensor(o[0]), &scale = tensor(o[2]);
    const int64_t per = integer(o[3]);
    need(x.dim() == 2 && x.size(1) <= HDMOE_NORM_MAX_D && per > 0 && x.size(0) % per == 0);
    like(dy, x, x.scalar_type(), x.sizes());
    like(scale, x, x.scalar_type(), {x.size(0) / per, x.size(1)});
    hdmoe_norm_grad_args a = {};
    a.gain_dtype = code(x), a.D = static_cast<int>(x.size(1)), a.rows = x.size(0), a.rows_per_group = per, a.one_plus = 1, a.eps = number(o[4]);
    void* const stream = stream_of(o[5]);
    at::Tensor dx, ds, dsh;
    int rc;
    {
      Unlocked u;
      ds = make_like(scale), dsh = make_like(scale);
      rc = norm_backward(a, dy, x, scale, dx, ds, dsh, stream);
    }
    return rc != 0 ? PyLong_FromLong(rc) : tuple({dx, ds, dsh});
  });
}

// ---- the router's balance loss ---------------------------------------------------------------------------------------

struct Balance {
  hdmoe_balance_args a = {};
  const at::Tensor &x, &w, &idx, &mask;
  Balance(PyObject* px, PyObject* pw, PyObject* pidx, PyObject* pmask, int64_t sequences, PyObject* palpha)
      : x(rows_of(px, true)), w(tensor(pw)), idx(tensor(pidx)), mask(optional(pmask)) {
    need(x.dim() == 2 && w.dim() == 2 && idx.dim() == 2);
    const int64_t T = x.size(0);
    like(w, x, x.scalar_type(), {w.size(0), x.size(1)});
    like(idx, x, at::kInt, {T, idx.size(1)});
    if (mask.defined()) need(mask.scalar_type() == at::kBool && mask.device() == x.device() && mask.is_contiguous() && mask.numel() == T);
    need(sequences > 0 && T % sequences == 0 && w.size(0) < (1 << 20) && idx.size(1) < (1 << 20));
    a.dtype = code(x), a.T = static_cast<int>(T), a.sequences = static_cast<int>(sequences), a.D = static_cast<int>(x.size(1));
    a.E = static_cast<int>(w.size(0)), a.k = static_cast<int>(idx.size(1)), a.alpha = number(palpha);
    a.x = data<void>(x), a.gate_w = data<void>(w), a.topk_idx = data<int32_t>(idx), a.mask = data<uint8_t>(mask);
  }
};

// (x, gate_w, topk_idx, alpha, sequences, mask, stream)
PyObject* do_gate_balance(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(7)
  return answer([&]() -> PyObject* {
    Balance c(o[0], o[1], o[2], o[5], integer(o[4]), o[3]);
    void* const stream = stream_of(o[6]);
    at::Tensor loss, counts, scores;
    int rc;
    {
      Unlocked u;
      loss = make(c.x, {}, at::kFloat), counts = make(c.x, {c.a.sequences, c.a.E}, at::kInt), scores = make(c.x, {c.a.T, c.a.E}, at::kFloat);
      c.a.loss = data<float>(loss), c.a.counts = data<int32_t>(counts), c.a.scores = data<void>(scores);
      const at::Tensor ws = room(c.a, c.x, balance_bytes(&c.a, 0));
      rc = balance(&c.a, stream);
    }
    return rc != 0 ? PyLong_FromLong(rc) : tuple({loss, counts, scores});
  });
}

// (dloss, x, gate_w, topk_idx, counts, scores, alpha, mask, dweight, stream)
PyObject* do_gate_balance_backward(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(10)
  return answer([&]() -> PyObject* {
    const at::Tensor &dloss = tensor(o[0]), &counts = tensor(o[4]), &scores = tensor(o[5]), &dweight = optional(o[8]);
    need(counts.dim() == 2);
    Balance c(o[1], o[2], o[3], o[7], counts.size(0), o[6]);
    like(dloss, c.x, at::kFloat, {});
    like(counts, c.x, at::kInt, {c.a.sequences, c.a.E});
    like(scores, c.x, at::kFloat, {c.a.T, c.a.E});
    if (dweight.defined()) like(dweight, c.x, c.x.scalar_type(), {c.a.T, c.a.k});
    c.a.dloss = data<float>(dloss), c.a.counts = data<int32_t>(counts), c.a.scores = data<void>(scores), c.a.dweight = data<void>(dweight);
    void* const stream = stream_of(o[9]);
    at::Tensor dx, dw;
    int rc;
    {
      Unlocked u;
      dx = make_like(c.x), dw = make_like(c.w);
      c.a.dx = data<void>(dx), c.a.dgate_w = data<void>(dw);
      const at::Tensor ws = room(c.a, c.x, balance_bytes(&c.a, 1));
      rc = balance_backward(&c.a, stream);
    }
    return rc != 0 ? PyLong_FromLong(rc) : tuple({dx, dw});
  });
}

// ---- adapters ----------------------------------------------------------------------------------------------------------

struct Adapters {
  hdmoe_adapter_args p = {};
  const at::Tensor &x, &a, &b;
  Adapters(PyObject* px, PyObject* pa, PyObject* pb, PyObject* pscale, PyObject* pindex) : x(rows_of(px, true)), a(tensor(pa)), b(tensor(pb)) {
    const at::Tensor &scale = tensor(pscale), &index = tensor(pindex);
    need(x.dim() >= 2 && a.dim() == 3 && b.dim() == 3);
    const int64_t n = a.size(0), R = a.size(1), K = x.size(-1), N = b.size(1), rows = x.numel() / K, requests = index.numel();
    like(a, x, x.scalar_type(), {n, R, K});
    like(b, x, x.scalar_type(), {n, N, R});
    like(scale, x, at::kFloat, {n});
    need(index.scalar_type() == at::kInt && index.device() == x.device() && index.is_contiguous() && requests > 0 && rows % requests == 0);
    need(n < (1 << 20) && R < (1 << 20) && N < (1ll << 30));
    p.dtype = code(x), p.rows = static_cast<int>(rows), p.requests = static_cast<int>(requests), p.K = static_cast<int>(K), p.N = static_cast<int>(N);
    p.n = static_cast<int>(n), p.R = static_cast<int>(R);
    p.x = data<void>(x), p.a = data<void>(a), p.b = data<void>(b), p.scale = data<float>(scale), p.index = data<int32_t>(index);
  }
  // rows like x's, N long
  void beside(const at::Tensor& t) const {
    need(t.scalar_type() == x.scalar_type() && t.device() == x.device() && t.dim() == x.dim() && t.size(-1) == p.N && t.is_contiguous());
    for (int64_t i = 0; i + 1 < x.dim(); ++i) need(t.size(i) == x.size(i));
  }
};

// (base, x, a, b, scale, index, out, fixed_k_cut, stream)
PyObject* do_add_adapters(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(9)
  return answer([&]() -> PyObject* {
    Adapters c(o[1], o[2], o[3], o[4], o[5]);
    const at::Tensor& base = tensor(o[0]);
    c.beside(base);
    if (o[6] != Py_None) c.beside(tensor(o[6]));
    const int fixed = PyObject_IsTrue(o[7]);
    need(fixed >= 0);
    c.p.fixed_k_cut = fixed;
    void* const stream = stream_of(o[8]);
    at::Tensor out = optional(o[6]);
    int rc;
    {
      Unlocked u;
      if (!out.defined()) out = make_like(base);
      c.p.base = data<void>(base), c.p.out = data<void>(out);
      const at::Tensor ws = room(c.p, c.x, adapters_bytes(&c.p, 0));
      rc = add_adapters(&c.p, stream);
    }
    if (rc != 0) return PyLong_FromLong(rc);
    if (o[6] == Py_None) return wrap(out);
    Py_INCREF(o[6]);
    return o[6];
  });
}

// (dy, x, a, b, scale, index, stream)
PyObject* do_add_adapters_backward(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(7)
  return answer([&]() -> PyObject* {
    Adapters c(o[1], o[2], o[3], o[4], o[5]);
    const at::Tensor& dy = tensor(o[0]);
    c.beside(dy);
    void* const stream = stream_of(o[6]);
    at::Tensor dx, da, db;
    int rc;
    {
      Unlocked u;
      dx = make_like(c.x), da = make_like(c.a), db = make_like(c.b);
      c.p.dy = data<void>(dy), c.p.dx = data<void>(dx), c.p.da = data<void>(da), c.p.db = data<void>(db);
      const at::Tensor ws = room(c.p, c.x, adapters_bytes(&c.p, 1));
      rc = add_adapters_backward(&c.p, stream);
    }
    return rc != 0 ? PyLong_FromLong(rc) : tuple({dx, da, db});
  });
}

// Addresses of the library's entry points: this module is not linked with it
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(9)
  layer_norm = reinterpret_cast<decltype(layer_norm)>(PyLong_AsVoidPtr(o[0]));
  layer_norm_bytes = reinterpret_cast<decltype(layer_norm_bytes)>(PyLong_AsVoidPtr(o[1]));
  layer_norm_backward = reinterpret_cast<decltype(layer_norm_backward)>(PyLong_AsVoidPtr(o[2]));
  balance_bytes = reinterpret_cast<decltype(balance_bytes)>(PyLong_AsVoidPtr(o[3]));
  balance = reinterpret_cast<decltype(balance)>(PyLong_AsVoidPtr(o[4]));
  balance_backward = reinterpret_cast<decltype(balance_backward)>(PyLong_AsVoidPtr(o[5]));
  adapters_bytes = reinterpret_cast<decltype(adapters_bytes)>(PyLong_AsVoidPtr(o[6]));
  add_adapters = reinterpret_cast<decltype(add_adapters)>(PyLong_AsVoidPtr(o[7]));
  add_adapters_backward = reinterpret_cast<decltype(add_adapters_backward)>(PyLong_AsVoidPtr(o[8]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<bind>("bind"),
                         method<do_layer_norm>("layer_norm"),
                         method<do_layer_norm_backward>("layer_norm_backward"),
                         method<do_ln_modulate_backward>("ln_modulate_backward"),
                         method<do_gate_balance>("gate_balance"),
                         method<do_gate_balance_backward>("gate_balance_backward"),
                         method<do_add_adapters>("add_adapters"),
                         method<do_add_adapters_backward>("add_adapters_backward"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_row_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version, hdmoe_version: whose headers this was compiled with; the caller compares them with the torch and the library that are there
PyMODINIT_FUNC PyInit__row_calls() {
  PyObject* const m = PyModule_Create(&module);
  if (m != nullptr && (PyModule_AddStringConstant(m, "torch_version", HDMOE_TORCH_VERSION) != 0 || PyModule_AddIntConstant(m, "hdmoe_version", HDMOE_VERSION) != 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
