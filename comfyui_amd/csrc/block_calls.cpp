// The calls of functional.py's block-scaled operators without the interpreter's share: on a few rows a call takes as long on the host as on the
// device, most of it for attributes of tensors (0.35 us a tensor from Python, 48 tensors in a feed-forward of 8 experts) and allocations (1.5
// us). A function here checks what its Python counterpart checks and makes the same library call, and answers None where anything is
// not as that takes it without more ado: wrong types or shapes, scales to be laid out anew, no rows. Python then goes its own way and has the
// words. Tensors are made with torch's allocator; the stream is the caller's current one and its device the current device.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>

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

decltype(&hdmoe_quant_block_fp8) cast_rows;
decltype(&hdmoe_block_workspace_bytes) workspace_bytes;
decltype(&hdmoe_block_linear) linear;
decltype(&hdmoe_block_swiglu) swiglu;

int64_t blocks(int64_t n) { return (n + 127) / 128; }

const at::Tensor& tensor(PyObject* o) {
  need(THPVariable_Check(o));
  return THPVariable_Unpack(o);
}

int code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return HDMOE_W_BF16;
    case at::kHalf: return HDMOE_W_F16;
    case at::kFloat8_e4m3fn: return HDMOE_W_E4M3FN;
    default: throw Otherwise();
  }
}

struct Call {
  hdmoe_block_args a = {};
  hdmoe_block_weights w[HDMOE_BLOCK_MAX_EXPERTS] = {};
  at::Tensor x, scale;     // activations, their scales
  int64_t rows, K, N = -1;
  int act;

  Call(PyObject* px, PyObject* ps) {
    x = tensor(px);
    act = code(x);
    need(x.is_cuda() && x.dim() == 2 && x.is_contiguous());
    rows = x.size(0);
    K = x.size(1);
    need(rows > 0 && rows < (1ll << 30) && K > 0 && K < (1ll << 30));
    need((act == HDMOE_W_E4M3FN) == (ps != Py_None));
    if (ps != Py_None) {
      scale = tensor(ps);
      const int64_t KB = blocks(K);
      need(scale.scalar_type() == at::kFloat && scale.device() == x.device() && scale.dim() == 2 && scale.size(0) == rows && scale.size(1) == KB &&
           (rows == 1 || scale.stride(0) == 1) && (KB == 1 || scale.stride(1) == rows));
    }
    a.a_dtype = act;
  }
  const void* matrix(PyObject* pw, PyObject* ps, const float*& s) {
    const at::Tensor &m = tensor(pw), &t = tensor(ps);
    need(m.scalar_type() == at::kFloat8_e4m3fn && m.device() == x.device() && m.dim() == 2 && m.is_contiguous());
    if (N < 0) N = m.size(0);
    need(N > 0 && N < (1ll << 30) && m.size(0) == N && m.size(1) == K);
    need(t.scalar_type() == at::kFloat && t.device() == x.device() && t.dim() == 2 && t.size(0) == blocks(N) && t.size(1) == blocks(K) && t.is_contiguous());
    s = static_cast<const float*>(t.const_data_ptr());
    return m.const_data_ptr();
  }
  // (weight, scale, bias) or, gate/up, (w1, scale1, w3, scale3)
  void entry(hdmoe_block_weights& e, PyObject* const* o, bool gate_up, int out) {
    e.weight = matrix(o[0], o[1], e.scale);
    if (gate_up) {
      e.weight3 = matrix(o[2], o[3], e.scale3);
    } else if (o[2] != Py_None) {
      const at::Tensor& b = tensor(o[2]);
      need(code(b) == out && out != HDMOE_W_E4M3FN && b.device() == x.device() && b.dim() == 1 && b.size(0) == N && b.is_contiguous());
      e.bias = b.const_data_ptr();
    }
  }
  const int32_t* numbers(PyObject* o, int64_t n) {
    const at::Tensor& t = tensor(o);
    need(t.scalar_type() == at::kInt && t.device() == x.device() && t.dim() == 1 && t.size(0) == n && t.is_contiguous());
    return static_cast<const int32_t*>(t.const_data_ptr());
  }
  // The experts' segments of the rows, read through perm or not; the number of rows of the output
  int64_t routed(PyObject* poffsets, PyObject* pexperts, PyObject* pperm, bool gate_up, int out) {
    need(PyList_Check(pexperts) || PyTuple_Check(pexperts));
    const Py_ssize_t E = PySequence_Fast_GET_SIZE(pexperts), width = gate_up ? 4 : 3;
    need(E >= 1 && E <= HDMOE_BLOCK_MAX_EXPERTS);
    for (Py_ssize_t i = 0; i < E; ++i) {
      PyObject* const o = PySequence_Fast_GET_ITEM(pexperts, i);
      need((PyList_Check(o) || PyTuple_Check(o)) && PySequence_Fast_GET_SIZE(o) == width);
      entry(w[i], PySequence_Fast_ITEMS(o), gate_up, out);
    }
    int64_t n = rows;
    if (pperm != Py_None) {
      n = rows * 2;
      a.perm = numbers(pperm, n);
      a.T = static_cast<int>(rows);
    }
    a.offsets = numbers(poffsets, E + 1);
    a.E = static_cast<int>(E);
    a.rows = static_cast<int>(n);
    a.K = static_cast<int>(K);
    a.N = static_cast<int>(N);
    a.experts = w;
    activations(a.routed);
    return n;
  }
  int64_t dense(PyObject* const* weights, bool gate_up, int out) {
    entry(w[0], weights, gate_up, out);
    a.rows_static = static_cast<int>(rows);
    a.K_static = static_cast<int>(K);
    a.N_static = static_cast<int>(N);
    a.shared = w;
    activations(a.fixed);
    return rows;
  }
  // The static group of another call of one group
  void with(const Call& d) {
    need(d.act == act && d.x.device() == x.device());
    a.rows_static = d.a.rows_static;
    a.K_static = d.a.K_static;
    a.N_static = d.a.N_static;
    a.shared = d.a.shared;
    a.fixed = d.a.fixed;
  }
  void activations(hdmoe_block_rows& r) {
    r.a = x.const_data_ptr();
    if (scale.defined()) {
      r.scale_a = static_cast<const float*>(scale.const_data_ptr());
      r.scale_a_stride = rows;
    }
  }
  at::Tensor make(int64_t n, int64_t m, at::ScalarType type) const {
    Unlocked u;
    return at::empty({n, m}, at::TensorOptions().dtype(type).device(x.device()));
  }
  at::Tensor scales(int64_t n, int64_t m) const {
    Unlocked u;
    return at::empty_strided({n, blocks(m)}, {1, n}, at::TensorOptions().dtype(at::kFloat).device(x.device()));
  }
  int run(bool gate_up, void* stream) {
    Unlocked u;
    at::Tensor room;
    if (gate_up || act != HDMOE_W_E4M3FN) {
      const size_t n = workspace_bytes(&a, gate_up);
      if (n > 0) {
        room = at::empty({static_cast<int64_t>(n)}, at::TensorOptions().dtype(at::kByte).device(x.device()));
        a.workspace = room.mutable_data_ptr();
        a.workspace_bytes = n;
      }
    }
    return gate_up ? swiglu(&a, stream) : linear(&a, stream);
  }
  // out_dtype as a code, or -1: bf16 for cast rows, else the rows' own type
  int type(PyObject* o) const {
    const long c = PyLong_AsLong(o);
    if (c == -1) return act == HDMOE_W_E4M3FN ? HDMOE_W_BF16 : act;
    need((c == HDMOE_W_BF16 || c == HDMOE_W_F16) && (act == HDMOE_W_E4M3FN || c == act));
    return static_cast<int>(c);
  }
};

PyObject* tuple(std::initializer_list<at::Tensor> tensors) {
  PyObject* const r = PyTuple_New(tensors.size());
  if (r == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
  return r;
}
PyObject* const* items(PyObject* o, Py_ssize_t n) {
  need((PyList_Check(o) || PyTuple_Check(o)) && PySequence_Fast_GET_SIZE(o) == n);
  return PySequence_Fast_ITEMS(o);
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
int truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  need(v >= 0);
  return v;
}

// (x, stream)
PyObject* do_cast(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(2)
  return answer([&]() -> PyObject* {
    const at::Tensor& x = tensor(o[0]);
    const int act = code(x);
    need(act != HDMOE_W_E4M3FN && x.is_cuda() && x.is_contiguous() && x.dim() > 0);
    const int64_t K = x.size(-1);
    need(K > 0 && K < (1ll << 30) && x.numel() > 0);
    const int64_t rows = x.numel() / K;
    void* const stream = stream_of(o[1]);
    at::Tensor q, s;
    int rc;
    {
      Unlocked u;
      q = at::empty(x.sizes(), at::TensorOptions().dtype(at::kFloat8_e4m3fn).device(x.device()));
      s = at::empty_strided({rows, blocks(K)}, {1, rows}, at::TensorOptions().dtype(at::kFloat).device(x.device()));
      rc = cast_rows(act, x.const_data_ptr(), rows, static_cast<int>(K), q.mutable_data_ptr(), static_cast<float*>(s.mutable_data_ptr()), rows, stream);
    }
    return rc != 0 ? PyLong_FromLong(rc) : tuple({q, s});
  });
}

// (x, weight, scale, bias, scale_x, out_dtype, fixed_k_cut, stream)
PyObject* do_linear(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(8)
  return answer([&]() -> PyObject* {
    Call c(o[0], o[4]);
    c.a.out_dtype = c.type(o[5]);
    c.a.fixed_k_cut = truth(o[6]);
    const int64_t n = c.dense(o + 1, false, c.a.out_dtype);
    const at::Tensor y = c.make(n, c.N, c.a.out_dtype == HDMOE_W_BF16 ? at::kBFloat16 : at::kHalf);
    c.a.fixed.out = y.mutable_data_ptr();
    const int rc = c.run(false, stream_of(o[7]));
    return rc != 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(y);
  });
}

// (a, offsets, experts, scale_a, out_dtype, perm, shared, a_static, scale_static, fixed_k_cut, stream)
PyObject* do_grouped_linear(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(11)
  return answer([&]() -> PyObject* {
    Call c(o[0], o[3]);
    c.a.out_dtype = c.type(o[4]);
    c.a.fixed_k_cut = truth(o[9]);
    const at::ScalarType type = c.a.out_dtype == HDMOE_W_BF16 ? at::kBFloat16 : at::kHalf;
    const int64_t n = c.routed(o[1], o[2], o[5], false, c.a.out_dtype);
    if (o[6] == Py_None) {
      const at::Tensor y = c.make(n, c.N, type);
      c.a.routed.out = y.mutable_data_ptr();
      const int rc = c.run(false, stream_of(o[10]));
      return rc != 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(y);
    }
    need(c.act == HDMOE_W_E4M3FN);   // (16-bit rows of two groups: cast before)
    Call d(o[7], o[8]);
    need(d.act == c.act && d.x.device() == c.x.device());   // before anything is allocated
    const int64_t m = d.dense(items(o[6], 3), false, c.a.out_dtype);
    const at::Tensor y = c.make(n, c.N, type), z = d.make(m, d.N, type);
    c.a.routed.out = y.mutable_data_ptr();
    d.a.fixed.out = z.mutable_data_ptr();
    c.with(d);
    const int rc = c.run(false, stream_of(o[10]));
    return rc != 0 ? PyLong_FromLong(rc) : tuple({y, z});
  });
}

// What a gate/up writes for n rows
struct Cast {
  at::Tensor h, s;
  Cast(const Call& c, hdmoe_block_rows& r, int64_t n) : h(c.make(n, c.N, at::kFloat8_e4m3fn)), s(c.scales(n, c.N)) {
    r.out = h.mutable_data_ptr();
    r.scale_out = static_cast<float*>(s.mutable_data_ptr());
    r.scale_out_stride = n;
  }
};

// (x, w1, scale1, w3, scale3, scale_x, fixed_k_cut, exact, stream)
PyObject* do_swiglu(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(9)
  return answer([&]() -> PyObject* {
    Call c(o[0], o[5]);
    c.a.out_dtype = HDMOE_W_BF16;
    c.a.fixed_k_cut = truth(o[6]);
    c.a.exact = truth(o[7]);
    const int64_t n = c.dense(o + 1, true, HDMOE_W_BF16);
    const Cast out(c, c.a.fixed, n);
    const int rc = c.run(true, stream_of(o[8]));
    return rc != 0 ? PyLong_FromLong(rc) : tuple({out.h, out.s});
  });
}

// (a, offsets, experts, scale_a, perm, shared, fixed_k_cut, exact, stream)
PyObject* do_grouped_swiglu(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(9)
  return answer([&]() -> PyObject* {
    Call c(o[0], o[3]);
    c.a.out_dtype = HDMOE_W_BF16;
    c.a.fixed_k_cut = truth(o[6]);
    c.a.exact = truth(o[7]);
    const int64_t n = c.routed(o[1], o[2], o[4], true, HDMOE_W_BF16);
    const Cast out(c, c.a.routed, n);
    if (o[5] == Py_None) {
      const int rc = c.run(true, stream_of(o[8]));
      return rc != 0 ? PyLong_FromLong(rc) : tuple({out.h, out.s});
    }
    Call d(o[0], o[3]);
    const int64_t m = d.dense(items(o[5], 4), true, HDMOE_W_BF16);
    const Cast shared(d, d.a.fixed, m);
    c.with(d);
    const int rc = c.run(true, stream_of(o[8]));
    return rc != 0 ? PyLong_FromLong(rc) : tuple({out.h, out.s, shared.h, shared.s});
  });
}

// Addresses of the library's entry points: this module is not linked with it
PyObject* bind(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HDMOE_ARGUMENTS(4)
  cast_rows = reinterpret_cast<decltype(cast_rows)>(PyLong_AsVoidPtr(o[0]));
  workspace_bytes = reinterpret_cast<decltype(workspace_bytes)>(PyLong_AsVoidPtr(o[1]));
  linear = reinterpret_cast<decltype(linear)>(PyLong_AsVoidPtr(o[2]));
  swiglu = reinterpret_cast<decltype(swiglu)>(PyLong_AsVoidPtr(o[3]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<bind>("bind"), method<do_cast>("cast"), method<do_linear>("linear"), method<do_grouped_linear>("grouped_linear"),
                         method<do_swiglu>("swiglu"), method<do_grouped_swiglu>("grouped_swiglu"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_block_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version, hdmoe_version: whose headers this was compiled with; the caller compares them with the torch and the library that are there
PyMODINIT_FUNC PyInit__block_calls() {
  PyObject* const m = PyModule_Create(&module);
  if (m != nullptr && (PyModule_AddStringConstant(m, "torch_version", HDMOE_TORCH_VERSION) != 0 || PyModule_AddIntConstant(m, "hdmoe_version", HDMOE_VERSION) != 0)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
