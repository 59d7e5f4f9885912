// host.cpp -- the module's launch path as a CPython extension: every ldr_* entry point, and those of the block operators
// (lbk_*), as a builtin that takes tensors, None, numbers and address tables as they are, and the allocations around a read, a
// block join and dropout. A launch through ctypes costs 4-5 us
// of argument conversion (up to 30 arguments, each tensor's address fetched in Python before), and a small pass is a few
// dozen of them: these cost about 1 us.
//
// The entry points' addresses come from the library the Python binding loaded (bind), so both always call the same one.

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>

#include <cstring>
#include <tuple>
#include <utility>

#include "loopback_block.h"
#include "loopback_read.h"

namespace {

// one argument of an entry point, converted from a Python object; set() leaves a Python error on failure
template <typename A> struct Arg;

template <typename P> struct Arg<P*> {   // a device address: a tensor's, an int, or None
  P* v = nullptr;
  bool set(PyObject* o) {
    if (o == Py_None) return true;
    if (THPVariable_Check(o)) {
      v = static_cast<P*>(THPVariable_Unpack(o).data_ptr());
      return true;
    }
    v = static_cast<P*>(PyLong_AsVoidPtr(o));
    return !(v == nullptr && PyErr_Occurred());
  }
};

// A table of addresses: a list or tuple of tensors and ints (at most LDR_MAX_SOURCES), an array of 64-bit integers
// (anything with a buffer, as the stack's cached tables), or a device array's address as an int.
template <> struct Arg<const uint64_t*> {
  const uint64_t* v = nullptr;
  uint64_t own[LDR_MAX_SOURCES];
  Py_buffer buf{};
  bool held = false;
  ~Arg() { if (held) PyBuffer_Release(&buf); }
  bool set(PyObject* o) {
    if (o == Py_None) return true;
    const bool list = PyList_CheckExact(o);
    if (list || PyTuple_CheckExact(o)) {
      const Py_ssize_t n = list ? PyList_GET_SIZE(o) : PyTuple_GET_SIZE(o);
      if (n > LDR_MAX_SOURCES) {
        PyErr_SetString(PyExc_ValueError, "an address table of more than LDR_MAX_SOURCES entries");
        return false;
      }
      for (Py_ssize_t i = 0; i < n; ++i) {
        Arg<void*> e;
        if (!e.set(list ? PyList_GET_ITEM(o, i) : PyTuple_GET_ITEM(o, i))) return false;
        own[i] = reinterpret_cast<uint64_t>(e.v);
      }
      v = own;
      return true;
    }
    if (PyLong_Check(o)) {
      v = static_cast<const uint64_t*>(PyLong_AsVoidPtr(o));
      return !(v == nullptr && PyErr_Occurred());
    }
    if (PyObject_GetBuffer(o, &buf, PyBUF_SIMPLE) != 0) return false;
    held = true;
    v = static_cast<const uint64_t*>(buf.buf);
    return true;
  }
};

template <> struct Arg<int64_t> {
  int64_t v = 0;
  bool set(PyObject* o) {
    v = PyLong_AsLongLong(o);
    return !(v == -1 && PyErr_Occurred());
  }
};
template <> struct Arg<int> {
  int v = 0;
  bool set(PyObject* o) {
    const long x = PyLong_AsLong(o);
    if (x == -1 && PyErr_Occurred()) return false;
    v = static_cast<int>(x);
    return true;
  }
};
template <> struct Arg<uint32_t> {
  uint32_t v = 0;
  bool set(PyObject* o) {
    const unsigned long long x = PyLong_AsUnsignedLongLong(o);
    if (x == static_cast<unsigned long long>(-1) && PyErr_Occurred()) return false;
    if (x > 0xffffffffull) {
      PyErr_SetString(PyExc_OverflowError, "a 32-bit unsigned argument");
      return false;
    }
    v = static_cast<uint32_t>(x);
    return true;
  }
};
template <> struct Arg<float> {
  float v = 0.f;
  bool set(PyObject* o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) return false;
    v = static_cast<float>(x);
    return true;
  }
};

template <typename... A, size_t... I>
PyObject* invoke(int (*f)(A...), PyObject* const* args, std::index_sequence<I...>) {
  std::tuple<Arg<A>...> t;
  if (!(std::get<I>(t).set(args[I]) && ...)) return nullptr;
  int code;
  Py_BEGIN_ALLOW_THREADS
  code = f(std::get<I>(t).v...);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(code);
}

// one entry point: its address once bound, and the builtin that calls it
template <typename F, int ID> struct Entry;
template <typename... A, int ID> struct Entry<int (*)(A...), ID> {
  static inline int (*fn)(A...) = nullptr;
  static PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (!fn || n != static_cast<Py_ssize_t>(sizeof...(A))) {
      PyErr_Format(PyExc_TypeError, fn ? "entry point takes %zd arguments, got %zd" : "entry point not bound",
                   static_cast<Py_ssize_t>(sizeof...(A)), n);
      return nullptr;
    }
    return invoke(fn, args, std::index_sequence_for<A...>());
    END_HANDLE_TH_ERRORS
  }
  static void bind(void* p) { fn = reinterpret_cast<int (*)(A...)>(p); }
};

#define LDR_ENTRIES(X)                                                                                           \
  X(rstd_fwd) X(rstd_bwd) X(write_dots) X(split_queries) X(dots_online) X(read_fwd) X(read_fwd_online)             \
  X(read_bwd1) X(read_bwd1_noalloc) X(reduce_rows) X(blend_sum) X(read_bwd2_list) X(dv_assemble) X(read_fwd_any)   \
  X(read_bwd1_any) X(dv_assemble_any) X(read_bwd2_list_any) X(blend_sum_any) X(write_rows) X(read_fwd_rows)        \
  X(read_bwd1_rows) X(dv_assemble_rows) X(read_bwd2_list_rows) X(blend_sum_rows)

#define LBK_ENTRIES(X)                                                                                            \
  X(dropout) X(join_fwd) X(join_bwd) X(pad_rows) X(ffn_gate_up) X(ffn_dgate_up) X(linear_fwd) X(linear_dx) X(linear_dw)

enum Id {
#define X(name) ID_##name,
  LDR_ENTRIES(X)
#undef X
#define X(name) ID_block_##name,
  LBK_ENTRIES(X)
#undef X
};
#define BLOCK_FN(name) Entry<decltype(&lbk_##name), ID_block_##name>::fn
int64_t (*join_scratch)(int64_t, int64_t, int64_t) = nullptr;

struct Binding { const char* name; void (*bind)(void*); };
const Binding bindings[] = {
#define X(name) {"ldr_" #name, &Entry<decltype(&ldr_##name), ID_##name>::bind},
    LDR_ENTRIES(X)
#undef X
#define X(name) {"lbk_" #name, &Entry<decltype(&lbk_##name), ID_block_##name>::bind},
    LBK_ENTRIES(X)
#undef X
    {"lbk_join_scratch", [](void* p) { join_scratch = reinterpret_cast<decltype(join_scratch)>(p); }},
};

// bind(name, address) of an entry point; False for a name this module has no builtin for
PyObject* host_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "bind(name, address)");
    return nullptr;
  }
  const char* name = PyUnicode_AsUTF8(args[0]);
  if (!name) return nullptr;
  void* p = PyLong_AsVoidPtr(args[1]);
  if (!p && PyErr_Occurred()) return nullptr;
  for (const Binding& b : bindings)
    if (std::strcmp(b.name, name) == 0) {
      b.bind(p);
      Py_RETURN_TRUE;
    }
  Py_RETURN_FALSE;
}

// alias(t, s): t[s] as a tensor of its own on t's storage (no autograd view of t, its own version counter)
PyObject* host_alias(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2 || !THPVariable_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "alias(tensor, index)");
    return nullptr;
  }
  const at::Tensor& t = THPVariable_Unpack(args[0]);
  int64_t s = PyLong_AsLongLong(args[1]);
  if (s == -1 && PyErr_Occurred()) return nullptr;
  if (s < 0 && t.dim() > 0) s += t.size(0);
  if (t.dim() < 1 || s < 0 || s >= t.size(0)) {
    PyErr_SetString(PyExc_IndexError, "alias: index out of range");
    return nullptr;
  }
  at::Tensor out = at::empty({0}, t.options());
  out.set_(t.storage(), t.storage_offset() + s * t.stride(0), t.sizes().slice(1), t.strides().slice(1));
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// read_buffers(like, n_tok, n, prob, prior, dots): a read's outputs (out, tc, prob or None, next prior or None, raw
// scores or None)
PyObject* host_read_buffers(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !THPVariable_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "read_buffers(like, n_tok, n, prob, prior, dots)");
    return nullptr;
  }
  const at::Tensor& like = THPVariable_Unpack(args[0]);
  const int64_t n_tok = PyLong_AsLongLong(args[1]), ns = PyLong_AsLongLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(like.device());
  PyObject* out = PyTuple_New(5);
  if (!out) return nullptr;
  try {
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(at::empty_like(like)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(at::empty({n_tok, ns}, f32)));
    auto opt = [&](int i, PyObject* flag, at::IntArrayRef shape) {
      PyObject* o = Py_None;
      if (flag == Py_True) o = THPVariable_Wrap(at::empty(shape, f32));
      else Py_INCREF(o);
      PyTuple_SET_ITEM(out, i, o);
    };
    opt(2, args[3], {n_tok, ns});
    opt(3, args[4], {ns});
    opt(4, args[5], {ns, n_tok});
  } catch (...) {
    Py_DECREF(out);
    throw;
  }
  return out;
  END_HANDLE_TH_ERRORS
}

// ---- block operators: the results' allocation and the launch in one call ------------------------------------------
const at::Tensor* tensor_of(PyObject* o) {   // None: no tensor
  if (o == Py_None) return nullptr;
  TORCH_CHECK_TYPE(THPVariable_Check(o), "a tensor or None");
  return &THPVariable_Unpack(o);
}
void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
PyObject* wrapped(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
int64_t int_of(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double float_of(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
template <typename F> void launch(const char* name, bool bound, F&& f) {
  TORCH_CHECK(bound, name, ": entry point not bound");
  int code;
  Py_BEGIN_ALLOW_THREADS
  code = f();
  Py_END_ALLOW_THREADS
  TORCH_CHECK(code == 0, name, ": refused or failed to launch (code ", code, ")");
}
template <size_t N> PyObject* tuple_of(const at::Tensor (&ts)[N]) {
  PyObject* out = PyTuple_New(N);
  if (!out) throw python_error();
  for (size_t i = 0; i < N; ++i) PyTuple_SET_ITEM(out, i, wrapped(ts[i]));
  return out;
}

// dropout(x, rng, site, drop, dtype, stream): contiguous x
PyObject* host_dropout(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "dropout(x, rng, site, drop, dtype, stream)");
  const at::Tensor &x = *tensor_of(args[0]), &rng = *tensor_of(args[1]);
  const int64_t site = int_of(args[2]), drop = int_of(args[3]), dtype = int_of(args[4]), stream = int_of(args[5]);
  at::Tensor out = at::empty_like(x);
  const int64_t d = x.size(-1), rows = x.numel() / d;
  launch("lbk_dropout", BLOCK_FN(dropout), [&] {
    return BLOCK_FN(dropout)(x.data_ptr(), static_cast<const int64_t*>(rng.data_ptr()), static_cast<uint32_t>(site),
                             static_cast<int>(drop), out.data_ptr(), rows, d, static_cast<int>(dtype),
                             reinterpret_cast<void*>(stream));
  });
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// join_fwd(x, y, post, gate, gate_rows, pre, rng, site, drop, scale, eps, dtype, stream, keep): (h, n, r_post, r_pre)
PyObject* host_join_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 14, "join_fwd(x, y, post, gate, gate_rows, pre, rng, site, drop, scale, eps, dtype, stream, keep)");
  const at::Tensor &x = *tensor_of(args[0]), &y = *tensor_of(args[1]);
  const at::Tensor *post = tensor_of(args[2]), *gate = tensor_of(args[3]), *pre = tensor_of(args[5]), *rng = tensor_of(args[6]);
  const int64_t gate_rows = int_of(args[4]), site = int_of(args[7]), drop = int_of(args[8]), dtype = int_of(args[11]),
                stream = int_of(args[12]);
  const float scale = static_cast<float>(float_of(args[9])), eps = static_cast<float>(float_of(args[10]));
  const bool keep = args[13] == Py_True;
  const int64_t d = x.size(-1), rows = x.numel() / d;
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(x.device());
  at::Tensor t[4] = {at::empty_like(x), pre ? at::empty_like(x) : at::Tensor(),
                     keep && post ? at::empty({rows}, f32) : at::Tensor(), keep && pre ? at::empty({rows}, f32) : at::Tensor()};
  launch("lbk_join_fwd", BLOCK_FN(join_fwd), [&] {
    return BLOCK_FN(join_fwd)(x.data_ptr(), y.data_ptr(), ptr(post), ptr(gate), gate_rows, ptr(pre),
                              drop ? static_cast<const int64_t*>(ptr(rng)) : nullptr, static_cast<uint32_t>(site),
                              static_cast<int>(drop), scale, eps, t[0].data_ptr(), ptr(t[1]), static_cast<float*>(ptr(t[2])),
                              static_cast<float*>(ptr(t[3])), rows, d, static_cast<int>(dtype), reinterpret_cast<void*>(stream));
  });
  return tuple_of(t);
  END_HANDLE_TH_ERRORS
}

// join_bwd(dh, dn, h, y, post, gate, gate_rows, pre, r_post, r_pre, rng, site, drop, scale, dtype, stream, need): (dx, dy, dpost,
// dgate, dpre), those of need's bits 1, 2, 4, 8, 16
PyObject* host_join_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 17, "join_bwd takes 17 arguments");
  const at::Tensor *dh = tensor_of(args[0]), *dn = tensor_of(args[1]), *h = tensor_of(args[2]), *post = tensor_of(args[4]),
                   *gate = tensor_of(args[5]), *pre = tensor_of(args[7]), *r_post = tensor_of(args[8]),
                   *r_pre = tensor_of(args[9]), *rng = tensor_of(args[10]);
  const at::Tensor& y = *tensor_of(args[3]);
  const int64_t gate_rows = int_of(args[6]), site = int_of(args[11]), drop = int_of(args[12]), dtype = int_of(args[14]),
                stream = int_of(args[15]), need = int_of(args[16]);
  const float scale = static_cast<float>(float_of(args[13]));
  const int64_t d = y.size(-1), rows = y.numel() / d;
  at::Tensor t[5] = {need & 1 ? at::empty_like(y) : at::Tensor(), need & 2 ? at::empty_like(y) : at::Tensor(),
                     need & 4 && post ? at::empty_like(*post) : at::Tensor(),
                     need & 8 && gate ? at::empty_like(*gate) : at::Tensor(),
                     need & 16 && pre && dn ? at::empty_like(*pre) : at::Tensor()};
  at::Tensor scratch;
  if (t[2].defined() || t[3].defined() || t[4].defined()) {
    TORCH_CHECK(join_scratch, "lbk_join_scratch: entry point not bound");
    scratch = at::empty({join_scratch(rows, d, gate_rows)}, at::TensorOptions().dtype(at::kFloat).device(y.device()));
  }
  launch("lbk_join_bwd", BLOCK_FN(join_bwd), [&] {
    return BLOCK_FN(join_bwd)(ptr(dh), ptr(dn), ptr(h), y.data_ptr(), ptr(post), ptr(gate), gate_rows, ptr(pre),
                              static_cast<const float*>(ptr(r_post)), static_cast<const float*>(ptr(r_pre)),
                              drop ? static_cast<const int64_t*>(ptr(rng)) : nullptr, static_cast<uint32_t>(site),
                              static_cast<int>(drop), scale, ptr(t[0]), ptr(t[1]), ptr(t[2]), ptr(t[3]), ptr(t[4]),
                              static_cast<float*>(ptr(scratch)), rows, d, static_cast<int>(dtype),
                              reinterpret_cast<void*>(stream));
  });
  return tuple_of(t);
  END_HANDLE_TH_ERRORS
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {
#define X(name) {#name, FAST((&Entry<decltype(&ldr_##name), ID_##name>::call)), METH_FASTCALL, nullptr},
    LDR_ENTRIES(X)
#undef X
#define X(name) {"lbk_" #name, FAST((&Entry<decltype(&lbk_##name), ID_block_##name>::call)), METH_FASTCALL, nullptr},
    LBK_ENTRIES(X)
#undef X
    {"dropout", FAST(&host_dropout), METH_FASTCALL, nullptr},
    {"join_fwd", FAST(&host_join_fwd), METH_FASTCALL, nullptr},
    {"join_bwd", FAST(&host_join_bwd), METH_FASTCALL, nullptr},
    {"bind", FAST(&host_bind), METH_FASTCALL, nullptr},
    {"alias", FAST(&host_alias), METH_FASTCALL, nullptr},
    {"read_buffers", FAST(&host_read_buffers), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "launch path of the Loopback read", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
