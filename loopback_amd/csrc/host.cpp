// host.cpp -- the module's launch path as a CPython extension: every ldr_* entry point as a builtin that takes tensors, None,
// numbers and address tables as they are, the allocations around a read, and the block operators (lbk_*) with the allocations
// and autograd nodes around them. A launch through ctypes costs 4-5 us of argument conversion (up to 30 arguments, each
// tensor's address fetched in Python before), and a small pass is a few dozen of them: these cost about 1 us.
//
// The entry points' addresses come from the library the Python binding loaded (bind), so both always call the same one.

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

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
#define BLOCK_FN(name) (Entry<decltype(&lbk_##name), ID_block_##name>::fn)
int64_t (*join_scratch)(int64_t, int64_t, int64_t) = nullptr;
int64_t (*linear_scratch)(int64_t, int64_t, int64_t) = nullptr;
int64_t (*ffn_saved_bytes)(int64_t, int64_t) = nullptr;

struct Binding { const char* name; void (*bind)(void*); };
const Binding bindings[] = {
#define X(name) {"ldr_" #name, &Entry<decltype(&ldr_##name), ID_##name>::bind},
    LDR_ENTRIES(X)
#undef X
#define X(name) {"lbk_" #name, &Entry<decltype(&lbk_##name), ID_block_##name>::bind},
    LBK_ENTRIES(X)
#undef X
    {"lbk_join_scratch", [](void* p) { join_scratch = reinterpret_cast<decltype(join_scratch)>(p); }},
    {"lbk_linear_scratch", [](void* p) { linear_scratch = reinterpret_cast<decltype(linear_scratch)>(p); }},
    {"lbk_ffn_saved_bytes", [](void* p) { ffn_saved_bytes = reinterpret_cast<decltype(ffn_saved_bytes)>(p); }},
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

// ---- block operators: the results' allocation and the launch in one call, and their autograd nodes ------------------
// The nodes are C++ ones: an ordinary backward then runs without Python (a Python node's costs the engine's thread some 40 us of
// waiting for the interpreter and calling). One that has to see torch operations -- it is itself differentiated, a dispatch mode,
// a transform or forward mode is on, its gradients are batched or of another kind -- calls the torch form in Python.
using OptTensor = std::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

OptTensor opt_tensor(PyObject* o) {   // None: no tensor
  if (o == Py_None) return std::nullopt;
  TORCH_CHECK_TYPE(THPVariable_Check(o), "a tensor or None");
  return THPVariable_Unpack(o);
}
const at::Tensor& tensor_of(PyObject* o) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), "a tensor");
  return THPVariable_Unpack(o);
}
void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const OptTensor& t) { return t ? ptr(*t) : nullptr; }
at::Tensor or_none(const OptTensor& t) { return t ? *t : at::Tensor(); }
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
void launched(const char* name, int code) {
  TORCH_CHECK(code == 0, name, ": refused or failed to launch (code ", code, ")");
}
PyObject* tuple_of(const variable_list& ts) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!out) throw python_error();
  for (size_t i = 0; i < ts.size(); ++i) PyTuple_SET_ITEM(out, i, wrapped(ts[i]));
  return out;
}
struct NoGil {   // the interpreter is free while this lives
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};
struct Gil {
  PyGILState_STATE state = PyGILState_Ensure();
  ~Gil() { PyGILState_Release(state); }
};

// the backwards' torch forms, Python functions of block_ops: dropout's, the join's and the feed-forward block's
PyObject* torch_forms[3] = {nullptr, nullptr, nullptr};

// torch_forms[which](*tensors, *numbers) with None for undefined tensors: its tuple of `results` tensors
variable_list torch_form(int which, const variable_list& tensors, std::initializer_list<int64_t> ints,
                         std::initializer_list<double> floats, size_t results) {
  Gil gil;
  TORCH_CHECK(torch_forms[which], "the block operators' torch forms are not bound");
  struct Ref {
    PyObject* o;
    ~Ref() { Py_XDECREF(o); }
  };
  auto fail = []() {
    python_error e;
    e.persist();
    throw e;
  };
  Ref args{PyTuple_New(static_cast<Py_ssize_t>(tensors.size() + ints.size() + floats.size()))};
  if (!args.o) fail();
  Py_ssize_t n = 0;
  for (const at::Tensor& t : tensors) PyTuple_SET_ITEM(args.o, n++, wrapped(t));
  for (int64_t v : ints) PyTuple_SET_ITEM(args.o, n++, PyLong_FromLongLong(v));
  for (double v : floats) PyTuple_SET_ITEM(args.o, n++, PyFloat_FromDouble(v));
  Ref got{PyObject_CallObject(torch_forms[which], args.o)};
  if (!got.o) fail();
  TORCH_CHECK(PyTuple_Check(got.o) && PyTuple_GET_SIZE(got.o) == static_cast<Py_ssize_t>(results), "a torch form's results");
  variable_list out(results);
  for (size_t i = 0; i < results; ++i) {
    PyObject* o = PyTuple_GET_ITEM(got.o, static_cast<Py_ssize_t>(i));
    if (o != Py_None) out[i] = tensor_of(o);
  }
  return out;
}

// whether a backward with these gradients runs on the kernels, for rows of `like`'s type and device, and its shape
bool on_kernels(const variable_list& grads, const at::Tensor& like, bool same_shape = true) {
  using c10::DispatchKey;
  if (at::GradMode::is_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
      c10::impl::tls_is_dispatch_key_included(DispatchKey::FuncTorchDynamicLayerFrontMode))
    return false;
  constexpr c10::DispatchKeySet other({DispatchKey::Python, DispatchKey::Batched, DispatchKey::FuncTorchBatched,
                                       DispatchKey::FuncTorchGradWrapper, DispatchKey::Functionalize, DispatchKey::ZeroTensor,
                                       DispatchKey::Conjugate, DispatchKey::Negative});
  for (const at::Tensor& g : grads)
    if (g.defined() && (g.layout() != at::kStrided || g.device() != like.device() || g.scalar_type() != like.scalar_type() ||
                        (same_shape && g.sizes() != like.sizes()) || g.key_set().has_any(other) || g._fw_grad(0).defined()))
      return false;
  return true;
}
// A backward launches where its results are allocated and its gradients copied: on the current stream of their GPU. The engine
// makes that the forward's stream; a node that is called by itself runs on its caller's.
int64_t stream_of(const at::Tensor& t) {
  return static_cast<int64_t>(reinterpret_cast<intptr_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream()));
}
// The kernels index a saved tensor by the forward's sizes; a saved-tensor hook may give back any other.
void as_saved(const at::Tensor& t, const at::Tensor& like, at::ScalarType type, int64_t rows, int64_t cols) {
  if (!t.defined()) return;
  TORCH_CHECK(t.layout() == at::kStrided && t.device() == like.device() && t.scalar_type() == type && t.dim() > 0 &&
                  t.numel() == rows * cols && t.size(-1) == cols,
              "a block operator's saved tensor came back from a hook with another shape, type or device: ", t.toString(), " ", t.sizes(),
              " on ", t.device());
}
int64_t code_of(at::ScalarType t) { return t == at::kFloat ? LDR_F32 : t == at::kBFloat16 ? LDR_BF16 : t == at::kHalf ? LDR_F16 : -1; }
at::Tensor rows_of(const at::Tensor& t) { return t.defined() && !t.is_contiguous() ? t.contiguous() : t; }

at::Tensor dropout_run(const at::Tensor& x, const at::Tensor& rng, int64_t site, int64_t drop, int64_t dtype, int64_t stream) {
  at::Tensor out = at::empty_like(x);
  const int64_t d = x.size(-1);
  TORCH_CHECK(BLOCK_FN(dropout), "lbk_dropout: entry point not bound");
  launched("lbk_dropout", BLOCK_FN(dropout)(x.data_ptr(), static_cast<const int64_t*>(rng.data_ptr()), static_cast<uint32_t>(site),
                                            static_cast<int>(drop), out.data_ptr(), x.numel() / d, d, static_cast<int>(dtype),
                                            reinterpret_cast<void*>(stream)));
  return out;
}

struct DropoutNode : torch::autograd::Function<DropoutNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& rng, int64_t site, int64_t drop,
                            int64_t dtype, int64_t stream) {
    ctx->save_for_backward({rng});
    ctx->saved_data["numbers"] = std::vector<int64_t>{site, drop};
    ctx->set_materialize_grads(false);
    return dropout_run(x, rng, site, drop, dtype, stream);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    const at::Tensor rng = ctx->get_saved_variables()[0];
    const std::vector<int64_t> n = ctx->saved_data["numbers"].toIntVector();
    const at::Tensor& g = grads[0];   // its own rows: nothing of the forward's sizes is indexed
    as_saved(rng, g, at::kLong, 1, 2);
    const int64_t code = code_of(g.scalar_type());
    if (!on_kernels(grads, g) || !g.is_cuda() || !rng.is_contiguous() || code < 0 || g.dim() == 0 || g.numel() == 0) {
      out[0] = torch_form(0, {g, rng}, {n[0], n[1]}, {}, 1)[0];
      return out;
    }
    const c10::DeviceGuard on(g.device());
    out[0] = dropout_run(rows_of(g), rng, n[0], n[1], code, stream_of(g));
    return out;
  }
};

variable_list join_run(const at::Tensor& x, const at::Tensor& y, const OptTensor& post, const OptTensor& gate, int64_t gate_rows,
                       const OptTensor& pre, const OptTensor& rng, int64_t site, int64_t drop, double scale, double eps,
                       int64_t dtype, int64_t stream, bool keep) {   // h, n, r_post, r_pre
  const int64_t d = x.size(-1), rows = x.numel() / d;
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(x.device());
  variable_list t{at::empty_like(x), pre ? at::empty_like(x) : at::Tensor(),
                  keep && post ? at::empty({rows}, f32) : at::Tensor(), keep && pre ? at::empty({rows}, f32) : at::Tensor()};
  TORCH_CHECK(BLOCK_FN(join_fwd), "lbk_join_fwd: entry point not bound");
  launched("lbk_join_fwd",
           BLOCK_FN(join_fwd)(x.data_ptr(), y.data_ptr(), ptr(post), ptr(gate), gate_rows, ptr(pre),
                              drop ? static_cast<const int64_t*>(ptr(rng)) : nullptr, static_cast<uint32_t>(site),
                              static_cast<int>(drop), static_cast<float>(scale), static_cast<float>(eps), t[0].data_ptr(), ptr(t[1]),
                              static_cast<float*>(ptr(t[2])), static_cast<float*>(ptr(t[3])), rows, d, static_cast<int>(dtype),
                              reinterpret_cast<void*>(stream)));
  return t;
}

struct JoinNode : torch::autograd::Function<JoinNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& y, const OptTensor& post,
                               const OptTensor& gate, const OptTensor& pre, const OptTensor& rng, int64_t gate_rows, int64_t site,
                               int64_t drop, double scale, double eps, int64_t dtype, int64_t stream) {
    variable_list t = join_run(x, y, post, gate, gate_rows, pre, rng, site, drop, scale, eps, dtype, stream, true);
    ctx->save_for_backward({pre ? x : at::Tensor(), y, or_none(post), or_none(gate), or_none(pre), t[2], t[3], or_none(rng)});
    ctx->saved_data["numbers"] = std::vector<int64_t>{gate_rows, site, drop, dtype, x.numel() / x.size(-1), x.size(-1)};
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    t.resize(pre ? 2 : 1);
    return t;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(13);
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &y = saved[1], &post = saved[2], &gate = saved[3], &pre = saved[4], &rng = saved[7];
    const at::Tensor dh = grads[0], dn = grads.size() > 1 ? grads[1] : at::Tensor();
    if (!dh.defined() && !dn.defined()) return out;
    const std::vector<int64_t> n = ctx->saved_data["numbers"].toIntVector();
    const double scale = ctx->saved_data["scale"].toDouble(), eps = ctx->saved_data["eps"].toDouble();
    const int64_t rows = n[4], d = n[5];
    const at::ScalarType type = y.scalar_type();
    TORCH_CHECK(code_of(type) == n[3], "the block join's y came back from a hook with another type: ", type);
    as_saved(saved[0], y, type, rows, d);
    as_saved(y, y, type, rows, d);
    as_saved(post, y, type, 1, d);
    as_saved(gate, y, type, (rows + n[0] - 1) / n[0], d);
    as_saved(pre, y, type, 1, d);
    as_saved(saved[5], y, at::kFloat, 1, rows);
    as_saved(saved[6], y, at::kFloat, 1, rows);
    as_saved(rng, y, at::kLong, 1, 2);
    // the tensors among the inputs are the node's edges, in order
    size_t edge = 0;
    const bool nx = ctx->needs_input_grad(edge++), ny = ctx->needs_input_grad(edge++);
    const bool npost = post.defined() && ctx->needs_input_grad(edge++), ngate = gate.defined() && ctx->needs_input_grad(edge++);
    const bool npre = pre.defined() && ctx->needs_input_grad(edge++) && dn.defined();
    if (!on_kernels({dh, dn}, y) || !y.is_cuda()) {
      const int64_t need = nx + 2 * ny + 4 * npost + 8 * ngate + 16 * npre;
      variable_list got = torch_form(1, {dh, dn, saved[0], y, post, gate, pre, rng}, {n[1], n[2], need}, {scale, eps}, 5);
      std::copy(got.begin(), got.end(), out.begin());
      return out;
    }
    const c10::DeviceGuard on(y.device());
    // the strides need not be those it was saved with
    variable_list s(saved.size());
    for (size_t i = 0; i < s.size(); ++i) s[i] = rows_of(saved[i]);
    const at::Tensor dhr = rows_of(dh), dnr = rows_of(dn);
    if (nx) out[0] = at::empty_like(s[1]);
    if (ny) out[1] = at::empty_like(s[1]);
    if (npost) out[2] = at::empty_like(s[2]);
    if (ngate) out[3] = at::empty_like(s[3]);
    if (npre) out[4] = at::empty_like(s[4]);
    at::Tensor scratch;
    if (npost || ngate || npre) {
      TORCH_CHECK(join_scratch, "lbk_join_scratch: entry point not bound");
      scratch = at::empty({join_scratch(rows, d, n[0])}, at::TensorOptions().dtype(at::kFloat).device(y.device()));
    }
    TORCH_CHECK(BLOCK_FN(join_bwd), "lbk_join_bwd: entry point not bound");
    launched("lbk_join_bwd",
             BLOCK_FN(join_bwd)(ptr(dhr), ptr(dnr), ptr(s[0]), s[1].data_ptr(), ptr(s[2]), ptr(s[3]), n[0], ptr(s[4]),
                                static_cast<const float*>(ptr(s[5])), static_cast<const float*>(ptr(s[6])),
                                n[2] ? static_cast<const int64_t*>(ptr(s[7])) : nullptr, static_cast<uint32_t>(n[1]),
                                static_cast<int>(n[2]), static_cast<float>(scale), ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(out[3]),
                                ptr(out[4]), static_cast<float*>(ptr(scratch)), rows, d, static_cast<int>(n[3]),
                                reinterpret_cast<void*>(stream_of(y))));
    return out;
  }
};

// ---- gated feed-forward block: y = (a(x Wg^T) * (x Wu^T)) Wd^T ------------------------------------------------------
struct Ffn {   // one call's sizes
  int64_t t, d, n, m, act, dtype, stream;
  int dt() const { return static_cast<int>(dtype); }
  void* st() const { return reinterpret_cast<void*>(stream); }
};
struct Rows {
  at::Tensor t;
  int64_t ld;
};
// contiguous rows as the tiled products take them: the tensor itself where its rows are aligned, else a copy that is
Rows operand(const at::Tensor& t, const Ffn& f) {
  const int64_t cols = t.size(-1), ld = (cols + 7) / 8 * 8;
  if (cols == ld && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) return {t, cols};
  const int64_t rows = t.numel() / cols;
  at::Tensor out = at::empty({rows, ld}, t.options());
  launched("lbk_pad_rows", BLOCK_FN(pad_rows)(t.data_ptr(), rows, cols, ld, out.data_ptr(), f.dt(), f.st()));
  return {out, ld};
}
at::Tensor scratch_of(int64_t columns, int64_t rows, int64_t summed, const at::Tensor& like) {
  const int64_t n = linear_scratch(columns, rows, summed);
  return n ? at::empty({n}, at::TensorOptions().dtype(at::kFloat).device(like.device())) : at::Tensor();
}

// y, the activations (rows of n rounded up to 8), the projections' saved values, and the aligned copies of x and the weights
// that were made (undefined where there was no need); `keep`: a backward follows that needs the saved values
variable_list ffn_run(const at::Tensor& x, const at::Tensor& wgu, const at::Tensor& wd, const Ffn& f, bool keep) {
  TORCH_CHECK(BLOCK_FN(ffn_gate_up) && BLOCK_FN(linear_fwd) && BLOCK_FN(pad_rows) && linear_scratch && ffn_saved_bytes,
              "lbk_ffn_*: entry points not bound");
  const int64_t n8 = (f.n + 7) / 8 * 8;
  at::Tensor act = at::empty({f.t, n8}, x.options()), saved;
  if (keep) saved = at::empty({ffn_saved_bytes(f.t, f.n)}, x.options().dtype(at::kByte));
  auto shape = x.sizes().vec();
  shape.back() = f.m;
  at::Tensor y = at::empty(shape, x.options());
  const bool few = f.t <= LBK_FEW_TOKENS;   // kernels that take any alignment
  const Rows xs = few && !keep ? Rows{x, f.d} : operand(x, f), gu = few && !keep ? Rows{wgu, f.d} : operand(wgu, f);
  launched("lbk_ffn_gate_up", BLOCK_FN(ffn_gate_up)(xs.t.data_ptr(), xs.ld, gu.t.data_ptr(), gu.ld, act.data_ptr(), n8, ptr(saved),
                                                    f.t, f.d, f.n, static_cast<int>(f.act), f.dt(), f.st()));
  const Rows down = few ? Rows{wd, f.n} : operand(wd, f);
  const at::Tensor scratch = few ? at::Tensor() : scratch_of(f.m, f.t, f.n, x);
  launched("lbk_linear_fwd", BLOCK_FN(linear_fwd)(act.data_ptr(), n8, down.t.data_ptr(), down.ld, y.data_ptr(), f.m,
                                                  static_cast<float*>(ptr(scratch)), f.t, f.n, f.m, f.dt(), f.st()));
  auto copy = [](const Rows& r, const at::Tensor& t) { return r.t.is_same(t) ? at::Tensor() : r.t; };
  return {y, act, saved, copy(xs, x), copy(gu, wgu), copy(down, wd)};
}

struct FfnNode : torch::autograd::Function<FfnNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wgu, const at::Tensor& wd, int64_t act,
                            int64_t dtype, int64_t stream) {
    const Ffn f{x.numel() / x.size(-1), x.size(-1), wd.size(1), wd.size(0), act, dtype, stream};
    const bool keep = x.requires_grad() || wgu.requires_grad();
    variable_list t = ffn_run(x, wgu, wd, f, keep);
    ctx->save_for_backward({x, wgu, wd, wd.requires_grad() ? t[1] : at::Tensor(), t[2], t[3], t[4], t[5]});
    ctx->saved_data["numbers"] = std::vector<int64_t>{f.t, f.d, f.n, f.m, act, dtype};
    ctx->set_materialize_grads(false);
    return t[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> v = ctx->saved_data["numbers"].toIntVector();
    Ffn f{v[0], v[1], v[2], v[3], v[4], v[5], 0};
    const at::ScalarType type = s[0].scalar_type();
    TORCH_CHECK(code_of(type) == f.dtype, "the feed-forward block's x came back from a hook with another type: ", type);
    const int64_t d8 = (f.d + 7) / 8 * 8, n8 = (f.n + 7) / 8 * 8;
    as_saved(s[0], s[0], type, f.t, f.d);
    as_saved(s[1], s[0], type, 2 * f.n, f.d);
    as_saved(s[2], s[0], type, f.m, f.n);
    as_saved(s[3], s[0], type, f.t, n8);
    as_saved(s[4], s[0], at::kByte, 1, ffn_saved_bytes(f.t, f.n));
    as_saved(s[5], s[0], type, f.t, d8);
    as_saved(s[6], s[0], type, 2 * f.n, d8);
    as_saved(s[7], s[0], type, f.m, n8);
    const bool nx = ctx->needs_input_grad(0), ngu = ctx->needs_input_grad(1), nd = ctx->needs_input_grad(2);
    if (!on_kernels(grads, s[0], false) || !s[0].is_cuda()) {
      const variable_list got = torch_form(2, {grads[0], s[0], s[1], s[2]}, {f.act, nx + 2 * ngu + 4 * nd}, {}, 3);
      std::copy(got.begin(), got.end(), out.begin());
      return out;
    }
    const c10::DeviceGuard on(s[0].device());
    f.stream = stream_of(s[0]);
    TORCH_CHECK(grads[0].dim() > 0 && grads[0].size(-1) == f.m && grads[0].numel() == f.t * f.m,
                "the feed-forward block's gradient has the wrong shape: ", grads[0].sizes());
    for (at::Tensor& t : s) t = rows_of(t);   // the strides need not be those it was saved with
    const Rows dy = operand(rows_of(grads[0]), f);
    auto kept = [&](int copy, int of) { return s[copy].defined() ? operand(s[copy], f) : operand(s[of], f); };
    if (nx || ngu) {
      at::Tensor saved = s[4];
      if (reinterpret_cast<uintptr_t>(saved.data_ptr()) % 16) saved = saved.clone();
      const int64_t ld = (2 * f.n + 7) / 8 * 8;
      const at::Tensor dgu = at::empty({f.t, ld}, s[0].options());
      const Rows down = kept(7, 2);
      launched("lbk_ffn_dgate_up", BLOCK_FN(ffn_dgate_up)(dy.t.data_ptr(), dy.ld, down.t.data_ptr(), down.ld, saved.data_ptr(),
                                                          dgu.data_ptr(), ld, f.t, f.n, f.m, f.dt(), f.st()));
      if (nx) {
        out[0] = at::empty_like(s[0]);
        const Rows gu = kept(6, 1);
        const at::Tensor scratch = scratch_of(f.d, f.t, 2 * f.n, dgu);
        launched("lbk_linear_dx", BLOCK_FN(linear_dx)(dgu.data_ptr(), ld, gu.t.data_ptr(), gu.ld, out[0].data_ptr(), f.d,
                                                      static_cast<float*>(ptr(scratch)), f.t, 2 * f.n, f.d, f.dt(), f.st()));
      }
      if (ngu) {
        out[1] = at::empty_like(s[1]);
        const Rows xs = kept(5, 0);
        const at::Tensor scratch = scratch_of(f.d, 2 * f.n, f.t, dgu);
        launched("lbk_linear_dw", BLOCK_FN(linear_dw)(dgu.data_ptr(), ld, xs.t.data_ptr(), xs.ld, static_cast<float*>(ptr(scratch)),
                                                      out[1].data_ptr(), f.t, 2 * f.n, f.d, f.dt(), f.st()));
      }
    }
    if (nd) {
      out[2] = at::empty_like(s[2]);
      const Rows act = operand(s[3], f);
      const at::Tensor scratch = scratch_of(f.n, f.m, f.t, act.t);
      launched("lbk_linear_dw", BLOCK_FN(linear_dw)(dy.t.data_ptr(), dy.ld, act.t.data_ptr(), act.ld,
                                                    static_cast<float*>(ptr(scratch)), out[2].data_ptr(), f.t, f.m, f.n, f.dt(), f.st()));
    }
    return out;
  }
};

// gated_ffn(x, w_gate_up, w_down, activation, dtype, stream, record): contiguous tensors
PyObject* host_gated_ffn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "gated_ffn(x, w_gate_up, w_down, activation, dtype, stream, record)");
  const at::Tensor &x = tensor_of(args[0]), &wgu = tensor_of(args[1]), &wd = tensor_of(args[2]);
  const int64_t act = int_of(args[3]), dtype = int_of(args[4]), stream = int_of(args[5]);
  const bool record = args[6] == Py_True;
  at::Tensor y;
  {
    NoGil free;
    if (record) y = FfnNode::apply(x, wgu, wd, act, dtype, stream);
    else y = ffn_run(x, wgu, wd, {x.numel() / x.size(-1), x.size(-1), wd.size(1), wd.size(0), act, dtype, stream}, false)[0];
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// dropout(x, rng, site, drop, dtype, stream, record): contiguous x
PyObject* host_dropout(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "dropout(x, rng, site, drop, dtype, stream, record)");
  const at::Tensor &x = tensor_of(args[0]), &rng = tensor_of(args[1]);
  const int64_t site = int_of(args[2]), drop = int_of(args[3]), dtype = int_of(args[4]), stream = int_of(args[5]);
  const bool record = args[6] == Py_True;
  at::Tensor out;
  {
    NoGil free;
    out = record ? DropoutNode::apply(x, rng, site, drop, dtype, stream) : dropout_run(x, rng, site, drop, dtype, stream);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// join(x, y, post, gate, gate_rows, pre, rng, site, drop, scale, eps, dtype, stream, record): (h, n or None), contiguous tensors
PyObject* host_join(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 14, "join(x, y, post, gate, gate_rows, pre, rng, site, drop, scale, eps, dtype, stream, record)");
  const at::Tensor &x = tensor_of(args[0]), &y = tensor_of(args[1]);
  const OptTensor post = opt_tensor(args[2]), gate = opt_tensor(args[3]), pre = opt_tensor(args[5]);
  const int64_t gate_rows = int_of(args[4]), site = int_of(args[7]), drop = int_of(args[8]), dtype = int_of(args[11]),
                stream = int_of(args[12]);
  const OptTensor rng = drop ? opt_tensor(args[6]) : std::nullopt;
  const double scale = float_of(args[9]), eps = float_of(args[10]);
  const bool record = args[13] == Py_True;
  variable_list t;
  {
    NoGil free;
    t = record ? JoinNode::apply(x, y, post, gate, pre, rng, gate_rows, site, drop, scale, eps, dtype, stream)
               : join_run(x, y, post, gate, gate_rows, pre, rng, site, drop, scale, eps, dtype, stream, false);
    t.resize(2);
  }
  return tuple_of(t);
  END_HANDLE_TH_ERRORS
}

// torch_forms(dropout, join, ffn): the Python functions that the nodes call where a backward has to be torch operations
PyObject* host_torch_forms(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3 || !PyCallable_Check(args[0]) || !PyCallable_Check(args[1]) || !PyCallable_Check(args[2])) {
    PyErr_SetString(PyExc_TypeError, "torch_forms(dropout, join, ffn)");
    return nullptr;
  }
  for (int i = 0; i < 3; ++i) {
    Py_INCREF(args[i]);
    Py_XDECREF(torch_forms[i]);
    torch_forms[i] = args[i];
  }
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef methods[] = {
#define X(name) {#name, FAST((&Entry<decltype(&ldr_##name), ID_##name>::call)), METH_FASTCALL, nullptr},
    LDR_ENTRIES(X)
#undef X
    {"dropout", FAST(&host_dropout), METH_FASTCALL, nullptr},
    {"join", FAST(&host_join), METH_FASTCALL, nullptr},
    {"gated_ffn", FAST(&host_gated_ffn), METH_FASTCALL, nullptr},
    {"torch_forms", FAST(&host_torch_forms), METH_FASTCALL, nullptr},
    {"bind", FAST(&host_bind), METH_FASTCALL, nullptr},
    {"alias", FAST(&host_alias), METH_FASTCALL, nullptr},
    {"read_buffers", FAST(&host_read_buffers), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "launch path of the Loopback read", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
