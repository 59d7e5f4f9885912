// host.cpp -- the module's launch path as a CPython extension: every ldr_* entry point as a builtin that takes tensors, None,
// numbers and address tables as they are, the allocations around a read, and the block operators (lbk_*) and the model's (lmo_*)
// with the allocations and autograd nodes around them. A launch through ctypes costs 4-5 us of argument conversion (up to 30 arguments, each
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
#include "loopback_model.h"
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

#define LMO_ENTRIES(X) X(layer_norm_fwd) X(layer_norm_bwd) X(distill_fwd) X(distill_bwd) X(diff_attn_fwd) X(diff_attn_bwd)

enum Id {
#define X(name) ID_##name,
  LDR_ENTRIES(X)
#undef X
#define X(name) ID_block_##name,
  LBK_ENTRIES(X)
#undef X
#define X(name) ID_model_##name,
  LMO_ENTRIES(X)
#undef X
};
#define BLOCK_FN(name) (Entry<decltype(&lbk_##name), ID_block_##name>::fn)
#define MODEL_FN(name) (Entry<decltype(&lmo_##name), ID_model_##name>::fn)
int64_t (*join_scratch)(int64_t, int64_t, int64_t) = nullptr;
int64_t (*linear_scratch)(int64_t, int64_t, int64_t) = nullptr;
int64_t (*ffn_saved_bytes)(int64_t, int64_t) = nullptr;
int64_t (*layer_norm_scratch)(int64_t, int64_t) = nullptr;
int64_t (*diff_attn_scratch)(const lmo_diff_shape*, int) = nullptr;
int64_t (*diff_attn_bwd_scratch)(const lmo_diff_shape*, int) = nullptr;

struct Binding { const char* name; void (*bind)(void*); };
const Binding bindings[] = {
#define X(name) {"ldr_" #name, &Entry<decltype(&ldr_##name), ID_##name>::bind},
    LDR_ENTRIES(X)
#undef X
#define X(name) {"lbk_" #name, &Entry<decltype(&lbk_##name), ID_block_##name>::bind},
    LBK_ENTRIES(X)
#undef X
#define X(name) {"lmo_" #name, &Entry<decltype(&lmo_##name), ID_model_##name>::bind},
    LMO_ENTRIES(X)
#undef X
    {"lmo_layer_norm_scratch", [](void* p) { layer_norm_scratch = reinterpret_cast<decltype(layer_norm_scratch)>(p); }},
    {"lmo_diff_attn_scratch", [](void* p) { diff_attn_scratch = reinterpret_cast<decltype(diff_attn_scratch)>(p); }},
    {"lmo_diff_attn_bwd_scratch", [](void* p) { diff_attn_bwd_scratch = reinterpret_cast<decltype(diff_attn_bwd_scratch)>(p); }},
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

// the backwards' torch forms, Python functions: of block_ops dropout's, the join's and the feed-forward block's, of model_ops
// layer norm's, the distillation loss's and differential attention's
constexpr int FORMS = 6, BLOCK_FORMS = 3;
PyObject* torch_forms[FORMS] = {};

// torch_forms[which](*tensors, *numbers) with None for undefined tensors: its tuple of `results` tensors
variable_list torch_form(int which, const variable_list& tensors, std::initializer_list<int64_t> ints,
                         std::initializer_list<double> floats, size_t results) {
  Gil gil;
  TORCH_CHECK(torch_forms[which], "the operators' torch forms are not bound");
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
              "an operator's saved tensor came back from a hook with another shape, type or device: ", t.toString(), " ", t.sizes(),
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

// ---- the model's operators: layer norm, the distillation loss, differential attention --------------------------------------------------------
// h (the rounded sum; undefined without add), y, and the rows' mean and rstd where a backward follows
variable_list layer_norm_run(const at::Tensor& x, const OptTensor& add, const OptTensor& w, const OptTensor& b, double eps,
                             int64_t dtype, int64_t stream, bool keep) {
  const int64_t d = x.size(-1), rows = x.numel() / d;
  variable_list t{add ? at::empty_like(x) : at::Tensor(), at::empty_like(x),
                  keep ? at::empty({rows, 2}, at::TensorOptions().dtype(at::kFloat).device(x.device())) : at::Tensor()};
  TORCH_CHECK(MODEL_FN(layer_norm_fwd), "lmo_layer_norm_fwd: entry point not bound");
  launched("lmo_layer_norm_fwd",
           MODEL_FN(layer_norm_fwd)(x.data_ptr(), ptr(add), ptr(w), ptr(b), ptr(t[0]), t[1].data_ptr(), static_cast<float*>(ptr(t[2])),
                                    rows, d, static_cast<float>(eps), static_cast<int>(dtype), reinterpret_cast<void*>(stream)));
  return t;
}

// (h, y) of rows x + add, or (x, y): the gradient that comes back along the first joins the norm's in one pass
struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& add, const OptTensor& w, const OptTensor& b,
                               double eps, int64_t dtype, int64_t stream) {
    variable_list t = layer_norm_run(x, add, w, b, eps, dtype, stream, true);
    if (!add) t[0] = x;
    ctx->save_for_backward({t[0], or_none(w), t[2]});
    ctx->saved_data["numbers"] = std::vector<int64_t>{x.numel() / x.size(-1), x.size(-1), dtype, add.has_value(), b.has_value()};
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    if (add && !x.requires_grad() && !add->requires_grad()) ctx->mark_non_differentiable({t[0]});
    t.resize(2);
    return t;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(7);
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &h = saved[0], &w = saved[1], &stats = saved[2], &dh = grads[0], &dy = grads[1];
    if (!dh.defined() && !dy.defined()) return out;
    const std::vector<int64_t> n = ctx->saved_data["numbers"].toIntVector();
    const double eps = ctx->saved_data["eps"].toDouble();
    const int64_t rows = n[0], d = n[1];
    const bool added = n[3];
    size_t edge = 0;   // the tensors among the inputs are the node's edges, in order
    const bool nx = ctx->needs_input_grad(edge++), nadd = added && ctx->needs_input_grad(edge++);
    const bool nw = w.defined() && ctx->needs_input_grad(edge++), nb = n[4] && ctx->needs_input_grad(edge++);
    auto give = [&](const at::Tensor& dx) {
      if (nx) out[0] = dx;
      if (nadd) out[1] = dx;
    };
    if (!dy.defined()) {   // only the residual stream goes on
      give(dh);
      return out;
    }
    const at::ScalarType type = h.scalar_type();
    TORCH_CHECK(code_of(type) == n[2], "the layer norm's rows came back from a hook with another type: ", type);
    as_saved(h, dy, type, rows, d);
    as_saved(w, h, type, 1, d);
    as_saved(stats, h, at::kFloat, rows, 2);
    if (!on_kernels({dh, dy}, h) || !h.is_cuda()) {
      const variable_list got = torch_form(3, {dh, dy, h, w}, {(nx || nadd) + 2 * nw + 4 * nb}, {eps}, 3);
      give(got[0]);
      out[2] = got[1];
      out[3] = got[2];
      return out;
    }
    const c10::DeviceGuard on(h.device());
    const at::Tensor hr = rows_of(h), wr = rows_of(w), sr = rows_of(stats), dhr = rows_of(dh), dyr = rows_of(dy);
    at::Tensor dx, scratch;
    if (nx || nadd) dx = at::empty_like(hr);
    if (nw) out[2] = at::empty({d}, hr.options());
    if (nb) out[3] = at::empty({d}, hr.options());
    if (nw || nb) {
      TORCH_CHECK(layer_norm_scratch, "lmo_layer_norm_scratch: entry point not bound");
      scratch = at::empty({layer_norm_scratch(rows, d)}, at::TensorOptions().dtype(at::kFloat).device(h.device()));
    }
    TORCH_CHECK(MODEL_FN(layer_norm_bwd), "lmo_layer_norm_bwd: entry point not bound");
    launched("lmo_layer_norm_bwd",
             MODEL_FN(layer_norm_bwd)(dyr.data_ptr(), hr.data_ptr(), ptr(wr), static_cast<const float*>(sr.data_ptr()), ptr(dhr), ptr(dx),
                                      ptr(out[2]), ptr(out[3]), static_cast<float*>(ptr(scratch)), rows, d, static_cast<int>(n[2]),
                                      reinterpret_cast<void*>(stream_of(h))));
    give(dx);
    return out;
  }
};

// layer_norm(x, add, w, b, eps, dtype, stream, record): (h or x, y), contiguous tensors
PyObject* host_layer_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8, "layer_norm(x, add, w, b, eps, dtype, stream, record)");
  const at::Tensor& x = tensor_of(args[0]);
  const OptTensor add = opt_tensor(args[1]), w = opt_tensor(args[2]), b = opt_tensor(args[3]);
  const double eps = float_of(args[4]);
  const int64_t dtype = int_of(args[5]), stream = int_of(args[6]);
  const bool record = args[7] == Py_True;
  variable_list t;
  {
    NoGil free;
    t = record ? LayerNormNode::apply(x, add, w, b, eps, dtype, stream) : layer_norm_run(x, add, w, b, eps, dtype, stream, false);
    t.resize(2);
    if (!t[0].defined()) t[0] = x;
  }
  return tuple_of(t);
  END_HANDLE_TH_ERRORS
}

struct DistillCall {   // one call's operands and sizes
  at::Tensor logits, top, ids, lse, labels;   // lse, labels: may be undefined
  double tau, hard;
  int64_t dtype, stream;
  int64_t vocab() const { return logits.size(-1); }
  int64_t rows() const { return logits.numel() / vocab(); }
  int64_t k() const { return top.size(-1); }
  int wide() const { return ids.scalar_type() == at::kLong; }
  int top_dtype() const { return static_cast<int>(code_of(top.scalar_type())); }
  void* st() const { return reinterpret_cast<void*>(stream); }
};

variable_list distill_run(const DistillCall& c) {   // loss, the rows' saved values, the gradient's factors
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(c.logits.device());
  variable_list t{at::empty({}, f32), at::empty({c.rows(), LMO_DISTILL_SAVED}, f32), at::empty({2}, f32)};
  TORCH_CHECK(MODEL_FN(distill_fwd), "lmo_distill_fwd: entry point not bound");
  launched("lmo_distill_fwd",
           MODEL_FN(distill_fwd)(c.logits.data_ptr(), c.top.data_ptr(), c.top_dtype(), c.ids.data_ptr(), c.wide(),
                                 static_cast<const float*>(ptr(c.lse)), static_cast<const int64_t*>(ptr(c.labels)),
                                 static_cast<float>(c.tau), static_cast<float>(c.hard), static_cast<float*>(t[1].data_ptr()),
                                 static_cast<float*>(t[2].data_ptr()), static_cast<float*>(t[0].data_ptr()), c.rows(), c.vocab(), c.k(),
                                 static_cast<int>(c.dtype), c.st()));
  return t;
}

struct DistillNode : torch::autograd::Function<DistillNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& top, const at::Tensor& ids,
                            const OptTensor& lse, const OptTensor& labels, double tau, double hard, int64_t dtype, int64_t stream) {
    const DistillCall c{logits, top, ids, or_none(lse), or_none(labels), tau, hard, dtype, stream};
    variable_list t = distill_run(c);
    ctx->save_for_backward({logits, top, ids, c.lse, c.labels, t[1], t[2]});
    ctx->saved_data["numbers"] = std::vector<int64_t>{c.rows(), c.vocab(), c.k(), dtype};
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["hard"] = hard;
    ctx->set_materialize_grads(false);
    return t[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    const at::Tensor& g = grads[0];
    if (!g.defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> n = ctx->saved_data["numbers"].toIntVector();
    const double tau = ctx->saved_data["tau"].toDouble(), hard = ctx->saved_data["hard"].toDouble();
    const at::Tensor& logits = s[0];
    TORCH_CHECK(code_of(logits.scalar_type()) == n[3], "the loss's logits came back from a hook with another type: ", logits.scalar_type());
    TORCH_CHECK(code_of(s[1].scalar_type()) >= 0 && (s[2].scalar_type() == at::kLong || s[2].scalar_type() == at::kInt),
                "the loss's teacher came back from a hook with another type");
    as_saved(logits, g, logits.scalar_type(), n[0], n[1]);
    as_saved(s[1], logits, s[1].scalar_type(), n[0], n[2]);
    as_saved(s[2], logits, s[2].scalar_type(), n[0], n[2]);
    if (s[3].defined()) as_saved(s[3].reshape({-1}), logits, at::kFloat, 1, n[0]);
    if (s[4].defined()) as_saved(s[4].reshape({-1}), logits, at::kLong, 1, n[0]);
    as_saved(s[5], logits, at::kFloat, n[0], LMO_DISTILL_SAVED);
    as_saved(s[6], logits, at::kFloat, 1, 2);
    if (!on_kernels(grads, s[6], false) || !logits.is_cuda() || g.numel() != 1) {
      out[0] = torch_form(4, {g, logits, s[1], s[2], s[3], s[4]}, {}, {tau, hard}, 1)[0];
      return out;
    }
    const c10::DeviceGuard on(logits.device());
    const DistillCall c{rows_of(logits), rows_of(s[1]), rows_of(s[2]), rows_of(s[3]), rows_of(s[4]), tau, hard, n[3], stream_of(logits)};
    const at::Tensor saved = rows_of(s[5]), coef = rows_of(s[6]);
    out[0] = at::empty_like(c.logits);
    TORCH_CHECK(MODEL_FN(distill_bwd), "lmo_distill_bwd: entry point not bound");
    launched("lmo_distill_bwd",
             MODEL_FN(distill_bwd)(c.logits.data_ptr(), c.top.data_ptr(), c.top_dtype(), c.ids.data_ptr(), c.wide(),
                                   static_cast<const int64_t*>(ptr(c.labels)), static_cast<float>(tau),
                                   static_cast<const float*>(saved.data_ptr()), static_cast<const float*>(coef.data_ptr()),
                                   static_cast<const float*>(g.data_ptr()), out[0].data_ptr(), c.rows(), c.vocab(), c.k(),
                                   c.lse.defined(), static_cast<int>(c.dtype), c.st()));
    return out;
  }
};

// distill(logits, top, ids, lse, labels, tau, hard, dtype, stream, record): the loss, contiguous tensors
PyObject* host_distill(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "distill(logits, top, ids, lse, labels, tau, hard, dtype, stream, record)");
  const at::Tensor &logits = tensor_of(args[0]), &top = tensor_of(args[1]), &ids = tensor_of(args[2]);
  const OptTensor lse = opt_tensor(args[3]), labels = opt_tensor(args[4]);
  const double tau = float_of(args[5]), hard = float_of(args[6]);
  const int64_t dtype = int_of(args[7]), stream = int_of(args[8]);
  const bool record = args[9] == Py_True;
  at::Tensor loss;
  {
    NoGil free;
    loss = record ? DistillNode::apply(logits, top, ids, lse, labels, tau, hard, dtype, stream)
                  : distill_run({logits, top, ids, or_none(lse), or_none(labels), tau, hard, dtype, stream})[0];
  }
  return THPVariable_Wrap(loss);
  END_HANDLE_TH_ERRORS
}

// q [b, tq, 2 h, dh], k [b, tk, 2 hk, dh], v [b, tk, hk, dv] as the kernels take them: themselves, or contiguous copies. A dimension
// of one may have any stride, which contiguous() keeps and nothing steps by: the kernels get 0 for it
at::Tensor attn_rows(const at::Tensor& t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) % 8 == 0 && (i == 0 || t.stride(i) <= (1 << 23))));
  if (ok) return t;
  at::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
lmo_strides strides_of(const at::Tensor& t) {
  const auto step = [&](int i) { return t.size(i) == 1 ? 0 : t.stride(i); };
  return {t.data_ptr(), step(0), step(1), step(2)};
}
lmo_strides lam_strides(const at::Tensor& t) {   // one value, one per head, or one per query and head
  return t.dim() == 3 ? lmo_strides{t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}
                      : lmo_strides{t.data_ptr(), 0, 0, t.dim() == 1 ? t.stride(0) : 0};
}
int lam_kind(const at::Tensor& t) { return t.dim() == 3 ? LMO_LAM_TOKEN : t.dim() == 1 ? LMO_LAM_HEAD : LMO_LAM_LAYER; }

struct DiffCall {
  at::Tensor q, k, v, lam, lengths, starts;   // the last two may be undefined
  bool causal;
  double scale;
  int64_t dtype, stream;
  lmo_diff_shape shape() const {
    return {q.size(0), q.size(1), k.size(1), q.size(2) / 2, v.size(2), q.size(3), v.size(3), causal, static_cast<float>(scale)};
  }
  int lam32() const { return lam.scalar_type() == at::kFloat; }
  const int32_t* len() const { return static_cast<const int32_t*>(ptr(lengths)); }
  const int32_t* start() const { return static_cast<const int32_t*>(ptr(starts)); }
  void* st() const { return reinterpret_cast<void*>(stream); }
};

variable_list diff_attn_run(const DiffCall& c, bool keep) {   // y, P2 v and the logarithms (undefined unless kept)
  const lmo_diff_shape s = c.shape();
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(c.q.device());
  variable_list t{at::empty({s.b, s.tq, s.h, s.dv}, c.q.options()), at::Tensor(), at::Tensor()};
  if (keep) {
    t[1] = at::empty_like(t[0]);
    t[2] = at::empty({2, s.b, s.h, s.tq}, f32);
  }
  TORCH_CHECK(MODEL_FN(diff_attn_fwd) && diff_attn_scratch, "lmo_diff_attn_fwd: entry point not bound");
  const int64_t n = diff_attn_scratch(&s, keep);
  const at::Tensor scratch = n ? at::empty({n}, f32) : at::Tensor();
  const at::Tensor q = attn_rows(c.q), k = attn_rows(c.k), v = attn_rows(c.v);
  const lmo_strides qs = strides_of(q), ks = strides_of(k), vs = strides_of(v), ls = lam_strides(c.lam);
  launched("lmo_diff_attn_fwd",
           MODEL_FN(diff_attn_fwd)(&qs, &ks, &vs, &ls, c.lam32(), c.len(), c.start(), t[0].data_ptr(), ptr(t[1]),
                                   static_cast<float*>(ptr(t[2])), static_cast<float*>(ptr(scratch)), &s, static_cast<int>(c.dtype), c.st()));
  return t;
}

struct DiffAttnNode : torch::autograd::Function<DiffAttnNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& lam,
                            const OptTensor& lengths, const OptTensor& starts, bool causal, double scale, int64_t dtype, int64_t stream) {
    const DiffCall c{q, k, v, lam, or_none(lengths), or_none(starts), causal, scale, dtype, stream};
    const variable_list t = diff_attn_run(c, true);
    ctx->save_for_backward({q, k, v, lam, c.lengths, c.starts, t[0], t[1], t[2]});
    const lmo_diff_shape s = c.shape();
    ctx->saved_data["numbers"] = std::vector<int64_t>{s.b, s.tq, s.tk, s.h, s.hk, s.dh, s.dv, dtype, causal, lam.dim(), lam.scalar_type() == at::kFloat};
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return t[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(10);
    const at::Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    const variable_list s = ctx->get_saved_variables();
    const std::vector<int64_t> n = ctx->saved_data["numbers"].toIntVector();
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t b = n[0], tq = n[1], tk = n[2], h = n[3], hk = n[4], dh = n[5], dv = n[6];
    const at::ScalarType type = s[0].scalar_type();
    TORCH_CHECK(code_of(type) == n[7], "the attention's queries came back from a hook with another type: ", type);
    auto sized = [&](const at::Tensor& t, at::ScalarType ty, at::IntArrayRef sizes) {
      if (!t.defined()) return;
      TORCH_CHECK(t.layout() == at::kStrided && t.device() == dy.device() && t.scalar_type() == ty && t.sizes() == sizes,
                  "an operator's saved tensor came back from a hook with another shape, type or device: ", t.toString(), " ", t.sizes(),
                  " on ", t.device());
    };
    sized(s[0], type, {b, tq, 2 * h, dh});
    sized(s[1], type, {b, tk, 2 * hk, dh});
    sized(s[2], type, {b, tk, hk, dv});
    const at::ScalarType lam_type = n[10] ? at::kFloat : type;
    if (n[9] == 0) sized(s[3], lam_type, {});
    else if (n[9] == 1) sized(s[3], lam_type, {h});
    else sized(s[3], lam_type, {b, tq, h});
    sized(s[4], at::kInt, {b});
    sized(s[5], at::kInt, {b});
    sized(s[6], type, {b, tq, h, dv});
    sized(s[7], type, {b, tq, h, dv});
    sized(s[8], at::kFloat, {2, b, h, tq});
    const bool nq = ctx->needs_input_grad(0), nk = ctx->needs_input_grad(1), nv = ctx->needs_input_grad(2), nl = ctx->needs_input_grad(3);
    if (!on_kernels(grads, s[6]) || !s[0].is_cuda()) {
      const variable_list got =
          torch_form(5, {dy, s[0], s[1], s[2], s[3], s[4], s[5]}, {n[8], nq + 2 * nk + 4 * nv + 8 * nl}, {scale}, 4);
      std::copy(got.begin(), got.end(), out.begin());
      return out;
    }
    const c10::DeviceGuard on(dy.device());
    auto aligned = [](const at::Tensor& t) {
      const at::Tensor r = rows_of(t);
      return reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 ? r.clone() : r;
    };
    const DiffCall c{attn_rows(s[0]), attn_rows(s[1]), attn_rows(s[2]), s[3], rows_of(s[4]), rows_of(s[5]), n[8] != 0, scale, n[7], stream_of(dy)};
    const at::Tensor y = aligned(s[6]), second = aligned(s[7]), lse = rows_of(s[8]), g = aligned(dy);
    const lmo_diff_shape sh = c.shape();
    const int kind = lam_kind(c.lam);
    TORCH_CHECK(MODEL_FN(diff_attn_bwd) && diff_attn_bwd_scratch, "lmo_diff_attn_bwd: entry point not bound");
    const at::Tensor scratch = at::empty({diff_attn_bwd_scratch(&sh, kind)}, at::TensorOptions().dtype(at::kFloat).device(dy.device()));
    const at::Tensor dq = at::empty({b, tq, 2 * h, dh}, g.options());
    at::Tensor dk, dval, dlam;
    if (nk || nv) {
      dk = at::empty({b, tk, 2 * hk, dh}, g.options());
      dval = at::empty({b, tk, hk, dv}, g.options());
    }
    if (nl) dlam = at::empty(c.lam.sizes(), c.lam.options());
    const lmo_strides qs = strides_of(c.q), ks = strides_of(c.k), vs = strides_of(c.v), ls = lam_strides(c.lam);
    launched("lmo_diff_attn_bwd",
             MODEL_FN(diff_attn_bwd)(&qs, &ks, &vs, &ls, c.lam32(), c.len(), c.start(), y.data_ptr(), second.data_ptr(),
                                     static_cast<const float*>(lse.data_ptr()), g.data_ptr(), dq.data_ptr(), ptr(dk), ptr(dval), ptr(dlam), kind,
                                     static_cast<float*>(scratch.data_ptr()), &sh, static_cast<int>(c.dtype), c.st()));
    if (nq) out[0] = dq;
    if (nk) out[1] = dk;
    if (nv) out[2] = dval;
    if (nl) out[3] = dlam;
    return out;
  }
};

// diff_attn(q, k, v, lam, lengths, starts, causal, scale, dtype, stream, record): y
PyObject* host_diff_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 11, "diff_attn(q, k, v, lam, lengths, starts, causal, scale, dtype, stream, record)");
  const at::Tensor &q = tensor_of(args[0]), &k = tensor_of(args[1]), &v = tensor_of(args[2]), &lam = tensor_of(args[3]);
  const OptTensor lengths = opt_tensor(args[4]), starts = opt_tensor(args[5]);
  const bool causal = args[6] == Py_True, record = args[10] == Py_True;
  const double scale = float_of(args[7]);
  const int64_t dtype = int_of(args[8]), stream = int_of(args[9]);
  at::Tensor y;
  {
    NoGil free;
    y = record ? DiffAttnNode::apply(q, k, v, lam, lengths, starts, causal, scale, dtype, stream)
               : diff_attn_run({q, k, v, lam, or_none(lengths), or_none(starts), causal, scale, dtype, stream}, false)[0];
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// the Python functions that the nodes call where a backward has to be torch operations, `count` of them from the first's place on
PyObject* set_forms(PyObject* const* args, Py_ssize_t n, int first, int count, const char* what) {
  bool ok = n == count;
  for (int i = 0; ok && i < count; ++i) ok = PyCallable_Check(args[i]);
  if (!ok) {
    PyErr_SetString(PyExc_TypeError, what);
    return nullptr;
  }
  for (int i = 0; i < count; ++i) {
    Py_INCREF(args[i]);
    Py_XDECREF(torch_forms[first + i]);
    torch_forms[first + i] = args[i];
  }
  Py_RETURN_NONE;
}
// torch_forms(dropout, join, ffn): the block operators'
PyObject* host_torch_forms(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return set_forms(args, n, 0, BLOCK_FORMS, "torch_forms(dropout, join, ffn)");
}
// model_forms(layer_norm, distill, diff_attn): the same of the model's operators
PyObject* host_model_forms(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return set_forms(args, n, BLOCK_FORMS, FORMS - BLOCK_FORMS, "model_forms(layer_norm, distill, diff_attn)");
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
    {"layer_norm", FAST(&host_layer_norm), METH_FASTCALL, nullptr},
    {"distill", FAST(&host_distill), METH_FASTCALL, nullptr},
    {"diff_attn", FAST(&host_diff_attn), METH_FASTCALL, nullptr},
    {"model_forms", FAST(&host_model_forms), METH_FASTCALL, nullptr},
    {"bind", FAST(&host_bind), METH_FASTCALL, nullptr},
    {"alias", FAST(&host_alias), METH_FASTCALL, nullptr},
    {"read_buffers", FAST(&host_read_buffers), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "launch path of the Loopback read", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
