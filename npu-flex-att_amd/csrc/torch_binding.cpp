// The cache and rotary entry points for torch tensors: argument checks, outputs and
// workspaces from torch's allocator, the tensors' device and its current stream, the
// C ABI call, and the rotation's autograd node.  Host code only.
//
// A decoding step makes these calls once per layer on problems of a few microseconds,
// where the same work in Python (about 12 us a call, and 120 us more for a backward
// pass that has to take the interpreter's lock on the engine's thread) is what the
// step would wait for.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <limits>
#include <string>

#include "../../include/flexatt.h"

namespace {
using at::Tensor;
using OptTensor = std::optional<Tensor>;

// ------------------------------------------------------------------- arguments --
[[noreturn]] void fail_assert(const char* what) {
  pybind11::gil_scoped_acquire gil;
  PyErr_SetString(PyExc_AssertionError, what);
  python_error e;
  e.persist();
  throw e;
}
// The reference's entry points assert matching shapes (npu_flash_attention.py:620-622).
#define FLEXATT_ASSERT(cond, what) \
  do {                             \
    if (!(cond)) fail_assert(what); \
  } while (0)

Tensor tensor_arg(PyObject* o, const char* name) {
  TORCH_CHECK(THPVariable_Check(o), name, " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}
OptTensor opt_tensor_arg(PyObject* o, const char* name) {
  if (o == Py_None) return std::nullopt;
  return tensor_arg(o, name);
}
double double_arg(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw python_error();
  return x;
}
bool bool_arg(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw python_error();
  return x != 0;
}
// A whole number, or the nearest of the two ends that 64 bits hold.
int64_t int_arg(PyObject* o) {
  PyObject* i = PyNumber_Index(o);
  if (!i) throw python_error();
  int over = 0;
  const int64_t x = PyLong_AsLongLongAndOverflow(i, &over);
  Py_DECREF(i);
  if (over) return over > 0 ? INT64_MAX : INT64_MIN;
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return x;
}
void want(Py_ssize_t n, Py_ssize_t k, const char* name) {
  TORCH_CHECK_TYPE(n == k, name, " takes ", k, " arguments, got ", n);
}

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return FLEXATT_F32;
    case at::kHalf: return FLEXATT_F16;
    case at::kBFloat16: return FLEXATT_BF16;
    default: TORCH_CHECK(false, "unsupported dtype ", t.scalar_type(), " (expected float32, float16 or bfloat16)");
  }
}

// A trace would record the outputs' allocation but not the kernel that fills them.
// (torch.compile breaks its graph at these calls and runs them as they are.)
void no_trace() {
  bool traced = torch::jit::tracer::isTracing();
  if (c10::impl::TorchDispatchModeTLS::any_modes_set())
    for (const auto key : {c10::impl::TorchDispatchModeKey::FAKE, c10::impl::TorchDispatchModeKey::PROXY,
                           c10::impl::TorchDispatchModeKey::FUNCTIONAL})
      traced = traced || c10::impl::TorchDispatchModeTLS::get_mode(key).has_value();
  TORCH_CHECK(!traced, "the rotary and cache calls cannot be traced (make_fx, export, jit.trace, fake tensors): "
                       "put the call into a torch.library.custom_op");
}

struct Named {
  const char* name;
  const Tensor* t;
};
// The kernels read and write through pointers: a derivative that an argument brings
// along would be dropped without a word.
void no_tangents(std::initializer_list<Named> all) {
  for (const Named& x : all)
    TORCH_CHECK(!x.t->_fw_grad(/*level=*/0).defined(), x.name,
                " carries a tangent: the rotary and cache operators have no forward-mode derivatives");
}
void no_derivatives(std::initializer_list<Named> all) {
  no_tangents(all);
  if (!at::GradMode::is_enabled()) return;
  for (const Named& x : all)
    TORCH_CHECK(!x.t->requires_grad(), x.name,
                " requires a gradient, which the call does not have: detach it, or call under torch.no_grad()");
}

// Four dimensions, the first one's type and device, a head dim with kernels.
void check_tensors(std::initializer_list<Named> all) {
  const Tensor& first = *all.begin()->t;
  for (const Named& x : all) {
    const Tensor& t = *x.t;
    TORCH_CHECK(t.is_cuda(), x.name, " must be on a ROCm GPU device (got ", t.device(), ")");
    TORCH_CHECK(t.scalar_type() == first.scalar_type(), x.name, " has dtype ", t.scalar_type(), ", expected ",
                first.scalar_type());
    TORCH_CHECK(t.device() == first.device(), x.name, " must be on ", first.device(), " (got ", t.device(), ")");
    TORCH_CHECK(t.dim() == 4, x.name, " must have four dimensions, got ", t.sizes());
    TORCH_CHECK(t.layout() == at::kStrided, x.name, " must be a strided tensor");
  }
  dtype_of(first);
  const int64_t d = first.size(3);
  TORCH_CHECK(d == 32 || d == 64 || d == 128 || d == 256, "unsupported head dim ", d, " (expected one of 32, 64, 128, 256)");
}

int32_t size32(int64_t x, const char* what) {
  TORCH_CHECK(x >= 0 && x <= INT32_MAX, what, " does not fit 32 bits");
  return (int32_t)x;
}

// An int32 [B] tensor of the call's device, contiguous.
Tensor per_sequence(const Tensor& t, const char* name, int64_t B, c10::Device dev) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B, name, " must be an int32 tensor [B] = [", B,
              "]");
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev, " (got ", t.device(), ")");
  return t.contiguous();
}

// True if the kernels can read t in place: innermost stride 1, rows on 16-byte boundaries.
bool kernel_ready(const Tensor& t) {
  const int64_t es = t.element_size();
  if ((t.size(3) > 1 && t.stride(3) != 1) || (uintptr_t)t.data_ptr() % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (t.stride(i) * es % 16) return false;
  return true;
}
Tensor prepare(const Tensor& t) {
  return kernel_ready(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}
void in_place(const Tensor& t, const char* name) {
  TORCH_CHECK(kernel_ready(t), name, " is written in place: its innermost stride must be 1 and its rows must start on "
              "16-byte boundaries");
}
// An output in its input's layout, contiguous where that one is not the kernels'.
Tensor out_like(const Tensor& t) {
  if (t.is_contiguous()) return at::empty(t.sizes(), t.options().requires_grad(false));
  Tensor o = at::empty_like(t);
  return kernel_ready(o) ? o : at::empty(t.sizes(), t.options().requires_grad(false));
}
flexatt_tensor view(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2), 1}; }

void* stream_of(c10::Device dev) { return (void*)c10::hip::getCurrentHIPStream(dev.index()).stream(); }
void check_status(int st, const char* what) {
  TORCH_CHECK(st == 0, what, " failed: ", flexatt_status_string(st), " (status ", st, ")");
}
// Written through its pointer: a graph that saved the tensor has to know.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Tensor workspace(size_t n, c10::Device dev) {
  if (n == 0 || n == SIZE_MAX) return Tensor();  // none needed, or a call that will be rejected
  return at::empty({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(dev));
}
void* data_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// -------------------------------------------------------------------- rotation --
Tensor check_frequencies(const Tensor& f, int64_t D, c10::Device dev) {
  TORCH_CHECK(f.scalar_type() == at::kDouble && f.dim() == 1,
              "inv_freq must be a float64 tensor with one entry per pair (see rotary_frequencies)");
  TORCH_CHECK(f.device() == dev, "inv_freq must be on ", dev, " (got ", f.device(), ")");
  TORCH_CHECK(2 * f.size(0) <= D, "inv_freq has ", f.size(0), " pairs, a head of ", D, " elements has ", D / 2);
  return f.contiguous();
}

flexatt_rotary rotary_struct(const Tensor& q, int64_t hkv, const Tensor& freq, const OptTensor& pos, bool interleaved,
                             double magnitude, bool inverse) {
  flexatt_rotary r = {};
  r.dtype = dtype_of(q);
  r.batch = size32(q.size(0), "batch");
  r.heads_q = size32(q.size(1), "Hq");
  r.heads_kv = size32(hkv, "Hkv");
  r.seqlen = size32(q.size(2), "S");
  r.head_dim = (int32_t)q.size(3);
  r.interleaved = interleaved;
  r.inverse = inverse;
  r.magnitude = (float)magnitude;
  TORCH_CHECK(std::isfinite(r.magnitude), "magnitude must be finite");
  if (freq.defined() && freq.numel() > 0) {
    r.rotary_dim = 2 * (int32_t)freq.numel();
    r.inv_freq = freq.const_data_ptr<double>();
  }
  if (pos) {
    const Tensor& p = *pos;
    TORCH_CHECK(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong,
                "positions must be an int32 or int64 tensor");
    TORCH_CHECK(p.device() == q.device(), "positions must be on ", q.device(), " (got ", p.device(), ")");
    const int64_t B = q.size(0), S = q.size(2);
    const bool one = p.dim() == 1 && p.size(0) == S;
    TORCH_CHECK(one || (p.dim() == 2 && p.size(1) == S && (p.size(0) == 1 || p.size(0) == B)),
                "positions must be [S] or [B, S] = [", B, ", ", S, "], got ", p.sizes());
    r.positions = p.data_ptr();
    r.position_bytes = (int32_t)p.element_size();
    r.position_stride_b = one || p.size(0) == 1 ? 0 : p.stride(0);
    r.position_stride_s = p.stride(one ? 0 : 1);
  }
  return r;
}

// (query', key'), key' undefined without a key.
std::pair<Tensor, Tensor> rotate(const Tensor& query, const Tensor& key, const Tensor& freq, const OptTensor& pos,
                                 bool interleaved, double magnitude, bool inverse) {
  no_trace();  // (a backward pass gets here too)
  const c10::Device dev = query.device();
  const c10::OptionalDeviceGuard guard(dev);
  const bool keyed = key.defined();
  const flexatt_rotary r = rotary_struct(query, keyed ? key.size(1) : 0, freq, pos, interleaved, magnitude, inverse);
  Tensor qo = out_like(query), ko = keyed ? out_like(key) : Tensor();
  if (query.numel() == 0 && (!keyed || key.numel() == 0)) return {qo, ko};
  const Tensor q = prepare(query), k = keyed ? prepare(key) : Tensor();
  const flexatt_tensor tq = view(q), tqo = view(qo);
  flexatt_tensor tk = {}, tko = {};
  if (keyed) tk = view(k), tko = view(ko);
  check_status(flexatt_rotary_apply(&r, &tq, keyed ? &tk : nullptr, &tqo, keyed ? &tko : nullptr, stream_of(dev)),
               "flexatt_rotary_apply");
  return {qo, ko};
}

// The rotation is linear, and its transpose turns the other way: the backward pass
// is this function again (so gradients of gradients work too).
struct Rotary : torch::autograd::Function<Rotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& query,
                                                const OptTensor& key, const Tensor& freq, const OptTensor& pos,
                                                bool interleaved, double magnitude, bool inverse) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({freq, pos ? *pos : Tensor()});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["inverse"] = inverse;
    auto [q, k] = rotate(query, key ? *key : Tensor(), freq, pos, interleaved, magnitude, inverse);
    if (k.defined()) return {q, k};
    return {q};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = ctx->saved_data["inverse"].toBool();
    const double magnitude = ctx->saved_data["magnitude"].toDouble();
    Tensor dq = grads[0], dk = grads.size() > 1 ? grads[1] : Tensor();
    const OptTensor pos = saved[1].defined() ? OptTensor(saved[1]) : std::nullopt;
    const auto turned = [&](const Tensor& a, const OptTensor& b) {
      return Rotary::apply(a, b, saved[0], pos, interleaved, magnitude, !inverse);
    };
    if (dq.defined() && dk.defined()) {
      const auto out = turned(dq, dk);
      dq = out[0];
      dk = out[1];
    } else if (dq.defined()) {
      dq = turned(dq, std::nullopt)[0];
    } else if (dk.defined()) {
      dk = turned(dk, std::nullopt)[0];
    }
    return {dq, dk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ---------------------------------------------------- norm of each head, rotation --
// A weight [D] of the call's dtype or fp32, on its device.
Tensor check_weight(const Tensor& w, const char* name, const Tensor& x) {
  TORCH_CHECK(w.device() == x.device(), name, " must be on ", x.device(), " (got ", w.device(), ")");
  TORCH_CHECK(w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type(), name, " has dtype ", w.scalar_type(),
              ", expected ", x.scalar_type(), " or float32");
  TORCH_CHECK(w.layout() == at::kStrided && w.dim() == 1 && w.size(0) == x.size(3), name, " must be [D] = [", x.size(3), "]");
  return w.contiguous();
}
void check_eps(double eps) {
  TORCH_CHECK((float)eps >= std::numeric_limits<float>::min() && std::isfinite((float)eps),
              "eps must be a positive number that 32 bits hold");
}
flexatt_norm norm_struct(const Tensor& wq, const Tensor& wk, double eps) {
  flexatt_norm n = {};
  const Tensor& any = wq.defined() ? wq : wk;
  n.weight_dtype = dtype_of(any);
  TORCH_CHECK(!wq.defined() || !wk.defined() || wq.scalar_type() == wk.scalar_type(),
              "query_weight and key_weight must have one dtype");
  n.eps = (float)eps;
  n.q_weight = data_or_null(wq);
  n.k_weight = data_or_null(wk);
  return n;
}

// (query', key'), key' undefined without a key.
std::pair<Tensor, Tensor> norm_rotate(const Tensor& query, const Tensor& key, const Tensor& wq, const Tensor& wk,
                                      const Tensor& freq, const OptTensor& pos, bool interleaved, double magnitude,
                                      double eps) {
  const c10::Device dev = query.device();
  const c10::OptionalDeviceGuard guard(dev);
  const bool keyed = key.defined();
  const flexatt_rotary r = rotary_struct(query, keyed ? key.size(1) : 0, freq, pos, interleaved, magnitude, false);
  const flexatt_norm n = norm_struct(wq, wk, eps);
  Tensor qo = out_like(query), ko = keyed ? out_like(key) : Tensor();
  if (query.numel() == 0 && (!keyed || key.numel() == 0)) return {qo, ko};
  const Tensor q = prepare(query), k = keyed ? prepare(key) : Tensor();
  const flexatt_tensor tq = view(q), tqo = view(qo);
  flexatt_tensor tk = {}, tko = {};
  if (keyed) tk = view(k), tko = view(ko);
  check_status(flexatt_norm_rotary_apply(&r, &n, &tq, keyed ? &tk : nullptr, &tqo, keyed ? &tko : nullptr, stream_of(dev)),
               "flexatt_norm_rotary_apply");
  return {qo, ko};
}

// The gradients of x and its weight, and of y and its own if there is one.
struct NormGrads {
  Tensor dx, dw, dy, dv;
};
NormGrads norm_rotate_grad(const Tensor& x, const Tensor& w, const Tensor& gx, const Tensor& y, const Tensor& v,
                           const Tensor& gy, const Tensor& freq, const OptTensor& pos, bool interleaved, double magnitude,
                           double eps) {
  no_trace();
  const c10::Device dev = x.device();
  const c10::OptionalDeviceGuard guard(dev);
  const bool two = y.defined();
  const flexatt_rotary r = rotary_struct(x, two ? y.size(1) : 0, freq, pos, interleaved, magnitude, false);
  const flexatt_norm n = norm_struct(w, v, eps);
  NormGrads g;
  g.dx = out_like(x);
  g.dw = at::empty(w.sizes(), w.options().requires_grad(false));
  if (two) g.dy = out_like(y), g.dv = at::empty(v.sizes(), v.options().requires_grad(false));
  if (x.numel() == 0) {
    g.dw.zero_();
    if (two) g.dv.zero_();
    return g;
  }
  const Tensor px = prepare(x), pg = prepare(gx), py = two ? prepare(y) : Tensor(), ph = two ? prepare(gy) : Tensor();
  const flexatt_tensor tx = view(px), tg = view(pg), td = view(g.dx);
  flexatt_tensor ty = {}, th = {}, te = {};
  if (two) ty = view(py), th = view(ph), te = view(g.dy);
  const size_t bytes = flexatt_norm_rotary_grad_workspace(&r);
  const Tensor ws = workspace(bytes, dev);
  check_status(flexatt_norm_rotary_grad(&r, &n, &tx, two ? &ty : nullptr, &tg, two ? &th : nullptr, &td,
                                        two ? &te : nullptr, g.dw.data_ptr(), data_or_null(g.dv), data_or_null(ws),
                                        ws.defined() ? bytes : 0, stream_of(dev)),
               "flexatt_norm_rotary_grad");
  return g;
}

struct NormRotary : torch::autograd::Function<NormRotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& query,
                                                const OptTensor& key, const Tensor& wq, const OptTensor& wk,
                                                const Tensor& freq, const OptTensor& pos, bool interleaved,
                                                double magnitude, double eps) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({query, key ? *key : Tensor(), wq, wk ? *wk : Tensor(), freq, pos ? *pos : Tensor()});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["eps"] = eps;
    auto [q, k] = norm_rotate(query, key ? *key : Tensor(), wq, wk ? *wk : Tensor(), freq, pos, interleaved, magnitude, eps);
    if (k.defined()) return {q, k};
    return {q};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool();
    const double magnitude = ctx->saved_data["magnitude"].toDouble(), eps = ctx->saved_data["eps"].toDouble();
    const Tensor gq = grads[0], gk = grads.size() > 1 ? grads[1] : Tensor();
    const OptTensor pos = saved[5].defined() ? OptTensor(saved[5]) : std::nullopt;
    // (a graph of this pass would end here without a word)
    TORCH_CHECK(!at::GradMode::is_enabled(), "norm_rotary_embedding has no gradients of its gradients (create_graph)");
    torch::autograd::variable_list out(9);
    const auto run = [&](const Tensor& x, const Tensor& w, const Tensor& g, const Tensor& y, const Tensor& v,
                         const Tensor& h) {
      return norm_rotate_grad(x, w, g, y, v, h, saved[4], pos, interleaved, magnitude, eps);
    };
    // (not for a frozen query or key, or one that this pass does not ask for; the tensors are inputs 0 to 3, or 0 and 1)
    const bool keyed = saved[1].defined();
    const bool q = gq.defined() && (ctx->needs_input_grad(0) || ctx->needs_input_grad(keyed ? 2 : 1));
    const bool k = gk.defined() && (ctx->needs_input_grad(1) || ctx->needs_input_grad(3));
    if (q && k) {
      const NormGrads r = run(saved[0], saved[2], gq, saved[1], saved[3], gk);
      out[0] = r.dx, out[2] = r.dw, out[1] = r.dy, out[3] = r.dv;
    } else if (q) {
      const NormGrads r = run(saved[0], saved[2], gq, Tensor(), Tensor(), Tensor());
      out[0] = r.dx, out[2] = r.dw;
    } else if (k) {
      const NormGrads r = run(saved[1], saved[3], gk, Tensor(), Tensor(), Tensor());
      out[1] = r.dx, out[3] = r.dw;
    }
    return out;
  }
};

PyObject* pair_of(const Tensor& a, const Tensor& b) {
  PyObject* t = PyTuple_New(2);
  if (!t) throw python_error();
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(a));
  if (b.defined()) {
    PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(b));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(t, 1, Py_None);
  }
  return t;
}

PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 6, "rotary");
  no_trace();
  const Tensor query = tensor_arg(a[0], "query");
  const OptTensor key = opt_tensor_arg(a[1], "key");
  Tensor freq = tensor_arg(a[2], "inv_freq");
  const OptTensor pos = opt_tensor_arg(a[3], "positions");
  const bool interleaved = bool_arg(a[4]);
  const double magnitude = double_arg(a[5]);
  no_derivatives({{"inv_freq", &freq}});
  if (key) {
    no_tangents({{"query", &query}, {"key", &*key}});
    check_tensors({{"query", &query}, {"key", &*key}});
    FLEXATT_ASSERT(key->size(0) == query.size(0) && key->size(2) == query.size(2) && key->size(3) == query.size(3),
                   "query and key must have the same batch, length and head dim");
    FLEXATT_ASSERT(key->size(1) > 0, "key must have a head");
  } else {
    no_tangents({{"query", &query}});
    check_tensors({{"query", &query}});
  }
  freq = check_frequencies(freq, query.size(3), query.device());
  Tensor qo, ko;
  {
    pybind11::gil_scoped_release no_gil;
    if (at::GradMode::is_enabled() && (query.requires_grad() || (key && key->requires_grad()))) {
      const auto out = Rotary::apply(query, key, freq, pos, interleaved, magnitude, false);
      qo = out[0];
      if (key) ko = out[1];
    } else {
      std::tie(qo, ko) = rotate(query, key ? *key : Tensor(), freq, pos, interleaved, magnitude, false);
    }
  }
  return pair_of(qo, ko);
  END_HANDLE_TH_ERRORS
}

PyObject* py_norm_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 9, "norm_rotary");
  no_trace();
  const Tensor query = tensor_arg(a[0], "query");
  const OptTensor key = opt_tensor_arg(a[1], "key");
  Tensor wq = tensor_arg(a[2], "query_weight");
  OptTensor wk = opt_tensor_arg(a[3], "key_weight");
  Tensor freq = tensor_arg(a[4], "inv_freq");
  const OptTensor pos = opt_tensor_arg(a[5], "positions");
  const bool interleaved = bool_arg(a[6]);
  const double magnitude = double_arg(a[7]), eps = double_arg(a[8]);
  no_derivatives({{"inv_freq", &freq}});
  no_tangents({{"query", &query}, {"query_weight", &wq}});
  TORCH_CHECK(key.has_value() == wk.has_value(), "key and key_weight go together");
  if (key) {
    no_tangents({{"key", &*key}, {"key_weight", &*wk}});
    check_tensors({{"query", &query}, {"key", &*key}});
    FLEXATT_ASSERT(key->size(0) == query.size(0) && key->size(2) == query.size(2) && key->size(3) == query.size(3),
                   "query and key must have the same batch, length and head dim");
    FLEXATT_ASSERT(key->size(1) > 0, "key must have a head");
    wk = check_weight(*wk, "key_weight", query);
  } else {
    check_tensors({{"query", &query}});
  }
  FLEXATT_ASSERT(query.size(1) > 0, "query must have a head");
  wq = check_weight(wq, "query_weight", query);
  check_eps(eps);
  freq = check_frequencies(freq, query.size(3), query.device());
  Tensor qo, ko;
  {
    pybind11::gil_scoped_release no_gil;
    if (at::GradMode::is_enabled() && (query.requires_grad() || wq.requires_grad() || (key && key->requires_grad()) ||
                                       (wk && wk->requires_grad()))) {
      const auto out = NormRotary::apply(query, key, wq, wk, freq, pos, interleaved, magnitude, eps);
      qo = out[0];
      if (key) ko = out[1];
    } else {
      std::tie(qo, ko) = norm_rotate(query, key ? *key : Tensor(), wq, wk ? *wk : Tensor(), freq, pos, interleaved,
                                     magnitude, eps);
    }
  }
  return pair_of(qo, ko);
  END_HANDLE_TH_ERRORS
}

// ----------------------------------------------------------------------- cache --
void check_cache(const Tensor& query, const Tensor& kc, const Tensor& vc) {
  FLEXATT_ASSERT(kc.sizes() == vc.sizes(), "key and value cache shapes must match");
  FLEXATT_ASSERT(kc.size(0) == query.size(0), "query and cache batch sizes must match");
  FLEXATT_ASSERT(kc.size(3) == query.size(3), "query and cache head dims must match");
  FLEXATT_ASSERT(kc.size(1) > 0 && query.size(1) % kc.size(1) == 0, "Hq must be divisible by Hkv");
}

// New tokens for a cache: what the appends check, and hand over.
struct Append {
  flexatt_rotary r;
  flexatt_norm n;
  bool normed = false, queried;
  Tensor q, k, v, qo, lengths, freq, wq, wk;
  flexatt_tensor tq, tk, tv, to, tkc, tvc;
  int32_t rows;
};
// False: there is nothing to write.
bool check_append(Append& x, const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& kc,
                  const Tensor& vc, const Tensor& lengths, const OptTensor& freq, const OptTensor& pos, bool interleaved,
                  double magnitude) {
  const int64_t B = query.size(0), S = query.size(2), D = query.size(3), hkv = kc.size(1), C = kc.size(2);
  const c10::Device dev = query.device();
  const std::array<int64_t, 4> shape = {B, hkv, S, D};
  FLEXATT_ASSERT(key.sizes() == at::IntArrayRef(shape) && value.sizes() == at::IntArrayRef(shape),
                 "key and value must be [B, Hkv, S, D]");
  x.lengths = per_sequence(lengths, "lengths", B, dev);
  x.freq = freq ? check_frequencies(*freq, D, dev) : Tensor();
  x.r = rotary_struct(query, hkv, x.freq, pos, interleaved, magnitude, false);
  in_place(kc, "key_cache");
  in_place(vc, "value_cache");
  TORCH_CHECK(C > 0, "the cache has no rows");
  x.rows = size32(C, "the cache's rows");
  x.qo = out_like(query);
  if (key.numel() == 0) return false;
  x.queried = query.size(1) > 0;
  x.q = prepare(query), x.k = prepare(key), x.v = prepare(value);
  x.tq = view(x.q), x.tk = view(x.k), x.tv = view(x.v), x.to = view(x.qo), x.tkc = view(kc), x.tvc = view(vc);
  return true;
}
// The norms' weights of an append (key's without a query head).
void check_append_norm(Append& x, const Tensor& query, const Tensor& wq, const Tensor& wk, double eps) {
  no_derivatives({{"query_weight", &wq}, {"key_weight", &wk}});
  x.wq = check_weight(wq, "query_weight", query);
  x.wk = check_weight(wk, "key_weight", query);
  check_eps(eps);
  x.n = norm_struct(query.size(1) > 0 ? x.wq : Tensor(), x.wk, eps);
  x.normed = true;
}

PyObject* py_rotary_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 10, "rotary_append");
  no_trace();
  const Tensor query = tensor_arg(a[0], "query"), key = tensor_arg(a[1], "key"), value = tensor_arg(a[2], "value");
  const Tensor kc = tensor_arg(a[3], "key_cache"), vc = tensor_arg(a[4], "value_cache");
  const Tensor lengths = tensor_arg(a[5], "lengths");
  const OptTensor freq = opt_tensor_arg(a[6], "inv_freq"), pos = opt_tensor_arg(a[7], "positions");
  const bool interleaved = bool_arg(a[8]);
  const double magnitude = double_arg(a[9]);
  if (freq) no_derivatives({{"inv_freq", &*freq}});
  no_derivatives({{"query", &query}, {"key", &key}, {"value", &value}, {"key_cache", &kc}, {"value_cache", &vc}});
  check_tensors({{"query", &query}, {"key", &key}, {"value", &value}, {"key_cache", &kc}, {"value_cache", &vc}});
  check_cache(query, kc, vc);
  const c10::Device dev = query.device();
  const c10::OptionalDeviceGuard guard(dev);
  Append x;
  if (check_append(x, query, key, value, kc, vc, lengths, freq, pos, interleaved, magnitude)) {
    check_status(flexatt_rotary_append(&x.r, x.queried ? &x.tq : nullptr, &x.tk, &x.tv, x.queried ? &x.to : nullptr,
                                       &x.tkc, &x.tvc, x.rows, x.lengths.const_data_ptr<int32_t>(), stream_of(dev)),
                 "flexatt_rotary_append");
    written(kc);
    written(vc);
  }
  return THPVariable_Wrap(x.qo);
  END_HANDLE_TH_ERRORS
}

PyObject* py_norm_rotary_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 13, "norm_rotary_append");
  no_trace();
  const Tensor query = tensor_arg(a[0], "query"), key = tensor_arg(a[1], "key"), value = tensor_arg(a[2], "value");
  const Tensor kc = tensor_arg(a[3], "key_cache"), vc = tensor_arg(a[4], "value_cache");
  const Tensor lengths = tensor_arg(a[5], "lengths");
  const Tensor wq = tensor_arg(a[6], "query_weight"), wk = tensor_arg(a[7], "key_weight");
  const OptTensor freq = opt_tensor_arg(a[8], "inv_freq"), pos = opt_tensor_arg(a[9], "positions");
  const bool interleaved = bool_arg(a[10]);
  const double magnitude = double_arg(a[11]), eps = double_arg(a[12]);
  if (freq) no_derivatives({{"inv_freq", &*freq}});
  no_derivatives({{"query", &query}, {"key", &key}, {"value", &value}, {"key_cache", &kc}, {"value_cache", &vc}});
  check_tensors({{"query", &query}, {"key", &key}, {"value", &value}, {"key_cache", &kc}, {"value_cache", &vc}});
  check_cache(query, kc, vc);
  const c10::Device dev = query.device();
  const c10::OptionalDeviceGuard guard(dev);
  Append x;
  check_append_norm(x, query, wq, wk, eps);
  if (check_append(x, query, key, value, kc, vc, lengths, freq, pos, interleaved, magnitude)) {
    check_status(flexatt_norm_rotary_append(&x.r, &x.n, x.queried ? &x.tq : nullptr, &x.tk, &x.tv,
                                            x.queried ? &x.to : nullptr, &x.tkc, &x.tvc, x.rows,
                                            x.lengths.const_data_ptr<int32_t>(), stream_of(dev)),
                 "flexatt_norm_rotary_append");
    written(kc);
    written(vc);
  }
  return THPVariable_Wrap(x.qo);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------- a cache of 8 bits --
int32_t code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat8_e4m3fn: return FLEXATT_E4M3;
    case at::kChar: return FLEXATT_INT8;
    default:
      TORCH_CHECK(false, "unsupported cache dtype ", t.scalar_type(), " (expected float8_e4m3fn or int8)");
  }
}
// Caches of one 8-bit dtype on `dev`, and their scales; `write`: they are written in place.
int32_t check_codes(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, c10::Device dev, bool write) {
  no_derivatives({{"key_cache", &kc}, {"value_cache", &vc}, {"key_scales", &ks}, {"value_scales", &vs}});
  for (const Named& x : {Named{"key_cache", &kc}, Named{"value_cache", &vc}}) {
    TORCH_CHECK(x.t->device() == dev, x.name, " must be on ", dev, " (got ", x.t->device(), ")");
    TORCH_CHECK(x.t->dim() == 4 && x.t->layout() == at::kStrided, x.name, " must be a strided tensor of four dimensions");
  }
  const int32_t code = code_of(kc);
  TORCH_CHECK(vc.scalar_type() == kc.scalar_type(), "value_cache has dtype ", vc.scalar_type(), ", expected ",
              kc.scalar_type());
  FLEXATT_ASSERT(kc.sizes() == vc.sizes(), "key and value cache shapes must match");
  for (const Named& x : {Named{"key_scales", &ks}, Named{"value_scales", &vs}}) {
    const Tensor& t = *x.t;
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.dim() == 3 && t.size(0) == kc.size(0) && t.size(1) == kc.size(1) &&
                    t.size(2) == kc.size(2) && t.device() == dev,
                x.name, " must be an fp32 [B, Hkv, C] = [", kc.size(0), ", ", kc.size(1), ", ", kc.size(2),
                "] tensor on ", dev);
    TORCH_CHECK(!write || t.is_contiguous(), x.name, " is written in place: it must be contiguous");
  }
  return code;
}

PyObject* py_quant_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 15, "quant_append");
  no_trace();
  const Tensor query = tensor_arg(a[0], "query"), key = tensor_arg(a[1], "key"), value = tensor_arg(a[2], "value");
  const Tensor kc = tensor_arg(a[3], "key_cache"), vc = tensor_arg(a[4], "value_cache");
  const Tensor ks = tensor_arg(a[5], "key_scales"), vs = tensor_arg(a[6], "value_scales");
  const Tensor lengths = tensor_arg(a[7], "lengths");
  const OptTensor freq = opt_tensor_arg(a[8], "inv_freq"), pos = opt_tensor_arg(a[9], "positions");
  const bool interleaved = bool_arg(a[10]);
  const double magnitude = double_arg(a[11]);
  const OptTensor wq = opt_tensor_arg(a[12], "query_weight"), wk = opt_tensor_arg(a[13], "key_weight");
  if (freq) no_derivatives({{"inv_freq", &*freq}});
  no_derivatives({{"query", &query}, {"key", &key}, {"value", &value}});
  check_tensors({{"query", &query}, {"key", &key}, {"value", &value}});
  const c10::Device dev = query.device();
  const int32_t code = check_codes(kc, vc, ks, vs, dev, true);
  check_cache(query, kc, vc);
  const c10::OptionalDeviceGuard guard(dev);
  Append x;
  TORCH_CHECK(wq.has_value() == wk.has_value(), "query_weight and key_weight go together");
  if (wk) check_append_norm(x, query, *wq, *wk, double_arg(a[14]));
  if (check_append(x, query, key, value, kc, vc, lengths, freq, pos, interleaved, magnitude)) {
    check_status(flexatt_quant_append(&x.r, x.normed ? &x.n : nullptr, code, x.queried ? &x.tq : nullptr, &x.tk, &x.tv,
                                      x.queried ? &x.to : nullptr, &x.tkc, &x.tvc, ks.mutable_data_ptr<float>(),
                                      vs.mutable_data_ptr<float>(), x.rows, x.lengths.const_data_ptr<int32_t>(),
                                      stream_of(dev)),
                 "flexatt_quant_append");
    for (const Tensor* t : {&kc, &vc, &ks, &vs}) written(*t);
  }
  return THPVariable_Wrap(x.qo);
  END_HANDLE_TH_ERRORS
}

PyObject* py_dequant(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 8, "dequant");
  no_trace();
  const Tensor kc = tensor_arg(a[0], "key_cache"), vc = tensor_arg(a[1], "value_cache");
  const Tensor ks = tensor_arg(a[2], "key_scales"), vs = tensor_arg(a[3], "value_scales");
  Tensor lengths = tensor_arg(a[4], "lengths");
  const bool fresh = a[6] == Py_None;
  TORCH_CHECK(kc.is_cuda(), "key_cache must be on a ROCm GPU device (got ", kc.device(), ")");
  const c10::Device dev = kc.device();
  const int32_t code = check_codes(kc, vc, ks, vs, dev, false);
  const c10::OptionalDeviceGuard guard(dev);
  const int64_t B = kc.size(0), H = kc.size(1), C = kc.size(2), D = kc.size(3);
  TORCH_CHECK(D == 32 || D == 64 || D == 128 || D == 256, "unsupported head dim ", D, " (expected one of 32, 64, 128, 256)");
  lengths = per_sequence(lengths, "lengths", B, dev);
  Tensor ko, vo;
  if (fresh) {
    TORCH_CHECK(THPDtype_Check(a[5]), "dtype must be a torch.dtype");
    const auto options = kc.options().dtype(((THPDtype*)a[5])->scalar_type);
    ko = at::empty({B, H, C, D}, options);
    vo = at::empty({B, H, C, D}, options);
    check_tensors({{"key", &ko}});
  } else {
    ko = tensor_arg(a[6], "out key");
    vo = tensor_arg(a[7], "out value");
    no_derivatives({{"out key", &ko}, {"out value", &vo}});
    check_tensors({{"out key", &ko}, {"out value", &vo}});
    TORCH_CHECK(ko.device() == dev && ko.sizes() == kc.sizes() && vo.sizes() == kc.sizes(),
                "out key and value must be [B, Hkv, C, D] = ", kc.sizes(), " on ", dev);
    in_place(ko, "out key");
    in_place(vo, "out value");
  }
  if (kc.numel() > 0) {
    flexatt_dequant p = {};
    p.dtype = dtype_of(ko);
    p.code = code;
    p.batch = size32(B, "batch");
    p.heads_kv = size32(H, "Hkv");
    p.cache_rows = size32(C, "the cache's rows");
    p.head_dim = (int32_t)D;
    p.fill = fresh;
    p.lengths = lengths.const_data_ptr<int32_t>();
    const Tensor k = prepare(kc), v = prepare(vc), sk = ks.contiguous(), sv = vs.contiguous();
    const flexatt_tensor tk = view(k), tv = view(v), tko = view(ko), tvo = view(vo);
    check_status(flexatt_dequant_rows(&p, &tk, &tv, sk.const_data_ptr<float>(), sv.const_data_ptr<float>(), &tko, &tvo,
                                      stream_of(dev)),
                 "flexatt_dequant_rows");
    if (!fresh) {
      written(ko);
      written(vo);
    }
  }
  if (fresh) return pair_of(ko, vo);
  return PyTuple_Pack(2, a[6], a[7]);
  END_HANDLE_TH_ERRORS
}

// Attention parameters as the attention entry points take them: a primitive is on
// for a positive value.
struct ScoreParams {
  float scale, cap;
  int32_t window;
};
ScoreParams score_params(PyObject* scale, PyObject* cap, PyObject* window, int64_t D) {
  ScoreParams s;
  s.scale = scale == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)double_arg(scale);
  const double c = cap == Py_None ? 0.0 : double_arg(cap);
  s.cap = c <= 0.0 ? 0.f : (float)c;  // (a NaN is passed on, and rejected)
  const int64_t w = window == Py_None ? 0 : int_arg(window);
  s.window = w <= 0 ? 0 : w > INT32_MAX ? INT32_MAX : (int32_t)w;
  return s;
}

// Drafted tokens over a cache of C rows: what the attention calls over one check, and
// hand over (m and d hold what p points to).
struct Drafted {
  flexatt_tree p;
  Tensor lengths, m, d, O, lse;
};
Drafted check_drafted(const Tensor& query, int64_t Hkv, int64_t C, const Tensor& lengths, const OptTensor& mask,
                      PyObject* window, const OptTensor& depth, PyObject* scale, PyObject* cap) {
  const int64_t B = query.size(0), Hq = query.size(1), T = query.size(2), D = query.size(3);
  const c10::Device dev = query.device();
  Drafted x = {};
  TORCH_CHECK(T <= C, T, " drafted tokens do not fit a cache of ", C, " rows");
  x.lengths = per_sequence(lengths, "lengths", B, dev);
  const ScoreParams s = score_params(scale, cap, window, D);
  flexatt_tree& p = x.p;
  p.dtype = dtype_of(query);
  p.batch = size32(B, "batch");
  p.heads_q = size32(Hq, "Hq");
  p.heads_kv = size32(Hkv, "Hkv");
  p.tokens = size32(T, "T");
  p.cache_rows = size32(C, "the cache's rows");
  p.head_dim = (int32_t)D;
  p.scale = s.scale;
  p.soft_cap = s.cap;
  p.sliding_window = s.window;
  p.lengths = x.lengths.const_data_ptr<int32_t>();
  if (mask) {
    Tensor& m = x.m;
    m = *mask;
    TORCH_CHECK(at::isIntegralType(m.scalar_type(), true), "tree_mask must be a bool or integer tensor");
    TORCH_CHECK((m.dim() == 2 || (m.dim() == 3 && (m.size(0) == 1 || m.size(0) == B))) && m.size(-1) == T &&
                    m.size(-2) == T,
                "tree_mask must be [T, T] or [B, T, T] with B=", B, " and T=", T, ", got ", m.sizes());
    TORCH_CHECK(m.device() == dev, "tree_mask must be on ", dev, " (got ", m.device(), ")");
    if (m.element_size() != 1) m = m.ne(0);
    m = m.contiguous();
    p.mask_batch = m.dim() == 3 ? (int32_t)m.size(0) : 1;
    p.tree_mask = (const uint8_t*)m.data_ptr();
  }
  if (s.window > 0) {
    TORCH_CHECK(depth || !mask, "sliding_window with a tree_mask needs depths");
    if (depth) {
      Tensor& d = x.d;
      d = *depth;
      TORCH_CHECK(d.scalar_type() == at::kInt && d.device() == dev, "depths must be an int32 tensor on ", dev);
      TORCH_CHECK((d.dim() == 1 || (d.dim() == 2 && (d.size(0) == 1 || d.size(0) == B))) && d.size(-1) == T,
                  "depths must be [T] or [B, T] = [", B, ", ", T, "], got ", d.sizes());
      d = d.expand({B, T}).contiguous();
      p.depths = d.const_data_ptr<int32_t>();
    }
  }
  x.O = out_like(query);
  x.lse = at::empty({B, Hq, T}, query.options().dtype(at::kFloat).requires_grad(false));
  return x;
}
// (the kernels' row offsets within a tile are 32 bits)
Tensor near_rows(const Tensor& t) {
  return t.size(2) == 1 || t.stride(2) * t.element_size() < 1 << 26 ? prepare(t) : t.contiguous();
}
PyObject* attended(const Drafted& x, bool return_lse) {
  if (return_lse) return pair_of(x.O, x.lse);
  return THPVariable_Wrap(x.O);
}

PyObject* py_tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 10, "tree_attention");
  no_trace();
  const Tensor query = tensor_arg(a[0], "query");
  const Tensor kc = tensor_arg(a[1], "key_cache"), vc = tensor_arg(a[2], "value_cache");
  const Tensor lengths = tensor_arg(a[3], "lengths");
  const OptTensor mask = opt_tensor_arg(a[4], "tree_mask"), depth = opt_tensor_arg(a[6], "depths");
  no_derivatives({{"query", &query}, {"key_cache", &kc}, {"value_cache", &vc}});
  check_tensors({{"query", &query}, {"key_cache", &kc}, {"value_cache", &vc}});
  check_cache(query, kc, vc);
  const c10::Device dev = query.device();
  const c10::OptionalDeviceGuard guard(dev);
  const Drafted x = check_drafted(query, kc.size(1), kc.size(2), lengths, mask, a[5], depth, a[7], a[8]);
  const bool return_lse = bool_arg(a[9]);
  if (query.numel() > 0) {
    const Tensor q = prepare(query), k = near_rows(kc), v = near_rows(vc);
    const size_t bytes = flexatt_tree_fwd_workspace(&x.p);
    const Tensor ws = workspace(bytes, dev);
    const flexatt_tensor tq = view(q), tk = view(k), tv = view(v), to = view(x.O);
    check_status(flexatt_tree_fwd(&x.p, &tq, &tk, &tv, &to, x.lse.mutable_data_ptr<float>(), data_or_null(ws),
                                  ws.defined() ? bytes : 0, stream_of(dev)),
                 "flexatt_tree_fwd");
  }
  return attended(x, return_lse);
  END_HANDLE_TH_ERRORS
}

PyObject* py_prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 12, "prefix_attention");
  no_trace();
  const Tensor query = tensor_arg(a[0], "query");
  const Tensor pk3 = tensor_arg(a[1], "prefix_key"), pv3 = tensor_arg(a[2], "prefix_value");
  const Tensor kc = tensor_arg(a[3], "key_cache"), vc = tensor_arg(a[4], "value_cache");
  const Tensor lengths = tensor_arg(a[5], "lengths");
  const OptTensor mask = opt_tensor_arg(a[6], "tree_mask"), depth = opt_tensor_arg(a[8], "depths");
  no_derivatives({{"query", &query}, {"prefix_key", &pk3}, {"prefix_value", &pv3}, {"key_cache", &kc}, {"value_cache", &vc}});
  FLEXATT_ASSERT(pk3.dim() == 3 && pv3.dim() == 3, "the prefix's key and value must be [Hkv, P, D]");
  const Tensor pk = pk3.unsqueeze(0), pv = pv3.unsqueeze(0);
  check_tensors({{"query", &query}, {"prefix_key", &pk}, {"prefix_value", &pv}, {"key_cache", &kc}, {"value_cache", &vc}});
  check_cache(query, kc, vc);
  FLEXATT_ASSERT(pk.sizes() == pv.sizes() && pk.size(1) == kc.size(1) && pk.size(3) == kc.size(3),
                 "the prefix's key and value must be [Hkv, P, D] with the cache's Hkv and D");
  const c10::Device dev = query.device();
  const c10::OptionalDeviceGuard guard(dev);
  const Drafted x = check_drafted(query, kc.size(1), kc.size(2), lengths, mask, a[7], depth, a[9], a[10]);
  const bool return_lse = bool_arg(a[11]);
  const int32_t rows = size32(pk.size(2), "the prefix's rows");
  if (query.numel() > 0) {
    const Tensor q = prepare(query), k = near_rows(kc), v = near_rows(vc);
    const flexatt_tensor tq = view(q), tk = view(k), tv = view(v), to = view(x.O);
    if (rows == 0) {  // nothing shared
      const size_t bytes = flexatt_tree_fwd_workspace(&x.p);
      const Tensor ws = workspace(bytes, dev);
      check_status(flexatt_tree_fwd(&x.p, &tq, &tk, &tv, &to, x.lse.mutable_data_ptr<float>(), data_or_null(ws),
                                    ws.defined() ? bytes : 0, stream_of(dev)),
                   "flexatt_tree_fwd");
    } else {
      const Tensor sk = near_rows(pk), sv = near_rows(pv);
      const flexatt_tensor tpk = view(sk), tpv = view(sv);
      const size_t bytes = flexatt_prefix_fwd_workspace(&x.p, rows);
      const Tensor ws = workspace(bytes, dev);
      check_status(flexatt_prefix_fwd(&x.p, rows, &tq, &tpk, &tpv, &tk, &tv, &to, x.lse.mutable_data_ptr<float>(),
                                      data_or_null(ws), ws.defined() ? bytes : 0, stream_of(dev)),
                   "flexatt_prefix_fwd");
    }
  }
  return attended(x, return_lse);
  END_HANDLE_TH_ERRORS
}

PyObject* py_quant_tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 12, "quant_tree_attention");
  no_trace();
  const Tensor query = tensor_arg(a[0], "query");
  const Tensor kc = tensor_arg(a[1], "key_cache"), vc = tensor_arg(a[2], "value_cache");
  const Tensor ks = tensor_arg(a[3], "key_scales"), vs = tensor_arg(a[4], "value_scales");
  const Tensor lengths = tensor_arg(a[5], "lengths");
  const OptTensor mask = opt_tensor_arg(a[6], "tree_mask"), depth = opt_tensor_arg(a[8], "depths");
  no_derivatives({{"query", &query}});
  check_tensors({{"query", &query}});
  const c10::Device dev = query.device();
  TORCH_CHECK(query.scalar_type() != at::kFloat, "a cache of 8 bits is attended by float16 or bfloat16 queries (for float32, "
              "read it back with dequantize_cache)");
  const int32_t code = check_codes(kc, vc, ks, vs, dev, false);
  check_cache(query, kc, vc);
  const c10::OptionalDeviceGuard guard(dev);
  const Drafted x = check_drafted(query, kc.size(1), kc.size(2), lengths, mask, a[7], depth, a[9], a[10]);
  const bool return_lse = bool_arg(a[11]);
  if (query.numel() > 0) {
    const Tensor q = prepare(query), k = near_rows(kc), v = near_rows(vc), sk = ks.contiguous(), sv = vs.contiguous();
    const size_t bytes = flexatt_quant_tree_fwd_workspace(&x.p);
    const Tensor ws = workspace(bytes, dev);
    const flexatt_tensor tq = view(q), tk = view(k), tv = view(v), to = view(x.O);
    check_status(flexatt_quant_tree_fwd(&x.p, code, &tq, &tk, &tv, sk.const_data_ptr<float>(), sv.const_data_ptr<float>(),
                                        &to, x.lse.mutable_data_ptr<float>(), data_or_null(ws), ws.defined() ? bytes : 0,
                                        stream_of(dev)),
                 "flexatt_quant_tree_fwd");
  }
  return attended(x, return_lse);
  END_HANDLE_TH_ERRORS
}

PyObject* py_weight_sums(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 10, "weight_sums");
  no_trace();
  const Tensor query = tensor_arg(a[0], "query"), key = tensor_arg(a[1], "key");
  FLEXATT_ASSERT(THPVariable_Check(a[2]), "lse must be [B, Hq, Sq]");
  Tensor lse = THPVariable_Unpack(a[2]);
  const OptTensor into = opt_tensor_arg(a[9], "into");
  no_derivatives({{"query", &query}, {"key", &key}, {"lse", &lse}});
  if (into) no_derivatives({{"into", &*into}});
  check_tensors({{"query", &query}, {"key", &key}});
  const int64_t B = query.size(0), Hq = query.size(1), Sq = query.size(2), D = query.size(3);
  const int64_t Hkv = key.size(1), Sk = key.size(2);
  const c10::Device dev = query.device();
  const c10::OptionalDeviceGuard guard(dev);
  FLEXATT_ASSERT(key.size(0) == B, "query and key batch sizes must match");
  FLEXATT_ASSERT(key.size(3) == D, "query and key head dims must match");
  FLEXATT_ASSERT(Hkv > 0 && Hq % Hkv == 0, "Hq must be divisible by Hkv");
  FLEXATT_ASSERT(lse.dim() == 3 && lse.size(0) == B && lse.size(1) == Hq && lse.size(2) == Sq, "lse must be [B, Hq, Sq]");
  TORCH_CHECK(lse.device() == dev, "lse must be on ", dev, " (got ", lse.device(), ")");
  lse = lse.to(at::kFloat).contiguous();
  const ScoreParams s = score_params(a[7], a[8], a[6], D);
  flexatt_weights p = {};
  p.dtype = dtype_of(query);
  p.batch = size32(B, "batch");
  p.heads_q = size32(Hq, "Hq");
  p.heads_kv = size32(Hkv, "Hkv");
  p.seqlen_q = size32(Sq, "Sq");
  p.seqlen_kv = size32(Sk, "Skv");
  p.head_dim = (int32_t)D;
  p.scale = s.scale;
  p.soft_cap = s.cap;
  p.causal = bool_arg(a[3]);
  p.sliding_window = s.window;
  Tensor starts, lengths, sums;
  if (THPVariable_Check(a[4])) {
    starts = per_sequence(THPVariable_Unpack(a[4]), "query_start", B, dev);
    p.query_starts = starts.const_data_ptr<int32_t>();
  } else {
    const int64_t x = int_arg(a[4]);
    TORCH_CHECK(x >= INT32_MIN && x <= INT32_MAX, "query_start must fit 32 bits");
    p.query_start = (int32_t)x;
  }
  if (const OptTensor x = opt_tensor_arg(a[5], "lengths")) {
    lengths = per_sequence(*x, "lengths", B, dev);
    p.lengths = lengths.const_data_ptr<int32_t>();
  }
  if (into) {
    sums = *into;
    TORCH_CHECK(sums.scalar_type() == at::kFloat && sums.dim() == 3 && sums.size(0) == B && sums.size(1) == Hkv &&
                    sums.size(2) == Sk && sums.device() == dev && sums.is_contiguous(),
                "into must be a contiguous fp32 [B, Hkv, Skv] = [", B, ", ", Hkv, ", ", Sk, "] tensor on ", dev);
    p.accumulate = 1;
  } else {
    sums = at::empty({B, Hkv, Sk}, query.options().dtype(at::kFloat).requires_grad(false));
  }
  if (sums.numel() > 0 && query.numel() == 0) {
    if (!into) sums.zero_();
  } else if (sums.numel() > 0) {
    const Tensor q = prepare(query), k = prepare(key);
    const size_t bytes = flexatt_weight_sums_workspace(&p);
    const Tensor ws = workspace(bytes, dev);
    const flexatt_tensor tq = view(q), tk = view(k);
    check_status(flexatt_weight_sums(&p, &tq, &tk, lse.const_data_ptr<float>(), sums.mutable_data_ptr<float>(),
                                     data_or_null(ws), ws.defined() ? bytes : 0, stream_of(dev)),
                 "flexatt_weight_sums");
    if (into) written(sums);
  }
  if (into) {
    Py_INCREF(a[9]);
    return a[9];
  }
  return THPVariable_Wrap(sums);
  END_HANDLE_TH_ERRORS
}

PyObject* py_evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want(n, 10, "evict");
  no_trace();
  const Tensor kc = tensor_arg(a[0], "key_cache"), vc = tensor_arg(a[1], "value_cache");
  Tensor scores = tensor_arg(a[2], "scores"), lengths = tensor_arg(a[3], "lengths");
  const bool fresh = a[7] == Py_None;
  Tensor ko, vo, so;
  no_derivatives({{"key_cache", &kc}, {"value_cache", &vc}, {"scores", &scores}});
  if (!fresh) {
    ko = tensor_arg(a[7], "out key");
    vo = tensor_arg(a[8], "out value");
    so = tensor_arg(a[9], "out scores");
    no_derivatives({{"out key", &ko}, {"out value", &vo}, {"out scores", &so}});
  }
  check_tensors({{"key_cache", &kc}, {"value_cache", &vc}});
  FLEXATT_ASSERT(kc.sizes() == vc.sizes(), "key and value cache shapes must match");
  const int64_t B = kc.size(0), H = kc.size(1), C = kc.size(2), D = kc.size(3);
  const c10::Device dev = kc.device();
  const c10::OptionalDeviceGuard guard(dev);
  TORCH_CHECK(kc.numel() > 0, "the cache has no rows");
  TORCH_CHECK(scores.scalar_type() == at::kFloat && scores.dim() == 3 && scores.size(0) == B && scores.size(1) == H &&
                  scores.size(2) == C && scores.device() == dev,
              "scores must be an fp32 [B, Hkv, C] = [", B, ", ", H, ", ", C, "] tensor on ", dev);
  scores = scores.contiguous();
  lengths = per_sequence(lengths, "lengths", B, dev);
  const int64_t keep = int_arg(a[4]), recent = int_arg(a[5]), sinks = int_arg(a[6]);
  TORCH_CHECK(keep >= 1 && keep <= INT32_MAX && recent >= 0 && sinks >= 0 && recent <= keep && sinks <= keep - recent,
              "keep must be at least 1, recent and sinks at least 0 and together at most keep");
  if (fresh) {
    ko = at::empty({B, H, keep, D}, kc.options().requires_grad(false));
    vo = at::empty({B, H, keep, D}, kc.options().requires_grad(false));
    so = at::empty({B, H, keep}, scores.options().requires_grad(false));
  } else {
    check_tensors({{"key_cache", &kc}, {"out key", &ko}, {"out value", &vo}});
    TORCH_CHECK(ko.size(0) == B && ko.size(1) == H && ko.size(3) == D && ko.sizes() == vo.sizes() && ko.size(2) >= keep,
                "out key and value must be [B, Hkv, at least keep, D] = [", B, ", ", H, ", ", keep, ", ", D, "]");
    in_place(ko, "out key");
    in_place(vo, "out value");
    TORCH_CHECK(so.scalar_type() == at::kFloat && so.dim() == 3 && so.size(0) == B && so.size(1) == H &&
                    so.size(2) == ko.size(2) && so.device() == dev && so.is_contiguous(),
                "out scores must be a contiguous fp32 [", B, ", ", H, ", ", ko.size(2), "] tensor on ", dev);
  }
  const auto ints = lengths.options();
  Tensor slots = at::empty({B, H, keep}, ints), fewer = at::empty({B}, ints);
  flexatt_evict p = {};
  p.dtype = dtype_of(kc);
  p.batch = size32(B, "batch");
  p.heads_kv = size32(H, "Hkv");
  p.cache_rows = size32(C, "the cache's rows");
  p.head_dim = (int32_t)D;
  p.keep = (int32_t)keep;
  p.recent = (int32_t)recent;
  p.sinks = (int32_t)sinks;
  p.out_rows = size32(ko.size(2), "the new cache's rows");
  p.fill = fresh;
  p.lengths = lengths.const_data_ptr<int32_t>();
  const Tensor k = prepare(kc), v = prepare(vc);
  const flexatt_tensor tk = view(k), tv = view(v), tko = view(ko), tvo = view(vo);
  check_status(flexatt_evict_rows(&p, &tk, &tv, scores.const_data_ptr<float>(), &tko, &tvo,
                                  so.mutable_data_ptr<float>(), slots.mutable_data_ptr<int32_t>(),
                                  fewer.mutable_data_ptr<int32_t>(), stream_of(dev)),
               "flexatt_evict_rows");
  if (!fresh)
    for (const Tensor* t : {&ko, &vo, &so}) written(*t);
  PyObject* out = PyTuple_New(5);
  if (!out) throw python_error();
  const Tensor* all[5] = {&ko, &vo, &so, &slots, &fewer};
  for (int i = 0; i < 5; ++i) {
    if (!fresh && i < 3) {
      Py_INCREF(a[7 + i]);
      PyTuple_SET_ITEM(out, i, a[7 + i]);
    } else {
      PyTuple_SET_ITEM(out, i, THPVariable_Wrap(*all[i]));
    }
  }
  return out;
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"rotary", (PyCFunction)(void (*)())py_rotary, METH_FASTCALL, nullptr},
    {"rotary_append", (PyCFunction)(void (*)())py_rotary_append, METH_FASTCALL, nullptr},
    {"tree_attention", (PyCFunction)(void (*)())py_tree_attention, METH_FASTCALL, nullptr},
    {"norm_rotary", (PyCFunction)(void (*)())py_norm_rotary, METH_FASTCALL, nullptr},
    {"norm_rotary_append", (PyCFunction)(void (*)())py_norm_rotary_append, METH_FASTCALL, nullptr},
    {"quant_append", (PyCFunction)(void (*)())py_quant_append, METH_FASTCALL, nullptr},
    {"dequant", (PyCFunction)(void (*)())py_dequant, METH_FASTCALL, nullptr},
    {"prefix_attention", (PyCFunction)(void (*)())py_prefix_attention, METH_FASTCALL, nullptr},
    {"quant_tree_attention", (PyCFunction)(void (*)())py_quant_tree_attention, METH_FASTCALL, nullptr},
    {"weight_sums", (PyCFunction)(void (*)())py_weight_sums, METH_FASTCALL, nullptr},
    {"evict", (PyCFunction)(void (*)())py_evict, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "flexatt_native", "libflexatt's cache and rotary calls for torch tensors.",
                       -1, kMethods};
}  // namespace

PyMODINIT_FUNC PyInit_flexatt_native() {
  PyObject* m = PyModule_Create(&kModule);
  if (m && PyModule_AddIntConstant(m, "ABI_VERSION", FLEXATT_ABI_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
