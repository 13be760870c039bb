// The usual calls of the selective scan, the causal convolution and the layer norm
// without an interpreted statement between the caller and the C entry: part of the
// Python module rnn_kernel_b200._host.
//
// Each function takes what its Python namesake takes, positionally, and gives its
// result, or None for a call that it leaves to Python: tensors that have to be
// copied first, calls that torch.jit.trace records, and all that is refused, which
// Python explains.  Gradients are autograd functions; their own derivatives raise.

#include "host_operators.h"

#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/object_ptr.h>

#include <atomic>
#include <climits>
#include <cmath>
#include <string>

#include "../../include/rnn_kernel_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// The library's entries, from bind().
struct {
  decltype(&gru_last_error) last_error;
  decltype(&gru_device_supported) device_supported;
  decltype(&gru_scan_stash_bytes) scan_stash_bytes;
  decltype(&gru_scan_workspace_bytes) scan_workspace_bytes;
  decltype(&gru_scan_forward) scan_forward;
  decltype(&gru_scan_backward) scan_backward;
  decltype(&gru_scan_step) scan_step;
  decltype(&gru_conv_workspace_bytes) conv_workspace_bytes;
  decltype(&gru_conv_forward) conv_forward;
  decltype(&gru_conv_backward) conv_backward;
  decltype(&gru_conv_step) conv_step;
  decltype(&gru_layer_norm_workspace_bytes) norm_workspace_bytes;
  decltype(&gru_layer_norm_forward) norm_forward;
  decltype(&gru_layer_norm_backward) norm_backward;
} lib;

void check(int status, const char* what) {
  TORCH_CHECK(status == 0, what, " failed (status ", status, "): ", lib.last_error());
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
const float* f32(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
float* out_f32(const Tensor& t) { return static_cast<float*>(out_ptr(t)); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor floats(const Tensor& like, int64_t bytes) { return at::empty({bytes / 4}, like.options().dtype(at::kFloat)); }

int code_of(at::ScalarType t) { return t == at::kFloat ? GRU_F32 : GRU_BF16; }
bool usual(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

bool supported(int device) {
  static std::atomic<signed char> known[64];  // 0: not asked yet
  if (device < 0 || device >= 64) return false;
  signed char k = known[device].load();
  if (k == 0) known[device].store(k = lib.device_supported(device) ? 1 : -1);
  return k > 0;
}

// Whether a call is of the usual kind: as many arguments as it takes, an entry to call, and
// no trace being recorded, which would hold the allocations alone.
template <typename F>
bool ready(Py_ssize_t n, Py_ssize_t takes, F entry) {
  return n == takes && entry && !torch::jit::tracer::isTracing();
}
// A plain tensor, or None where that is allowed (an undefined one then).
bool take(PyObject* o, Tensor* t, bool none_too = false) {
  if (o == Py_None) return none_too;
  if (!THPVariable_CheckExact(o)) return false;
  *t = THPVariable_Unpack(o);
  return t->layout() == at::kStrided && !t->is_neg();
}
// Whether the C structs' sizes hold x's.
bool counted(const Tensor& x) {
  for (const int64_t n : x.sizes())
    if (n > INT_MAX) return false;
  return true;
}
bool on(const Tensor& t, const Tensor& like, at::ScalarType type) {
  return t.device() == like.device() && t.scalar_type() == type;
}
// Absent, or of that type and size, and dense.
bool vector_of(const Tensor& t, const Tensor& like, at::ScalarType type, int64_t n) {
  return !t.defined() || (on(t, like, type) && t.dim() == 1 && t.size(0) == n && t.is_contiguous());
}
bool dense_last(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1; }
// The same, with tokens less than 2^31 bytes apart.
bool near(const Tensor& t) { return dense_last(t) && t.stride(1) * t.element_size() < (int64_t(1) << 31); }

template <typename... T>
bool differentiated(const T&... t) {
  return at::GradMode::is_enabled() && ((t.defined() && t.requires_grad()) || ...);
}

PyObject* one(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* two(const Tensor& a, const Tensor& b) {
  THPObjectPtr r(PyTuple_New(2));
  if (!r) throw python_error();
  PyTuple_SET_ITEM(r.get(), 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(r.get(), 1, THPVariable_Wrap(b));
  return r.release();
}

std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
Tensor given(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// Passes gradients on; their own derivative raises, where without it they would
// count as constants.
struct NoSecond : Function<NoSecond> {
  static variable_list forward(AutogradContext* ctx, Tensor anchor, std::string name, variable_list grads) {
    ctx->saved_data["name"] = name;
    variable_list out;
    for (const Tensor& g : grads) out.push_back(g.clone());
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list) {
    TORCH_CHECK(false, ctx->saved_data["name"].toStringRef(), " has no second derivative.");
  }
};
variable_list first_derivatives(const char* name, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (const Tensor& g : grads)
    if (g.defined()) some.push_back(g);
  Tensor anchor = at::empty({0});
  anchor.requires_grad_(true);
  some = NoSecond::apply(anchor, std::string(name), some);
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = some[k++];
  return grads;
}

// ---- layer norm ---------------------------------------------------------------

gru_norm_args norm_args(const Tensor& x, const Tensor& s, const Tensor& weight, double eps) {
  const int64_t D = weight.size(0);
  gru_norm_args a{};
  a.dtype = code_of(x.scalar_type()), a.residual_dtype = code_of(s.scalar_type()), a.weight_dtype = code_of(weight.scalar_type());
  a.width = (int)D, a.eps = (float)eps;
  a.rows = x.numel() / D, a.row_stride = a.residual_row_stride = D;
  return a;
}

void norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, double eps, Tensor* out,
                  Tensor* sum, Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  const gru_norm_args a = norm_args(x, residual.defined() ? residual : x, weight, eps);
  *out = at::empty(x.sizes(), x.options());
  if (residual.defined()) *sum = at::empty(x.sizes(), residual.options());
  if (stats) *stats = at::empty({3, a.rows}, x.options().dtype(at::kFloat));
  check(lib.norm_forward(&a, ptr(x), ptr(residual), ptr(weight), ptr(bias), out_ptr(*out), out_ptr(*sum),
                         stats ? out_f32(*stats) : nullptr, stream_of(x)),
        "gru_layer_norm_forward");
}

struct LayerNorm : Function<LayerNorm> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor weight, std::optional<Tensor> bias,
                               std::optional<Tensor> residual, double eps) {
    Tensor out, sum, stats;
    norm_forward(x, weight, given(bias), given(residual), eps, &out, &sum, &stats);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({sum.defined() ? sum : x, weight, stats});
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->saved_data["has"] = (int64_t)(bias.has_value() | (residual.has_value() << 1));
    return sum.defined() ? variable_list{out, sum} : variable_list{out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &weight = saved[1], &stats = saved[2];
    const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
    const int64_t has = ctx->saved_data["has"].toInt();
    const c10::DeviceGuard guard(s.device());
    Tensor dout = grads[0].defined() ? grads[0].contiguous() : at::zeros(s.sizes(), s.options().dtype(type));
    Tensor dsum = has & 2 ? dense(grads[1]) : Tensor();
    Tensor dx = at::empty(s.sizes(), s.options().dtype(type)), dres;
    // a sum hands the same gradient to both of its terms, as torch's addition does, if they have one type
    if (has & 2 && s.scalar_type() != type) dres = at::empty(s.sizes(), s.options());
    Tensor dw = at::empty_like(weight), db = has & 1 ? at::empty_like(weight) : Tensor();
    const gru_norm_args a = norm_args(dx, s, weight, 0.0);
    const size_t bytes = lib.norm_workspace_bytes(&a);
    Tensor ws = floats(s, (int64_t)bytes);
    check(lib.norm_backward(&a, ptr(s), ptr(weight), f32(stats), ptr(dout), ptr(dsum), out_ptr(dx), out_ptr(dres), out_ptr(dw),
                            out_ptr(db), out_ptr(ws), bytes, stream_of(s)),
          "gru_layer_norm_backward");
    variable_list g = first_derivatives("layer_norm", {dx, dw, db, dres});
    return {g[0], g[1], g[2], has & 2 ? (dres.defined() ? g[3] : g[0]) : Tensor(), Tensor()};
  }
};

// ---- selective scan -----------------------------------------------------------

gru_scan_args scan_args(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& skip,
                        const Tensor& z, const Tensor& bias, bool softplus, const Tensor& state) {
  gru_scan_args a{};
  const bool all = x.dim() == 3;  // else one token
  a.dtype = code_of(x.scalar_type());
  a.B = (int)x.size(0), a.T = all ? (int)x.size(1) : 1, a.D = (int)A.size(0), a.N = (int)A.size(1), a.G = (int)B.size(-2);
  a.dt_softplus = softplus;
  a.x = ptr(x), a.dt = ptr(dt), a.b = ptr(B), a.c = ptr(C), a.z = ptr(z);
  a.a = f32(A), a.skip = f32(skip), a.dt_bias = f32(bias), a.initial_state = f32(state);
  auto rows = [&](long* s, const Tensor& t) {
    if (t.defined()) s[0] = t.stride(0), s[1] = all ? t.stride(1) : 0;
  };
  rows(a.x_stride, x), rows(a.dt_stride, dt), rows(a.z_stride, z), rows(a.b_stride, B), rows(a.c_stride, C);
  a.b_stride[2] = B.stride(-2), a.c_stride[2] = C.stride(-2);
  return a;
}

// Whether all of a call's tensors are as the C entry takes them; lead: dimensions
// before the channels.
bool scan_usual(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& skip,
                const Tensor& z, const Tensor& bias, const Tensor& state, int64_t lead) {
  const auto type = x.scalar_type();
  if (!x.is_cuda() || !usual(type) || x.dim() != lead + 1 || !counted(x) || A.dim() != 2 || B.dim() != lead + 2) return false;
  const int64_t D = x.size(-1), G = B.size(-2), N = B.size(-1);
  if (D < 1 || G < 1 || D % G || N < 1 || N > 64) return false;
  if (!on(dt, x, type) || dt.sizes() != x.sizes() || (z.defined() && (!on(z, x, type) || z.sizes() != x.sizes()))) return false;
  if (!on(B, x, type) || !on(C, x, type) || B.sizes() != C.sizes() || B.sizes().slice(0, lead) != x.sizes().slice(0, lead)) return false;
  if (!on(A, x, at::kFloat) || A.size(0) != D || A.size(1) != N || !A.is_contiguous()) return false;
  if (!vector_of(skip, x, at::kFloat, D) || !vector_of(bias, x, at::kFloat, D)) return false;
  if (state.defined() && (!on(state, x, at::kFloat) || state.dim() != 3 || state.size(0) != x.size(0) || state.size(1) != D ||
                          state.size(2) != N || !state.is_contiguous()))
    return false;
  for (const Tensor* t : {&x, &dt, &B, &C, &z})
    if (t->defined() && !(lead == 2 ? near(*t) : dense_last(*t))) return false;
  return supported(x.device().index());
}

void scan_forward(const gru_scan_args& a, const Tensor& x, const Tensor& A, Tensor* out, Tensor* last, Tensor* stash) {
  const c10::DeviceGuard guard(x.device());
  *out = at::empty({a.B, a.T, a.D}, x.options());
  *last = at::empty({a.B, a.D, a.N}, A.options());
  const size_t kept = stash ? lib.scan_stash_bytes(&a) : 0, bytes = lib.scan_workspace_bytes(&a, 0);
  if (stash) *stash = floats(A, (int64_t)kept);
  Tensor ws = bytes ? floats(A, (int64_t)bytes) : Tensor();
  check(lib.scan_forward(&a, out_ptr(*out), out_f32(*last), stash ? out_ptr(*stash) : nullptr, kept, out_ptr(ws), bytes, stream_of(x)),
        "gru_scan_forward");
}

struct Scan : Function<Scan> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, std::optional<Tensor> skip,
                               std::optional<Tensor> z, std::optional<Tensor> bias, bool softplus, std::optional<Tensor> state) {
    Tensor out, last, stash;
    scan_forward(scan_args(x, dt, A, B, C, given(skip), given(z), given(bias), softplus, given(state)), x, A, &out, &last, &stash);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, dt, A, B, C, given(skip), given(z), given(bias), stash});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["state"] = state.has_value() && state->requires_grad();
    return {out, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &A = s[2], &skip = s[5], &z = s[6], &bias = s[7], &stash = s[8];
    const gru_scan_args a = scan_args(x, s[1], A, s[3], s[4], skip, z, bias, ctx->saved_data["softplus"].toBool(), Tensor());
    const c10::DeviceGuard guard(x.device());
    Tensor dout = dense(grads[0]), dlast = dense(grads[1]);
    auto wide = [&] { return at::empty({a.B, a.T, a.D}, x.options()); };
    auto few = [&] { return at::empty({a.B, a.T, a.G, a.N}, x.options()); };
    Tensor dx = wide(), ddt = wide(), dz = z.defined() ? wide() : Tensor(), dB = few(), dC = few(), dA = at::empty_like(A);
    Tensor dskip = skip.defined() ? at::empty_like(skip) : Tensor(), dbias = bias.defined() ? at::empty_like(bias) : Tensor();
    Tensor dstate = ctx->saved_data["state"].toBool() ? at::empty({a.B, a.D, a.N}, A.options()) : Tensor();
    const size_t kept = lib.scan_stash_bytes(&a), bytes = lib.scan_workspace_bytes(&a, 1);
    Tensor ws = floats(A, (int64_t)bytes);
    check(lib.scan_backward(&a, ptr(dout), f32(dlast), ptr(stash), kept, out_ptr(dx), out_ptr(ddt), out_f32(dA), out_ptr(dB),
                            out_ptr(dC), out_f32(dskip), out_ptr(dz), out_f32(dbias), out_f32(dstate), out_ptr(ws), bytes,
                            stream_of(x)),
          "gru_scan_backward");
    variable_list g = first_derivatives("selective_scan", {dx, ddt, dA, dB, dC, dskip, dz, dbias, dstate});
    return {g[0], g[1], g[2], g[3], g[4], g[5], g[6], g[7], Tensor(), g[8]};
  }
};

// ---- causal convolution -------------------------------------------------------

gru_conv_args conv_args(const Tensor& x, const Tensor& weight, const Tensor& bias, int activation, const Tensor& state) {
  gru_conv_args a{};
  const bool all = x.dim() == 3;
  a.dtype = code_of(x.scalar_type()), a.weight_dtype = code_of(weight.scalar_type());
  a.B = (int)x.size(0), a.T = all ? (int)x.size(1) : 1, a.D = (int)weight.size(0), a.W = (int)weight.size(1);
  a.activation = activation;
  a.x = ptr(x), a.weight = ptr(weight), a.bias = ptr(bias), a.initial_state = ptr(state);
  a.x_stride[0] = x.stride(0), a.x_stride[1] = all ? x.stride(1) : 0;
  return a;
}
bool conv_usual(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& state, int64_t lead) {
  const auto type = x.scalar_type();
  if (!x.is_cuda() || !usual(type) || x.dim() != lead + 1 || !counted(x) || weight.dim() != 2) return false;
  const int64_t D = x.size(-1), W = weight.size(1);
  const auto wtype = weight.scalar_type();
  if (D < 1 || W < 2 || W > 8 || weight.size(0) != D || !weight.is_contiguous() || weight.device() != x.device()) return false;
  if ((wtype != type && wtype != at::kFloat) || !vector_of(bias, x, wtype, D)) return false;
  if (state.defined() && (!on(state, x, type) || state.dim() != 3 || state.size(0) != x.size(0) || state.size(1) != W - 1 ||
                          state.size(2) != D || !state.is_contiguous()))
    return false;
  return dense_last(x) && supported(x.device().index());
}

void conv_forward(const gru_conv_args& a, const Tensor& x, Tensor* out, Tensor* last) {
  const c10::DeviceGuard guard(x.device());
  *out = at::empty({a.B, a.T, a.D}, x.options());
  *last = at::empty({a.B, a.W - 1, a.D}, x.options());
  check(lib.conv_forward(&a, out_ptr(*out), out_ptr(*last), stream_of(x)), "gru_conv_forward");
}

struct Conv : Function<Conv> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor weight, std::optional<Tensor> bias, int64_t activation,
                               std::optional<Tensor> state) {
    Tensor out, last;
    conv_forward(conv_args(x, weight, given(bias), (int)activation, given(state)), x, &out, &last);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, given(bias), given(state)});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["state"] = state.has_value() && state->requires_grad();
    return {out, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &weight = s[1], &bias = s[2], &state = s[3];
    const gru_conv_args a = conv_args(x, weight, bias, (int)ctx->saved_data["activation"].toInt(), state);
    const c10::DeviceGuard guard(x.device());
    Tensor dout = dense(grads[0]), dlast = dense(grads[1]);
    Tensor dx = at::empty({a.B, a.T, a.D}, x.options()), dw = at::empty_like(weight);
    Tensor db = bias.defined() ? at::empty_like(bias) : Tensor(), ds = ctx->saved_data["state"].toBool() ? at::empty_like(state) : Tensor();
    const size_t bytes = lib.conv_workspace_bytes(&a);
    Tensor ws = floats(x, (int64_t)bytes);
    check(lib.conv_backward(&a, ptr(dout), ptr(dlast), out_ptr(dx), out_ptr(dw), out_ptr(db), out_ptr(ds), out_ptr(ws), bytes,
                            stream_of(x)),
          "gru_conv_backward");
    variable_list g = first_derivatives("causal_conv", {dx, dw, db, ds});
    return {g[0], g[1], g[2], Tensor(), g[3]};
  }
};

// ---- what Python calls ---------------------------------------------------------

// An activation's code: 0 None, 1 "silu", -1 anything else.
int activation_of(PyObject* o) {
  if (o == Py_None) return 0;
  return PyUnicode_Check(o) && PyUnicode_CompareWithASCIIString(o, "silu") == 0 ? 1 : -1;
}

bool changed_in_place(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return true;
}

// layer_norm(x, weight, bias, eps, residual)
PyObject* layer_norm(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, weight, bias, residual;
  if (!ready(n, 5, lib.norm_forward) || !take(o[0], &x) || !take(o[1], &weight) || !take(o[2], &bias, true) ||
      !PyFloat_Check(o[3]) || !take(o[4], &residual, true))
    Py_RETURN_NONE;
  const double eps = PyFloat_AS_DOUBLE(o[3]);
  const auto type = x.scalar_type(), wtype = weight.scalar_type();
  if (!x.is_cuda() || !usual(type) || x.dim() < 1 || !x.is_contiguous() || !(eps >= 0.0) || !std::isfinite(eps)) Py_RETURN_NONE;
  const int64_t D = x.size(-1);
  if (D < 1 || D > 16384 || (wtype != type && wtype != at::kFloat) || !vector_of(weight, x, wtype, D) || !vector_of(bias, x, wtype, D))
    Py_RETURN_NONE;
  if (residual.defined() && (residual.device() != x.device() || residual.sizes() != x.sizes() || !residual.is_contiguous() ||
                             (residual.scalar_type() != type && residual.scalar_type() != at::kFloat)))
    Py_RETURN_NONE;
  if (!supported(x.device().index())) Py_RETURN_NONE;
  variable_list r;
  {
    pybind11::gil_scoped_release no_gil;
    if (differentiated(x, weight, bias, residual)) {
      r = LayerNorm::apply(x, weight, maybe(bias), maybe(residual), eps);
    } else {
      r.resize(2);
      norm_forward(x, weight, bias, residual, eps, &r[0], &r[1], nullptr);
    }
  }
  return residual.defined() ? two(r[0], r[1]) : one(r[0]);
  END_HANDLE_TH_ERRORS
}

// selective_scan(x, dt, A, B, C, skip, z, dt_bias, dt_softplus, initial_state)
PyObject* selective_scan(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, dt, A, B, C, skip, z, bias, state;
  if (!ready(n, 10, lib.scan_forward) || !take(o[0], &x) || !take(o[1], &dt) || !take(o[2], &A) || !take(o[3], &B) || !take(o[4], &C) ||
      !take(o[5], &skip, true) || !take(o[6], &z, true) || !take(o[7], &bias, true) || !PyBool_Check(o[8]) || !take(o[9], &state, true))
    Py_RETURN_NONE;
  if (!scan_usual(x, dt, A, B, C, skip, z, bias, state, 2)) Py_RETURN_NONE;
  const bool softplus = o[8] == Py_True;
  variable_list r;
  {
    pybind11::gil_scoped_release no_gil;
    if (differentiated(x, dt, A, B, C, skip, z, bias, state)) {
      r = Scan::apply(x, dt, A, B, C, maybe(skip), maybe(z), maybe(bias), softplus, maybe(state));
    } else {
      r.resize(2);
      scan_forward(scan_args(x, dt, A, B, C, skip, z, bias, softplus, state), x, A, &r[0], &r[1], nullptr);
    }
  }
  return two(r[0], r[1]);
  END_HANDLE_TH_ERRORS
}

// selective_step(x, dt, A, B, C, state, skip, z, dt_bias, dt_softplus)
PyObject* selective_step(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, dt, A, B, C, skip, z, bias, state;
  if (!ready(n, 10, lib.scan_step) || !take(o[0], &x) || !take(o[1], &dt) || !take(o[2], &A) || !take(o[3], &B) || !take(o[4], &C) ||
      !take(o[5], &state) || !take(o[6], &skip, true) || !take(o[7], &z, true) || !take(o[8], &bias, true) || !PyBool_Check(o[9]))
    Py_RETURN_NONE;
  if (!scan_usual(x, dt, A, B, C, skip, z, bias, state, 1)) Py_RETURN_NONE;
  const gru_scan_args a = scan_args(x, dt, A, B, C, skip, z, bias, o[9] == Py_True, Tensor());
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(x.device());
    out = at::empty({a.B, a.D}, x.options());
    check(lib.scan_step(&a, out_f32(state), out_ptr(out), stream_of(x)), "gru_scan_step");
    changed_in_place(state);
  }
  return one(out);
  END_HANDLE_TH_ERRORS
}

// causal_conv(x, weight, bias, activation, initial_state)
PyObject* causal_conv(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, weight, bias, state;
  if (!ready(n, 5, lib.conv_forward) || !take(o[0], &x) || !take(o[1], &weight) || !take(o[2], &bias, true) || !take(o[4], &state, true))
    Py_RETURN_NONE;
  const int activation = activation_of(o[3]);
  if (activation < 0 || !conv_usual(x, weight, bias, state, 2)) Py_RETURN_NONE;
  variable_list r;
  {
    pybind11::gil_scoped_release no_gil;
    if (differentiated(x, weight, bias, state)) {
      r = Conv::apply(x, weight, maybe(bias), (int64_t)activation, maybe(state));
    } else {
      r.resize(2);
      conv_forward(conv_args(x, weight, bias, activation, state), x, &r[0], &r[1]);
    }
  }
  return two(r[0], r[1]);
  END_HANDLE_TH_ERRORS
}

// causal_conv_step(x, weight, state, bias, activation)
PyObject* causal_conv_step(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor x, weight, bias, state;
  if (!ready(n, 5, lib.conv_step) || !take(o[0], &x) || !take(o[1], &weight) || !take(o[2], &state) || !take(o[3], &bias, true)) Py_RETURN_NONE;
  const int activation = activation_of(o[4]);
  if (activation < 0 || !conv_usual(x, weight, bias, state, 1)) Py_RETURN_NONE;
  const gru_conv_args a = conv_args(x, weight, bias, activation, Tensor());
  Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(x.device());
    out = at::empty({a.B, a.D}, x.options());
    check(lib.conv_step(&a, out_ptr(state), out_ptr(out), stream_of(x)), "gru_conv_step");
    changed_in_place(state);
  }
  return one(out);
  END_HANDLE_TH_ERRORS
}

// bind({entry's name: its address}): where the library was loaded.
PyObject* bind(PyObject*, PyObject* table) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(PyDict_Check(table), "bind: a dict of addresses");
  auto address = [&](const char* name) {
    PyObject* v = PyDict_GetItemString(table, name);
    TORCH_CHECK(v && PyLong_Check(v), "bind: no address of ", name);
    return PyLong_AsVoidPtr(v);
  };
#define GRU_BIND(field, name) lib.field = reinterpret_cast<decltype(&name)>(address(#name))
  GRU_BIND(last_error, gru_last_error);
  GRU_BIND(device_supported, gru_device_supported);
  GRU_BIND(scan_stash_bytes, gru_scan_stash_bytes);
  GRU_BIND(scan_workspace_bytes, gru_scan_workspace_bytes);
  GRU_BIND(scan_forward, gru_scan_forward);
  GRU_BIND(scan_backward, gru_scan_backward);
  GRU_BIND(scan_step, gru_scan_step);
  GRU_BIND(conv_workspace_bytes, gru_conv_workspace_bytes);
  GRU_BIND(conv_forward, gru_conv_forward);
  GRU_BIND(conv_backward, gru_conv_backward);
  GRU_BIND(conv_step, gru_conv_step);
  GRU_BIND(norm_workspace_bytes, gru_layer_norm_workspace_bytes);
  GRU_BIND(norm_forward, gru_layer_norm_forward);
  GRU_BIND(norm_backward, gru_layer_norm_backward);
#undef GRU_BIND
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define GRU_FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {GRU_FAST(layer_norm),  GRU_FAST(selective_scan), GRU_FAST(selective_step),
                         GRU_FAST(causal_conv), GRU_FAST(causal_conv_step), {"bind", bind, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

}  // namespace

PyMethodDef* operator_methods() { return methods; }
