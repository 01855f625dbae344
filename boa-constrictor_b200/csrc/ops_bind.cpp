// Host side of boa_b200.ops: argument checks, outputs and workspaces from
// torch's allocator, torch's current stream, gradients, and the calls of the
// library's C entry points.  A one-token call is mostly host time, which is why
// this is C++: 11-22 us a call from Python through ctypes, about 5 us from here.
//
// The entry points' addresses come from the library that boa_b200._native
// loads, so this module holds no kernels and links to none.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <sstream>
#include <stdexcept>
#include <string>

#include "boa_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kStates = 16;

// ------------------------------------------------------------------- errors
struct Refused {            // bad arguments: ValueError, or RuntimeError for the wrong device
  PyObject* type;
  std::string text;
};
struct Failed : std::runtime_error {   // an error code of the library: BoaError (RuntimeError inside backward)
  int code;
  std::string plain;                   // BoaError adds the code itself
  Failed(int c, const std::string& p) : std::runtime_error(with_code(c, p)), code(c), plain(p) {}
  static std::string with_code(int c, const std::string& p) {
    return "[boa_b200 error " + std::to_string(c) + "] " + p;
  }
};

void put(std::ostringstream& s, const char* v) { s << v; }
void put(std::ostringstream& s, int64_t v) { s << v; }
void put(std::ostringstream& s, int v) { s << v; }
void put(std::ostringstream& s, at::ScalarType t) { s << c10::toString(t); }
void put(std::ostringstream& s, const c10::Device& d) { s << d.str(); }
void put(std::ostringstream& s, at::IntArrayRef v) {
  s << '(';
  for (size_t i = 0; i < v.size(); ++i) s << (i ? ", " : "") << v[i];
  s << ')';
}
template <typename... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (put(s, a), ...);
  return s.str();
}
[[noreturn]] void refuse(const std::string& what) { throw Refused{PyExc_ValueError, what}; }

// ------------------------------------------------------------- entry points
struct Api {
  bool ready = false;
  decltype(&boa_last_error) last_error;
  decltype(&boa_layer_norm) layer_norm;
  decltype(&boa_layer_norm_workspace_bytes) layer_norm_workspace_bytes;
  decltype(&boa_layer_norm_backward) layer_norm_backward;
  decltype(&boa_causal_conv) causal_conv;
  decltype(&boa_causal_conv_workspace_bytes) causal_conv_workspace_bytes;
  decltype(&boa_causal_conv_backward) causal_conv_backward;
  decltype(&boa_causal_conv_step) causal_conv_step;
  decltype(&boa_ssm_checkpoint_bytes) ssm_checkpoint_bytes;
  decltype(&boa_ssm_workspace_bytes) ssm_workspace_bytes;
  decltype(&boa_ssm_scan) ssm_scan;
  decltype(&boa_ssm_scan_backward) ssm_scan_backward;
  decltype(&boa_ssm_step) ssm_step;
} api;
PyObject* loader = nullptr;     // called once, on first use: {name: address}
PyObject* boa_error = nullptr;  // boa_b200._native.BoaError

struct PythonError {};          // a Python error is set

template <typename F>
void address(PyObject* d, const char* name, F& f) {
  PyObject* v = PyDict_GetItemString(d, name);
  if (!v) {
    PyErr_Format(PyExc_RuntimeError, "libboa_b200.so has no %s", name);
    throw PythonError{};
  }
  f = reinterpret_cast<F>(PyLong_AsVoidPtr(v));
}

void need_api() {
  if (api.ready) return;
  PyObject* d = loader ? PyObject_CallNoArgs(loader) : nullptr;
  if (!d) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "_boa_ops: bind() was not called");
    throw PythonError{};
  }
  address(d, "boa_last_error", api.last_error);
  address(d, "boa_layer_norm", api.layer_norm);
  address(d, "boa_layer_norm_workspace_bytes", api.layer_norm_workspace_bytes);
  address(d, "boa_layer_norm_backward", api.layer_norm_backward);
  address(d, "boa_causal_conv", api.causal_conv);
  address(d, "boa_causal_conv_workspace_bytes", api.causal_conv_workspace_bytes);
  address(d, "boa_causal_conv_backward", api.causal_conv_backward);
  address(d, "boa_causal_conv_step", api.causal_conv_step);
  address(d, "boa_ssm_checkpoint_bytes", api.ssm_checkpoint_bytes);
  address(d, "boa_ssm_workspace_bytes", api.ssm_workspace_bytes);
  address(d, "boa_ssm_scan", api.ssm_scan);
  address(d, "boa_ssm_scan_backward", api.ssm_scan_backward);
  address(d, "boa_ssm_step", api.ssm_step);
  Py_DECREF(d);
  api.ready = true;
}

void check(int rc, const char* name) {
  if (rc != BOA_OK) throw Failed(rc, text(name, ": ", api.last_error()));
}

// ---------------------------------------------------------------- arguments
int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? BOA_DTYPE_F32 : t == at::kBFloat16 ? BOA_DTYPE_BF16 : t == at::kHalf ? BOA_DTYPE_F16 : -1;
}
void check_kind(const char* who, const Tensor& x) {
  if (dtype_code(x.scalar_type()) < 0)
    refuse(text(who, ": x must be float32, bfloat16 or float16, not ", x.scalar_type()));
  for (const int64_t n : x.sizes())      // the entry points take 32-bit sizes
    if (n > INT32_MAX) refuse(text(who, ": every size of x must be below 2^31, got ", x.sizes()));
}
void check_shape(const char* who, const char* name, const Tensor& t, at::IntArrayRef want) {
  if (t.sizes() != want) refuse(text(who, ": ", name, " must have shape ", want, ", got ", t.sizes()));
}
void check_same(const char* who, const char* name, const Tensor& x, const Tensor& t) {
  if (t.scalar_type() != x.scalar_type())
    refuse(text(who, ": ", name, " must have the type of x (", x.scalar_type(), "), got ", t.scalar_type()));
}
void check_device(const char* who, const Tensor& x, std::initializer_list<const Tensor*> others) {
  if (!x.is_cuda()) throw Refused{PyExc_RuntimeError, text(who, " runs on CUDA devices only (no CPU path)")};
  for (const Tensor* t : others)
    if (t->defined() && t->device() != x.device())
      throw Refused{PyExc_RuntimeError,
                    text(who, ": all tensors must be on ", x.device(), ", got one on ", t->device())};
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
bool misaligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0; }

// Memory as the values are: a view that torch marks as negated holds the other sign.
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// A parameter as contiguous, 16-byte aligned fp32 (differentiable).
Tensor param(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor r = plain(t.scalar_type() == at::kFloat ? t : t.to(at::kFloat));
  if (!r.is_contiguous()) r = r.contiguous();
  return misaligned(r) ? r.clone() : r;
}
// Channels contiguous; other strides stay as they are.
Tensor rows(const Tensor& t) {
  return plain(!t.defined() || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous());
}
Tensor whole(const Tensor& t) { return t.defined() ? plain(t.contiguous()) : t; }
// An input of a step apart from the state that the step changes in place: one that shares its memory would be read by
// some threads after others have written it.
Tensor apart(const Tensor& t, const Tensor& state) {
  if (!t.defined() || t.numel() == 0 || state.numel() == 0) return t;
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  const char *begin = static_cast<const char*>(t.data_ptr()), *end = begin + (last + 1) * (int64_t)t.element_size();
  const char *from = static_cast<const char*>(state.data_ptr()), *to = from + state.nbytes();
  return begin < to && from < end ? t.clone(at::MemoryFormat::Contiguous) : t;
}
Tensor int_lens(const char* who, const Tensor& lens, int64_t batch, int64_t length) {
  if (!lens.defined()) return lens;
  if (lens.scalar_type() != at::kInt && lens.scalar_type() != at::kLong)
    refuse(text(who, ": lens must be int32 or int64, not ", lens.scalar_type()));
  check_shape(who, "lens", lens, {batch});
  return (lens.scalar_type() == at::kInt ? lens : lens.clamp(0, length).to(at::kInt)).contiguous();
}
// A tangent (torch.autograd.forward_ad) is no requires_grad: without this the
// raw call would drop it, and a dropped tangent reads as a derivative of zero.
void reverse_mode_only(const char* who, std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined())
      throw Refused{PyExc_RuntimeError,
                    text(who, " has no forward-mode derivative: take derivatives with backward() or torch.autograd.grad")};
}
// torch.jit.trace cannot see into a call: it would record its result as a constant.
void no_tracing(const char* who) {
  if (torch::jit::tracer::isTracing())
    throw Refused{PyExc_RuntimeError, text(who, " cannot be traced: its result would become a constant")};
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
Tensor like(const Tensor& t) { return t.defined() ? fresh(t.sizes(), t.scalar_type(), t) : Tensor(); }
Tensor bytes(size_t n, const Tensor& x) { return n ? fresh({(int64_t)n}, at::kByte, x) : Tensor(); }
void* stream_of(const Tensor& x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }
// The library selects the device; this puts the caller's back.
struct OnDevice {
  c10::cuda::CUDAGuard guard;
  explicit OnDevice(const Tensor& x) : guard((c10::DeviceIndex)x.get_device()) {}
};
// Optional inputs cross Function::apply as optionals: it asks plain ones for their device.
using Opt = std::optional<Tensor>;
Opt opt(const Tensor& t) { return t.defined() ? Opt(t) : Opt(); }
Tensor val(const Opt& o) { return o.has_value() ? *o : Tensor(); }

// For a backward call with the incoming gradients `up` and the saved inputs.
void first_order_only(const char* who, const variable_list& up, const variable_list& saved) {
  if (at::GradMode::is_enabled())
    throw std::runtime_error(text(who, " has no second derivative: call backward without create_graph"));
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const variable_list* v : {&up, &saved})
    for (const Tensor& t : *v)
      if (t.defined() && t._fw_grad(/*level=*/0).defined())
        throw std::runtime_error(text(who, " has no second derivative: its backward takes no forward-mode tangents"));
}
// dy as the kernels read it; zeros when only the final state was used
Tensor upstream(const Tensor& dy, const Tensor& x) {
  return dy.defined() ? rows(dy) : at::zeros(x.sizes(), x.options());
}

// --------------------------------------------------------------- layer norm
Tensor norm_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
  OnDevice on(x);
  const int64_t n = x.size(0), width = x.size(1);
  Tensor y = fresh({n, width}, x.scalar_type(), x);
  if (stats) *stats = fresh({n, 2}, at::kFloat, x);
  check(api.layer_norm(n, (int)width, dtype_code(x.scalar_type()), ptr(x), x.stride(0), fptr(w), fptr(b), (float)eps,
                       ptr(y), stats ? fptr(*stats) : nullptr, x.get_device(), stream_of(x)),
        "boa_layer_norm");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opt& b_, double eps) {
    const Tensor b = val(b_);
    Tensor stats, y = norm_forward(x, w, b, eps, &stats);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["bias"] = b.defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const variable_list s = ctx->get_saved_variables();
    first_order_only("layer_norm", up, s);
    const Tensor &x = s[0], &w = s[1], &stats = s[2];
    OnDevice on(x);
    const Tensor dy = rows(up[0]);
    const int64_t n = x.size(0), width = x.size(1);
    const int kind = dtype_code(x.scalar_type());
    Tensor dx = like(x), dw = like(w), db = ctx->saved_data["bias"].toBool() ? like(w) : Tensor();
    const size_t need = api.layer_norm_workspace_bytes(n, (int)width, kind);
    Tensor ws = bytes(need, x);
    check(api.layer_norm_backward(n, (int)width, kind, ptr(x), x.stride(0), ptr(dy), dy.stride(0), fptr(w), fptr(stats),
                                  ptr(dx), fptr(dw), fptr(db), ptr(ws), need, x.get_device(), stream_of(x)),
          "boa_layer_norm_backward");
    return {dx, dw, db, Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps) {
  const char* who = "layer_norm";
  check_kind(who, x);
  if (x.dim() < 1 || x.size(-1) < 1)
    refuse(text(who, ": x needs a last axis of at least one element, got shape ", x.sizes()));
  const int64_t width = x.size(-1);
  check_shape(who, "weight", weight, {width});
  if (bias.defined()) check_shape(who, "bias", bias, {width});
  no_tracing(who);
  reverse_mode_only(who, {&x, &weight, &bias});
  check_device(who, x, {&weight, &bias});
  const Tensor w = param(weight), b = param(bias);
  const Tensor flat = rows(x.dim() == 2 ? x : x.reshape({-1, width}));
  const Tensor y = wants_grad({&x, &w, &b}) ? LayerNorm::apply(flat, w, opt(b), eps) : norm_forward(flat, w, b, eps, nullptr);
  return x.dim() == 2 ? y : y.view(x.sizes());
}

// ------------------------------------------------------- causal convolution
boa_conv_args conv_args(const Tensor& x, const Tensor& w, const Tensor& b, bool silu, const Tensor& state,
                        const Tensor& lens) {
  boa_conv_args a{};
  a.dtype = dtype_code(x.scalar_type());
  a.batch = (int)x.size(0);
  a.channels = (int)x.size(-1);
  a.width = (int)w.size(1);
  a.silu = silu;
  a.device = x.get_device();
  a.x = ptr(x);
  a.x_bs = x.stride(0);
  if (x.dim() == 3) {
    a.length = (int)x.size(1);
    a.x_ts = x.stride(1);
  }
  a.weight = fptr(w);
  a.bias = fptr(b);
  a.state = ptr(state);
  a.lens = static_cast<const int32_t*>(ptr(lens));
  return a;
}

variable_list conv_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& state, const Tensor& lens,
                           bool silu, bool return_state) {
  OnDevice on(x);
  Tensor y = like(x), out;
  if (return_state) out = fresh({x.size(0), w.size(1) - 1, x.size(2)}, x.scalar_type(), x);
  boa_conv_args a = conv_args(x, w, b, silu, state, lens);
  a.y = ptr(y);
  a.state_out = ptr(out);
  check(api.causal_conv(&a, stream_of(x)), "boa_causal_conv");
  return return_state ? variable_list{y, out} : variable_list{y};
}

struct CausalConv : torch::autograd::Function<CausalConv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opt& b_,
                               const Opt& state_, const Opt& lens_, bool silu, bool return_state) {
    const Tensor b = val(b_), state = val(state_), lens = val(lens_);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, b, state, lens});
    ctx->saved_data["silu"] = silu;
    return conv_forward(x, w, b, state, lens, silu, return_state);
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const variable_list s = ctx->get_saved_variables();
    first_order_only("causal_conv", up, s);
    const Tensor &x = s[0], &w = s[1], &b = s[2], &state = s[3];
    OnDevice on(x);
    boa_conv_args a = conv_args(x, w, b, ctx->saved_data["silu"].toBool(), state, s[4]);
    const Tensor dy = upstream(up[0], x);
    const Tensor dout = up.size() > 1 && up[1].defined() ? whole(up[1]) : Tensor();
    Tensor dx = like(x), dw = like(w), db = like(b), ds = like(state);
    a.dy = ptr(dy);
    a.dy_bs = dy.stride(0);
    a.dy_ts = dy.stride(1);
    a.dstate_out = ptr(dout);
    a.dx = ptr(dx);
    a.dweight = fptr(dw);
    a.dbias = fptr(db);
    a.dstate = ptr(ds);
    a.workspace_bytes = api.causal_conv_workspace_bytes(&a);
    Tensor ws = bytes(a.workspace_bytes, x);
    a.workspace = ptr(ws);
    check(api.causal_conv_backward(&a, stream_of(x)), "boa_causal_conv_backward");
    return {dx, dw, db, ds, Tensor(), Tensor(), Tensor()};
  }
};

Tensor conv_weight(const char* who, const Tensor& weight, int64_t channels) {
  Tensor w = weight;
  if (w.dim() == 3 && w.size(1) == 1) w = w.select(1, 0);     // nn.Conv1d(groups=channels).weight
  if (w.dim() != 2 || w.size(0) != channels || w.size(1) < 2 || w.size(1) > 4)
    refuse(text(who, ": weight must be [", channels, ", width] or [", channels,
                ", 1, width] with width 2, 3 or 4, got ", weight.sizes()));
  return w;
}

variable_list causal_conv(const Tensor& x_, const Tensor& weight, const Tensor& bias, bool silu, const Tensor& state_,
                          const Tensor& lens_, bool return_state) {
  const char* who = "causal_conv";
  check_kind(who, x_);
  if (x_.dim() != 3 || x_.size(2) < 1) refuse(text(who, ": x must be [batch, length, channels], got ", x_.sizes()));
  const int64_t n = x_.size(0), length = x_.size(1), e = x_.size(2);
  Tensor w = conv_weight(who, weight, e);
  if (bias.defined()) check_shape(who, "bias", bias, {e});
  if (state_.defined()) {
    check_shape(who, "state", state_, {n, w.size(1) - 1, e});
    check_same(who, "state", x_, state_);
  }
  const Tensor lens = int_lens(who, lens_, n, length);
  no_tracing(who);
  reverse_mode_only(who, {&x_, &weight, &bias, &state_});
  check_device(who, x_, {&w, &bias, &state_, &lens});
  w = param(w);
  const Tensor b = param(bias), x = rows(x_), state = whole(state_);
  if (wants_grad({&x, &w, &b, &state})) return CausalConv::apply(x, w, opt(b), opt(state), opt(lens), silu, return_state);
  return conv_forward(x, w, b, state, lens, silu, return_state);
}

Tensor causal_conv_step(const Tensor& x_, const Tensor& state, const Tensor& weight, const Tensor& bias, bool silu) {
  const char* who = "causal_conv_step";
  check_kind(who, x_);
  if (x_.dim() != 2 || x_.size(1) < 1) refuse(text(who, ": x must be [batch, channels], got ", x_.sizes()));
  const int64_t n = x_.size(0), e = x_.size(1);
  Tensor w = conv_weight(who, weight, e);
  if (bias.defined()) check_shape(who, "bias", bias, {e});
  check_shape(who, "state", state, {n, w.size(1) - 1, e});
  check_same(who, "state", x_, state);
  if (!state.is_contiguous() || state.is_neg()) refuse(text(who, ": state is updated in place and must be contiguous"));
  no_tracing(who);
  reverse_mode_only(who, {&x_, &state, &weight, &bias});
  check_device(who, x_, {&state, &w, &bias});
  if (wants_grad({&x_, &state, &w, &bias}))
    throw Refused{PyExc_RuntimeError,
                  text(who, " has no gradient: call it under torch.no_grad(), or use causal_conv")};
  w = apart(param(w), state);
  const Tensor b = apart(param(bias), state), x = apart(rows(x_), state);
  OnDevice on(x);
  Tensor y = like(x);
  boa_conv_args a = conv_args(x, w, b, silu, Tensor(), Tensor());
  a.y = ptr(y);
  a.state_out = ptr(state);
  state.unsafeGetTensorImpl()->bump_version();
  check(api.causal_conv_step(&a, stream_of(x)), "boa_causal_conv_step");
  return y;
}

// --------------------------------------------- selective state space scan
struct SsmIn {
  Tensor x, dt, A, B, C, D, z, bias, state, lens;
};

boa_ssm_args ssm_args(const SsmIn& i, bool softplus) {
  boa_ssm_args a{};
  const Tensor& x = i.x;
  a.dtype = dtype_code(x.scalar_type());
  a.batch = (int)x.size(0);
  a.channels = (int)x.size(-1);
  a.states = (int)i.A.size(1);
  a.softplus = softplus;
  a.device = x.get_device();
  a.x = ptr(x);
  a.dt = ptr(i.dt);
  a.z = ptr(i.z);
  a.B = ptr(i.B);
  a.C = ptr(i.C);
  a.x_bs = x.stride(0);
  a.dt_bs = i.dt.stride(0);
  a.B_bs = i.B.stride(0);
  a.C_bs = i.C.stride(0);
  if (i.z.defined()) a.z_bs = i.z.stride(0);
  if (x.dim() == 3) {
    a.length = (int)x.size(1);
    a.x_ts = x.stride(1);
    a.dt_ts = i.dt.stride(1);
    a.B_ts = i.B.stride(1);
    a.C_ts = i.C.stride(1);
    if (i.z.defined()) a.z_ts = i.z.stride(1);
  }
  a.A = fptr(i.A);
  a.D = fptr(i.D);
  a.dt_bias = fptr(i.bias);
  a.state = fptr(i.state);
  a.lens = static_cast<const int32_t*>(ptr(i.lens));
  return a;
}

variable_list ssm_forward(const SsmIn& i, bool softplus, bool return_state, Tensor* checkpoints) {
  const Tensor& x = i.x;
  OnDevice on(x);
  boa_ssm_args a = ssm_args(i, softplus);
  Tensor y = like(x), out;
  if (return_state) out = fresh({x.size(0), x.size(2), kStates}, at::kFloat, x);
  if (checkpoints) *checkpoints = bytes(api.ssm_checkpoint_bytes(&a), x);
  a.workspace_bytes = api.ssm_workspace_bytes(&a, 0);
  Tensor ws = bytes(a.workspace_bytes, x);
  a.y = ptr(y);
  a.state_out = fptr(out);
  a.checkpoints = checkpoints ? fptr(*checkpoints) : nullptr;
  a.workspace = ptr(ws);
  check(api.ssm_scan(&a, stream_of(x)), "boa_ssm_scan");
  return return_state ? variable_list{y, out} : variable_list{y};
}

struct SsmScan : torch::autograd::Function<SsmScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A,
                               const Tensor& B, const Tensor& C, const Opt& D_, const Opt& z_, const Opt& bias_,
                               const Opt& state_, const Opt& lens_, bool softplus, bool return_state) {
    ctx->set_materialize_grads(false);
    const Tensor D = val(D_), z = val(z_), bias = val(bias_), state = val(state_), lens = val(lens_);
    Tensor checkpoints;
    variable_list out = ssm_forward({x, dt, A, B, C, D, z, bias, state, lens}, softplus, return_state, &checkpoints);
    ctx->save_for_backward({x, dt, A, B, C, D, z, bias, state, lens, checkpoints});
    ctx->saved_data["softplus"] = softplus;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const variable_list s = ctx->get_saved_variables();
    first_order_only("ssm_scan", up, s);
    const SsmIn i{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9]};
    const Tensor& x = i.x;
    OnDevice on(x);
    boa_ssm_args a = ssm_args(i, ctx->saved_data["softplus"].toBool());
    const Tensor dy = upstream(up[0], x);
    const Tensor dout = up.size() > 1 && up[1].defined() ? whole(up[1]) : Tensor();
    Tensor dx = like(x), ddt = like(i.dt), dA = like(i.A), dB = like(i.B), dC = like(i.C), dD = like(i.D),
           dz = like(i.z), dbias = like(i.bias), ds = like(i.state);
    a.checkpoints = fptr(s[10]);
    a.dy = ptr(dy);
    a.dy_bs = dy.stride(0);
    a.dy_ts = dy.stride(1);
    a.dstate_out = fptr(dout);
    a.dx = ptr(dx);
    a.ddt = ptr(ddt);
    a.dz = ptr(dz);
    a.dB = ptr(dB);
    a.dC = ptr(dC);
    a.dA = fptr(dA);
    a.dD = fptr(dD);
    a.ddt_bias = fptr(dbias);
    a.dstate = fptr(ds);
    a.workspace_bytes = api.ssm_workspace_bytes(&a, 1);
    Tensor ws = bytes(a.workspace_bytes, x);
    a.workspace = ptr(ws);
    check(api.ssm_scan_backward(&a, stream_of(x)), "boa_ssm_scan_backward");
    return {dx, ddt, dA, dB, dC, dD, dz, dbias, ds, Tensor(), Tensor(), Tensor()};
  }
};

void ssm_check(const char* who, const SsmIn& i, int64_t dims) {
  const Tensor& x = i.x;
  check_kind(who, x);
  if (x.dim() != dims || x.size(-1) < 1)
    refuse(text(who, ": x must be [batch, ", dims == 3 ? "length, " : "", "channels], got ", x.sizes()));
  const int64_t e = x.size(-1);
  check_shape(who, "dt", i.dt, x.sizes());
  check_shape(who, "A", i.A, {e, kStates});
  std::vector<int64_t> bc(x.sizes().begin(), x.sizes().end());
  bc.back() = kStates;
  check_shape(who, "B", i.B, bc);
  check_shape(who, "C", i.C, bc);
  if (i.D.defined()) check_shape(who, "D", i.D, {e});
  if (i.bias.defined()) check_shape(who, "dt_bias", i.bias, {e});
  if (i.z.defined()) {
    check_shape(who, "z", i.z, x.sizes());
    check_same(who, "z", x, i.z);
  }
  check_same(who, "dt", x, i.dt);
  check_same(who, "B", x, i.B);
  check_same(who, "C", x, i.C);
  if (i.state.defined()) {
    check_shape(who, "state", i.state, {x.size(0), e, kStates});
    if (i.state.scalar_type() != at::kFloat)
      refuse(text(who, ": state must be float32, not ", i.state.scalar_type()));
  }
}

void ssm_prepare(SsmIn& i) {
  i.A = param(i.A);
  i.D = param(i.D);
  i.bias = param(i.bias);
  i.x = rows(i.x);
  i.dt = rows(i.dt);
  i.B = rows(i.B);
  i.C = rows(i.C);
  i.z = rows(i.z);
}

variable_list ssm_scan(SsmIn i, bool softplus, bool return_state) {
  const char* who = "ssm_scan";
  ssm_check(who, i, 3);
  i.lens = int_lens(who, i.lens, i.x.size(0), i.x.size(1));
  no_tracing(who);
  reverse_mode_only(who, {&i.x, &i.dt, &i.A, &i.B, &i.C, &i.D, &i.z, &i.bias, &i.state});
  check_device(who, i.x, {&i.dt, &i.A, &i.B, &i.C, &i.D, &i.z, &i.bias, &i.state, &i.lens});
  ssm_prepare(i);
  i.state = param(i.state);
  if (wants_grad({&i.x, &i.dt, &i.A, &i.B, &i.C, &i.D, &i.z, &i.bias, &i.state}))
    return SsmScan::apply(i.x, i.dt, i.A, i.B, i.C, opt(i.D), opt(i.z), opt(i.bias), opt(i.state), opt(i.lens), softplus,
                          return_state);
  return ssm_forward(i, softplus, return_state, nullptr);
}

Tensor ssm_step(SsmIn i, bool softplus) {
  const char* who = "ssm_step";
  ssm_check(who, i, 2);
  if (!i.state.is_contiguous() || i.state.is_neg() || misaligned(i.state))
    refuse(text(who, ": state is updated in place and must be contiguous and 16-byte aligned"));
  no_tracing(who);
  reverse_mode_only(who, {&i.x, &i.dt, &i.state, &i.A, &i.B, &i.C, &i.D, &i.z, &i.bias});
  check_device(who, i.x, {&i.dt, &i.state, &i.A, &i.B, &i.C, &i.D, &i.z, &i.bias});
  if (wants_grad({&i.x, &i.dt, &i.state, &i.A, &i.B, &i.C, &i.D, &i.z, &i.bias}))
    throw Refused{PyExc_RuntimeError, text(who, " has no gradient: call it under torch.no_grad(), or use ssm_scan")};
  ssm_prepare(i);
  for (Tensor* t : {&i.x, &i.dt, &i.A, &i.B, &i.C, &i.D, &i.z, &i.bias}) *t = apart(*t, i.state);
  OnDevice on(i.x);
  Tensor y = like(i.x);
  boa_ssm_args a = ssm_args(i, softplus);
  a.state = nullptr;
  a.y = ptr(y);
  a.state_out = fptr(i.state);
  i.state.unsafeGetTensorImpl()->bump_version();
  check(api.ssm_step(&a, stream_of(i.x)), "boa_ssm_step");
  return y;
}

// ------------------------------------------------------------------- Python
const Tensor& arg(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
    throw PythonError{};
  }
  return THPVariable_Unpack(o);
}
Tensor maybe(PyObject* o, const char* name) { return o == Py_None ? Tensor() : arg(o, name); }
bool flag(PyObject* o) {
  const int r = PyObject_IsTrue(o);
  if (r < 0) throw PythonError{};
  return r;
}
PyObject* give(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* give(const variable_list& v) {
  if (v.size() == 1) return THPVariable_Wrap(v[0]);
  PyObject* r = PyTuple_New((Py_ssize_t)v.size());
  for (size_t i = 0; r && i < v.size(); ++i) PyTuple_SET_ITEM(r, (Py_ssize_t)i, THPVariable_Wrap(v[i]));
  return r;
}

// Runs f() and turns its C++ exceptions into Python ones.
template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F f) {
  HANDLE_TH_ERRORS
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "_boa_ops: %zd arguments, %zd wanted", got, want);
    return nullptr;
  }
  try {
    need_api();
    return give(f());
  } catch (const PythonError&) {
    return nullptr;
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  } catch (const Failed& e) {
    if (PyObject* v = PyObject_CallFunction(boa_error, "is", e.code, e.plain.c_str())) {
      PyErr_SetObject(boa_error, v);
      Py_DECREF(v);
    }
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&] {
    const double eps = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) throw PythonError{};
    return layer_norm(arg(a[0], "x"), arg(a[1], "weight"), maybe(a[2], "bias"), eps);
  });
}
PyObject* py_causal_conv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&] {
    return causal_conv(arg(a[0], "x"), arg(a[1], "weight"), maybe(a[2], "bias"), flag(a[3]), maybe(a[4], "state"),
                       maybe(a[5], "lens"), flag(a[6]));
  });
}
PyObject* py_causal_conv_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&] {
    return causal_conv_step(arg(a[0], "x"), arg(a[1], "state"), arg(a[2], "weight"), maybe(a[3], "bias"), flag(a[4]));
  });
}
PyObject* py_ssm_scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 12, [&] {
    return ssm_scan({arg(a[0], "x"), arg(a[1], "dt"), arg(a[2], "A"), arg(a[3], "B"), arg(a[4], "C"), maybe(a[5], "D"),
                     maybe(a[6], "z"), maybe(a[7], "dt_bias"), maybe(a[9], "state"), maybe(a[10], "lens")},
                    flag(a[8]), flag(a[11]));
  });
}
PyObject* py_ssm_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 10, [&] {
    return ssm_step({arg(a[0], "x"), arg(a[1], "dt"), arg(a[3], "A"), arg(a[4], "B"), arg(a[5], "C"),
                     maybe(a[6], "D"), maybe(a[7], "z"), maybe(a[8], "dt_bias"), arg(a[2], "state"), Tensor()},
                    flag(a[9]));
  });
}
// held_on_default_stream(parameters): whether an autograd graph that is still alive would accumulate into one of them on
// its device's default stream, which cannot take part in a capture.
PyObject* py_held(PyObject*, PyObject* list) {
  HANDLE_TH_ERRORS
  PyObject* seq = PySequence_Fast(list, "a sequence of tensors");
  if (!seq) return nullptr;
  bool held = false;
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq) && !held; ++i) {
    PyObject* o = PySequence_Fast_GET_ITEM(seq, i);
    if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) continue;
    const Tensor& t = THPVariable_Unpack(o);
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = node ? node->stream() : std::nullopt;
    held = stream && *stream == c10::cuda::getDefaultCUDAStream(t.get_device()).unwrap();
  }
  Py_DECREF(seq);
  return PyBool_FromLong(held);
  END_HANDLE_TH_ERRORS
}
// bind(loader, BoaError)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "bind(loader, error)");
    return nullptr;
  }
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  Py_XDECREF(loader);
  Py_XDECREF(boa_error);
  loader = a[0];
  boa_error = a[1];
  api.ready = false;
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"bind", fast(py_bind), METH_FASTCALL, "the entry points' loader and the error class"},
    {"layer_norm", fast(py_layer_norm), METH_FASTCALL, "x, weight, bias, eps"},
    {"causal_conv", fast(py_causal_conv), METH_FASTCALL, "x, weight, bias, silu, state, lens, return_state"},
    {"causal_conv_step", fast(py_causal_conv_step), METH_FASTCALL, "x, state, weight, bias, silu"},
    {"ssm_scan", fast(py_ssm_scan), METH_FASTCALL, "x, dt, A, B, C, D, z, dt_bias, softplus, state, lens, return_state"},
    {"ssm_step", fast(py_ssm_step), METH_FASTCALL, "x, dt, state, A, B, C, D, z, dt_bias, softplus"},
    {"held_on_default_stream", py_held, METH_O, "parameters"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_boa_ops", "host side of boa_b200.ops", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__boa_ops(void) { return PyModule_Create(&module); }
