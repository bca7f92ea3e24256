// binding.cpp -- libafc_ops.so for torch tensors on a GPU (module _ops_torch, behind rlfluidcontrol_amd.ops): checks, outputs and
// workspaces from torch's allocator, the current stream of the tensors' device, and the backward passes as autograd functions.
// In C++ because the calls are short: at the sizes of the learner the kernels of a training step take some 40 us, and the same
// work in Python took 240.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../../include/afc_ops.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct OpsFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};
py::object *g_error_class = nullptr;

void ok(int rc) {
  if (rc != AFC_OK) throw OpsFailure(std::string(afc_ops_last_error()) + " (" + std::to_string(rc) + ")");
}

void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

int dtype_of(const Tensor &t) { return t.scalar_type() == at::kFloat ? AFC_F32 : t.scalar_type() == at::kBFloat16 ? AFC_BF16 : AFC_F16; }
bool known(const Tensor &t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

// ---- checks: ValueError with the same rules as the Python side has for tensors on the CPU ----
void tensor(const char *name, const Tensor &t, at::IntArrayRef shape, at::ScalarType dtype, const at::Device &device) {
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " has shape ", t.sizes(), ", expected ", shape);
  TORCH_CHECK_VALUE(t.scalar_type() == dtype, name, " is ", t.scalar_type(), ", expected ", dtype);
  TORCH_CHECK_VALUE(t.device() == device, name, " is on ", t.device(), ", expected ", device);
  TORCH_CHECK_VALUE(t.layout() == at::kStrided, name, " must be a strided tensor");
}
void sequence(const char *name, const Tensor &t, at::IntArrayRef shape, at::ScalarType dtype, const at::Device &device) {
  tensor(name, t, shape, dtype, device);
  TORCH_CHECK_VALUE(t.size(-1) <= 1 || t.stride(-1) == 1 || t.numel() == 0, name, " must be contiguous along its last axis");
}
void optional(const char *name, const Maybe &t, at::IntArrayRef shape, at::ScalarType dtype, const at::Device &device) {
  if (t) tensor(name, *t, shape, dtype, device);
}
void input(const Tensor &x, int dims) {
  TORCH_CHECK_VALUE(x.dim() == dims, "x must have ", dims, " axes, it has ", x.dim());
  TORCH_CHECK_VALUE(known(x), "x is ", x.scalar_type(), ": float32, bfloat16 or float16 is expected");
  TORCH_CHECK_VALUE(x.is_cuda(), "x is on ", x.device(), ": a GPU is expected");
  TORCH_CHECK_VALUE(x.size(-1) >= 1, "x has no channels");
}
bool wants(const Tensor &t) { return t.defined() && t.requires_grad(); }
bool wants(const Maybe &t) { return t && t->requires_grad(); }
template <class... T>
bool wants_grad(const T &...t) {
  return at::GradMode::is_enabled() && (wants(t) || ...);
}
// which of a function's tensor arguments want a gradient, as bits in their order (the edges of a node leave out what is not given)
template <class... T>
int64_t wanted(const T &...t) {
  int64_t bits = 0, bit = 1;
  ((bits |= wants(t) ? bit : 0, bit <<= 1), ...);
  return bits;
}
template <class... T>
void no_grad(const T &...t) {
  TORCH_CHECK_VALUE(!wants_grad(t...), "a step has no gradient: call it under torch.no_grad(), or the whole-sequence form");
}

Tensor value(const Maybe &t) { return t ? *t : Tensor(); }
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }

// A kernel knows nothing of forward-mode derivatives: what it writes would have none, which PyTorch takes for zero.
bool has_tangent(const Tensor &t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const Maybe &t) { return t && has_tangent(*t); }
// Nor does a tracer see it: torch.jit.trace and make_fx would record the allocation of an output and not what fills it.
void not_traced() {
  const bool traced = torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() ||
                      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch);
  TORCH_CHECK_NOT_IMPLEMENTED(!traced, "these operators cannot be traced on a GPU: a tracer sees their outputs' memory and not what fills it");
}
// x.conj().imag and the like are views whose sign is applied when PyTorch reads them; the memory has the other one
bool is_negated(const Tensor &t) { return t.defined() && t.is_neg(); }
bool is_negated(const Maybe &t) { return t && is_negated(*t); }
template <class... T>
void as_stored(const T &...t) {
  TORCH_CHECK_VALUE(!(is_negated(t) || ...), "a tensor is a view that negates its memory (resolve_neg() gives a plain one)");
}
template <class... T>
void no_tangent(const T &...t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(t) || ...), "these operators have no forward-mode derivative on a GPU (a tensor carries a tangent)");
}

// the bytes from a tensor's first element to its last
struct Span {
  uintptr_t from, to;
  explicit Span(const Tensor &t) : from((uintptr_t)t.data_ptr()), to(from) {
    if (t.numel() == 0) return;
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    to += (uintptr_t)(last + 1) * t.element_size();
  }
};
// a state that is updated in place is read and written by many threads at once
void own_memory(const Tensor &state, const char *name, const Tensor &t) {
  if (!t.defined()) return;
  const Span a(state), b(t);
  TORCH_CHECK_VALUE(a.from == a.to || b.from == b.to || a.to <= b.from || b.to <= a.from, "state shares memory with ", name);
}
// what a kernel has written behind autograd's back: a graph that saved the old values refuses to use them
void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor dense(const Tensor &t) { return t.defined() ? t.resolve_neg().contiguous() : t; }
Tensor dense(const Maybe &t) { return t ? dense(*t) : Tensor(); }
Tensor last_contiguous(const Tensor &t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t.resolve_neg() : dense(t); }
template <class T = void>
T *ptr(const Tensor &t) {
  return t.defined() ? (T *)t.data_ptr() : nullptr;
}
afc_seq seq(const Tensor &t) {
  afc_seq s = {};
  if (!t.defined()) return s;
  s.data = t.data_ptr();
  s.stride_batch = t.stride(0);
  if (t.dim() > 2) s.stride_length = t.stride(1);
  if (t.dim() > 3) s.stride_group = t.stride(2);
  return s;
}
afc_seq token(const Tensor &t) {  // [batch, width] or [batch, groups, state]
  afc_seq s = {};
  if (!t.defined()) return s;
  s.data = t.data_ptr();
  s.stride_batch = t.stride(0);
  if (t.dim() > 2) s.stride_group = t.stride(1);
  return s;
}
Tensor fresh(const Tensor &like) { return at::empty(like.sizes(), like.options()); }
Tensor fresh_if(const Tensor &like, bool wanted) { return like.defined() && wanted ? fresh(like) : Tensor(); }
Tensor space(const Tensor &x, uint64_t bytes) { return at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)); }

void first_order_only(const Tensor &dy, const Tensor &dlast) {
  not_traced();
  no_tangent(dy, dlast);
  TORCH_CHECK(!at::GradMode::is_enabled(), "the gradients of these operators have no gradient of their own (create_graph=True)");
}

// ---- convolution ----
void check_filter(const Tensor &weight, const Maybe &bias, int64_t width, const at::Device &device) {
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) >= 2 && weight.size(1) <= 4, "weight must be [width, taps] with 2 to 4 taps, it is ", weight.sizes());
  tensor("weight", weight, {width, weight.size(1)}, at::kFloat, device);
  optional("bias", bias, {width}, at::kFloat, device);
}

afc_conv_args conv_args(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &state, const Tensor &lengths, bool silu) {
  afc_conv_args p = {};
  p.device = x.device().index();
  p.dtype = dtype_of(x);
  p.taps = (int)weight.size(1);
  p.silu = silu;
  p.batch = x.size(0), p.length = x.size(1), p.width = x.size(2);
  p.x = seq(x);
  p.weight = ptr<float>(weight), p.bias = ptr<float>(bias);
  p.initial_state = ptr(state), p.lengths = ptr<int32_t>(lengths);
  return p;
}

void check_conv(const Tensor &x, const Tensor &weight, const Maybe &bias, const Maybe &state, const Maybe &lengths) {
  sequence("x", x, x.sizes(), x.scalar_type(), x.device());
  check_filter(weight, bias, x.size(2), x.device());
  optional("initial_state", state, {x.size(0), weight.size(1) - 1, x.size(2)}, x.scalar_type(), x.device());
  optional("lengths", lengths, {x.size(0)}, at::kInt, x.device());
}

variable_list conv_forward(const Tensor &x, const Tensor &weight, const Tensor &bias, const Tensor &state, const Tensor &lengths, bool silu, bool want_last) {
  Tensor y = at::empty(x.sizes(), x.options()), last;
  afc_conv_args p = conv_args(x, weight, bias, state, lengths, silu);
  p.y = seq(y);
  if (want_last) {
    last = at::empty({x.size(0), weight.size(1) - 1, x.size(2)}, x.options());
    p.final_state = ptr(last);
  }
  ok(afc_conv(&p, stream_of(x)));
  return want_last ? variable_list{y, last} : variable_list{y};
}

struct Conv : torch::autograd::Function<Conv> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const Maybe &bias, const Maybe &state, const Maybe &lengths, bool silu,
                               bool want_last) {
    const Tensor w = dense(weight), b = dense(bias), s = dense(state), n = dense(lengths);
    ctx->save_for_backward({x, w, b, s, n});
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["wanted"] = wanted(x, weight, bias, state);
    ctx->set_materialize_grads(false);
    return conv_forward(x, w, b, s, n, silu, want_last);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(7);
    Tensor dy = grads[0], dlast = grads.size() > 1 ? grads[1] : Tensor();
    first_order_only(dy, dlast);
    if (!dy.defined() && !dlast.defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], weight = dense(saved[1]), bias = dense(saved[2]), state = dense(saved[3]), lengths = dense(saved[4]);
    // (hooks of saved tensors may hand back others than they were given)
    input(x, 3);
    as_stored(x);
    check_conv(x, weight, maybe(bias), maybe(state), maybe(lengths));
    dy = dy.defined() ? last_contiguous(dy) : at::zeros(x.sizes(), x.options());
    if (dlast.defined()) dlast = dense(dlast);
    tensor("the adjoint of y", dy, x.sizes(), x.scalar_type(), x.device());
    optional("the adjoint of the final state", maybe(dlast), {x.size(0), weight.size(1) - 1, x.size(2)}, x.scalar_type(), x.device());
    const int64_t need = ctx->saved_data["wanted"].toInt();
    const Tensor dx = fresh(x), dw = fresh_if(weight, need & 2), db = fresh_if(bias, need & 4), ds = fresh_if(state, need & 8);
    afc_conv_args p = conv_args(x, weight, bias, state, lengths, ctx->saved_data["silu"].toBool());
    p.dy = seq(dy), p.dfinal_state = ptr(dlast), p.dx = seq(dx);
    p.dweight = ptr<float>(dw), p.dbias = ptr<float>(db), p.dinitial_state = ptr(ds);
    Tensor ws;
    if (dw.defined() || db.defined()) {
      ok(afc_conv_workspace(&p, &p.workspace_bytes));
      ws = space(x, p.workspace_bytes);
      p.workspace = ptr(ws);
    }
    ok(afc_conv_grad(&p, stream_of(x)));
    out[0] = dx, out[1] = dw, out[2] = db, out[3] = ds;
    return out;
  }
};

variable_list causal_conv(const Tensor &x, const Tensor &weight, const Maybe &bias, bool silu, const Maybe &state, const Maybe &lengths, bool want_last) {
  not_traced();
  no_tangent(x, weight, bias, state);
  as_stored(x);
  input(x, 3);
  check_conv(x, weight, bias, state, lengths);
  if (wants_grad(x, weight, bias, state)) return Conv::apply(x, weight, bias, state, lengths, silu, want_last);
  return conv_forward(x, dense(weight), dense(bias), dense(state), dense(lengths), silu, want_last);
}

Tensor causal_conv_step(const Tensor &x, const Tensor &state, const Tensor &weight, const Maybe &bias, bool silu) {
  not_traced();
  no_tangent(x, state, weight, bias);
  as_stored(x, state);
  input(x, 2);
  sequence("x", x, x.sizes(), x.scalar_type(), x.device());
  check_filter(weight, bias, x.size(1), x.device());
  tensor("state", state, {x.size(0), weight.size(1) - 1, x.size(1)}, x.scalar_type(), x.device());
  TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous");
  own_memory(state, "x", x), own_memory(state, "weight", weight), own_memory(state, "bias", value(bias));
  no_grad(x, state, weight, bias);
  const Tensor w = dense(weight), b = dense(bias), y = at::empty(x.sizes(), x.options());
  afc_conv_args p = {};
  p.device = x.device().index();
  p.dtype = dtype_of(x);
  p.taps = (int)w.size(1);
  p.silu = silu;
  p.batch = x.size(0), p.length = 1, p.width = x.size(1);
  p.x = token(x), p.y = token(y);
  p.weight = ptr<float>(w), p.bias = ptr<float>(b);
  p.initial_state = p.final_state = ptr(state);
  ok(afc_conv_step(&p, stream_of(x)));
  written(state);
  return y;
}

// ---- scan ----
struct ScanInputs {
  Tensor x, dt, A, B, C, D, z, dt_bias;
};

// B and C get an axis of groups where they have none; `rows`: the axes in front of width
void check_scan(ScanInputs &in) {
  const Tensor &x = in.x;
  const at::Device dev = x.device();
  const auto type = x.scalar_type();
  const int64_t lead = x.dim() - 1, W = x.size(-1);
  sequence("x", x, x.sizes(), type, dev);
  sequence("dt", in.dt, x.sizes(), type, dev);
  if (in.z.defined()) sequence("z", in.z, x.sizes(), type, dev);
  TORCH_CHECK_VALUE(in.A.dim() == 2 && in.A.size(1) >= 1 && in.A.size(1) <= 64, "A must be [width, state] with a state of 1 to 64, it is ", in.A.sizes());
  const int64_t N = in.A.size(1);
  tensor("A", in.A, {W, N}, at::kFloat, dev);
  if (in.D.defined()) tensor("D", in.D, {W}, at::kFloat, dev);
  if (in.dt_bias.defined()) tensor("dt_bias", in.dt_bias, {W}, at::kFloat, dev);
  for (Tensor *t : {&in.B, &in.C}) {
    TORCH_CHECK_VALUE(t->dim() == lead + 1 || t->dim() == lead + 2, t == &in.B ? "B" : "C", " must be [..., state] or [..., groups, state], it is ", t->sizes());
    if (t->dim() == lead + 1) *t = t->unsqueeze(-2);
  }
  const int64_t G = in.B.size(-2);
  TORCH_CHECK_VALUE(G >= 1 && W % G == 0, G, " groups do not divide the width ", W);
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
  shape.push_back(G), shape.push_back(N);
  sequence("B", in.B, shape, type, dev);
  sequence("C", in.C, shape, type, dev);
}

void check_scan_rows(const Tensor &x, const Tensor &A, const Maybe &state, const Maybe &lengths) {
  optional("initial_state", state, {x.size(0), x.size(2), A.size(1)}, at::kFloat, x.device());
  optional("lengths", lengths, {x.size(0)}, at::kInt, x.device());
}

afc_scan_args scan_args(const ScanInputs &in, const Tensor &state, const Tensor &lengths, bool softplus) {
  const Tensor &x = in.x;
  afc_scan_args p = {};
  p.device = x.device().index();
  p.dtype = dtype_of(x);
  p.softplus = softplus;
  p.state = (int)in.A.size(1);
  p.batch = x.size(0), p.length = x.size(1), p.width = x.size(2), p.groups = in.B.size(2);
  p.x = seq(x), p.dt = seq(in.dt), p.b = seq(in.B), p.c = seq(in.C), p.z = seq(in.z);
  p.a = ptr<float>(in.A), p.d = ptr<float>(in.D), p.dt_bias = ptr<float>(in.dt_bias);
  p.initial_state = ptr<float>(state), p.lengths = ptr<int32_t>(lengths);
  return p;
}

variable_list scan_forward(const ScanInputs &in, const Tensor &state, const Tensor &lengths, bool softplus, bool want_last, Tensor *checkpoints) {
  const Tensor &x = in.x;
  Tensor y = at::empty(x.sizes(), x.options()), last, ws;
  afc_scan_args p = scan_args(in, state, lengths, softplus);
  p.y = seq(y);
  if (want_last) {
    last = at::empty({x.size(0), x.size(2), in.A.size(1)}, x.options().dtype(at::kFloat));
    p.final_state = ptr<float>(last);
  }
  uint64_t kept, grad;
  ok(afc_scan_workspace(&p, &kept, &p.workspace_bytes, &grad));
  if (checkpoints) {
    *checkpoints = space(x, kept);
    p.checkpoints = ptr<float>(*checkpoints);
  }
  if (p.workspace_bytes) {
    ws = space(x, p.workspace_bytes);
    p.workspace = ptr(ws);
  }
  ok(afc_scan(&p, stream_of(x)));
  return want_last ? variable_list{y, last} : variable_list{y};
}

struct Scan : torch::autograd::Function<Scan> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Maybe &D, const Maybe &z,
                               const Maybe &dt_bias, const Maybe &state, const Maybe &lengths, bool softplus, bool want_last) {
    const ScanInputs in = {x, dt, dense(A), B, C, dense(D), value(z), dense(dt_bias)};
    const Tensor s = dense(state), n = dense(lengths);
    Tensor checkpoints;
    variable_list out = scan_forward(in, s, n, softplus, want_last, &checkpoints);
    ctx->save_for_backward({in.x, in.dt, in.A, in.B, in.C, in.D, in.z, in.dt_bias, s, n, checkpoints});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["wanted"] = wanted(x, dt, A, B, C, D, z, dt_bias, state);
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list out(12);
    Tensor dy = grads[0], dlast = grads.size() > 1 ? grads[1] : Tensor();
    first_order_only(dy, dlast);
    if (!dy.defined() && !dlast.defined()) return out;
    const variable_list v = ctx->get_saved_variables();
    ScanInputs in = {v[0], v[1], dense(v[2]), v[3], v[4], dense(v[5]), v[6], dense(v[7])};
    const Tensor &x = in.x, state = dense(v[8]), lengths = dense(v[9]), checkpoints = dense(v[10]);
    input(x, 3);
    as_stored(x, in.dt, in.B, in.C, in.z);
    check_scan(in);
    check_scan_rows(x, in.A, maybe(state), maybe(lengths));
    dy = dy.defined() ? last_contiguous(dy) : at::zeros(x.sizes(), x.options());
    if (dlast.defined()) dlast = dense(dlast);
    tensor("the adjoint of y", dy, x.sizes(), x.scalar_type(), x.device());
    optional("the adjoint of the final state", maybe(dlast), {x.size(0), x.size(2), in.A.size(1)}, at::kFloat, x.device());
    out[0] = fresh(x), out[1] = fresh(in.dt), out[3] = fresh(in.B), out[4] = fresh(in.C);
    const int64_t need = ctx->saved_data["wanted"].toInt();
    out[2] = fresh_if(in.A, need & 4), out[5] = fresh_if(in.D, need & 32), out[6] = fresh_if(in.z, need & 64);
    out[7] = fresh_if(in.dt_bias, need & 128), out[8] = fresh_if(state, need & 256);
    afc_scan_args p = scan_args(in, state, lengths, ctx->saved_data["softplus"].toBool());
    p.checkpoints = ptr<float>(checkpoints);
    p.dy = seq(dy), p.dfinal_state = ptr<float>(dlast);
    p.dx = seq(out[0]), p.ddt = seq(out[1]), p.db = seq(out[3]), p.dc = seq(out[4]), p.dz = seq(out[6]);
    p.da = ptr<float>(out[2]), p.dd = ptr<float>(out[5]), p.ddt_bias = ptr<float>(out[7]), p.dinitial_state = ptr<float>(out[8]);
    uint64_t kept, scan;
    ok(afc_scan_workspace(&p, &kept, &scan, &p.workspace_bytes));
    tensor("the states of the forward pass", checkpoints, {(int64_t)kept}, at::kByte, x.device());
    const Tensor ws = space(x, p.workspace_bytes);
    p.workspace = ptr(ws);
    ok(afc_scan_grad(&p, stream_of(x)));
    return out;
  }
};

variable_list selective_scan(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Maybe &D, const Maybe &z, const Maybe &dt_bias,
                             bool softplus, const Maybe &state, const Maybe &lengths, bool want_last) {
  not_traced();
  no_tangent(x, dt, A, B, C, D, z, dt_bias, state);
  as_stored(x, dt, B, C, z);
  input(x, 3);
  ScanInputs in = {x, dt, A, B, C, value(D), value(z), value(dt_bias)};
  check_scan(in);
  check_scan_rows(x, A, state, lengths);
  if (wants_grad(x, dt, A, B, C, D, z, dt_bias, state)) return Scan::apply(x, dt, A, in.B, in.C, D, z, dt_bias, state, lengths, softplus, want_last);
  in.A = dense(in.A), in.D = dense(D), in.dt_bias = dense(dt_bias);
  return scan_forward(in, dense(state), dense(lengths), softplus, want_last, nullptr);
}

Tensor selective_scan_step(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Tensor &state, const Maybe &D, const Maybe &z,
                           const Maybe &dt_bias, bool softplus) {
  not_traced();
  no_tangent(x, dt, A, B, C, state, D, z, dt_bias);
  as_stored(x, dt, B, C, state, z);
  input(x, 2);
  ScanInputs in = {x, dt, A, B, C, value(D), value(z), value(dt_bias)};
  check_scan(in);
  tensor("state", state, {x.size(0), x.size(1), A.size(1)}, at::kFloat, x.device());
  TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous");
  own_memory(state, "x", x), own_memory(state, "dt", dt), own_memory(state, "B", in.B), own_memory(state, "C", in.C), own_memory(state, "z", in.z);
  own_memory(state, "A", A), own_memory(state, "D", in.D), own_memory(state, "dt_bias", in.dt_bias);
  no_grad(x, dt, A, B, C, state, D, z, dt_bias);
  const Tensor a = dense(A), d = dense(D), bias = dense(dt_bias), y = at::empty(x.sizes(), x.options());
  afc_scan_args p = {};
  p.device = x.device().index();
  p.dtype = dtype_of(x);
  p.softplus = softplus;
  p.state = (int)a.size(1);
  p.batch = x.size(0), p.length = 1, p.width = x.size(1), p.groups = in.B.size(1);
  p.x = token(x), p.dt = token(dt), p.b = token(in.B), p.c = token(in.C), p.z = token(in.z), p.y = token(y);
  p.a = ptr<float>(a), p.d = ptr<float>(d), p.dt_bias = ptr<float>(bias);
  p.initial_state = p.final_state = ptr<float>(state);
  ok(afc_scan_step(&p, stream_of(x)));
  written(state);
  return y;
}

// ---- gradient norm ----
bool without_gaps(const Tensor &t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

// max_norm < 0: only the norm
Tensor clip(const std::vector<Tensor> &grads, double max_norm, const std::optional<std::vector<Tensor>> &out) {
  const bool scale = max_norm >= 0;
  const size_t n = grads.size();
  not_traced();
  for (const Tensor &g : grads) no_tangent(g), as_stored(g);
  if (out)
    for (const Tensor &o : *out) no_tangent(o), as_stored(o);
  TORCH_CHECK_VALUE(n > 0 && (!out || out->size() == n), "out has another number of tensors than grads");
  const at::Device dev = grads[0].device();
  TORCH_CHECK_VALUE(dev.is_cuda(), "gradients are on ", dev, ": a GPU is expected");
  std::vector<void *> in(n), to(n);
  std::vector<int64_t> numel(n);
  std::vector<int32_t> in_dtype(n), out_dtype(n);
  auto check = [&](const Tensor &g) {
    TORCH_CHECK_VALUE(known(g), "a gradient is ", g.scalar_type(), ": float32, bfloat16 or float16 is expected");
    TORCH_CHECK_VALUE(g.device() == dev, "gradients on ", dev, " and on ", g.device());
    TORCH_CHECK_VALUE(g.layout() == at::kStrided && without_gaps(g), "a gradient has gaps or repeated elements in memory");
    TORCH_CHECK_VALUE(!(scale && at::GradMode::is_enabled() && g.requires_grad()), "a gradient to be scaled requires a gradient itself");
  };
  for (size_t i = 0; i < n; ++i) {
    const Tensor &g = grads[i], &o = out ? (*out)[i] : g;
    check(g);
    if (out) {
      check(o);
      TORCH_CHECK_VALUE(g.sizes() == o.sizes() && g.strides() == o.strides(), "an output has shape ", o.sizes(), " and strides ", o.strides(), ", its gradient ", g.sizes(),
                        " and ", g.strides());
    }
    in[i] = g.data_ptr(), to[i] = o.data_ptr();
    numel[i] = g.numel();
    in_dtype[i] = dtype_of(g), out_dtype[i] = dtype_of(o);
  }
  const Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat).requires_grad(false));
  afc_clip_args p = {};
  p.device = dev.index();
  p.count = (int32_t)n;
  p.in = in.data(), p.numel = numel.data(), p.in_dtype = in_dtype.data();
  if (scale) p.out = to.data(), p.out_dtype = out_dtype.data(), p.max_norm = (float)max_norm;
  p.norm = ptr<float>(norm);
  ok(afc_clip_workspace(&p, &p.workspace_bytes));
  const Tensor ws = space(norm, p.workspace_bytes);
  p.workspace = ptr(ws);
  ok(afc_clip(&p, stream_of(norm)));
  if (scale)
    for (const Tensor &t : out ? *out : grads) written(t);
  return norm;
}

}  // namespace

PYBIND11_MODULE(_ops_torch, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const OpsFailure &e) {
      PyErr_SetString(g_error_class ? g_error_class->ptr() : PyExc_RuntimeError, e.what());
    }
  });
  m.def("set_error_class", [](py::object cls) { g_error_class = new py::object(std::move(cls)); });
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("clip", &clip);
}
