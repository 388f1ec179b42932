// The state space layer's operators (causal convolution, selective scan, linear with residual) as torch calls over the C-ABI:
// checks of arguments, outputs and workspaces from torch's allocator, autograd Functions.  Host code only; one call from Python
// into C++ an operator.  Workspaces are allocated call by call and not kept: these operators may be captured into a graph,
// and a captured address must not be handed to another call meanwhile.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <unordered_set>
#include <vector>

#include "timeband_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using OptT = std::optional<Tensor>;

constexpr int ACT_NONE = 0, ACT_GELU = 5;

void ok(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (code ", rc, "): ", tb_last_error()); }
Tensor opt(const OptT& t) { return t.has_value() ? *t : Tensor(); }
OptT maybe(const Tensor& t) { return t.defined() ? OptT(t) : std::nullopt; }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const float* fptr(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
float* out_fptr(const Tensor& t) { return static_cast<float*>(out_ptr(t)); }
void* stream(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

// the first call on a device: the library looks it over (refuses other parts than gfx950)
void first_use(int dev) {
  static std::atomic<bool> seen[64];
  if (dev < 64 && seen[dev].load(std::memory_order_acquire)) return;
  ok(tb_init(dev), "tb_init");
  if (dev < 64) seen[dev].store(true, std::memory_order_release);
}

// Device and element type of a call: the type's code
int check(const char* what, const Tensor& lead, std::initializer_list<const Tensor*> others) {
  auto on_gpu = [&](const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "timeband_amd ops run on the GPU only (got a CPU tensor); there is no CPU fallback in the product path");
  };
  on_gpu(lead);
  for (const Tensor* t : others) {
    if (!t->defined()) continue;
    on_gpu(*t);
    TORCH_CHECK(t->device() == lead.device(), what, ": tensors are on ", lead.device(), " and ", t->device());
    TORCH_CHECK(t->scalar_type() == lead.scalar_type(), what, ": expected ", lead.scalar_type(), " throughout, got ", t->scalar_type());
  }
  const int code = code_of(lead);
  TORCH_CHECK(code >= 0, what, ": ", lead.scalar_type(), " is not supported (float32, bfloat16, float16)");
  return code;
}

void shape(const char* what, const char* name, const Tensor& t, at::IntArrayRef want) {
  if (t.defined()) TORCH_CHECK(t.sizes() == want, what, ": ", name, ": expected shape ", want, ", got ", t.sizes());
}

Tensor par32(const char* what, const char* name, const Tensor& t, at::IntArrayRef want, const Tensor& lead) {
  if (!t.defined()) return t;
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.sizes() == want && t.device() == lead.device(), what, ": ", name, ": expected float32 ", want, " on ",
              lead.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
  return t.contiguous();
}

Tensor last_dense(const Tensor& t) { return !t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

Tensor lengths_of(const char* what, const Tensor& t, int64_t B, const Tensor& lead) {
  if (!t.defined()) return t;
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B && t.device() == lead.device(), what, ": lengths must be int32 (", B, ",) on ",
              lead.device());
  return t.contiguous();
}

Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

int fits(const char* what, int64_t v) {
  TORCH_CHECK(v <= INT_MAX, what, ": a size of ", v, " is not supported");
  return (int)v;
}

bool wanted(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Dual tensors (torch.autograd.forward_ad): without requires_grad a call passes its autograd Function by, and its result would have no
// tangent, which counts as a zero one.
void no_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts) TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, ": forward-mode derivatives are not supported");
}

void inference_only(const char* what, std::initializer_list<const Tensor*> ts) {
  TORCH_CHECK(!wanted(ts), what, " updates its state in place and has no gradient: call it under torch.no_grad()");
}

// what a step wrote over counts as changed: a recorded call that saved it refuses its backward pass (tensors made for inference only
// have no count)
void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A backward pass ends by making its stream wait for the streams that its leaves' accumulation nodes were made on.  Under
// capture such a node from outside (an eager graph of the same leaf that somebody still holds) ties the capture to work
// that is not part of it, and the process ends inside the runtime when the capture does.  Refused here, before anything is
// recorded: every accumulation node behind the inputs has to be of the capturing stream.
void check_capture(std::initializer_list<const Tensor*> inputs) {
  std::vector<torch::autograd::Node*> todo;
  std::unordered_set<torch::autograd::Node*> seen;
  std::vector<std::shared_ptr<torch::autograd::Node>> held;
  c10::StreamId cur = 0;
  bool asked = false;
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad()) continue;
    if (!asked) {
      const auto s = c10::hip::getCurrentHIPStream(t->get_device());
      hipStreamCaptureStatus status;
      C10_HIP_CHECK(hipStreamIsCapturing(s.stream(), &status));
      if (status == hipStreamCaptureStatusNone) return;
      cur = s.unwrap().id();
      asked = true;
    }
    auto n = t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn();
    if (n && seen.insert(n.get()).second) {
      todo.push_back(n.get());
      held.push_back(std::move(n));
    }
  }
  while (!todo.empty()) {
    torch::autograd::Node* n = todo.back();
    todo.pop_back();
    if (n->next_edges().empty() && n->num_inputs() == 1 && n->name() == "torch::autograd::AccumulateGrad") {
      const auto s = n->stream();
      TORCH_CHECK(!s.has_value() || s->id() == cur,
                  "timeband_amd: a backward pass cannot be captured while an autograd graph of the same leaf, made outside the "
                  "capture, is alive: drop (or detach) what earlier calls returned");
    }
    for (const auto& e : n->next_edges())
      if (e.function && seen.insert(e.function.get()).second) todo.push_back(e.function.get());
  }
}

// gradients have no gradient of their own: asking for one is an error, not a zero
tensor_list once(tensor_list g) {
  if (!at::GradMode::is_enabled()) return g;
  auto stop = std::make_shared<torch::autograd::DelayedError>("timeband_amd: this operator's gradient cannot be differentiated again", g.size());
  tensor_list out = (*stop)(tensor_list(g));
  for (size_t i = 0; i < g.size(); ++i)
    if (!g[i].defined()) out[i] = Tensor();
  return out;
}

// ---- convolution -------------------------------------------------------------------------------------------------------
struct ConvOut {
  Tensor y, state;
};

ConvOut conv_forward(const Tensor& x, const Tensor& w, const Tensor& b, int act, const Tensor& state, const Tensor& lengths, bool want_state) {
  c10::DeviceGuard guard(x.device());
  const int64_t B = x.size(0), T = x.size(1), D = x.size(2), K = w.size(1);
  ConvOut r;
  r.y = at::empty({B, T, D}, x.options());
  if (want_state) r.state = at::empty({B, K - 1, D}, x.options());
  ok(tb_conv_fwd(ptr(x), x.stride(0), x.stride(1), ptr(w), ptr(b), w.scalar_type() == at::kFloat, ptr(state), static_cast<const int*>(ptr(lengths)),
                 out_ptr(r.y), out_ptr(r.state), fits("causal_conv", B), fits("causal_conv", T), fits("causal_conv", D), (int)K, act, code_of(x), stream(x)),
     "tb_conv_fwd");
  return r;
}

struct ConvFn : public torch::autograd::Function<ConvFn> {
  static tensor_list forward(AutogradContext* ctx, Tensor x, Tensor w, OptT b_, int64_t act, OptT state_, OptT lengths_, bool want_state) {
    Tensor b = opt(b_), state = opt(state_), lengths = opt(lengths_);
    ConvOut r = conv_forward(x, w, b, (int)act, state, lengths, want_state);
    ctx->save_for_backward({x, w, b, state, lengths});
    ctx->saved_data["act"] = act;
    ctx->saved_data["need"] = std::vector<bool>{x.requires_grad(), w.requires_grad(), b.defined() && b.requires_grad()};
    ctx->set_materialize_grads(false);
    if (!want_state) return {r.y};
    ctx->mark_non_differentiable({r.state});
    return {r.y, r.state};
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    tensor_list g(7);
    if (!grads[0].defined()) return g;
    auto sv = ctx->get_saved_variables();
    const Tensor &x = sv[0], &w = sv[1], &b = sv[2], &state = sv[3], &lengths = sv[4];
    auto need = ctx->saved_data["need"].toBoolList();
    c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), T = x.size(1), D = x.size(2), K = w.size(1);
    if (B == 0 || T == 0) {
      if (need[0]) g[0] = at::zeros_like(x);
      if (need[1]) g[1] = at::zeros_like(w);
      if (need[2]) g[2] = at::zeros_like(b);
      return once(std::move(g));
    }
    Tensor dy = grads[0].contiguous(), dx = at::empty({B, T, D}, x.options());
    if (need[1]) g[1] = at::empty({D, K}, w.options());
    if (need[2]) g[2] = at::empty({D}, b.options());
    Tensor ws = bytes(tb_conv_bwd_workspace_bytes((int)B, (int)T, (int)D, (int)K, code_of(x)), x);
    ok(tb_conv_bwd(ptr(dy), ptr(x), x.stride(0), x.stride(1), ptr(w), ptr(b), w.scalar_type() == at::kFloat, ptr(state),
                   static_cast<const int*>(ptr(lengths)), out_ptr(dx), out_ptr(g[1]), out_ptr(g[2]), (int)B, (int)T, (int)D, (int)K,
                   (int)ctx->saved_data["act"].toInt(), code_of(x), out_ptr(ws), ws.numel(), stream(x)),
       "tb_conv_bwd");
    if (need[0]) g[0] = dx;
    return once(std::move(g));
  }
};

void conv_params(const char* what, Tensor& w, Tensor& b, int64_t D, const Tensor& x) {
  TORCH_CHECK(w.dim() == 2 && w.size(0) == D, what, ": weight must be (", D, ", taps), got ", w.sizes());
  for (const Tensor* t : {&w, &b})
    if (t->defined())
      TORCH_CHECK(t->device() == x.device() && (t->scalar_type() == at::kFloat || t->scalar_type() == x.scalar_type()) && t->scalar_type() == w.scalar_type(),
                  what, ": weight and bias must both be ", x.scalar_type(), " or both Float, on ", x.device());
  shape(what, "bias", b, {D});
  w = w.contiguous();
  if (b.defined()) b = b.contiguous();
}

py::object causal_conv(Tensor x, Tensor w, OptT bias, int64_t act, OptT state_, OptT lengths_, bool return_state) {
  const char* what = "causal_conv";
  Tensor b = opt(bias), state = opt(state_);
  no_tangents(what, {&x, &w, &b, &state});
  check(what, x, {&state});
  TORCH_CHECK(x.dim() == 3, "causal_conv: x must be (B, T, D)");
  const int64_t B = x.size(0), D = x.size(2);
  conv_params(what, w, b, D, x);
  shape(what, "state", state, {B, w.size(1) - 1, D});
  TORCH_CHECK(!wanted({&state}), "causal_conv: no gradient runs through the state (detach it)");
  Tensor lengths = lengths_of(what, opt(lengths_), B, x);
  x = last_dense(x);
  if (state.defined()) state = state.contiguous();
  {
    c10::DeviceGuard guard(x.device());
    first_use(x.get_device());
  }
  Tensor y, s;
  if (wanted({&x, &w, &b})) {
    check_capture({&x, &w, &b});
    tensor_list r = ConvFn::apply(x, w, maybe(b), act, maybe(state), maybe(lengths), return_state);
    y = r[0];
    if (return_state) s = r[1];
  } else {
    ConvOut r = conv_forward(x, w, b, (int)act, state, lengths, return_state);
    y = r.y;
    s = r.state;
  }
  return return_state ? py::object(py::make_tuple(y, s)) : py::cast(y);
}

Tensor causal_conv_step(Tensor x, Tensor state, Tensor w, OptT bias, int64_t act) {
  const char* what = "causal_conv_step";
  Tensor b = opt(bias);
  no_tangents(what, {&x, &w, &b, &state});
  const int code = check(what, x, {&state});
  TORCH_CHECK(x.dim() == 2, "causal_conv_step: x must be (B, D)");
  const int64_t B = x.size(0), D = x.size(1);
  conv_params(what, w, b, D, x);
  const int64_t K = w.size(1);
  shape(what, "state", state, {B, K - 1, D});
  inference_only(what, {&x, &state, &w, &b});
  TORCH_CHECK(K < 2 || ((D < 2 || state.stride(2) == 1) && (K < 3 || state.stride(1) == D)),
              "causal_conv_step: the rows of state must be dense (it is updated in place)");
  TORCH_CHECK(B < 2 || state.stride(0) >= (K - 1) * D, "causal_conv_step: the rows of state overlap");
  x = last_dense(x);
  c10::DeviceGuard guard(x.device());
  first_use(x.get_device());
  Tensor y = at::empty({B, D}, x.options());
  ok(tb_conv_step(ptr(x), x.stride(0), out_ptr(state), state.stride(0), ptr(w), ptr(b), w.scalar_type() == at::kFloat, out_ptr(y), fits(what, B),
                  fits(what, D), (int)K, (int)act, code, stream(x)),
     "tb_conv_step");
  changed(state);
  return y;
}

// ---- scan ----------------------------------------------------------------------------------------------------------------
struct ScanIn {
  Tensor u, dt, A, Bm, Cm, D, z, bias, h0, lengths;
  bool softplus;
};
struct ScanOut {
  Tensor out, hT, states;
};
struct Strides {
  long v[14];
};

Strides strides_of(const Tensor& u, const Tensor& dt, const Tensor& z, const Tensor& B, const Tensor& C) {
  return {{u.stride(0), u.stride(1), dt.stride(0), dt.stride(1), z.defined() ? z.stride(0) : 0, z.defined() ? z.stride(1) : 0, B.stride(0), B.stride(1),
           B.stride(2), C.stride(0), C.stride(1), C.stride(2), 0, 0}};
}

ScanOut scan_forward(const ScanIn& q, bool want_state, bool train) {
  c10::DeviceGuard guard(q.u.device());
  const char* what = "selective_scan";
  const int B = fits(what, q.u.size(0)), T = fits(what, q.u.size(1)), D = fits(what, q.u.size(2)), G = (int)q.Bm.size(2), N = (int)q.Bm.size(3);
  ScanOut r;
  r.out = at::empty({B, T, D}, q.u.options());
  if (want_state) r.hT = at::empty({B, D, N}, q.A.options());
  if (B && T) {
    if (train) r.states = bytes(tb_scan_states_bytes(B, T, D, N), q.u);
    Tensor ws = bytes(tb_scan_workspace_bytes(B, T, D, N, G, 0), q.u);
    const Strides st = strides_of(q.u, q.dt, q.z, q.Bm, q.Cm);
    ok(tb_scan_fwd(ptr(q.u), ptr(q.dt), ptr(q.z), ptr(q.Bm), ptr(q.Cm), st.v, fptr(q.A), fptr(q.D), fptr(q.bias), q.softplus, fptr(q.h0),
                   static_cast<const int*>(ptr(q.lengths)), out_ptr(r.out), out_fptr(r.hT), out_fptr(r.states), B, T, D, N, G, code_of(q.u), out_ptr(ws),
                   ws.numel(), stream(q.u)),
       "tb_scan_fwd");
  } else if (want_state) {
    if (q.h0.defined()) r.hT.copy_(q.h0);
    else r.hT.zero_();
  }
  return r;
}

struct ScanFn : public torch::autograd::Function<ScanFn> {
  static tensor_list forward(AutogradContext* ctx, Tensor u, Tensor dt, Tensor A, Tensor Bm, Tensor Cm, OptT D_, OptT z_, OptT bias_, OptT h0_,
                             OptT lengths_, bool softplus, bool want_state) {
    Tensor D = opt(D_), z = opt(z_), bias = opt(bias_), h0 = opt(h0_), lengths = opt(lengths_);
    std::vector<bool> need;
    for (const Tensor* t : {&u, &dt, &A, &Bm, &Cm, &D, &z, &bias, &h0}) need.push_back(t->defined() && t->requires_grad());
    ScanOut r = scan_forward({u, dt, A, Bm, Cm, D, z, bias, h0, lengths, softplus}, want_state, true);
    ctx->save_for_backward({u, dt, A, Bm, Cm, D, z, bias, lengths, r.states});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["need"] = need;
    ctx->set_materialize_grads(false);
    if (!want_state) return {r.out};
    return {r.out, r.hT};
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    tensor_list g(12);
    Tensor dout = grads[0], dhT = grads.size() > 1 ? grads[1] : Tensor();
    if (!dout.defined() && !dhT.defined()) return g;
    auto sv = ctx->get_saved_variables();
    const Tensor &u = sv[0], &dt = sv[1], &A = sv[2], &Bm = sv[3], &Cm = sv[4], &Dp = sv[5], &z = sv[6], &bias = sv[7], &lengths = sv[8], &states = sv[9];
    auto need = ctx->saved_data["need"].toBoolList();
    c10::DeviceGuard guard(u.device());
    const int B = (int)u.size(0), T = (int)u.size(1), D = (int)u.size(2), G = (int)Bm.size(2), N = (int)Bm.size(3);
    const bool empty = !B || !T;
    for (int i = 0; i < 8; ++i)
      if (need[i]) g[i] = empty ? at::zeros(sv[i].sizes(), sv[i].options()) : at::empty(sv[i].sizes(), sv[i].options());
    if (empty) {
      if (need[8]) g[8] = dhT.defined() ? dhT.clone() : at::zeros({B, D, N}, A.options());
      return once(std::move(g));
    }
    if (need[8]) g[8] = at::empty({B, D, N}, A.options());
    dout = dout.defined() ? last_dense(dout) : at::zeros({B, T, D}, u.options());
    if (dhT.defined()) dhT = dhT.contiguous();
    Tensor ws = bytes(tb_scan_workspace_bytes(B, T, D, N, G, 1), u);
    Strides st = strides_of(u, dt, z, Bm, Cm);
    st.v[12] = dout.stride(0);
    st.v[13] = dout.stride(1);
    ok(tb_scan_bwd(ptr(dout), ptr(u), ptr(dt), ptr(z), ptr(Bm), ptr(Cm), st.v, fptr(A), fptr(Dp), fptr(bias), ctx->saved_data["softplus"].toBool(),
                   static_cast<const int*>(ptr(lengths)), fptr(states), fptr(dhT), out_ptr(g[0]), out_ptr(g[1]), out_ptr(g[6]), out_ptr(g[3]),
                   out_ptr(g[4]), out_fptr(g[2]), out_fptr(g[5]), out_fptr(g[7]), out_fptr(g[8]), B, T, D, N, G, code_of(u), out_ptr(ws), ws.numel(),
                   stream(u)),
       "tb_scan_bwd");
    return once(std::move(g));
  }
};

py::object selective_scan(Tensor u, Tensor dt, Tensor A, Tensor Bm, Tensor Cm, OptT D_, OptT z_, OptT bias_, bool softplus, OptT h0_, OptT lengths_,
                          bool return_state) {
  const char* what = "selective_scan";
  Tensor z = opt(z_), D = opt(D_), bias = opt(bias_), h0 = opt(h0_);
  no_tangents(what, {&u, &dt, &A, &Bm, &Cm, &D, &z, &bias, &h0});
  check(what, u, {&dt, &Bm, &Cm, &z});
  TORCH_CHECK(u.dim() == 3, "selective_scan: u must be (B, T, D)");
  const int64_t B = u.size(0), T = u.size(1), Dn = u.size(2);
  shape(what, "dt", dt, u.sizes());
  shape(what, "z", z, u.sizes());
  if (Bm.dim() == 3) Bm = Bm.unsqueeze(2);
  if (Cm.dim() == 3) Cm = Cm.unsqueeze(2);
  TORCH_CHECK(Bm.dim() == 4 && Bm.size(0) == B && Bm.size(1) == T && Cm.sizes() == Bm.sizes(), "selective_scan: B and C must be (", B, ", ", T, ", N) or (",
              B, ", ", T, ", G, N)");
  const int64_t G = Bm.size(2), N = Bm.size(3);
  TORCH_CHECK(G > 0 && Dn % G == 0, "selective_scan: ", Dn, " channels do not divide into ", G, " groups");
  A = par32(what, "A", A, {Dn, N}, u);
  D = par32(what, "D", D, {Dn}, u);
  bias = par32(what, "dt_bias", bias, {Dn}, u);
  h0 = par32(what, "h0", h0, {B, Dn, N}, u);
  Tensor lengths = lengths_of(what, opt(lengths_), B, u);
  u = last_dense(u);
  dt = last_dense(dt);
  z = last_dense(z);
  Bm = last_dense(Bm);
  Cm = last_dense(Cm);
  {
    c10::DeviceGuard guard(u.device());
    first_use(u.get_device());
  }
  Tensor out, hT;
  if (wanted({&u, &dt, &A, &Bm, &Cm, &D, &z, &bias, &h0})) {
    check_capture({&u, &dt, &A, &Bm, &Cm, &D, &z, &bias, &h0});
    tensor_list r = ScanFn::apply(u, dt, A, Bm, Cm, maybe(D), maybe(z), maybe(bias), maybe(h0), maybe(lengths), softplus, return_state);
    out = r[0];
    if (return_state) hT = r[1];
  } else {
    ScanOut r = scan_forward({u, dt, A, Bm, Cm, D, z, bias, h0, lengths, softplus}, return_state, false);
    out = r.out;
    hT = r.hT;
  }
  return return_state ? py::object(py::make_tuple(out, hT)) : py::cast(out);
}

Tensor selective_scan_step(Tensor state, Tensor u, Tensor dt, Tensor A, Tensor Bm, Tensor Cm, OptT D_, OptT z_, OptT bias_, bool softplus) {
  const char* what = "selective_scan_step";
  Tensor z = opt(z_), D = opt(D_), bias = opt(bias_);
  no_tangents(what, {&state, &u, &dt, &A, &Bm, &Cm, &D, &z, &bias});
  const int code = check(what, u, {&dt, &Bm, &Cm, &z});
  TORCH_CHECK(u.dim() == 2, "selective_scan_step: u must be (B, D)");
  const int64_t B = u.size(0), Dn = u.size(1);
  shape(what, "dt", dt, u.sizes());
  shape(what, "z", z, u.sizes());
  if (Bm.dim() == 2) Bm = Bm.unsqueeze(1);
  if (Cm.dim() == 2) Cm = Cm.unsqueeze(1);
  TORCH_CHECK(Bm.dim() == 3 && Bm.size(0) == B && Cm.sizes() == Bm.sizes(), "selective_scan_step: B and C must be (", B, ", N) or (", B, ", G, N)");
  const int64_t G = Bm.size(1), N = Bm.size(2);
  TORCH_CHECK(G > 0 && Dn % G == 0, "selective_scan_step: ", Dn, " channels do not divide into ", G, " groups");
  A = par32(what, "A", A, {Dn, N}, u);
  D = par32(what, "D", D, {Dn}, u);
  bias = par32(what, "dt_bias", bias, {Dn}, u);
  TORCH_CHECK(state.scalar_type() == at::kFloat && state.sizes() == at::IntArrayRef({B, Dn, N}) && state.device() == u.device(),
              "selective_scan_step: state must be float32 (", B, ", ", Dn, ", ", N, ") on ", u.device());
  inference_only(what, {&state, &u, &dt, &A, &Bm, &Cm, &D, &z, &bias});
  TORCH_CHECK((N < 2 || state.stride(2) == 1) && (Dn < 2 || state.stride(1) == N), "selective_scan_step: the rows of state must be dense (it is updated in place)");
  TORCH_CHECK(B < 2 || state.stride(0) >= Dn * N, "selective_scan_step: the rows of state overlap");
  u = last_dense(u);
  dt = last_dense(dt);
  z = last_dense(z);
  Bm = last_dense(Bm);
  Cm = last_dense(Cm);
  c10::DeviceGuard guard(u.device());
  first_use(u.get_device());
  Tensor out = at::empty({B, Dn}, u.options());
  const long st[7] = {u.stride(0), dt.stride(0), z.defined() ? z.stride(0) : 0, Bm.stride(0), Bm.stride(1), Cm.stride(0), Cm.stride(1)};
  ok(tb_scan_step(out_fptr(state), state.stride(0), ptr(u), ptr(dt), ptr(z), ptr(Bm), ptr(Cm), st, fptr(A), fptr(D), fptr(bias), softplus, out_ptr(out),
                  fits(what, B), fits(what, Dn), (int)N, (int)G, code, stream(u)),
     "tb_scan_step");
  changed(state);
  return out;
}

// ---- linear --------------------------------------------------------------------------------------------------------------
Tensor linres_forward(const Tensor& x, const Tensor& W, const Tensor& b, int act, const Tensor& res, Tensor* z) {
  c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0);
  const int K = fits("linear_residual", x.size(1)), N = fits("linear_residual", W.size(0)), code = code_of(x);
  Tensor y = at::empty({M, N}, x.options());
  if (z && act) *z = at::empty({M, N}, x.options().dtype(at::kFloat));
  Tensor ws = bytes(tb_linres_fwd_workspace_bytes(ptr(x), x.stride(0), ptr(W), W.stride(0), M, K, N, code), x);
  ok(tb_linres_fwd(ptr(x), x.stride(0), ptr(W), W.stride(0), ptr(b), ptr(res), res.defined() ? res.stride(0) : 0, out_ptr(y),
                   z ? out_fptr(*z) : nullptr, M, K, N, act, code, out_ptr(ws), ws.numel(), stream(x)),
     "tb_linres_fwd");
  return y;
}

struct LinResFn : public torch::autograd::Function<LinResFn> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor W, OptT b_, int64_t act, OptT res_) {
    Tensor b = opt(b_), res = opt(res_);
    const bool products = x.requires_grad() || W.requires_grad() || (b.defined() && b.requires_grad());
    Tensor z;
    Tensor y = linres_forward(x, W, b, (int)act, res, products ? &z : nullptr);
    ctx->saved_data["act"] = act;
    ctx->saved_data["need"] = std::vector<bool>{x.requires_grad(), W.requires_grad(), b.defined() && b.requires_grad(), res.defined() && res.requires_grad()};
    if (products) ctx->save_for_backward({x, W, z});
    return y;
  }
  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    tensor_list g(5);
    auto need = ctx->saved_data["need"].toBoolList();
    if (need[3]) g[4] = grads[0];
    if (!need[0] && !need[1] && !need[2]) return g;
    auto sv = ctx->get_saved_variables();
    const Tensor &x = sv[0], &W = sv[1], &z = sv[2];
    c10::DeviceGuard guard(x.device());
    const int64_t M = x.size(0);
    const int K = (int)x.size(1), N = (int)W.size(0), code = code_of(x);
    auto make = [&](at::IntArrayRef s) { return M ? at::empty(s, x.options()) : at::zeros(s, x.options()); };
    if (need[0]) g[0] = make({M, K});
    if (need[1]) g[1] = make({N, K});
    if (need[2]) g[2] = make({N});
    if (M) {
      Tensor dy = last_dense(grads[0]);
      const int act = (int)ctx->saved_data["act"].toInt();
      Tensor ws = bytes(tb_linres_bwd_workspace_bytes(ptr(dy), dy.stride(0), ptr(x), x.stride(0), act, need[0], need[1], need[2], M, K, N, code), x);
      ok(tb_linres_bwd(ptr(dy), dy.stride(0), ptr(x), x.stride(0), ptr(W), W.stride(0), fptr(z), act, out_ptr(g[0]), out_ptr(g[1]), out_ptr(g[2]), M, K, N, code, out_ptr(ws), ws.numel(), stream(x)),
         "tb_linres_bwd");
    }
    return once(std::move(g));
  }
};

Tensor linear_residual(Tensor x, Tensor W, OptT b_, int64_t act, OptT res_) {
  const char* what = "linear_residual";
  Tensor b = opt(b_), res = opt(res_);
  no_tangents(what, {&x, &W, &b, &res});
  check(what, x, {&W, &b, &res});
  TORCH_CHECK(x.dim() >= 1 && W.dim() == 2 && W.size(1) == x.size(-1) && W.size(0) >= 1 && W.size(1) >= 1, "linear_residual: weight ", W.sizes(),
              " does not match the input ", x.sizes());
  const int64_t N = W.size(0), K = W.size(1);
  shape(what, "b", b, {N});
  std::vector<int64_t> want(x.sizes().begin(), x.sizes().end());
  want.back() = N;
  shape(what, "residual", res, want);
  TORCH_CHECK(act >= ACT_NONE && act <= ACT_GELU, "linear_residual: activation ", act, " is not supported");
  if (x.dim() != 2) x = x.reshape({-1, K});
  x = last_dense(x);
  if (res.defined()) {
    if (res.dim() != 2) res = res.reshape({-1, N});
    res = last_dense(res);
  }
  W = last_dense(W);
  if (b.defined()) b = b.contiguous();
  {
    c10::DeviceGuard guard(x.device());
    first_use(x.get_device());
  }
  Tensor y;
  if (wanted({&x, &W, &b, &res})) {
    check_capture({&x, &W, &b, &res});
    y = LinResFn::apply(x, W, maybe(b), act, maybe(res));
  } else {
    y = linres_forward(x, W, b, (int)act, res, nullptr);
  }
  return want.size() == 2 ? y : y.view(want);
}

}  // namespace

void tb_bind_ssm(py::module_& m) {
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("linear_residual", &linear_residual);
}
