// torch.ops.mineral.{linear_attention, linear_attention_step, group_norm_act, linear_act}: the operators of include/mineral_memory.h
// as PyTorch operators with their gradients.  Host code only: checks of the arguments, allocation of outputs and workspaces through
// torch's allocator, the launch on the current stream of the tensors' device.  In C++ because a call that acts for a few
// environments takes less on the GPU than the interpreter needs to get there (17 us a call and 160 us for a call with its
// gradient from Python on MI355X, measured with kernels of under 10 us).
//
// Every kernel is reached through the dispatcher, the forward pass below autograd and the backward pass from the autograd node: tracers,
// dispatch modes, tensor subclasses and lazily negated tensors then see one operator instead of its allocations.  Operators whose names
// begin with an underscore are the halves of a differentiable call.  Shape functions for tensors without data are in memory_ops.py.
//
// CPU tensors go through the same checks and are then refused: there is no CPU kernel.
#include "../../include/mineral_memory.h"
#include "../../include/mineral_ppo.h"

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/InferenceMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <string>
#include <tuple>

namespace {

using at::Tensor;
using OptT = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

#define NEED(what, ok, ...) TORCH_CHECK_VALUE(ok, what, ": ", __VA_ARGS__)

const Tensor none;
const Tensor& of(const OptT& t) { return t.has_value() ? *t : none; }
OptT opt(const Tensor& t) { return t.defined() ? OptT(t) : OptT(); }

int dtype_of(const char* what, const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MRL_F32;
    case at::kBFloat16: return MRL_BF16;
    case at::kHalf: return MRL_F16;
    default: TORCH_CHECK_VALUE(false, what, ": dtype ", t.scalar_type(), " (float32, bfloat16 or float16)");
  }
}

void same_device(const char* what, const Tensor& t, std::initializer_list<const Tensor*> others) {
  for (const Tensor* o : others) NEED(what, !o->defined() || o->device() == t.device(), "tensors on ", t.device(), " and ", o->device());
}

void check(int rc, const char* what) {
  if (rc == MRL_OK) return;
  const std::string msg = mrl_last_error();
  TORCH_CHECK_VALUE(rc != MRL_EINVAL, what, ": ", msg);
  TORCH_CHECK(false, what, " failed (", rc, "): ", msg);
}

const void* cp(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mp(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

Tensor new_like(const Tensor& t, at::IntArrayRef shape) { return at::empty(shape, t.options().memory_format(at::MemoryFormat::Contiguous).requires_grad(false)); }
Tensor new_floats(const Tensor& t, at::IntArrayRef shape) { return at::empty(shape, t.options().dtype(at::kFloat).requires_grad(false)); }

struct Workspace {
  Tensor t;
  int64_t n;
  Workspace(const char* what, int64_t bytes, const Tensor& like) : n(bytes) {
    if (n < 0) check((int)n, what);
    if (n > 0) t = at::empty({n}, like.options().dtype(at::kByte).requires_grad(false));
  }
  void* p() const { return mp(t); }
};

// the last dimension contiguous; every other stride stays
Tensor rows_of(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
// contiguous, on a 16-byte address
Tensor aligned(const Tensor& t) {
  const Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.const_data_ptr()) & 15) ? c.clone() : c;
}
Tensor contiguous(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Forward-mode derivatives are refused instead of dropped.
void no_tangent(const char* what, std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), what, ": no forward-mode derivative");
}

// The operator `name` as a typed handle, and a call of it below autograd.
template <typename Signature> c10::TypedOperatorHandle<Signature> op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}
using BelowAutograd = at::AutoDispatchBelowAutograd;

void once(const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(), what, ": differentiable once; its gradient under create_graph=True has none of its own");
}

[[noreturn]] void no_cpu(const char* what) { TORCH_CHECK_NOT_IMPLEMENTED(false, what, ": tensors have to be on the GPU, there is no CPU kernel"); }

// Of tensors in the order of the bits of `needs`: those whose bit is set, and back to where they belong.
std::vector<Tensor> asked(int64_t needs, std::initializer_list<Tensor> all) {
  std::vector<Tensor> r;
  int i = 0;
  for (const Tensor& t : all)
    if (needs >> i++ & 1) r.push_back(t);
  return r;
}
void place(int64_t needs, const std::vector<Tensor>& got, std::initializer_list<Tensor*> to) {
  size_t n = 0;
  int i = 0;
  for (Tensor* t : to)
    if (needs >> i++ & 1) *t = got[n++];
}

// ---- linear attention ------------------------------------------------------------------------------------------------------------
struct Attention {
  mrl_attention a;
  Tensor q, k, v, log_decay, resets, state;   // what `a` points into

  Attention(const char* what, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& l_, const Tensor& r_, const Tensor& s_, double scale, bool step) {
    a.dtype = dtype_of(what, q_);
    NEED(what, k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type(), "q, k and v of one type, got ", q_.scalar_type(), ", ", k_.scalar_type(), ", ",
         v_.scalar_type());
    const int64_t dims = step ? 3 : 4;
    bool ok = q_.dim() == dims && k_.sizes() == q_.sizes() && v_.dim() == dims;
    for (int64_t i = 0; ok && i + 1 < dims; ++i) ok = v_.size(i) == q_.size(i);
    NEED(what, ok, "q and k [batch, ", step ? "" : "steps, ", "heads, dim_k] and v [.., dim_v], got ", q_.sizes(), ", ", k_.sizes(), ", ", v_.sizes());
    same_device(what, q_, {&k_, &v_, &l_, &r_, &s_});
    a.batch = q_.size(0);
    a.steps = step ? 1 : q_.size(1);
    const int64_t H = q_.size(-2), K = q_.size(-1), V = v_.size(-1);
    NEED(what, H >= 1 && H < (1 << 30) && K >= 1 && K <= MRL_ATTENTION_MAX_DIM && V >= 1 && V <= MRL_ATTENTION_MAX_DIM, H, " heads of dim_k ", K, ", dim_v ", V, " (1..",
         MRL_ATTENTION_MAX_DIM, " each)");
    a.heads = (int32_t)H; a.dim_k = (int32_t)K; a.dim_v = (int32_t)V;
    NEED(what, l_.scalar_type() == at::kFloat && l_.dim() == 1 && l_.size(0) == H, "log_decay: float32 [", H, "], got ", l_.scalar_type(), " ", l_.sizes());
    if (r_.defined()) {
      const bool shape = step ? r_.dim() == 1 && r_.size(0) == a.batch : r_.dim() == 2 && r_.size(0) == a.batch && r_.size(1) == a.steps;
      NEED(what, (r_.scalar_type() == at::kBool || r_.scalar_type() == at::kByte) && shape, "resets: bool or uint8 [batch", step ? "" : ", steps", "], got ", r_.scalar_type(),
           " ", r_.sizes());
      resets = r_.contiguous();
    }
    if (s_.defined()) {
      NEED(what, s_.scalar_type() == at::kFloat && s_.dim() == 4 && s_.size(0) == a.batch && s_.size(1) == H && s_.size(2) == K && s_.size(3) == V,
           "state: float32 [batch, heads, dim_k, dim_v], got ", s_.scalar_type(), " ", s_.sizes());
      if (step) NEED(what, s_.is_contiguous(), "state is updated in place and has to be contiguous");
      state = s_.contiguous();
    }
    q = rows_of(q_); k = rows_of(k_); v = rows_of(v_);
    log_decay = l_.contiguous();
    const Tensor* t[3] = {&q, &k, &v};
    int64_t* st[3] = {a.q_stride, a.k_stride, a.v_stride};
    for (int i = 0; i < 3; ++i) {
      st[i][0] = t[i]->stride(0);
      st[i][1] = step ? 0 : t[i]->stride(1);
      st[i][2] = t[i]->stride(-2);
    }
    a.q = cp(q); a.k = cp(k); a.v = cp(v);
    a.log_decay = static_cast<const float*>(cp(log_decay));
    a.resets = static_cast<const uint8_t*>(cp(resets));
    a.initial_state = step ? nullptr : static_cast<const float*>(cp(state));
    a.scale = (float)scale;
  }
  Tensor new_state() const { return new_floats(q, {a.batch, a.heads, a.dim_k, a.dim_v}); }
};

std::tuple<Tensor, Tensor> linear_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& l, const OptT& r, const OptT& s, double scale) {
  const char* what = "linear_attention";
  const Attention d(what, q, k, v, l, of(r), of(s), scale, false);
  c10::DeviceGuard guard(q.device());
  Tensor out = new_like(v, v.sizes()), final = d.new_state();
  const Workspace ws(what, mrl_linear_attention_workspace_bytes(&d.a, 0), q);
  check(mrl_linear_attention(&d.a, mp(out), static_cast<float*>(mp(final)), ws.p(), ws.n, stream_of(q)), what);
  return {out, final};
}
using AttentionSig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptT&, const OptT&, double);

// The gradients that `needs` names (1 q, 2 k, 4 v, 8 initial state), in this order.
std::vector<Tensor> attention_backward(const OptT& dout_, const OptT& dfinal_, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& l, const OptT& r, const OptT& s,
                                       double scale, int64_t needs) {
  const char* what = "linear_attention_backward";
  const Attention d(what, q, k, v, l, of(r), of(s), scale, false);
  c10::DeviceGuard guard(q.device());
  const Tensor dout = dout_.has_value() ? rows_of(*dout_) : at::zeros_like(v, at::MemoryFormat::Contiguous), dfinal = contiguous(of(dfinal_));
  const int64_t st[3] = {dout.stride(0), dout.stride(1), dout.stride(2)};
  Tensor dq, dk, ds;
  if (needs & 1) dq = new_like(q, q.sizes());
  if (needs & 2) dk = new_like(k, k.sizes());
  Tensor dv = needs & 12 ? new_like(v, v.sizes()) : Tensor();             // the state's gradient comes with it
  if (needs & 8) ds = d.new_state();
  const Workspace ws(what, mrl_linear_attention_workspace_bytes(&d.a, 1), q);
  check(mrl_linear_attention_backward(&d.a, cp(dout), st, static_cast<const float*>(cp(dfinal)), mp(dq), mp(dk), mp(dv), static_cast<float*>(mp(ds)), ws.p(), ws.n, stream_of(q)),
        what);
  return asked(needs, {dq, dk, dv, ds});
}
using AttentionBackwardSig = std::vector<Tensor>(const OptT&, const OptT&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptT&, const OptT&, double, int64_t);

struct LinearAttention : Function<LinearAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& l, const OptT& r, const OptT& s, double scale,
                               int64_t needs) {
    static const auto fwd = op<AttentionSig>("mineral::linear_attention");
    const BelowAutograd below;
    ctx->set_materialize_grads(false);
    auto [out, final] = fwd.call(q, k, v, l, r, s, scale);
    ctx->save_for_backward({q, k, v, l, of(r), of(s)});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["needs"] = needs;
    return {out, final};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static const auto bwd = op<AttentionBackwardSig>("mineral::_linear_attention_backward");
    once("linear_attention");
    no_tangent("linear_attention", {&g[0], &g[1]});
    variable_list res(8);
    if (!g[0].defined() && !g[1].defined()) return res;
    const BelowAutograd below;
    const auto t = ctx->get_saved_variables();
    const int64_t needs = ctx->saved_data["needs"].toInt();
    const auto got = bwd.call(opt(g[0]), opt(g[1]), t[0], t[1], t[2], t[3], opt(t[4]), opt(t[5]), ctx->saved_data["scale"].toDouble(), needs);
    place(needs, got, {&res[0], &res[1], &res[2], &res[5]});
    return res;
  }
};

std::tuple<Tensor, Tensor> linear_attention_autograd(c10::DispatchKeySet ks, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& l, const OptT& r, const OptT& s,
                                                     double scale) {
  no_tangent("linear_attention", {&q, &k, &v, &l, &of(s)});
  if (!wants_grad({&q, &k, &v, &l, &of(s)})) {
    static const auto fwd = op<AttentionSig>("mineral::linear_attention");
    const BelowAutograd below;
    return fwd.redispatch(ks & c10::after_autograd_keyset, q, k, v, l, r, s, scale);
  }
  TORCH_CHECK_NOT_IMPLEMENTED(!l.requires_grad(), "linear_attention: the decays are constants of the heads; log_decay has no gradient");
  const int64_t needs = q.requires_grad() | k.requires_grad() << 1 | v.requires_grad() << 2 | (of(s).defined() && s->requires_grad()) << 3;
  const auto o = LinearAttention::apply(q, k, v, l, r, s, scale, needs);
  return {o[0], o[1]};
}
std::tuple<Tensor, Tensor> linear_attention_cpu(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& l, const OptT& r, const OptT& s, double scale) {
  const Attention d("linear_attention", q, k, v, l, of(r), of(s), scale, false);
  no_cpu("linear_attention");
}

Tensor linear_attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& l, const Tensor& state, const OptT& r, double scale) {
  const char* what = "linear_attention_step";
  const Attention d(what, q, k, v, l, of(r), state, scale, true);
  if (q.is_cpu()) no_cpu(what);
  c10::DeviceGuard guard(q.device());
  Tensor out = new_like(v, v.sizes());
  check(mrl_linear_attention_step(&d.a, static_cast<float*>(mp(state)), mp(out), stream_of(q)), what);
  return out;
}
using StepSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptT&, double);

Tensor linear_attention_step_autograd(c10::DispatchKeySet ks, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& l, const Tensor& state, const OptT& r, double scale) {
  static const auto fwd = op<StepSig>("mineral::linear_attention_step");
  no_tangent("linear_attention_step", {&q, &k, &v, &l, &state});
  TORCH_CHECK_NOT_IMPLEMENTED(!wants_grad({&q, &k, &v, &l, &state}),
                              "linear_attention_step: no gradient (linear_attention over the rollout has one); call it under torch.no_grad()");
  const BelowAutograd below;
  return fwd.redispatch(ks & c10::after_autograd_keyset, q, k, v, l, state, r, scale);
}
// Reached in inference mode too, where autograd is not: what a step overwrites is marked as written.
Tensor linear_attention_step_inplace(c10::DispatchKeySet ks, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& l, const Tensor& state, const OptT& r, double scale) {
  static const auto fwd = op<StepSig>("mineral::linear_attention_step");
  TORCH_CHECK(!state.is_inference() || c10::InferenceMode::is_enabled(), "linear_attention_step: a state made in inference mode is updated there only");
  Tensor out;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    out = fwd.redispatch(ks & c10::after_ADInplaceOrView_keyset, q, k, v, l, state, r, scale);
  }
  state.unsafeGetTensorImpl()->bump_version();
  return out;
}
// torch's own fallback for lazily negated tensors serves operators that return what they overwrite; this one returns something else.
Tensor linear_attention_step_negated(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& l, const Tensor& state, const OptT& r, double scale) {
  static const auto fwd = op<StepSig>("mineral::linear_attention_step");
  const Tensor s = state.resolve_neg();
  Tensor out = fwd.call(q.resolve_neg(), k.resolve_neg(), v.resolve_neg(), l.resolve_neg(), s, r, scale);
  if (state.is_neg()) state.copy_(s);
  return out;
}

// ---- activations -------------------------------------------------------------------------------------------------------------------
int act_of(const char* what, const std::optional<std::string_view>& name) {
  if (!name.has_value()) return MRL_ACT_NONE;
  static constexpr std::pair<std::string_view, int> known[] = {{"SiLU", MRL_ACT_SILU}, {"ELU", MRL_ACT_ELU}, {"ReLU", MRL_ACT_RELU}, {"Tanh", MRL_ACT_TANH}, {"GELU", MRL_ACT_GELU}};
  for (const auto& k : known)
    if (*name == k.first) return k.second;
  TORCH_CHECK_NOT_IMPLEMENTED(false, what, ": act_type=", std::string(*name), " (built: None, SiLU, ELU, ReLU, Tanh, GELU)");
}

// ---- group norm ----------------------------------------------------------------------------------------------------------------------
mrl_group_norm norm_of(const char* what, const Tensor& x, int64_t groups, const Tensor& w, const Tensor& b, double eps, int act) {
  mrl_group_norm p;
  p.dtype = dtype_of(what, x);
  NEED(what, x.dim() >= 2, "x [batch, ..., channels], got ", x.sizes());
  const int64_t C = x.size(-1);
  NEED(what, groups >= 1 && C >= 1 && C <= (1 << 24) && C % groups == 0, C, " channels are not ", groups, " groups");
  NEED(what, eps >= 0.0, "eps ", eps);
  same_device(what, x, {&w, &b});
  p.param_dtype = p.dtype;
  for (const Tensor* t : {&w, &b})
    if (t->defined()) {
      NEED(what, t->dim() == 1 && t->size(0) == C && (t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat), "weight and bias: [", C, "] of ", x.scalar_type(),
           " or float32, got ", t->scalar_type(), " ", t->sizes());
      p.param_dtype = dtype_of(what, *t);
    }
  NEED(what, !w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "weight and bias of one type");
  p.batch = x.size(0);
  p.pixels = 1;
  for (int64_t i = 1; i + 1 < x.dim(); ++i) p.pixels *= x.size(i);
  p.channels = (int32_t)C; p.groups = (int32_t)groups; p.act = act; p.eps = (float)eps;
  return p;
}

std::tuple<Tensor, Tensor> norm_forward(const Tensor& x_, int64_t groups, const Tensor& w_, const Tensor& b_, double eps, int act, bool keep) {
  const char* what = "group_norm_act";
  const mrl_group_norm p = norm_of(what, x_, groups, w_, b_, eps, act);
  c10::DeviceGuard guard(x_.device());
  const Tensor x = aligned(x_), w = contiguous(w_), b = contiguous(b_);
  Tensor y = new_like(x, x.sizes()), stats = keep ? new_floats(x, {2, p.batch, groups}) : Tensor();
  const Workspace ws(what, mrl_group_norm_act_workspace_bytes(&p, 0), x);
  float* mean = keep ? static_cast<float*>(mp(stats)) : nullptr;
  check(mrl_group_norm_act(&p, cp(x), cp(w), cp(b), mp(y), mean, keep ? mean + p.batch * groups : nullptr, ws.p(), ws.n, stream_of(x)), what);
  return {y, stats};
}

using Name = std::optional<std::string_view>;

Tensor group_norm_act(const Tensor& x, int64_t groups, const OptT& w, const OptT& b, double eps, Name act) {
  return std::get<0>(norm_forward(x, groups, of(w), of(b), eps, act_of("group_norm_act", act), false));
}
using NormSig = Tensor(const Tensor&, int64_t, const OptT&, const OptT&, double, Name);

std::tuple<Tensor, Tensor> group_norm_act_stats(const Tensor& x, int64_t groups, const OptT& w, const OptT& b, double eps, int64_t act) {
  return norm_forward(x, groups, of(w), of(b), eps, (int)act, true);
}
using NormStatsSig = std::tuple<Tensor, Tensor>(const Tensor&, int64_t, const OptT&, const OptT&, double, int64_t);

// The gradients that `needs` names (1 x, 2 weight, 4 bias), in this order.
std::vector<Tensor> group_norm_act_backward(const Tensor& dy_, const Tensor& x_, const Tensor& stats, const OptT& w_, const OptT& b_, int64_t groups, double eps, int64_t act,
                                            int64_t needs) {
  const char* what = "group_norm_act_backward";
  const mrl_group_norm p = norm_of(what, x_, groups, of(w_), of(b_), eps, (int)act);
  c10::DeviceGuard guard(x_.device());
  const Tensor x = aligned(x_), dy = aligned(dy_), w = contiguous(of(w_)), b = contiguous(of(b_));
  Tensor dx = new_like(x, x.sizes()), dw, db;
  if (needs & 6) {
    const auto o = x.options().dtype(p.param_dtype == MRL_F32 ? at::kFloat : x.scalar_type()).requires_grad(false);
    const bool empty = x.numel() == 0;
    dw = empty ? at::zeros({p.channels}, o) : at::empty({p.channels}, o);
    db = empty ? at::zeros({p.channels}, o) : at::empty({p.channels}, o);
  }
  if (x.numel() > 0) {
    const Workspace ws(what, mrl_group_norm_act_workspace_bytes(&p, 1), x);
    const float* mean = static_cast<const float*>(cp(stats));
    check(mrl_group_norm_act_backward(&p, cp(x), cp(dy), cp(w), cp(b), mean, mean + p.batch * p.groups, mp(dx), mp(dw), mp(db), ws.p(), ws.n, stream_of(x)), what);
  }
  return asked(needs, {dx, dw, db});
}
using NormBackwardSig = std::vector<Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptT&, const OptT&, int64_t, double, int64_t, int64_t);

struct GroupNormAct : Function<GroupNormAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptT& w, const OptT& b, int64_t groups, double eps, int64_t act, int64_t needs) {
    static const auto fwd = op<NormStatsSig>("mineral::_group_norm_act_stats");
    const BelowAutograd below;
    auto [y, stats] = fwd.call(x, groups, w, b, eps, act);
    ctx->save_for_backward({x, stats, of(w), of(b)});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["act"] = act;
    ctx->saved_data["needs"] = needs;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static const auto bwd = op<NormBackwardSig>("mineral::_group_norm_act_backward");
    once("group_norm_act");
    no_tangent("group_norm_act", {&g[0]});
    const BelowAutograd below;
    const auto t = ctx->get_saved_variables();
    const int64_t needs = ctx->saved_data["needs"].toInt();
    variable_list res(7);
    const auto got = bwd.call(g[0], t[0], t[1], opt(t[2]), opt(t[3]), ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["act"].toInt(), needs);
    place(needs, got, {&res[0], &res[1], &res[2]});
    return res;
  }
};

Tensor group_norm_act_autograd(c10::DispatchKeySet ks, const Tensor& x, int64_t groups, const OptT& w, const OptT& b, double eps, Name act) {
  no_tangent("group_norm_act", {&x, &of(w), &of(b)});
  if (!wants_grad({&x, &of(w), &of(b)})) {
    static const auto fwd = op<NormSig>("mineral::group_norm_act");
    const BelowAutograd below;
    return fwd.redispatch(ks & c10::after_autograd_keyset, x, groups, w, b, eps, act);
  }
  const int64_t needs = x.requires_grad() | (of(w).defined() && w->requires_grad()) << 1 | (of(b).defined() && b->requires_grad()) << 2;
  return GroupNormAct::apply(x, w, b, groups, eps, (int64_t)act_of("group_norm_act", act), needs);
}
Tensor group_norm_act_cpu(const Tensor& x, int64_t groups, const OptT& w, const OptT& b, double eps, Name act) {
  norm_of("group_norm_act", x, groups, of(w), of(b), eps, act_of("group_norm_act", act));
  no_cpu("group_norm_act");
}
std::tuple<Tensor, Tensor> group_norm_act_stats_cpu(const Tensor& x, int64_t groups, const OptT& w, const OptT& b, double eps, int64_t act) {
  norm_of("group_norm_act", x, groups, of(w), of(b), eps, (int)act);
  no_cpu("group_norm_act");
}

// ---- linear layer ----------------------------------------------------------------------------------------------------------------------
struct Linear {
  mrl_linear p;
  Tensor x;       // as rows

  Linear(const char* what, const Tensor& x_, const Tensor& w, const Tensor& b, const Tensor& r, int act) {
    p.dtype = dtype_of(what, x_);
    NEED(what, x_.dim() >= 1 && w.dim() == 2 && w.size(1) == x_.size(-1), "x [.., inputs] and weight [outputs, inputs], got ", x_.sizes(), ", ", w.sizes());
    const int64_t K = x_.size(-1), N = w.size(0);
    same_device(what, x_, {&w, &b, &r});
    const std::pair<const char*, const Tensor*> named[] = {{"weight", &w}, {"bias", &b}, {"residual", &r}};
    for (const auto& n : named)
      NEED(what, !n.second->defined() || n.second->scalar_type() == x_.scalar_type(), n.first, ": ", x_.scalar_type(), " like x, got ", n.second->scalar_type());
    NEED(what, K <= (1 << 24) && N <= (1 << 24), "weight of ", w.sizes());
    NEED(what, !b.defined() || (b.dim() == 1 && b.size(0) == N), "bias: [", N, "], got ", b.sizes());
    int64_t rows = 1;
    for (int64_t i = 0; i + 1 < x_.dim(); ++i) rows *= x_.size(i);
    bool same = !r.defined() || (r.dim() == x_.dim() && r.size(-1) == N);
    for (int64_t i = 0; same && r.defined() && i + 1 < x_.dim(); ++i) same = r.size(i) == x_.size(i);
    NEED(what, same, "residual: the output's shape, got ", r.sizes(), " beside x ", x_.sizes(), " and ", N, " outputs; expand a broadcast one");
    x = x_.dim() == 2 ? x_ : x_.reshape({rows, K});
    if ((K != 1 && x.stride(1) != 1) || (rows > 1 && x.stride(0) < K)) x = x.contiguous();
    p.rows = rows; p.x_stride = rows > 1 ? x.stride(0) : K;
    p.inputs = (int32_t)K; p.outputs = (int32_t)N; p.act = act;
  }
  at::DimVector out_shape(const Tensor& x_) const {
    at::DimVector s(x_.sizes().begin(), x_.sizes().end());
    s.back() = p.outputs;
    return s;
  }
};

std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w_, const Tensor& b_, const Tensor& r_, int act, bool keep) {
  const char* what = "linear_act";
  const Linear d(what, x, w_, b_, r_, act);
  c10::DeviceGuard guard(x.device());
  const Tensor w = w_.contiguous(), b = contiguous(b_), r = contiguous(r_);
  const auto shape = d.out_shape(x);
  Tensor y = new_like(x, shape), slope = keep && act != MRL_ACT_NONE ? new_like(x, shape) : Tensor();   // 16 or 32 bits each, like x
  check(mrl_linear_act(&d.p, cp(d.x), cp(w), cp(b), cp(r), mp(y), mp(slope), stream_of(x)), what);
  return {y, slope};
}

Tensor linear_act(const Tensor& x, const Tensor& w, const OptT& b, const OptT& r, Name act) {
  return std::get<0>(linear_forward(x, w, of(b), of(r), act_of("linear_act", act), false));
}
using LinearSig = Tensor(const Tensor&, const Tensor&, const OptT&, const OptT&, Name);

std::tuple<Tensor, Tensor> linear_act_slope(const Tensor& x, const Tensor& w, const OptT& b, const OptT& r, int64_t act) {
  TORCH_CHECK_VALUE(act != MRL_ACT_NONE, "linear_act: no activation, no slope");
  return linear_forward(x, w, of(b), of(r), (int)act, true);
}
using LinearSlopeSig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const OptT&, const OptT&, int64_t);

// The gradients that `needs` names (1 x, 2 weight, 4 bias), in this order.
std::vector<Tensor> linear_act_backward(const Tensor& dy_, const Tensor& x, const Tensor& w_, const OptT& slope, int64_t act, int64_t needs) {
  const char* what = "linear_act_backward";
  const Linear d(what, x, w_, none, none, (int)act);
  c10::DeviceGuard guard(x.device());
  Tensor dx, dw, db;
  if (needs & 1) dx = new_like(x, x.sizes());
  if (needs & 2) dw = new_like(w_, w_.sizes());
  if (needs & 4) db = new_like(x, {d.p.outputs});
  if (d.p.outputs == 0) {
    if (dx.defined()) dx.zero_();
  } else {
    const Tensor w = w_.contiguous(), dy = dy_.contiguous();
    const Workspace ws(what, mrl_linear_act_backward_workspace_bytes(&d.p), dy);
    check(mrl_linear_act_backward(&d.p, cp(d.x), cp(w), cp(of(slope)), cp(dy), mp(dx), mp(dw), mp(db), ws.p(), ws.n, stream_of(dy)), what);
  }
  return asked(needs, {dx, dw, db});
}
using LinearBackwardSig = std::vector<Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptT&, int64_t, int64_t);

struct LinearAct : Function<LinearAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptT& b, const OptT& r, Name name, int64_t needs) {
    const int act = act_of("linear_act", name);
    const BelowAutograd below;
    Tensor y, slope;
    if (act != MRL_ACT_NONE && needs & 7) {
      static const auto fwd = op<LinearSlopeSig>("mineral::_linear_act_slope");
      std::tie(y, slope) = fwd.call(x, w, b, r, act);
    } else {
      static const auto fwd = op<LinearSig>("mineral::linear_act");
      y = fwd.call(x, w, b, r, name);
    }
    ctx->save_for_backward({x, w, slope});
    ctx->saved_data["act"] = (int64_t)act;
    ctx->saved_data["needs"] = needs;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    static const auto bwd = op<LinearBackwardSig>("mineral::_linear_act_backward");
    once("linear_act");
    no_tangent("linear_act", {&g[0]});
    variable_list res(6);
    const int64_t needs = ctx->saved_data["needs"].toInt();
    if (needs & 8) res[3] = g[0];
    if (!(needs & 7)) return res;
    const BelowAutograd below;
    const auto t = ctx->get_saved_variables();
    const auto got = bwd.call(g[0], t[0], t[1], opt(t[2]), ctx->saved_data["act"].toInt(), needs & 7);
    place(needs & 7, got, {&res[0], &res[1], &res[2]});
    return res;
  }
};

Tensor linear_act_autograd(c10::DispatchKeySet ks, const Tensor& x, const Tensor& w, const OptT& b, const OptT& r, Name act) {
  no_tangent("linear_act", {&x, &w, &of(b), &of(r)});
  if (!wants_grad({&x, &w, &of(b), &of(r)})) {
    static const auto fwd = op<LinearSig>("mineral::linear_act");
    const BelowAutograd below;
    return fwd.redispatch(ks & c10::after_autograd_keyset, x, w, b, r, act);
  }
  const int64_t needs = x.requires_grad() | w.requires_grad() << 1 | (of(b).defined() && b->requires_grad()) << 2 | (of(r).defined() && r->requires_grad()) << 3;
  return LinearAct::apply(x, w, b, r, act, needs);
}
Tensor linear_act_cpu(const Tensor& x, const Tensor& w, const OptT& b, const OptT& r, Name act) {
  const Linear d("linear_act", x, w, of(b), of(r), act_of("linear_act", act));
  no_cpu("linear_act");
}
std::tuple<Tensor, Tensor> linear_act_slope_cpu(const Tensor& x, const Tensor& w, const OptT& b, const OptT& r, int64_t act) {
  const Linear d("linear_act", x, w, of(b), of(r), (int)act);
  no_cpu("linear_act");
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(mineral, m) {
  m.set_python_module("mineral_amd.memory_ops");            // where the shape functions are
  m.def("linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? resets=None, Tensor? initial_state=None, float scale=1.0) -> (Tensor, Tensor)");
  m.def("linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, Tensor? resets=None, float scale=1.0) -> Tensor");
  m.def("group_norm_act(Tensor x, int num_groups, Tensor? weight=None, Tensor? bias=None, float eps=1e-05, str? act_type=None) -> Tensor");
  m.def("linear_act(Tensor x, Tensor weight, Tensor? bias=None, Tensor? residual=None, str? act_type=None) -> Tensor");
  // the halves of a differentiable call
  m.def("_linear_attention_backward(Tensor? d_out, Tensor? d_final, Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? resets, Tensor? initial_state, float scale, int needs) -> Tensor[]");
  m.def("_group_norm_act_stats(Tensor x, int num_groups, Tensor? weight, Tensor? bias, float eps, int act) -> (Tensor, Tensor)");
  m.def("_group_norm_act_backward(Tensor dy, Tensor x, Tensor stats, Tensor? weight, Tensor? bias, int num_groups, float eps, int act, int needs) -> Tensor[]");
  m.def("_linear_act_slope(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int act) -> (Tensor, Tensor)");
  m.def("_linear_act_backward(Tensor dy, Tensor x, Tensor weight, Tensor? slope, int act, int needs) -> Tensor[]");
}
TORCH_LIBRARY_IMPL(mineral, CUDA, m) {
  m.impl("linear_attention", linear_attention);
  m.impl("linear_attention_step", linear_attention_step);
  m.impl("group_norm_act", group_norm_act);
  m.impl("linear_act", linear_act);
  m.impl("_linear_attention_backward", attention_backward);
  m.impl("_group_norm_act_stats", group_norm_act_stats);
  m.impl("_group_norm_act_backward", group_norm_act_backward);
  m.impl("_linear_act_slope", linear_act_slope);
  m.impl("_linear_act_backward", linear_act_backward);
}
TORCH_LIBRARY_IMPL(mineral, Autograd, m) {
  m.impl("linear_attention", linear_attention_autograd);
  m.impl("linear_attention_step", linear_attention_step_autograd);
  m.impl("group_norm_act", group_norm_act_autograd);
  m.impl("linear_act", linear_act_autograd);
}
TORCH_LIBRARY_IMPL(mineral, ADInplaceOrView, m) { m.impl("linear_attention_step", linear_attention_step_inplace); }
TORCH_LIBRARY_IMPL(mineral, Negative, m) { m.impl("linear_attention_step", linear_attention_step_negated); }
TORCH_LIBRARY_IMPL(mineral, CPU, m) {
  m.impl("linear_attention", linear_attention_cpu);
  m.impl("linear_attention_step", linear_attention_step);
  m.impl("group_norm_act", group_norm_act_cpu);
  m.impl("linear_act", linear_act_cpu);
  m.impl("_group_norm_act_stats", group_norm_act_stats_cpu);
  m.impl("_linear_act_slope", linear_act_slope_cpu);
}
