// The state-space sequence operators as torch functions with autograd (module vit_amd._ssm, used by vit_amd/ssm.py) on the C
// entry points of librvit.  In C++ because these operators are also called one token at a time and in training steps of short
// windows, where the checks, allocations and argument conversions of a Python wrapper and a Python autograd node take
// several times the kernels' time (a token's scan: 13.4 us, here 5.5, its launch alone 4; a training step of 64 windows of 8 tokens,
// fp32: 207 us, here 105, its kernels 56).
// Nothing is kept from one call for the next.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/rvit.h"

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef optional<Tensor> Opt;

namespace {

// ---- arguments ----
Tensor get(const Opt& t) { return t.has_value() ? *t : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int64_t stride(const Tensor& t, int d) { return t.defined() ? t.stride(d) : 0; }
int dtype(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? RVIT_BF16 : RVIT_F32; }
bool any_type(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
void* stream(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
Tensor like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor bytes(int64_t n, const Tensor& t) { return at::empty({n}, t.options().dtype(at::kByte)); }

void done(int status, const char* what) {
  TORCH_CHECK_VALUE(status != RVIT_EINVAL, what, ": ", rvit_last_error());
  TORCH_CHECK(status == 0, what, " failed with status ", status, ": ", rvit_last_error());
}

void check_f32(const Tensor& t, at::IntArrayRef shape, const char* op, const char* name) {
  TORCH_CHECK_VALUE(!t.defined() || (t.scalar_type() == at::kFloat && t.sizes() == shape && t.is_contiguous()), op, ": ", name, " must be contiguous float32 ",
                    shape, ", got ", t.scalar_type(), " ", t.sizes());
}
void check_like(const Tensor& t, const Tensor& x, at::IntArrayRef shape, const char* op, const char* name) {
  TORCH_CHECK_VALUE(!t.defined() || (t.scalar_type() == x.scalar_type() && t.sizes() == shape && t.is_contiguous()), op, ": ", name, " must be contiguous ",
                    x.scalar_type(), " ", shape, ", got ", t.scalar_type(), " ", t.sizes());
}
void check_lengths(const Tensor& t, int64_t B, const char* op) {
  TORCH_CHECK_VALUE(!t.defined() || (t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == B && t.is_contiguous()), op,
                    ": lengths must be contiguous int32 [", B, "], got ", t.scalar_type(), " ", t.sizes());
}
// (a result of a kernel has no tangent, which reads as a tangent of zero)
void no_tangent(const char* op, const Tensor& t) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), op, ": no forward-mode derivatives (torch.autograd.forward_ad)");
}
void check_gpu(const char* op, std::initializer_list<Tensor> ts) {
  // (a trace holds torch operations: the allocation of a result, and nothing that fills it)
  TORCH_CHECK(!torch::jit::tracer::isTracing(), op, ": torch.jit.trace cannot record it");
  const at::Device dev = ts.begin()->device();
  for (const Tensor& t : ts) {
    TORCH_CHECK_VALUE(!t.defined() || t.device() == dev, op, ": tensors on ", dev, " and ", t.device());
    no_tangent(op, t);
  }
  TORCH_CHECK(dev.is_cuda(), "vit_amd ops run only on the GPU (HIP); got a CPU tensor. There is no CPU fallback.");
}
int size(int64_t n, const char* op) {
  TORCH_CHECK_VALUE(n < (1ll << 31), op, ": a dimension of ", n);
  return (int)n;
}
// t with its last `inner` dimensions packed (a copy only where they are not)
Tensor packed(const Tensor& t, int inner) {
  if (!t.defined()) return t;
  int64_t step = 1;
  for (int d = 1; d <= inner && d <= t.dim(); ++d) {
    if (t.size(-d) != 1 && t.stride(-d) != step) return t.contiguous();
    step *= t.size(-d);
  }
  return t;
}
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
void no_gradient(const char* op, std::initializer_list<Tensor> ts) {
  TORCH_CHECK(!wants_grad(ts), op, ": has no gradient, and an input requires one (torch.no_grad(), or detach it)");
}
void first_order(const char* op, const variable_list& g) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": no second derivatives (create_graph=True)");
  for (const Tensor& t : g) no_tangent(op, t);
}
// a state that a kernel advanced in place: a graph that saved it must notice
void advanced(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Opt some(const Tensor& t) { return t.defined() ? Opt(t) : Opt(); }

// ---- short causal convolution ----
void conv_shapes(const char* op, const Tensor& x, const Tensor& w, const Tensor& bias, bool step) {
  TORCH_CHECK_VALUE(x.dim() == (step ? 2 : 3) && any_type(x), op, ": x must be bf16 / f32 ", step ? "[B,C]" : "[B,T,C]", ", got ", x.scalar_type(), " ", x.sizes());
  const int64_t C = x.size(-1);
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == C && w.size(1) >= 2 && w.size(1) <= 6 && C >= 1, op, ": weight must be [C=", C, ", 2..6], got ",
                    w.sizes());
  check_f32(w, w.sizes(), op, "weight");
  check_f32(bias, {C}, op, "bias");
}

std::pair<Tensor, Tensor> conv_run(const Tensor& x, const Tensor& w, const Tensor& bias, bool silu, const Tensor& state, const Tensor& lengths, bool want_state) {
  const c10::DeviceGuard guard(x.device());
  const int64_t B = x.size(0), T = x.size(1), C = x.size(2), K = w.size(1);
  Tensor y = like(x), after;
  if (want_state) after = at::empty({B, K - 1, C}, x.options());
  if (B == 0 || T == 0) {      // no tokens: nothing runs, the kept inputs stay
    if (want_state) state.defined() ? after.copy_(state) : after.zero_();
    return {y, after};
  }
  done(rvit_ssm_conv_fwd(ptr(x), x.stride(0), x.stride(1), w.data_ptr<float>(), (const float*)ptr(bias), ptr(state), (const int*)ptr(lengths), ptr(y), ptr(after),
                         dtype(x), size(B, "causal_conv"), size(T, "causal_conv"), size(C, "causal_conv"), (int)K, silu, stream(x)),
       "rvit_ssm_conv_fwd");
  return {y, after};
}

struct Conv : torch::autograd::Function<Conv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opt& bias_, bool silu, const Opt& state_, const Opt& lengths_,
                               bool want_state) {
    const Tensor bias = get(bias_), state = get(state_), lengths = get(lengths_);
    const char* op = "causal_conv";
    int64_t nb = 0;      // (what the backward pass cannot take is refused here)
    if (x.numel())
      done(rvit_ssm_conv_bwd_workspace(&nb, size(x.size(0), op), size(x.size(1), op), size(x.size(2), op), (int)w.size(1)), "rvit_ssm_conv_bwd_workspace");
    auto out = conv_run(x, w, bias, silu, state, lengths, want_state);
    ctx->save_for_backward({x, w, bias, state, lengths});
    ctx->saved_data["silu"] = silu;
    ctx->set_materialize_grads(false);
    if (want_state) return {out.first, out.second};
    return {out.first};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("causal_conv", g);
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &bias = s[2], &state = s[3], &lengths = s[4];
    const c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2), K = w.size(1);
    Tensor dx = like(x), dw = like(w), db = bias.defined() ? like(bias) : Tensor(), ds = state.defined() ? like(state) : Tensor();
    const Tensor dafter = g.size() > 1 ? dense(g[1]) : Tensor();
    if (B == 0 || T == 0) {
      dw.zero_();
      if (db.defined()) db.zero_();
      if (ds.defined()) dafter.defined() ? ds.copy_(dafter) : ds.zero_();
    } else {
      const Tensor dy = g[0].defined() ? packed(g[0], 1) : at::zeros(x.sizes(), x.options());
      int64_t nb = 0;
      done(rvit_ssm_conv_bwd_workspace(&nb, (int)B, (int)T, (int)C, (int)K), "rvit_ssm_conv_bwd_workspace");
      const Tensor ws = bytes(nb, x);
      done(rvit_ssm_conv_bwd(ptr(x), x.stride(0), x.stride(1), w.data_ptr<float>(), (const float*)ptr(bias), ptr(state), (const int*)ptr(lengths), ptr(dy),
                             dy.stride(0), dy.stride(1), ptr(dafter), ptr(dx), dw.data_ptr<float>(), (float*)ptr(db), ptr(ds), ptr(ws), nb, dtype(x), (int)B, (int)T,
                             (int)C, (int)K, ctx->saved_data["silu"].toBool(), stream(x)),
           "rvit_ssm_conv_bwd");
    }
    return {dx, dw, db, Tensor(), ds, Tensor(), Tensor()};
  }
};

std::pair<Tensor, Opt> conv(Tensor x, const Tensor& w, const Opt& bias_, bool silu, const Opt& state_, const Opt& lengths_, bool want_state) {
  const Tensor bias = get(bias_), state = dense(get(state_)), lengths = get(lengths_);
  conv_shapes("causal_conv", x, w, bias, false);
  check_like(state, x, {x.size(0), w.size(1) - 1, x.size(2)}, "causal_conv", "state");
  check_lengths(lengths, x.size(0), "causal_conv");
  check_gpu("causal_conv", {x, w, bias, state, lengths});
  x = packed(x, 1);
  if (wants_grad({x, w, bias, state})) {
    const variable_list out = Conv::apply(x, w, some(bias), silu, some(state), some(lengths), want_state);
    return {out[0], want_state ? Opt(out[1]) : Opt()};
  }
  auto out = conv_run(x, w, bias, silu, state, lengths, want_state);
  return {out.first, some(out.second)};
}

Tensor conv_step(Tensor x, const Tensor& w, const Opt& bias_, const Tensor& state, bool silu) {
  const Tensor bias = get(bias_);
  conv_shapes("causal_conv_step", x, w, bias, true);
  check_like(state, x, {x.size(0), w.size(1) - 1, x.size(1)}, "causal_conv_step", "state");
  no_gradient("causal_conv_step", {x, w, bias, state});
  check_gpu("causal_conv_step", {x, w, bias, state});
  const c10::DeviceGuard guard(x.device());
  x = packed(x, 1);
  const Tensor y = like(x);
  if (x.size(0) == 0) return y;
  done(rvit_ssm_conv_step(ptr(x), x.stride(0), w.data_ptr<float>(), (const float*)ptr(bias), ptr(state), ptr(y), dtype(x), size(x.size(0), "causal_conv_step"),
                          size(x.size(1), "causal_conv_step"), (int)w.size(1), silu, stream(x)),
       "rvit_ssm_conv_step");
  advanced(state);
  return y;
}

// ---- selective scan ----
struct Dims {
  int B, T, H, P, G, N;
  Dims(const Tensor& x, const Tensor& Bm, bool step)
      : B(size(x.size(0), "selective_scan")), T(step ? 1 : size(x.size(1), "selective_scan")), H(size(x.size(-2), "selective_scan")),
        P(size(x.size(-1), "selective_scan")), G((int)Bm.size(-2)), N((int)Bm.size(-1)) {}
};

void scan_shapes(const char* op, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm, const Tensor& D, const Tensor& z,
                 const Tensor& dt_bias, bool step) {
  const int lead = step ? 1 : 2;
  TORCH_CHECK_VALUE(x.dim() == lead + 2 && any_type(x), op, ": x must be bf16 / f32 ", step ? "[B,H,P]" : "[B,T,H,P]", ", got ", x.scalar_type(), " ", x.sizes());
  TORCH_CHECK_VALUE(Bm.dim() == lead + 2 && Bm.sizes() == Cm.sizes() && Bm.sizes().slice(0, lead) == x.sizes().slice(0, lead), op, ": Bm and Cm must be ",
                    step ? "[B,G,N]" : "[B,T,G,N]", ", got ", Bm.sizes(), " and ", Cm.sizes());
  const int64_t H = x.size(-2), P = x.size(-1), G = Bm.size(-2), N = Bm.size(-1);
  TORCH_CHECK_VALUE(H >= 1 && P >= 1 && G >= 1 && N >= 1 && H % G == 0 && N <= 128, op, ": ", H, " heads in ", G, " groups, ", P, " channels, ", N,
                    " states (at most 128)");
  TORCH_CHECK_VALUE(dt.sizes() == x.sizes().slice(0, lead + 1), op, ": dt must be ", x.sizes().slice(0, lead + 1), ", got ", dt.sizes());
  TORCH_CHECK_VALUE(!z.defined() || z.sizes() == x.sizes(), op, ": z must be ", x.sizes(), ", got ", z.sizes());
  for (const Tensor* t : {&dt, &Bm, &Cm, &z})
    TORCH_CHECK_VALUE(!t->defined() || t->scalar_type() == x.scalar_type(), op, ": x, dt, Bm, Cm, z of one dtype, got ", x.scalar_type(), " and ", t->scalar_type());
  check_f32(A, {H}, op, "A");
  check_f32(D, {H}, op, "D");
  check_f32(dt_bias, {H}, op, "dt_bias");
}

struct ScanOut { Tensor y, after, v, states; };

ScanOut scan_run(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm, const Tensor& D, const Tensor& z, const Tensor& dt_bias,
                 const Tensor& state, const Tensor& lengths, bool want_state, bool train) {
  const c10::DeviceGuard guard(x.device());
  ScanOut o;
  o.y = like(x);
  if (x.size(0) == 0) {      // no samples: nothing runs
    if (want_state) o.after = at::empty({0, x.size(2), x.size(3), Bm.size(3)}, A.options());
    return o;
  }
  const Dims d(x, Bm, false);
  int64_t fwd = 0, floats = 0, bwd = 0;
  done(rvit_ssm_scan_plan(&fwd, &floats, train ? &bwd : nullptr, d.B, d.T, d.H, d.P, d.G, d.N), "rvit_ssm_scan_plan");
  if (want_state) o.after = at::empty({d.B, d.H, d.P, d.N}, A.options());
  if (train && z.defined()) o.v = at::empty(x.sizes(), A.options());
  if (train) o.states = at::empty({floats}, A.options());
  const Tensor ws = fwd > 16 ? bytes(fwd, x) : Tensor();
  done(rvit_ssm_scan_fwd(ptr(x), x.stride(0), x.stride(1), ptr(dt), dt.stride(0), dt.stride(1), A.data_ptr<float>(), ptr(Bm), Bm.stride(0), Bm.stride(1), ptr(Cm),
                         Cm.stride(0), Cm.stride(1), (const float*)ptr(D), ptr(z), stride(z, 0), stride(z, 1), (const float*)ptr(dt_bias), (const float*)ptr(state),
                         (const int*)ptr(lengths), ptr(o.y), (float*)ptr(o.v), (float*)ptr(o.after), (float*)ptr(o.states), ptr(ws), fwd, dtype(x), d.B, d.T, d.H, d.P, d.G,
                         d.N, stream(x)),
       "rvit_ssm_scan_fwd");
  return o;
}

struct Scan : torch::autograd::Function<Scan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& Bm, const Tensor& Cm, const Opt& D_,
                               const Opt& z_, const Opt& dt_bias_, const Opt& state_, const Opt& lengths_, bool want_state) {
    const Tensor D = get(D_), z = get(z_), dt_bias = get(dt_bias_), state = get(state_), lengths = get(lengths_);
    const ScanOut o = scan_run(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, want_state, true);
    ctx->save_for_backward({x, dt, A, Bm, Cm, D, z, dt_bias, lengths, o.v, o.states});
    ctx->saved_data["state"] = state.defined();
    ctx->set_materialize_grads(false);
    if (want_state) return {o.y, o.after};
    return {o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("selective_scan", g);
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &dt = s[1], &A = s[2], &Bm = s[3], &Cm = s[4], &D = s[5], &z = s[6], &dt_bias = s[7], &lengths = s[8], &v = s[9], &states = s[10];
    const c10::DeviceGuard guard(x.device());
    const Dims d(x, Bm, false);
    Tensor dx = like(x), ddt = like(dt), dB = like(Bm), dC = like(Cm), dA = like(A);
    Tensor dz = z.defined() ? like(x) : Tensor(), dD = D.defined() ? like(D) : Tensor(), dbias = dt_bias.defined() ? like(dt_bias) : Tensor();
    Tensor ds = ctx->saved_data["state"].toBool() ? at::empty({d.B, d.H, d.P, d.N}, A.options()) : Tensor();
    const Tensor dafter = g.size() > 1 ? dense(g[1]) : Tensor();
    if (d.B == 0 || d.T == 0) {
      for (const Tensor& t : {dA, dD, dbias})
        if (t.defined()) t.zero_();
      if (ds.defined()) dafter.defined() ? ds.copy_(dafter) : ds.zero_();
    } else {
      const Tensor dy = g[0].defined() ? packed(g[0], 2) : at::zeros(x.sizes(), x.options());
      int64_t nb = 0;
      done(rvit_ssm_scan_plan(nullptr, nullptr, &nb, d.B, d.T, d.H, d.P, d.G, d.N), "rvit_ssm_scan_plan");
      const Tensor ws = bytes(nb, x);
      done(rvit_ssm_scan_bwd(ptr(x), x.stride(0), x.stride(1), ptr(dt), dt.stride(0), dt.stride(1), A.data_ptr<float>(), ptr(Bm), Bm.stride(0), Bm.stride(1), ptr(Cm),
                             Cm.stride(0), Cm.stride(1), (const float*)ptr(D), ptr(z), stride(z, 0), stride(z, 1), (const float*)ptr(dt_bias),
                             (const int*)ptr(lengths), (const float*)ptr(v), (const float*)ptr(states), ptr(dy), dy.stride(0), dy.stride(1), (const float*)ptr(dafter), ptr(dx),
                             ptr(ddt), dA.data_ptr<float>(), ptr(dB), ptr(dC), (float*)ptr(dD), ptr(dz), (float*)ptr(dbias), (float*)ptr(ds), ptr(ws), nb, dtype(x),
                             d.B, d.T, d.H, d.P, d.G, d.N, stream(x)),
           "rvit_ssm_scan_bwd");
    }
    return {dx, ddt, dA, dB, dC, dD, dz, dbias, ds, Tensor(), Tensor()};
  }
};

std::pair<Tensor, Opt> scan(Tensor x, Tensor dt, const Tensor& A, Tensor Bm, Tensor Cm, const Opt& D_, const Opt& z_, const Opt& dt_bias_, const Opt& state_,
                            const Opt& lengths_, bool want_state) {
  const Tensor D = get(D_), dt_bias = get(dt_bias_), state = dense(get(state_)), lengths = get(lengths_);
  Tensor z = get(z_);
  scan_shapes("selective_scan", x, dt, A, Bm, Cm, D, z, dt_bias, false);
  check_f32(state, {x.size(0), x.size(2), x.size(3), Bm.size(3)}, "selective_scan", "state");
  check_lengths(lengths, x.size(0), "selective_scan");
  check_gpu("selective_scan", {x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths});
  x = packed(x, 2);
  dt = packed(dt, 1);
  Bm = packed(Bm, 2);
  Cm = packed(Cm, 2);
  z = packed(z, 2);
  if (wants_grad({x, dt, A, Bm, Cm, D, z, dt_bias, state})) {
    const variable_list out = Scan::apply(x, dt, A, Bm, Cm, some(D), some(z), some(dt_bias), some(state), some(lengths), want_state);
    return {out[0], want_state ? Opt(out[1]) : Opt()};
  }
  const ScanOut o = scan_run(x, dt, A, Bm, Cm, D, z, dt_bias, state, lengths, want_state, false);
  return {o.y, some(o.after)};
}

Tensor scan_step(Tensor x, Tensor dt, const Tensor& A, Tensor Bm, Tensor Cm, const Tensor& state, const Opt& D_, const Opt& z_, const Opt& dt_bias_) {
  const Tensor D = get(D_), dt_bias = get(dt_bias_);
  Tensor z = get(z_);
  scan_shapes("selective_scan_step", x, dt, A, Bm, Cm, D, z, dt_bias, true);
  check_f32(state, {x.size(0), x.size(1), x.size(2), Bm.size(2)}, "selective_scan_step", "state");
  no_gradient("selective_scan_step", {x, dt, A, Bm, Cm, D, z, dt_bias, state});
  check_gpu("selective_scan_step", {x, dt, A, Bm, Cm, D, z, dt_bias, state});
  const c10::DeviceGuard guard(x.device());
  x = packed(x, 2);
  dt = packed(dt, 1);
  Bm = packed(Bm, 2);
  Cm = packed(Cm, 2);
  z = packed(z, 2);
  const Dims d(x, Bm, true);
  const Tensor y = like(x);
  if (d.B == 0) return y;
  done(rvit_ssm_scan_step(ptr(x), x.stride(0), ptr(dt), dt.stride(0), A.data_ptr<float>(), ptr(Bm), Bm.stride(0), ptr(Cm), Cm.stride(0), (const float*)ptr(D), ptr(z),
                          stride(z, 0), (const float*)ptr(dt_bias), (float*)ptr(state), ptr(y), dtype(x), d.B, d.H, d.P, d.G, d.N, stream(x)),
       "rvit_ssm_scan_step");
  advanced(state);
  return y;
}

// ---- norms around a block ----
int sandwich_shapes(const Tensor& residual, const Tensor& y, const Tensor& pw, const Tensor& pb, const Tensor& nw, const Tensor& nb, const Tensor& gate) {
  const char* op = "sandwich_norm";
  TORCH_CHECK_VALUE(any_type(residual) && any_type(y) && residual.sizes() == y.sizes(), op, ": residual and y must be bf16 / f32 of one shape, got ",
                    residual.scalar_type(), " ", residual.sizes(), " and ", y.scalar_type(), " ", y.sizes());
  const int64_t E = y.dim() ? y.size(-1) : 0;
  TORCH_CHECK_VALUE(y.dim() >= 2 && E >= 1 && E <= 4096, op, ": y must be [..., E] with E <= 4096, got ", y.sizes());
  check_f32(pw, {E}, op, "post_weight");
  check_f32(pb, {E}, op, "post_bias");
  check_f32(nw, {E}, op, "pre_weight");
  check_f32(nb, {E}, op, "pre_bias");
  if (!gate.defined()) return 0;
  TORCH_CHECK_VALUE(gate.scalar_type() == at::kFloat || gate.scalar_type() == y.scalar_type(), op, ": gate must be float32 or ", y.scalar_type(), ", got ",
                    gate.scalar_type());
  if (gate.dim() == 1 && gate.size(0) == E) return 1;
  if (gate.sizes() == y.sizes()) return 3;
  TORCH_CHECK_VALUE(y.dim() == 3 && gate.dim() == 2 && gate.size(0) == y.size(0) && gate.size(1) == E, op, ": gate must be [E], [B,E] (with y [B,T,E]) or like y ",
                    y.sizes(), ", got ", gate.sizes());
  return y.size(1) == 1 ? 3 : 2;      // (samples of one row: the rows' own gates)
}

std::pair<Tensor, Tensor> sandwich_run(const Tensor& residual, const Tensor& y, const Tensor& pw, const Tensor& pb, const Tensor& nw, const Tensor& nb,
                                       const Tensor& gate, int kind, double scale, bool rms, double eps, const Tensor& stats) {
  const c10::DeviceGuard guard(y.device());
  Tensor h = like(residual), n = like(y);
  const int64_t E = y.size(-1), rows = y.numel() / E;
  if (rows)
    done(rvit_sandwich_norm_fwd(ptr(residual), dtype(residual), ptr(y), dtype(y), ptr(gate), kind, gate.defined() ? dtype(gate) : RVIT_F32, (float)scale,
                                pw.data_ptr<float>(), (const float*)ptr(pb), nw.data_ptr<float>(), (const float*)ptr(nb), (float)eps, rms, ptr(h), ptr(n),
                                (float*)ptr(stats), rows, size(y.size(-2), "sandwich_norm"), (int)E, stream(y)),
         "rvit_sandwich_norm_fwd");
  return {h, n};
}

struct Sandwich : torch::autograd::Function<Sandwich> {
  static variable_list forward(AutogradContext* ctx, const Tensor& residual, const Tensor& y, const Tensor& pw, const Opt& pb_, const Tensor& nw, const Opt& nb_,
                               const Opt& gate_, int64_t kind, double scale, bool rms, double eps) {
    const Tensor pb = get(pb_), nb = get(nb_), gate = get(gate_);
    const int64_t rows = y.numel() / y.size(-1);
    int64_t nbytes = 0;      // (what the backward pass cannot take is refused here)
    if (rows)
      done(rvit_sandwich_norm_bwd_workspace(&nbytes, rows, size(y.size(-2), "sandwich_norm"), (int)y.size(-1), (int)kind), "rvit_sandwich_norm_bwd_workspace");
    const Tensor stats = at::empty({rows, 4}, pw.options());
    const auto out = sandwich_run(residual, y, pw, pb, nw, nb, gate, (int)kind, scale, rms, eps, stats);
    ctx->save_for_backward({residual, y, pw, pb, nw, nb, gate, stats});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["rms"] = rms;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    return {out.first, out.second};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("sandwich_norm", g);
    const auto s = ctx->get_saved_variables();
    const Tensor &residual = s[0], &y = s[1], &pw = s[2], &pb = s[3], &nw = s[4], &nb = s[5], &gate = s[6], &stats = s[7];
    const c10::DeviceGuard guard(y.device());
    const Tensor dh = g[0].defined() ? g[0].contiguous() : at::zeros(residual.sizes(), residual.options());
    const Tensor dn = g[1].defined() ? g[1].contiguous() : at::zeros(y.sizes(), y.options());
    Tensor dres = like(residual), dy = like(y), dpw = like(pw), dnw = like(nw);
    Tensor dpb = pb.defined() ? like(pb) : Tensor(), dnb = nb.defined() ? like(nb) : Tensor(), dg = gate.defined() ? like(gate) : Tensor();
    const int64_t E = y.size(-1), rows = y.numel() / E;
    if (rows == 0) {
      for (const Tensor& t : {dpw, dnw, dpb, dnb, dg})
        if (t.defined()) t.zero_();
    } else {
      const int kind = (int)ctx->saved_data["kind"].toInt(), T = (int)y.size(-2);
      int64_t nbytes = 0;
      done(rvit_sandwich_norm_bwd_workspace(&nbytes, rows, T, (int)E, kind), "rvit_sandwich_norm_bwd_workspace");
      const Tensor ws = bytes(nbytes, y);
      done(rvit_sandwich_norm_bwd(ptr(residual), dtype(residual), ptr(y), dtype(y), ptr(gate), kind, gate.defined() ? dtype(gate) : RVIT_F32,
                                  (float)ctx->saved_data["scale"].toDouble(), pw.data_ptr<float>(), (const float*)ptr(pb), nw.data_ptr<float>(),
                                  (const float*)ptr(nb), (float)ctx->saved_data["eps"].toDouble(), ctx->saved_data["rms"].toBool(), stats.data_ptr<float>(), ptr(dh),
                                  ptr(dn), ptr(dres), ptr(dy), ptr(dg), dpw.data_ptr<float>(), (float*)ptr(dpb), dnw.data_ptr<float>(), (float*)ptr(dnb), ptr(ws),
                                  nbytes, rows, T, (int)E, stream(y)),
           "rvit_sandwich_norm_bwd");
    }
    return {dres, dy, dpw, dpb, dnw, dnb, dg, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::pair<Tensor, Tensor> sandwich(const Tensor& residual_, const Tensor& y_, const Tensor& pw, const Opt& pb_, const Tensor& nw, const Opt& nb_, const Opt& gate_,
                                   double scale, bool rms, double eps) {
  const Tensor pb = get(pb_), nb = get(nb_), gate = dense(get(gate_));
  const int kind = sandwich_shapes(residual_, y_, pw, pb, nw, nb, gate);
  check_gpu("sandwich_norm", {residual_, y_, pw, pb, nw, nb, gate});
  const Tensor residual = residual_.contiguous(), y = y_.contiguous();
  if (wants_grad({residual, y, pw, pb, nw, nb, gate})) {
    const variable_list out = Sandwich::apply(residual, y, pw, some(pb), nw, some(nb), some(gate), (int64_t)kind, scale, rms, eps);
    return {out[0], out[1]};
  }
  return sandwich_run(residual, y, pw, pb, nw, nb, gate, kind, scale, rms, eps, Tensor());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("abi", [] { return RVIT_ABI_VERSION; });
  m.def("conv", &conv);
  m.def("conv_step", &conv_step);
  m.def("scan", &scan);
  m.def("scan_step", &scan_step);
  m.def("sandwich", &sandwich);
}
