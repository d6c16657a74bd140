// gbx_torch.cpp -- the policy operators of include/gbx_hip.h for torch tensors:
// argument checks, outputs, scratch memory, gradients and streams.
//
// A step of a few envs is a few microseconds of GPU work, and a small
// rollout's gradient runs on autograd's own thread: this glue is C++ because
// in Python it takes longer than the kernels do.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <vector>

#include "gbx_hip.h"

namespace {

using at::IntArrayRef;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

struct HipFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void check(int64_t rc) {
  if (rc >= 0) return;
  const std::string what = gbx_last_error();
  TORCH_CHECK_VALUE(rc != GBX_E_INVALID && rc != GBX_E_UNSUPPORTED, what);
  throw HipFailure(what);
}

// ---------------------------------------------------------------- arguments

int elem_of(at::ScalarType t) {
  return t == at::kFloat ? GBX_F32 : t == at::kBFloat16 ? GBX_BF16 : t == at::kHalf ? GBX_F16 : -1;
}
int input(const char* name, const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor, got one on ", t.device());
  const int elem = elem_of(t.scalar_type());
  TORCH_CHECK_VALUE(elem >= 0, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  return elem;
}
Tensor rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
void same_place(const char* name, const Tensor& t, const Tensor& like, IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.device() == like.device(), name, ": expected a tensor on ", like.device(), ", got one on ", t.device());
  TORCH_CHECK_VALUE(t.sizes() == shape, name, ": expected shape ", shape, ", got ", t.sizes());
}
// of x's type and device and the given shape, last dimension contiguous
Tensor like(const char* name, const Tensor& t, const Tensor& x, IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type(), name, ": expected ", x.scalar_type(), ", got ", t.scalar_type());
  same_place(name, t, x, shape);
  return rows(t);
}
Maybe like(const char* name, const Maybe& t, const Tensor& x, IntArrayRef shape) {
  return t ? Maybe(like(name, *t, x, shape)) : t;
}
// a parameter in 32 bits (autograd sees the cast), contiguous
Tensor param(const char* name, const Tensor& t, const Tensor& x, IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.is_floating_point(), name, ": expected a floating-point tensor, got ", t.scalar_type());
  same_place(name, t, x, shape);
  return (t.scalar_type() == at::kFloat ? t : t.to(at::kFloat)).contiguous();
}
Maybe param(const char* name, const Maybe& t, const Tensor& x, IntArrayRef shape) {
  return t ? Maybe(param(name, *t, x, shape)) : t;
}
Maybe starts(const Maybe& t, const Tensor& x, IntArrayRef shape) {
  if (!t) return t;
  TORCH_CHECK_VALUE(t->scalar_type() == at::kBool || t->scalar_type() == at::kByte, "resets: expected bool or uint8, got ", t->scalar_type());
  same_place("resets", *t, x, shape);
  return t->contiguous();
}
Tensor state_of(const Tensor& t, const Tensor& x, at::ScalarType kind, IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.scalar_type() == kind, "state: expected ", kind, ", got ", t.scalar_type());
  same_place("state", t, x, shape);
  return t;
}
bool wants_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}
const Tensor* opt(const Maybe& t) { return t ? &*t : nullptr; }
// (a tangent would be dropped where no autograd function is called: a derivative
// of zero)
void no_tangent(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors) TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(0).defined(), what, " has no forward-mode derivative");
}
Tensor given(const Maybe& t) { return t ? *t : Tensor(); }  // undefined: not given
// (autograd's functions take what is not given as no argument, not as an undefined tensor)
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
void no_grad(const char* what, std::initializer_list<const Tensor*> tensors) {
  TORCH_CHECK(!wants_grad(tensors), what, " has no gradient: call it under torch.no_grad() or with detached tensors");
}
void check_width(const Tensor& weight) {
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) >= 2 && weight.size(1) <= 4, "weight: expected [channels, 2 to 4], got ", weight.sizes());
}
int32_t narrow(const char* name, int64_t v) {
  TORCH_CHECK_VALUE(v <= INT32_MAX, name, ": ", v, " is out of range");
  return (int32_t)v;
}

// ------------------------------------------------------------------ launches

const void* in(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const float* fin(const Tensor& t) { return (const float*)in(t); }
float* fout(const Tensor& t) { return (float*)out(t); }
const uint8_t* bytes(const Tensor& t) { return (const uint8_t*)in(t); }
void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
Tensor floats(const Tensor& x, IntArrayRef shape) { return at::empty(shape, x.options().dtype(at::kFloat)); }
Tensor blank(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }
Tensor zeros(const Tensor& t) { return t.defined() ? at::zeros(t.sizes(), t.options()) : Tensor(); }
// after no steps: what was there before, or zeros
Tensor unmoved(const Tensor& state, const Tensor& like) { return state.defined() ? state.clone() : zeros(like); }
// scratch memory, from the caching allocator like the outputs
Tensor work(const Tensor& x, int64_t count) {
  check(count);
  return count ? floats(x, {count}) : Tensor();
}
// Tells autograd that t changes in place; before the launch, since it raises
// where t may not (an inference tensor outside inference mode).
void will_change(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }
void once() { TORCH_CHECK(!at::GradMode::is_enabled(), "the policy operators are differentiable once: no create_graph"); }

// ------------------------------------------------------------------ the norm

// [..., D] as rows [R, D]
Tensor flat(const Tensor& t) {
  const Tensor r = rows(t);
  return r.dim() == 2 ? r : r.reshape({-1, r.size(-1)});
}
Tensor norm_forward(int elem, const Tensor& x, const Tensor& weight, const Tensor& residual, double eps, const Tensor& y, const Tensor& scale, int group) {
  const c10::DeviceGuard guard(x.device());
  const Tensor summed = residual.defined() ? blank(x) : Tensor();
  if (x.numel() == 0) return summed;
  const Tensor xr = flat(x), rr = residual.defined() ? flat(residual) : Tensor();
  check(gbx_rms_norm(xr.size(0), narrow("channels", x.size(-1)), elem, (float)eps, in(xr), xr.stride(0), in(rr), rr.defined() ? rr.stride(0) : 0,
                     fin(weight), out(y), out(summed), fout(scale), group, stream(x)));
  return summed;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& residual_, double eps, int64_t elem) {
    const Tensor residual = given(residual_);
    ctx->set_materialize_grads(false);
    const Tensor y = blank(x), summed = norm_forward((int)elem, x, weight, residual, eps, y, Tensor(), 0);
    ctx->save_for_backward({residual.defined() ? summed : x, weight});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["elem"] = elem;
    ctx->saved_data["plain"] = !residual.defined();
    return residual.defined() ? variable_list{y, summed} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const auto saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &weight = saved[1];
    const bool plain = ctx->saved_data["plain"].toBool();
    const Tensor dsummed = plain ? Tensor() : grads[1];
    Tensor dx, dweight;
    if (!grads[0].defined() || s.numel() == 0) {  // the sum alone was used, or there are no rows
      dx = dsummed.defined() ? dsummed : at::zeros_like(s);
      dweight = at::zeros_like(weight);
    } else {
      const c10::DeviceGuard guard(s.device());
      const int32_t dim = (int32_t)s.size(-1);
      const Tensor sr = flat(s), dy = flat(grads[0]), ds = dsummed.defined() ? flat(dsummed) : Tensor();
      dx = blank(s);
      dweight = blank(weight);
      const Tensor scratch = work(s, gbx_rms_norm_grad_work(sr.size(0), dim));
      check(gbx_rms_norm_grad(sr.size(0), dim, (int)ctx->saved_data["elem"].toInt(), (float)ctx->saved_data["eps"].toDouble(), in(sr), sr.stride(0), in(dy),
                              dy.stride(0), in(ds), ds.defined() ? ds.stride(0) : 0, fin(weight), out(dx), fout(dweight), fout(scratch), stream(s)));
    }
    return {dx, dweight, plain ? Tensor() : dx, Tensor(), Tensor()};
  }
};

std::vector<Tensor> rms_norm(const Tensor& x, const Tensor& weight, const Maybe& residual, double eps) {
  const int elem = input("x", x);
  no_tangent("rms_norm", {&x, &weight, opt(residual)});
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x: expected [..., channels], got ", x.sizes());
  const Tensor w = param("weight", weight, x, {x.size(-1)}), r = given(like("residual", residual, x, x.sizes()));
  if (wants_grad({&x, &w, &r})) return RmsNorm::apply(x, w, maybe(r), eps, (int64_t)elem);
  const Tensor y = blank(x), summed = norm_forward(elem, x, w, r, eps, y, Tensor(), 0);
  return residual ? std::vector<Tensor>{y, summed} : std::vector<Tensor>{y};
}

std::vector<Tensor> rms_norm_fp8(const Tensor& x, const Tensor& weight, const Maybe& residual, double eps, int64_t group) {
  const int elem = input("x", x);
  no_grad("rms_norm_fp8", {&x, &weight, opt(residual)});
  no_tangent("rms_norm_fp8", {&x, &weight, opt(residual)});
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x: expected [..., channels], got ", x.sizes());
  const Tensor w = param("weight", weight, x, {x.size(-1)}), r = given(like("residual", residual, x, x.sizes()));
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
  if (group) shape.push_back((x.size(-1) + group - 1) / group);
  const Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)), scale = floats(x, shape);
  const Tensor summed = norm_forward(elem, x, w, r, eps, q, scale, (int)group);
  return residual ? std::vector<Tensor>{q, scale, summed} : std::vector<Tensor>{q, scale};
}

// ----------------------------------------------------- the causal convolution

struct CausalConv : torch::autograd::Function<CausalConv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias_, const Maybe& state_, const Maybe& resets_, int64_t silu, int64_t elem) {
    const Tensor bias = given(bias_), state = given(state_), resets = given(resets_);
    ctx->set_materialize_grads(false);
    const c10::DeviceGuard guard(x.device());
    const Tensor y = blank(x);
    Tensor last = at::empty({x.size(1), weight.size(1) - 1, x.size(2)}, x.options());
    if (x.numel() == 0) {
      last = unmoved(state, last);
    } else {
      check(gbx_causal_conv(narrow("steps", x.size(0)), narrow("envs", x.size(1)), narrow("channels", x.size(2)), (int)weight.size(1), (int)elem, (int)silu, in(x),
                            x.stride(0), x.stride(1), fin(weight), fin(bias), in(state), bytes(resets), out(y), out(last), stream(x)));
    }
    ctx->save_for_backward({x, weight, bias, state, resets});
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["elem"] = elem;
    ctx->mark_non_differentiable({last});
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    variable_list result(7);
    if (!grads[0].defined()) return result;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &state = saved[3], &resets = saved[4];
    const c10::DeviceGuard guard(x.device());
    if (x.numel() == 0) {
      for (int i = 0; i < 3; ++i) result[i] = zeros(saved[i]);
      return result;
    }
    const int32_t steps = (int32_t)x.size(0), envs = (int32_t)x.size(1), dim = (int32_t)x.size(2), width = (int32_t)weight.size(1);
    const Tensor dy = rows(grads[0]), dx = blank(x), dweight = blank(weight), dbias = blank(bias);
    const Tensor scratch = work(x, gbx_causal_conv_grad_work(steps, envs, dim, width));
    check(gbx_causal_conv_grad(steps, envs, dim, width, (int)ctx->saved_data["elem"].toInt(), (int)ctx->saved_data["silu"].toInt(), in(x), x.stride(0), x.stride(1), fin(weight),
                               fin(bias), in(state), bytes(resets), in(dy), dy.stride(0), dy.stride(1), out(dx), fout(dweight), fout(dbias), fout(scratch), stream(x)));
    result[0] = dx, result[1] = dweight, result[2] = dbias;
    return result;
  }
};

std::vector<Tensor> causal_conv(const Tensor& x_, const Tensor& weight, const Maybe& bias, const Maybe& state, const Maybe& resets, bool silu) {
  const int elem = input("x", x_);
  no_tangent("causal_conv", {&x_, &weight, opt(bias), opt(state)});
  TORCH_CHECK_VALUE(x_.dim() == 3 && x_.size(2) >= 1, "x: expected [steps, envs, channels], got ", x_.sizes());
  check_width(weight);
  const Tensor x = rows(x_);
  const int64_t steps = x.size(0), envs = x.size(1), dim = x.size(2), width = weight.size(1);
  const Tensor w = param("weight", weight, x, {dim, width}), b = given(param("bias", bias, x, {dim}));
  TORCH_CHECK_VALUE(!wants_grad({opt(state)}), "state carries no gradient: detach it");
  const Tensor before = state ? state_of(*state, x, x.scalar_type(), {envs, width - 1, dim}).contiguous() : Tensor();
  const Tensor begins = given(starts(resets, x, {steps, envs}));
  return CausalConv::apply(x, w, maybe(b), maybe(before), maybe(begins), (int64_t)silu, (int64_t)elem);
}

Tensor causal_conv_step(const Tensor& x_, const Tensor& weight, const Maybe& bias, const Tensor& state, const Maybe& resets, bool silu) {
  const int elem = input("x", x_);
  no_grad("causal_conv_step", {&x_, &weight, opt(bias), &state});
  no_tangent("causal_conv_step", {&x_, &weight, opt(bias), &state});
  TORCH_CHECK_VALUE(x_.dim() == 2 && x_.size(1) >= 1, "x: expected [envs, channels], got ", x_.sizes());
  check_width(weight);
  const Tensor x = rows(x_);
  const int64_t envs = x.size(0), dim = x.size(1), width = weight.size(1);
  const Tensor w = param("weight", weight, x, {dim, width}), b = given(param("bias", bias, x, {dim}));
  state_of(state, x, x.scalar_type(), {envs, width - 1, dim});
  TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous: it is updated in place");
  const Tensor begins = given(starts(resets, x, {envs})), y = blank(x);
  if (envs) {
    const c10::DeviceGuard guard(x.device());
    will_change(state);
    check(gbx_causal_conv_step(narrow("envs", envs), narrow("channels", dim), (int)width, elem, silu, in(x), x.stride(0), fin(w), fin(b), out(state), bytes(begins), out(y), stream(x)));
  }
  return y;
}

// -------------------------------------------------------- the selective scan

struct Scan {  // checked operands; undefined: not given
  Tensor x, dt, a, b, c, skip, z, bias, resets;
};
gbx_scan_in scan_in(const Scan& s, bool softplus, int elem) {
  const bool one = s.x.dim() == 2;  // a single step
  const auto step = [&](const Tensor& t) { return !t.defined() || one ? 0 : t.stride(0); };
  const auto env = [&](const Tensor& t) { return !t.defined() ? 0 : t.stride(one ? 0 : 1); };
  gbx_scan_in g{};
  g.steps = one ? 1 : narrow("steps", s.x.size(0)), g.envs = narrow("envs", s.x.size(-2)), g.dim = narrow("channels", s.x.size(-1));
  g.groups = narrow("groups", s.b.size(-2)), g.states = (int32_t)s.a.size(1), g.elem = elem, g.softplus = softplus;
  g.x = in(s.x), g.dt = in(s.dt), g.z = in(s.z), g.b = in(s.b), g.c = in(s.c);
  g.x_step = step(s.x), g.x_env = env(s.x), g.dt_step = step(s.dt), g.dt_env = env(s.dt), g.z_step = step(s.z), g.z_env = env(s.z);
  g.b_step = step(s.b), g.b_env = env(s.b), g.b_group = s.b.stride(-2), g.c_step = step(s.c), g.c_env = env(s.c), g.c_group = s.c.stride(-2);
  g.a = fin(s.a), g.skip = fin(s.skip), g.bias = fin(s.bias), g.resets = bytes(s.resets);
  return g;
}
Scan scan_operands(const Tensor& x_, const Tensor& dt, const Tensor& a, const Tensor& b_, const Tensor& c_, const Maybe& skip, const Maybe& z, const Maybe& bias, const Maybe& resets) {
  const Tensor x = rows(x_), b = b_.dim() == x.dim() ? b_.unsqueeze(-2) : b_, c = c_.dim() == x.dim() ? c_.unsqueeze(-2) : c_;
  const int64_t dim = x.size(-1);
  TORCH_CHECK_VALUE(a.dim() == 2 && a.size(1) >= 1 && a.size(1) <= 32, "A: expected [channels, 1 to 32 states], got ", a.sizes());
  TORCH_CHECK_VALUE(b.dim() == x.dim() + 1 && b.size(-2) >= 1 && dim % b.size(-2) == 0, "B: expected [..., groups, states] with groups dividing ", dim, ", got ", b.sizes());
  std::vector<int64_t> each(x.sizes().begin(), x.sizes().end() - 1);
  const std::vector<int64_t> lead = each;
  each.push_back(b.size(-2));
  each.push_back(a.size(1));
  return {x, like("dt", dt, x, x.sizes()), param("A", a, x, {dim, a.size(1)}), like("B", b, x, each), like("C", c, x, each),
          given(param("D", skip, x, {dim})), given(like("z", z, x, x.sizes())), given(param("dt_bias", bias, x, {dim})), given(starts(resets, x, lead))};
}
variable_list scan_forward(const Scan& s, const Tensor& state, bool softplus, int elem, bool save) {
  const c10::DeviceGuard guard(s.x.device());
  const int64_t steps = s.x.size(0), envs = s.x.size(1), dim = s.x.size(2), states = s.a.size(1);
  const Tensor y = blank(s.x), last = floats(s.x, {envs, dim, states}), saved = save ? floats(s.x, {(steps + 7) / 8, envs, states, dim}) : Tensor();
  if (s.x.numel() == 0) return {y, unmoved(state, last), saved};
  const gbx_scan_in g = scan_in(s, softplus, elem);
  const Tensor scratch = work(s.x, gbx_selective_scan_work(&g));
  check(gbx_selective_scan(&g, fin(state), out(y), fout(last), fout(saved), fout(scratch), stream(s.x)));
  return {y, last, saved};
}

struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Maybe& skip_, const Maybe& z_,
                               const Maybe& bias_, const Maybe& state, const Maybe& resets_, bool softplus, int64_t elem) {
    const Tensor skip = given(skip_), z = given(z_), bias = given(bias_), resets = given(resets_);
    ctx->set_materialize_grads(false);
    const variable_list r = scan_forward({x, dt, a, b, c, skip, z, bias, resets}, given(state), softplus, (int)elem, true);
    ctx->save_for_backward({x, dt, a, b, c, skip, z, bias, resets, r[2]});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["elem"] = elem;
    ctx->mark_non_differentiable({r[1]});
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    variable_list result(12);
    if (!grads[0].defined()) return result;
    const auto v = ctx->get_saved_variables();
    const Scan s{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8]};
    const c10::DeviceGuard guard(s.x.device());
    if (s.x.numel() == 0) {
      for (int i = 0; i < 8; ++i) result[i] = zeros(v[i]);
      return result;
    }
    const gbx_scan_in g = scan_in(s, ctx->saved_data["softplus"].toBool(), (int)ctx->saved_data["elem"].toInt());
    const Tensor dy = rows(grads[0]);
    for (int i = 0; i < 8; ++i) result[i] = blank(v[i]);
    const Tensor scratch = work(s.x, gbx_selective_scan_grad_work(&g));
    check(gbx_selective_scan_grad(&g, fin(v[9]), in(dy), dy.stride(0), dy.stride(1), out(result[0]), out(result[1]), out(result[6]), out(result[3]), out(result[4]), fout(result[2]),
                                  fout(result[5]), fout(result[7]), fout(scratch), stream(s.x)));
    return result;
  }
};

std::vector<Tensor> selective_scan(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Maybe& skip, const Maybe& z, const Maybe& bias, bool softplus,
                                   const Maybe& state, const Maybe& resets) {
  const int elem = input("x", x);
  no_tangent("selective_scan", {&x, &dt, &a, &b, &c, opt(skip), opt(z), opt(bias), opt(state)});
  TORCH_CHECK_VALUE(x.dim() == 3 && x.size(2) >= 1, "x: expected [steps, envs, channels], got ", x.sizes());
  const Scan s = scan_operands(x, dt, a, b, c, skip, z, bias, resets);
  TORCH_CHECK_VALUE(!wants_grad({opt(state)}), "state carries no gradient: detach it");
  const std::vector<int64_t> kept{x.size(1), x.size(2), s.a.size(1)};
  const Tensor before = state ? state_of(*state, x, at::kFloat, kept).contiguous() : Tensor();
  if (wants_grad({&s.x, &s.dt, &s.a, &s.b, &s.c, &s.skip, &s.z, &s.bias}))
    return SelectiveScan::apply(s.x, s.dt, s.a, s.b, s.c, maybe(s.skip), maybe(s.z), maybe(s.bias), maybe(before), maybe(s.resets), softplus, (int64_t)elem);
  const variable_list r = scan_forward(s, before, softplus, elem, false);
  return {r[0], r[1]};
}

Tensor selective_scan_step(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Maybe& skip, const Maybe& z, const Tensor& state, const Maybe& bias,
                           bool softplus, const Maybe& resets) {
  const int elem = input("x", x);
  no_grad("selective_scan_step", {&x, &dt, &a, &b, &c, opt(skip), opt(z), &state, opt(bias)});
  no_tangent("selective_scan_step", {&x, &dt, &a, &b, &c, opt(skip), opt(z), &state, opt(bias)});
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) >= 1, "x: expected [envs, channels], got ", x.sizes());
  const Scan s = scan_operands(x, dt, a, b, c, skip, z, bias, resets);
  state_of(state, x, at::kFloat, {x.size(0), x.size(1), s.a.size(1)});
  TORCH_CHECK_VALUE(state.is_contiguous(), "state must be contiguous: it is updated in place");
  const Tensor y = blank(x);
  if (x.size(0)) {
    const c10::DeviceGuard guard(x.device());
    const gbx_scan_in g = scan_in(s, softplus, elem);
    will_change(state);
    check(gbx_selective_scan_step(&g, fout(state), out(y), stream(x)));
  }
  return y;
}

// --------------------------------------------------------------------- AdamW

// What does not change from step to step of a parameter group.
struct AdamwPlan {
  std::vector<int64_t> sizes, starts;
  Tensor exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale;  // scales undefined: 32 bits

  AdamwPlan(std::vector<int64_t> sizes_, std::vector<int64_t> starts_, const Tensor& m, const Tensor& v, const Maybe& ms, const Maybe& vs)
      : sizes(std::move(sizes_)), starts(std::move(starts_)), exp_avg(m), exp_avg_sq(v), exp_avg_scale(given(ms)), exp_avg_sq_scale(given(vs)) {}

  // One step of the parameters `which` (all: empty).  False, and nothing done,
  // if their types differ or one has no gradient.
  bool step(const std::vector<Tensor>& params, const std::vector<int64_t>& which, const Maybe& grad_scale, double beta1, double beta2, double step_size, double inv_root2, double eps,
            double keep, uint32_t key) const {
    TORCH_CHECK_VALUE(params.size() == sizes.size(), "the optimizer was made for ", sizes.size(), " parameters, got ", params.size());
    const size_t count = which.empty() ? params.size() : which.size();
    std::vector<Tensor> grads;
    std::vector<uint64_t> p_at, g_at;
    std::vector<int64_t> n, at;
    grads.reserve(count), p_at.reserve(count), g_at.reserve(count), n.reserve(count), at.reserve(count);
    at::ScalarType kind{}, grad_kind{};
    for (size_t k = 0; k < count; ++k) {
      const size_t i = which.empty() ? k : (size_t)which[k];
      const Tensor& p = params.at(i);
      TORCH_CHECK_VALUE(p.numel() == sizes[i] && p.is_contiguous() && p.device() == exp_avg.device() && elem_of(p.scalar_type()) >= 0,
                        "a parameter has another size, layout, type or device than when the optimizer was made");
      const Tensor& g = p.grad();
      if (!g.defined()) return false;
      TORCH_CHECK_VALUE(g.layout() == at::kStrided && (g.scalar_type() == p.scalar_type() || g.scalar_type() == at::kFloat) && g.device() == p.device() && g.numel() == p.numel(),
                        "a gradient of ", g.scalar_type(), " (", g.layout(), ") on ", g.device(), " does not go with ", p.scalar_type(), " on ", p.device());
      if (k == 0) kind = p.scalar_type(), grad_kind = g.scalar_type();
      if (p.scalar_type() != kind || g.scalar_type() != grad_kind) return false;
      grads.push_back(g.contiguous());
      p_at.push_back((uint64_t)p.mutable_data_ptr());
      g_at.push_back((uint64_t)grads.back().const_data_ptr());
      n.push_back(sizes[i]);
      at.push_back(starts[i]);
    }
    if (count == 0) return true;
    if (grad_scale)
      TORCH_CHECK_VALUE(grad_scale->scalar_type() == at::kFloat && grad_scale->numel() == 1 && grad_scale->device() == exp_avg.device(),
                        "grad_scale must be one float32 element on the parameters' device");
    const c10::DeviceGuard guard(exp_avg.device());
    gbx_adamw_in a{};
    a.count = (int32_t)count, a.elem = elem_of(kind), a.grad_elem = elem_of(grad_kind), a.state_bits = exp_avg_scale.defined() ? 8 : 32;
    a.params = p_at.data(), a.grads = g_at.data(), a.sizes = n.data(), a.starts = at.data();
    a.exp_avg = out(exp_avg), a.exp_avg_sq = out(exp_avg_sq), a.exp_avg_scale = fout(exp_avg_scale), a.exp_avg_sq_scale = fout(exp_avg_sq_scale);
    a.grad_scale = grad_scale ? fin(*grad_scale) : nullptr;
    a.beta1 = beta1, a.beta2 = beta2, a.step_size = step_size, a.inv_root2 = inv_root2, a.eps = eps, a.keep = keep, a.key = key;
    for (size_t k = 0; k < count; ++k) will_change(params[which.empty() ? k : (size_t)which[k]]);
    check(gbx_adamw(&a, stream(exp_avg)));
    return true;
  }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  using Unlocked = py::call_guard<py::gil_scoped_release>;
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const HipFailure& e) {
      PyErr_SetString(py::module_::import("gbxcule_amd._lib").attr("GbxError").ptr(), e.what());
    }
  });
  m.def("rms_norm", &rms_norm, Unlocked());
  m.def("rms_norm_fp8", &rms_norm_fp8, Unlocked());
  m.def("causal_conv", &causal_conv, Unlocked());
  m.def("causal_conv_step", &causal_conv_step, Unlocked());
  m.def("selective_scan", &selective_scan, Unlocked());
  m.def("selective_scan_step", &selective_scan_step, Unlocked());
  py::class_<AdamwPlan>(m, "AdamwPlan")
      .def(py::init<std::vector<int64_t>, std::vector<int64_t>, const Tensor&, const Tensor&, const Maybe&, const Maybe&>())
      .def("step", &AdamwPlan::step, Unlocked());
}
