// The public token operators (attention, layer_norm, linear) over the C ABI: argument checks, memory and autograd in C++, so
// that a call on a few tokens costs its launches and not the interpreter (one LayerNorm of 16 rows, forward: 16 us through
// Python wrappers, of which the launch is 3; forward and backward: 131 us).  Compiled by build.py against torch.
//
// Everything is enqueued on the current HIP stream of the tensors' device; results and scratch come from torch's caching
// allocator.  The backward passes are first-order: autograd runs one with grad mode on only for create_graph=True, which
// is refused instead of dropping the second-order terms silently.  Forward-mode derivatives and traces are refused too.
#include <torch/extension.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <cmath>
#include "../../include/cgrna.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> Maybe;

void check(int status, const char* what) {
  if (status == CG_OK) return;
  const char* kind = status == CG_ERR_BAD_ARG ? "bad argument" : status == CG_ERR_UNSUPPORTED ? "unsupported"
                     : status == CG_ERR_WORKSPACE ? "workspace too small" : nullptr;
  if (kind) TORCH_CHECK(false, what, ": ", kind);
  TORCH_CHECK(false, what, ": hipError ", status);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
int code_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? CG_BF16 : CG_F32; }
Tensor bytes(size_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}
Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor fresh(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options()); }

std::string type_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? "torch.float32" : t.scalar_type() == at::kBFloat16 ? "torch.bfloat16"
         : std::string(c10::toString(t.scalar_type()));
}

void first_order_only() {
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "cycle-gan-rna_amd: this module's backward is first-order only; differentiating through it with "
              "create_graph=True is not supported (the second-order terms would be dropped silently).");
}

void typed(const char* name, const Tensor& x) {
  TORCH_CHECK_VALUE(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, name,
                    ": float32 or bfloat16 tensors, not ", type_of(x));
}
void same(const char* name, const Tensor& x, const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.device() == x.device(), name, ": ", what, " is on ", t.device(), ", the input on ", x.device());
  TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type(), name, ": ", what, " is ", type_of(t), ", the input ", type_of(x));
}
void on_hip(const char* name, const Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "cycle-gan-rna_amd runs on a HIP device only (", name, " got a tensor on ", x.device(), ")");
}
// What goes past these functions unseen: they hand addresses to kernels, so a tangent would be dropped without a word, and a
// trace would hold the allocation of the result but not what fills it.
void only_run(const char* name, std::initializer_list<Tensor> inputs) {
  typedef c10::impl::TorchDispatchModeTLS Modes;
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(), name,
              ": cannot be traced (the trace would replay memory that nothing has written)");
  for (const Tensor& t : inputs)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), name,
                ": no forward-mode derivatives (the tangent would be dropped silently)");
}
bool fits_int(int64_t n) { return n <= INT32_MAX; }
// autograd takes an absent tensor as an absent optional, and counts the edges of those that are there
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor tensor(const Maybe& t) { return t ? *t : Tensor(); }
struct Wanted {      // which of a Function's tensor arguments want a gradient, asked in the order of the arguments
  AutogradContext* ctx;
  size_t edge;
  bool next(bool there) { return there && ctx->needs_input_grad(edge++); }
};

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// ---- attention -----------------------------------------------------------------------------------------------------
// t (B, S, heads, D), or a dense copy where the kernels' 16-byte pieces do not fit its address and strides.
Tensor pieces(const Tensor& t) {
  const int64_t e = 16 / t.element_size();
  const bool ok = t.stride(3) == 1 && ((uintptr_t)t.data_ptr() & 15) == 0 && (t.size(0) <= 1 || t.stride(0) % e == 0) &&
                  (t.size(2) <= 1 || t.stride(2) % e == 0) &&
                  (t.size(1) <= 1 || (t.stride(1) % e == 0 && t.stride(1) * t.element_size() * 64 < (int64_t(1) << 31)));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

#define STRIDED(t) ptr(t), (t).stride(0), (t).stride(1), (t).stride(2)

struct AttnShape {
  int B, H, Hkv, Sq, Sk, D, dt;
  AttnShape(const Tensor& q, const Tensor& k)
      : B(q.size(0)), H(q.size(2)), Hkv(k.size(2)), Sq(q.size(1)), Sk(k.size(1)), D(q.size(3)), dt(code_of(q)) {}
};

// For the backward pass: log2 of the sum of exp(s), and in bf16 what the rounding of o left (delta = sum_d do o is formed from both)
struct Kept { Tensor lse2, low; };

Tensor attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& words, double scale, bool causal,
                         Kept* keep) {
  const AttnShape s(q, k);
  Tensor o = fresh(q.sizes(), q);
  if (keep) keep->lse2 = floats({s.B, s.H, s.Sq}, q);
  if (keep && s.dt == CG_BF16) keep->low = fresh(q.sizes(), q);
  const Tensor ws = bytes(cg_attention_fwd_workspace_bytes(s.B, s.H, s.Hkv, s.Sq, s.Sk, s.D, s.dt), q);
  check(cg_attention_fwd_low(ptr(o), keep ? ptr(keep->low) : nullptr, keep ? (float*)ptr(keep->lse2) : nullptr, STRIDED(q),
                             STRIDED(k), STRIDED(v), ptr(words), s.B, s.H, s.Hkv, s.Sq, s.Sk, s.D, (float)scale, causal, s.dt,
                             ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(q)),
        "cg_attention_fwd_low");
  return o;
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q0, const Tensor& k0, const Tensor& v0, const Maybe& words_,
                        double scale, bool causal) {
    const Tensor words = tensor(words_), q = pieces(q0), k = pieces(k0), v = pieces(v0);
    Kept keep;
    Tensor o = attention_forward(q, k, v, words, scale, causal, &keep);
    ctx->save_for_backward({q, k, v, o, keep.low, keep.lse2, words});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &o = saved[3], &low = saved[4], &lse2 = saved[5], &words = saved[6];
    const c10::OptionalDeviceGuard guard(q.device());
    const Tensor g = pieces(grads[0]);
    const AttnShape s(q, k);
    Tensor dq = fresh(q.sizes(), q), dk = fresh(k.sizes(), q), dv = fresh(k.sizes(), q);
    const Tensor ws = bytes(cg_attention_bwd_workspace_bytes(s.B, s.H, s.Hkv, s.Sq, s.Sk, s.D, s.dt), q);
    check(cg_attention_bwd_low(ptr(dq), ptr(dk), ptr(dv), STRIDED(g), ptr(o), ptr(low), (const float*)ptr(lse2), STRIDED(q),
                               STRIDED(k), STRIDED(v), ptr(words), s.B, s.H, s.Hkv, s.Sq, s.Sk, s.D,
                               (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["causal"].toBool(), s.dt, ptr(ws),
                               ws.defined() ? ws.numel() : 0, stream_of(q)),
          "cg_attention_bwd_low");
    return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
  }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, bool causal, const Maybe& key_mask, c10::optional<double> scale_) {
  const char* name = "attention";
  typed(name, q);
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "attention: q (B, Sq, H, D) and k, v (B, Sk, Hkv, D), not ",
                    q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  same(name, q, k, "k");
  same(name, q, v, "v");
  const int64_t b = q.size(0), h = q.size(2), d = q.size(3), sk = k.size(1);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(0) == b && k.size(3) == d && k.size(2) > 0 && h > 0 && h % k.size(2) == 0,
                    "attention: q ", q.sizes(), " does not go with k ", k.sizes(), " and v ", v.sizes());
  const int step = q.scalar_type() == at::kFloat ? 4 : 8;
  TORCH_CHECK_VALUE(d > 0 && d <= 128 && d % step == 0, "attention: head dimensions up to 128 in steps of ", step, " for ",
                    type_of(q), ", not ", d);
  TORCH_CHECK_VALUE(fits_int(b) && fits_int(h) && fits_int(q.size(1)) && fits_int(sk), "attention: sizes of 2^31 and more");
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)d);
  TORCH_CHECK_VALUE(scale > 1e-37 && scale < 1e37, "attention: scale has to be a positive number, not ", scale);
  if (key_mask) {
    const Tensor& m = *key_mask;
    TORCH_CHECK_VALUE((m.scalar_type() == at::kBool || m.scalar_type() == at::kByte) && m.dim() == 2 && m.size(0) == b && m.size(1) == sk,
                      "attention: key_mask has to be (", b, ", ", sk, ") bool, not ", m.sizes(), " ", type_of(m));
    TORCH_CHECK_VALUE(m.device() == q.device(), "attention: key_mask is on ", m.device(), ", q on ", q.device());
  }
  only_run(name, {q, k, v});
  on_hip(name, q);
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor words;
  if (key_mask) {
    const Tensor m = key_mask->stride(1) == 1 ? *key_mask : key_mask->contiguous();
    words = at::empty({b, (sk + 63) / 64}, q.options().dtype(at::kLong));
    check(cg_attention_mask_words(ptr(words), (const uint8_t*)m.data_ptr(), m.stride(0), b, sk, stream_of(q)), "cg_attention_mask_words");
  }
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return AttentionFn::apply(q, k, v, maybe(words), scale, causal);
  return attention_forward(pieces(q), pieces(k), pieces(v), words, scale, causal, nullptr);
}

// ---- rows ----------------------------------------------------------------------------------------------------------
constexpr int64_t LINEAR_LD = 1 << 21;      // the dense layer's longest row pitch: a tile's rows lie within 2^31 bytes

// t (..., n) as (M, n) rows whose elements are next to each other, that do not overlap and lie at most `most` elements
// apart; a copy only where needed.
Tensor rows(const Tensor& t, int64_t n, int64_t most = INT64_MAX) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, n});
  if (r.size(0) == 0) return fresh({0, n}, t);
  const bool ok = (r.stride(1) == 1 || n == 1) && (r.size(0) == 1 || (r.stride(0) >= n && r.stride(0) <= most));
  return ok ? r : r.contiguous();
}
int64_t ld(const Tensor& t, int64_t n) { return t.defined() && t.size(0) > 1 ? t.stride(0) : n; }
#define ROWS(t, n) ptr(t), ld(t, n)

// ---- LayerNorm -----------------------------------------------------------------------------------------------------
struct LnOut { Tensor x, r, y, s, stats; };

LnOut ln_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, double eps, bool keep) {
  LnOut f;
  const int64_t n = x.size(-1);
  f.x = rows(x, n);
  const int64_t m = f.x.size(0);
  TORCH_CHECK_VALUE(fits_int(m), "layer_norm: 2^31 rows and more");
  f.y = fresh(x.sizes(), x);
  if (residual.defined()) {
    f.r = rows(residual, n);
    f.s = fresh(x.sizes(), x);
  }
  if (keep) f.stats = floats({2, m}, x);
  float* mean = keep ? (float*)ptr(f.stats) : nullptr;
  const Tensor& p = weight.defined() ? weight : bias;
  check(cg_ln_fwd(ptr(f.y), n, ptr(f.s), n, ROWS(f.x, n), ROWS(f.r, n), ptr(weight), ptr(bias), (float)eps, mean,
                  keep ? mean + m : nullptr, m, n, code_of(x), code_of(p.defined() ? p : x), stream_of(x)),
        "cg_ln_fwd");
  return f;
}

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight_, const Maybe& bias_,
                               const Maybe& residual_, double eps) {
    const Tensor weight = tensor(weight_), bias = tensor(bias_), residual = tensor(residual_);
    LnOut f = ln_forward(x, weight, bias, residual, eps, true);
    ctx->set_materialize_grads(false);
    ctx->saved_data["types"] = (int64_t)((bias.defined() ? (bias.scalar_type() == at::kBFloat16 ? 2 : 1) : 0));
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["residual"] = residual.defined();
    // A float32 sum is kept as it is stored; from a bf16 one, half a rounding step off, the weight's gradient would be
    // 1.4 times as far off as its own rounding: there x and the residual are read again
    if (!f.s.defined() || x.scalar_type() == at::kBFloat16) {
      ctx->save_for_backward({f.x, f.r, weight, f.stats});
    } else {
      ctx->save_for_backward({f.s, Tensor(), weight, f.stats});
    }
    if (!f.s.defined()) return {f.y};
    return {f.y, f.s};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order_only();
    const auto saved = ctx->get_saved_variables();
    const int64_t n = saved[0].size(-1), types = ctx->saved_data["types"].toInt();
    const c10::OptionalDeviceGuard guard(saved[0].device());
    const Tensor s = rows(saved[0], n), &r = saved[1], &weight = saved[2], &stats = saved[3];
    const int64_t m = s.size(0);
    Wanted wanted{ctx, 0};
    const bool nx = wanted.next(true), nw = wanted.next(weight.defined()), nb = wanted.next(types != 0),
               nr = wanted.next(ctx->saved_data["residual"].toBool());
    const Tensor dy = grads[0].defined() ? rows(grads[0], n) : at::zeros({m, n}, s.options());
    const Tensor ds = grads.size() > 1 && grads[1].defined() ? rows(grads[1], n) : Tensor();
    Tensor dx, dw, db, ws;
    if (nx || nr) dx = fresh(ctx->saved_data["shape"].toIntVector(), s);
    if (nw) dw = fresh(weight.sizes(), weight);
    if (nb) db = at::empty({n}, s.options().dtype(types == 2 ? at::kBFloat16 : at::kFloat));
    if (nw || nb) ws = bytes(cg_ln_bwd_workspace_bytes(m, n, code_of(s)), s);
    if (dx.defined() || ws.defined()) {
      const int wcode = nb ? (types == 2 ? CG_BF16 : CG_F32) : code_of(weight.defined() ? weight : s);
      check(cg_ln_bwd(ptr(dx), n, ROWS(dy, n), ROWS(ds, n), ROWS(s, n), ROWS(r, n), ptr(weight), (const float*)ptr(stats),
                      (const float*)ptr(stats) + m, ptr(dw), ptr(db), m, n, code_of(s), wcode, ptr(ws),
                      ws.defined() ? ws.numel() : 0, stream_of(s)),
            "cg_ln_bwd");
    }
    return {nx ? dx : Tensor(), dw, db, nr ? dx : Tensor(), Tensor()};
  }
};

py::object layer_norm(const Tensor& x, const Maybe& weight_, const Maybe& bias_, const Maybe& residual_, double eps) {
  const char* name = "layer_norm";
  typed(name, x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, "layer_norm: a last axis of at least one element, not shape ", x.sizes());
  const int64_t n = x.size(-1);
  TORCH_CHECK_VALUE(n <= int64_t(1) << 30, "layer_norm: up to 2^30 columns, not ", n);
  Tensor weight = tensor(weight_), bias = tensor(bias_);
  const Tensor residual = tensor(residual_);
  if (residual.defined()) {
    same(name, x, residual, "residual");
    TORCH_CHECK_VALUE(residual.sizes() == x.sizes(), "layer_norm: residual ", residual.sizes(), " for x ", x.sizes());
  }
  for (const auto& p : {std::make_pair("weight", weight), std::make_pair("bias", bias)}) {
    if (!p.second.defined()) continue;
    TORCH_CHECK_VALUE(p.second.dim() == 1 && p.second.size(0) == n, "layer_norm: ", p.first, " ", p.second.sizes(), " for a last axis of ", n);
    TORCH_CHECK_VALUE(p.second.device() == x.device() && (p.second.scalar_type() == x.scalar_type() || p.second.scalar_type() == at::kFloat),
                      "layer_norm: ", p.first, " is ", type_of(p.second), " on ", p.second.device(), ", x ", type_of(x), " on ", x.device());
  }
  if (weight.defined() && bias.defined())
    TORCH_CHECK_VALUE(weight.scalar_type() == bias.scalar_type(), "layer_norm: weight is ", type_of(weight), ", bias ", type_of(bias));
  TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "layer_norm: eps has to be a number that is not negative, not ", eps);
  only_run(name, {x, weight, bias, residual});
  on_hip(name, x);
  const c10::OptionalDeviceGuard guard(x.device());
  if (weight.defined()) weight = weight.contiguous();
  if (bias.defined()) bias = bias.contiguous();
  Tensor y, s;
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual))) {
    const variable_list out = LayerNormFn::apply(x, maybe(weight), maybe(bias), maybe(residual), eps);
    y = out[0];
    if (out.size() > 1) s = out[1];
  } else {
    const LnOut f = ln_forward(x, weight, bias, residual, eps, false);
    y = f.y, s = f.s;
  }
  if (!s.defined()) return py::cast(y);
  return py::make_tuple(y, s);
}

// ---- dense layer ---------------------------------------------------------------------------------------------------
Tensor linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual, at::IntArrayRef shape, int act,
                      double slope, Tensor* z) {
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  TORCH_CHECK_VALUE(fits_int(m) && fits_int(n) && fits_int(k), "linear: 2^31 rows or columns and more");
  Tensor y = fresh(shape, x);
  if (z) *z = fresh({m, n}, x);
  const Tensor r = residual.defined() ? rows(residual, n, LINEAR_LD) : Tensor();
  const Tensor ws = bytes(cg_linear_fwd_workspace_bytes(m, n, k, code_of(x)), x);
  check(cg_linear_fwd(ptr(y), n, z ? ptr(*z) : nullptr, n, ROWS(x, k), ROWS(w, k), ptr(bias), ROWS(r, n), m, n, k, act, (float)slope,
                      code_of(x), ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(x)),
        "cg_linear_fwd");
  return y;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias_, const Maybe& residual_,
                        int64_t act, double slope) {
    const Tensor bias = tensor(bias_), residual = tensor(residual_);
    const int64_t n = weight.size(0), k = weight.size(1);
    const Tensor x2 = rows(x, k, LINEAR_LD), w2 = rows(weight, k, LINEAR_LD);
    auto shape = x.sizes().vec();
    ctx->saved_data["shape"] = shape;
    ctx->saved_data["act"] = act;
    ctx->saved_data["slope"] = slope;
    ctx->saved_data["bias"] = bias.defined();
    ctx->saved_data["residual"] = residual.defined();
    shape.back() = n;
    Tensor z;
    Tensor y = linear_forward(x2, w2, bias, residual, shape, act, slope, act != CG_ACT_NONE ? &z : nullptr);
    ctx->save_for_backward({x2, w2, z});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order_only();
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &z = saved[2];
    const c10::OptionalDeviceGuard guard(x.device());
    const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
    Wanted wanted{ctx, 0};
    const bool nx = wanted.next(true), nw = wanted.next(true), nb = wanted.next(ctx->saved_data["bias"].toBool()),
               nr = wanted.next(ctx->saved_data["residual"].toBool());
    Tensor dx, dw, db;
    if (nx) dx = fresh(ctx->saved_data["shape"].toIntVector(), x);
    if (nw) dw = fresh({n, k}, x);
    if (nb) db = fresh({n}, x);
    if (nx || nw || nb) {
      const Tensor dy = rows(grads[0], n, LINEAR_LD);
      const Tensor ws = bytes(cg_linear_bwd_workspace_bytes(m, n, k, code_of(x)), x);
      check(cg_linear_bwd(ptr(dx), k, ptr(dw), ptr(db), ROWS(dy, n), ROWS(z, n), ROWS(x, k), ROWS(w, k), m, n, k,
                          ctx->saved_data["act"].toInt(), (float)ctx->saved_data["slope"].toDouble(), code_of(x), ptr(ws),
                          ws.numel(), stream_of(x)),
            "cg_linear_bwd");
    }
    return {dx, dw, db, nr ? grads[0] : Tensor(), Tensor(), Tensor()};
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const Maybe& bias_, const std::string& activation, double slope, const Maybe& residual_) {
  const char* name = "linear";
  typed(name, x);
  TORCH_CHECK_VALUE(weight.dim() == 2 && x.dim() >= 1 && x.size(-1) == weight.size(1) && weight.numel() > 0, "linear: x ", x.sizes(),
                    " does not go with weight ", weight.sizes());
  const int64_t n = weight.size(0), k = weight.size(1);
  same(name, x, weight, "weight");
  Tensor bias = tensor(bias_);
  const Tensor residual = tensor(residual_);
  if (bias.defined()) {
    same(name, x, bias, "bias");
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == n, "linear: bias ", bias.sizes(), " for ", n, " outputs");
  }
  auto shape = x.sizes().vec();
  shape.back() = n;
  if (residual.defined()) {
    same(name, x, residual, "residual");
    TORCH_CHECK_VALUE(residual.sizes() == at::IntArrayRef(shape), "linear: residual ", residual.sizes(), " for an output ", shape);
  }
  const int act = activation == "none" ? CG_ACT_NONE : activation == "leaky" ? CG_ACT_LEAKY : activation == "gelu" ? CG_ACT_GELU
                  : activation == "silu" ? CG_ACT_SILU : -1;
  TORCH_CHECK_VALUE(act >= 0, "linear: activation has to be 'none', 'leaky', 'gelu' or 'silu', not '", activation, "'");
  TORCH_CHECK_VALUE(std::isfinite(slope), "linear: slope has to be a number, not ", slope);
  only_run(name, {x, weight, bias, residual});
  on_hip(name, x);
  const c10::OptionalDeviceGuard guard(x.device());
  if (bias.defined()) bias = bias.contiguous();
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual)))
    return LinearFn::apply(x, weight, maybe(bias), maybe(residual), act, slope);
  return linear_forward(rows(x, k, LINEAR_LD), rows(weight, k, LINEAR_LD), bias, residual, shape, act, slope, nullptr);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("attention", &attention);
  m.def("layer_norm", &layer_norm);
  m.def("linear", &linear);
}
