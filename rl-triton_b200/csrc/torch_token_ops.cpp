// torch_token_ops.cpp -- the token-level policy operators (namespace rl_triton)
// with their gradients.
//
// Four operators are differentiable: token_logprobs and policy_loss_logits (by the
// logits), policy_loss and preference_loss (by the log-probabilities), once each
// and in reverse mode.  Each has an
// autograd function here that calls operators of its own (names with a leading
// underscore: the kernels proper) through the dispatcher, so that fake tensors
// and torch.compile see the same calls.  The functions are in C++ because a
// training step on a small batch is bound by the host.
//
// The losses' gradients are written by the forward call, for an incoming
// gradient of grad_scale; the backward call hands that buffer out, and writes
// it anew only when the incoming gradient differs (the device compares: the
// host is not synchronised).  A second backward pass over a retained graph
// gets a buffer of its own.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/record_function.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/custom_class.h>
#include <torch/library.h>

#include <map>
#include <mutex>
#include <tuple>
#include <utility>

#include "rlscan.h"
#include "torch_shared.h"

namespace {

using namespace rls_torch;
using at::Tensor;
using OptT = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

const float* F(const Tensor& t) { return t.data_ptr<float>(); }
const float* F(const OptT& t) { return t && t->defined() ? t->data_ptr<float>() : nullptr; }
float* W(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr<float>() : nullptr; }
OptT opt(const Tensor& t) { return t.defined() ? OptT(t) : OptT(); }
Tensor plain(const OptT& t) { return t ? *t : Tensor(); }

// ---- inputs ----------------------------------------------------------------------
// Looks at every tensor's device, then spares the library its queries for the
// calls in this scope.
class Placed {
 public:
  template <class... Ts>
  explicit Placed(const Tensor& first, const Ts&... rest) {
    TORCH_CHECK(first.is_cuda(), "inputs must be on CUDA");
    (same(first, rest), ...);
    before_ = rls_assume_device(first.device().index());
  }
  ~Placed() { rls_assume_device(before_); }
  Placed(const Placed&) = delete;
  Placed& operator=(const Placed&) = delete;

 private:
  static void same(const Tensor& first, const Tensor& t) {
    TORCH_CHECK(!t.defined() || t.device() == first.device(), "all tensors of one call must be on ", first.device(),
                "; got a tensor on ", t.device());
  }
  static void same(const Tensor& first, const OptT& t) {
    if (t) same(first, *t);
  }
  int before_;
};

// The kernels go by the sizes and types that a call names, so every tensor of a call is
// held against them: the operators can be called without the functions in front of them.
void shaped(const Tensor& t, at::IntArrayRef sizes, const char* name) {
  TORCH_CHECK(t.sizes() == sizes, name, ": expected shape ", sizes, ", got ", t.sizes());
}
void real(const Tensor& t, at::IntArrayRef sizes, const char* name) {
  shaped(t, sizes, name);
  TORCH_CHECK(t.is_floating_point(), name, ": expected floating point, got ", t.scalar_type());
}
void real(const OptT& t, at::IntArrayRef sizes, const char* name) {
  if (t && t->defined()) real(*t, sizes, name);
}
void masks(const OptT& t, at::IntArrayRef sizes, const char* name) {
  if (!t || !t->defined()) return;
  shaped(*t, sizes, name);
  TORCH_CHECK(!t->is_complex(), name, ": expected bool, integers or floats, got ", t->scalar_type());
}
void scalar(const Tensor& t, const char* name) {
  TORCH_CHECK(t.numel() == 1 && t.is_floating_point(), name, ": expected one floating-point number");
}
// Advantages, one a step or one a row.
void advantages_ok(const Tensor& t, int64_t n, int64_t steps) {
  const int64_t sizes[2] = {n, steps};
  real(t, at::IntArrayRef(sizes, t.dim() == 1 ? 1 : 2), "advantages");
}
// What an operator of this file wrote for its backward call.
void kept(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const char* name) {
  shaped(t, sizes, name);
  TORCH_CHECK(t.scalar_type() == type && t.is_contiguous(), name, ": expected contiguous ", type);
}

struct MaskArg {
  OptT t;
  int kind = RLS_MASK_NONE;
  const void* ptr() const { return t ? t->data_ptr() : nullptr; }
};

MaskArg mask_arg(const OptT& mask) {
  MaskArg m;
  if (!mask || !mask->defined()) return m;
  Tensor t = *mask;
  switch (t.scalar_type()) {
    case at::kBool: case at::kByte: case at::kChar: m.kind = RLS_MASK_U8; break;
    case at::kFloat: m.kind = RLS_MASK_F32; break;
    case at::kBFloat16: m.kind = RLS_MASK_BF16; break;
    case at::kInt: m.kind = RLS_MASK_I32; break;
    case at::kLong: m.kind = RLS_MASK_I64; break;
    default: t = t.ne(0); m.kind = RLS_MASK_U8;
  }
  m.t = t.is_contiguous() ? t : t.contiguous();
  if (m.t->numel() == 0) { m.t = OptT(); m.kind = RLS_MASK_NONE; }
  return m;
}

// Logits as the kernels take them: any env and step strides, the vocabulary
// contiguous.
Tensor logits_arg(const Tensor& t) {
  return t.size(2) <= 1 || t.stride(2) == 1 ? t : t.contiguous();
}
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? RLS_BF16 : RLS_F32; }
Tensor tokens_arg(const Tensor& t) {
  Tensor c = t.scalar_type() == at::kLong ? t : t.to(at::kLong);
  return c.is_contiguous() ? c : c.contiguous();
}

// The buffer of a logits gradient.  It takes the logits' own strides where they
// leave no more than a quarter of the buffer unused (a slice of the steps, a
// vocabulary cut from a padded one): if the logits start on a 16-byte boundary too, every
// row then has the alignment of its logits, which the kernels need for 16-byte stores.
Tensor op_grad_buffer(const Tensor& logits) {
  TORCH_CHECK(logits.dim() == 3, "logits: expected shape [num_envs, seq_len, vocab], got ", logits.sizes());
  const int64_t n = logits.size(0), t = logits.size(1), v = logits.size(2);
  const int64_t es = logits.stride(0), ss = logits.stride(1);
  if (logits.numel() == 0 || (v > 1 && logits.stride(2) != 1)) return at::empty(logits.sizes(), logits.options());
  const bool apart = (t == 1 || ss >= v) && (n == 1 || es >= (t - 1) * ss + v);
  const int64_t span = (n - 1) * es + (t - 1) * ss + v;
  if (!apart || span > n * t * v + n * t * v / 4 || logits.is_contiguous())
    return at::empty(logits.sizes(), logits.options());
  return at::empty_strided(logits.sizes(), logits.strides(), logits.options());
}

// In the place of an output that a call does not have: an empty tensor, made once a
// device, type and output (an allocation less for each; no two outputs share one).
enum Missing { kEntropy, kStatistics, kNorm, kRows, kGradient, kOrder };
Tensor none(const Tensor& t, Missing what, at::ScalarType type = at::kFloat) {
  static std::mutex mu;
  static std::map<std::tuple<int, int, at::ScalarType>, Tensor> made;
  std::lock_guard<std::mutex> lock(mu);
  Tensor& n = made[{(int)t.device().index(), (int)what, type}];
  if (!n.defined()) {
    c10::InferenceMode normal(false);  // it may be saved for a backward call later
    n = at::empty({0}, at::TensorOptions().device(t.device()).dtype(type));
  }
  return n;
}

struct LogitsArgs {
  Tensor x, tokens;
  MaskArg mask;
  int64_t n, t, v;
  LogitsArgs(const Tensor& logits, const Tensor& tok, const OptT& m)
      : x(logits_arg(checked(logits, tok, m))), tokens(tokens_arg(tok)), mask(mask_arg(m)), n(x.size(0)), t(x.size(1)),
        v(x.size(2)) {}
  static const Tensor& checked(const Tensor& logits, const Tensor& tok, const OptT& m) {
    TORCH_CHECK(logits.dim() == 3, "logits: expected shape [num_envs, seq_len, vocab], got ", logits.sizes());
    TORCH_CHECK(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16,
                "logits: expected float32 or bfloat16, got ", logits.scalar_type());
    const at::IntArrayRef steps = logits.sizes().slice(0, 2);
    shaped(tok, steps, "tokens");
    TORCH_CHECK(c10::isIntegralType(tok.scalar_type(), /*includeBool=*/false), "tokens: expected integers, got ",
                tok.scalar_type());
    masks(m, steps, "mask");
    return logits;
  }
  // What the forward call kept of the rows, and a buffer for their gradient.
  void check_kept(const Tensor& order, const Tensor& stats) const {
    if (order.numel()) kept(order, {n * t + 1}, at::kInt, "order");
    if (v > RLS_SHORT_VOCAB || stats.numel()) kept(stats, {n, t, RLS_ROW_STATS}, at::kFloat, "row_stats");
  }
  void check_grad(const Tensor& g) const {
    shaped(g, x.sizes(), "grad");
    TORCH_CHECK(g.scalar_type() == x.scalar_type(), "grad: expected ", x.scalar_type(), ", got ", g.scalar_type());
    TORCH_CHECK(v <= 1 || g.numel() == 0 || g.stride(2) == 1, "grad: the vocabulary must be contiguous");
  }
  // Long rows with a mask go by an order of the rows, made once for both directions.
  Tensor order_buffer() const {
    const bool some = mask.t && v > RLS_SHORT_VOCAB && n * t <= 0x7ffffffe;
    return some ? at::empty({n * t + 1}, x.options().dtype(at::kInt)) : none(x, kOrder, at::kInt);
  }
  Tensor order() const {
    Tensor o = order_buffer();
    if (!o.numel()) return o;
    Tensor ws = workspace_for(x.device(), stream_of(x), 1 << 20);
    check(rls_row_order(mask.ptr(), mask.kind, n, t, o.data_ptr<int32_t>(), ws.data_ptr(), (size_t)ws.numel(),
                        stream_of(x)),
          "rls_row_order");
    return o;
  }
};
int32_t* I(const Tensor& t) { return t.numel() ? t.data_ptr<int32_t>() : nullptr; }

Tensor like(const Tensor& t, at::IntArrayRef sizes) { return at::empty(sizes, t.options().dtype(at::kFloat)); }

// What a long row keeps for the backward call.
Tensor row_stats(const LogitsArgs& a, bool keep) {
  return keep && a.v > RLS_SHORT_VOCAB ? like(a.x, {a.n, a.t, RLS_ROW_STATS}) : none(a.x, kRows);
}

// ---- log-probabilities -------------------------------------------------------------
// (logprobs, entropy or empty, the rows' statistics or empty, their order or empty)
std::tuple<Tensor, Tensor, Tensor, Tensor> op_logprobs(const Tensor& logits, const Tensor& tokens, const OptT& mask,
                                               double temperature, bool entropy, bool keep) {
  const Placed placed(logits, tokens, mask);
  const LogitsArgs a(logits, tokens, mask);
  Tensor lp = like(a.x, {a.n, a.t});
  Tensor ent = entropy ? like(a.x, {a.n, a.t}) : none(a.x, kEntropy);
  Tensor stats = row_stats(a, keep), order = a.order();
  check(rls_token_logprobs(a.x.data_ptr(), a.x.stride(0), a.x.stride(1), a.tokens.data_ptr<int64_t>(), a.mask.ptr(),
                           a.mask.kind, I(order), W(lp), W(ent), W(stats), a.n, a.t, a.v, temperature, dtype_of(a.x),
                           stream_of(a.x)),
        "rls_token_logprobs");
  return {lp, ent, stats, order};
}

Tensor op_logprobs_backward(const Tensor& logits, const Tensor& tokens, const OptT& mask, const Tensor& order,
                            const Tensor& stats,
                            const OptT& g_lp, const OptT& g_ent, double temperature) {
  const Placed placed(logits, tokens, mask, order, stats, g_lp, g_ent);
  const LogitsArgs a(logits, tokens, mask);
  a.check_kept(order, stats);
  real(g_lp, {a.n, a.t}, "g_logprobs");
  real(g_ent, {a.n, a.t}, "g_entropy");
  const OptT gl = f32(g_lp), ge = f32(g_ent);
  Tensor g = op_grad_buffer(a.x);
  check(rls_token_logprobs_backward(a.x.data_ptr(), a.x.stride(0), a.x.stride(1), a.tokens.data_ptr<int64_t>(),
                                    a.mask.ptr(), a.mask.kind, I(order), W(stats), F(gl), F(ge), g.data_ptr(), g.stride(0),
                                    g.stride(1), a.n, a.t, a.v, temperature, dtype_of(a.x), stream_of(a.x)),
        "rls_token_logprobs_backward");
  return g;
}

// ---- policy loss ---------------------------------------------------------------------
rls_policy_t policy_of(double clip_low, double clip_high, double dual_clip, double kl_coef, int64_t kl,
                       double entropy_coef, int64_t reduction) {
  rls_policy_t p{};
  p.clip_low = clip_low;
  p.clip_high = clip_high;
  p.dual_clip = dual_clip;
  p.kl_coef = (float)kl_coef;
  p.entropy_coef = (float)entropy_coef;
  p.kl_kind = (int)kl;
  p.reduction = (int)reduction;
  return p;
}

Tensor norm_for(const MaskArg& m, const Tensor& ref, int64_t n, int64_t reduction) {
  return m.t && reduction != RLS_REDUCE_SUM ? like(ref, {n + 1}) : none(ref, kNorm);
}

// A policy loss's inputs besides the log-probabilities or logits of [n, t] steps.
void policy_inputs_ok(const Tensor& old_lp, const Tensor& adv, const OptT& ref, int64_t n, int64_t t) {
  real(old_lp, {n, t}, "old_logprobs");
  advantages_ok(adv, n, t);
  real(ref, {n, t}, "ref_logprobs");
}
void norm_ok(const Tensor& norm, const MaskArg& m, int64_t n, int64_t reduction) {
  if (m.t && reduction != RLS_REDUCE_SUM) kept(norm, {n + 1}, at::kFloat, "norm");
}
void logprobs_ok(const Tensor& lp, const OptT& mask) {
  TORCH_CHECK(lp.dim() == 2, "logprobs: expected shape [num_envs, seq_len], got ", lp.sizes());
  real(lp, lp.sizes(), "logprobs");
  masks(mask, lp.sizes(), "mask");
}

Tensor policy_workspace(const Tensor& t) { return workspace_for(t.device(), stream_of(t), 1 << 20); }

// (loss, statistics [5], norm, gradient or an empty tensor)
std::tuple<Tensor, Tensor, Tensor, Tensor> op_policy(const Tensor& logprobs, const Tensor& old_logprobs,
                                                     const Tensor& advantages, const OptT& mask, const OptT& ref,
                                                     double clip_low, double clip_high, double dual_clip,
                                                     double kl_coef, int64_t kl, int64_t reduction, double grad_scale,
                                                     bool need_stats, bool need_grad) {
  const Placed placed(logprobs, old_logprobs, advantages, mask, ref);
  logprobs_ok(logprobs, mask);
  policy_inputs_ok(old_logprobs, advantages, ref, logprobs.size(0), logprobs.size(1));
  const Tensor lp = f32(logprobs), old_lp = f32(old_logprobs), adv = f32(advantages);
  const OptT rf = f32(ref);
  const MaskArg m = mask_arg(mask);
  const int64_t n = lp.size(0), t = lp.size(1);
  const rls_policy_t p = policy_of(clip_low, clip_high, dual_clip, kl_coef, kl, 0.0, reduction);
  Tensor loss = like(lp, {}), stats = need_stats ? like(lp, {5}) : none(lp, kStatistics), norm = norm_for(m, lp, n, reduction);
  Tensor grad = need_grad ? like(lp, {n, t}) : none(lp, kGradient);
  Tensor ws = policy_workspace(lp);
  check(rls_policy_loss(F(lp), F(old_lp), F(adv), adv.dim() == 1, F(rf), m.ptr(), m.kind, &p, (float)grad_scale,
                        W(norm), loss.data_ptr<float>(), W(stats), W(grad), n, t, ws.data_ptr(),
                        (size_t)ws.numel(), stream_of(lp)),
        "rls_policy_loss");
  return {loss, stats, norm, grad};
}

void op_policy_backward_(Tensor& grad, const Tensor& logprobs, const Tensor& old_logprobs, const Tensor& advantages,
                         const OptT& mask, const OptT& ref, const Tensor& norm, const Tensor& grad_loss,
                         double clip_low, double clip_high, double dual_clip, double kl_coef, int64_t kl,
                         int64_t reduction, double grad_scale, bool force) {
  const Placed placed(grad, logprobs, old_logprobs, advantages, mask, ref, norm, grad_loss);
  logprobs_ok(logprobs, mask);
  policy_inputs_ok(old_logprobs, advantages, ref, logprobs.size(0), logprobs.size(1));
  kept(grad, logprobs.sizes(), at::kFloat, "grad");
  scalar(grad_loss, "grad_loss");
  const Tensor lp = f32(logprobs), old_lp = f32(old_logprobs), adv = f32(advantages), g = f32(grad_loss);
  const OptT rf = f32(ref);
  const MaskArg m = mask_arg(mask);
  norm_ok(norm, m, lp.size(0), reduction);
  const rls_policy_t p = policy_of(clip_low, clip_high, dual_clip, kl_coef, kl, 0.0, reduction);
  check(rls_policy_loss_backward(F(lp), F(old_lp), F(adv), adv.dim() == 1, F(rf), m.ptr(), m.kind, &p,
                                 (float)grad_scale, F(g), force, W(norm), W(grad), lp.size(0), lp.size(1),
                                 stream_of(lp)),
        "rls_policy_loss_backward");
}

// (loss, logprobs, entropy or empty, statistics [5], norm, the rows' order and statistics, gradient or empty)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> op_policy_logits(
    const Tensor& logits, const Tensor& tokens, const Tensor& old_logprobs, const Tensor& advantages,
    const OptT& mask, const OptT& ref, double clip_low, double clip_high, double dual_clip, double kl_coef, int64_t kl,
    double entropy_coef, bool need_stats, double temperature, int64_t reduction, double grad_scale, bool need_grad) {
  const Placed placed(logits, tokens, old_logprobs, advantages, mask, ref);
  const LogitsArgs a(logits, tokens, mask);
  policy_inputs_ok(old_logprobs, advantages, ref, a.n, a.t);
  const Tensor old_lp = f32(old_logprobs), adv = f32(advantages);
  const OptT rf = f32(ref);
  const rls_policy_t p = policy_of(clip_low, clip_high, dual_clip, kl_coef, kl, entropy_coef, reduction);
  Tensor loss = like(a.x, {}), stats = need_stats ? like(a.x, {5}) : none(a.x, kStatistics), norm = norm_for(a.mask, a.x, a.n, reduction);
  Tensor lp = like(a.x, {a.n, a.t}), rows = row_stats(a, true), order = a.order_buffer();
  Tensor ent = need_stats || entropy_coef != 0.0 ? like(a.x, {a.n, a.t}) : none(a.x, kEntropy);
  Tensor g = need_grad ? op_grad_buffer(a.x) : none(a.x, kGradient, a.x.scalar_type());
  Tensor ws = policy_workspace(a.x);
  check(rls_policy_loss_logits(a.x.data_ptr(), a.x.stride(0), a.x.stride(1), a.tokens.data_ptr<int64_t>(), F(old_lp),
                               F(adv), adv.dim() == 1, F(rf), a.mask.ptr(), a.mask.kind, I(order), &p, (float)grad_scale,
                               W(norm), W(lp), W(ent), W(rows), loss.data_ptr<float>(), W(stats),
                               need_grad ? g.data_ptr() : nullptr, need_grad ? g.stride(0) : 0,
                               need_grad ? g.stride(1) : 0, a.n, a.t, a.v, temperature, dtype_of(a.x),
                               ws.data_ptr(), (size_t)ws.numel(), stream_of(a.x)),
        "rls_policy_loss_logits");
  return {loss, lp, ent, stats, norm, order, rows, g};
}

void op_policy_logits_backward_(Tensor& grad, const Tensor& logits, const Tensor& tokens, const Tensor& old_logprobs,
                                const Tensor& advantages, const OptT& mask, const OptT& ref, const Tensor& norm,
                                const Tensor& order, const Tensor& rows, const Tensor& grad_loss, double clip_low,
                                double clip_high, double dual_clip, double kl_coef, int64_t kl, double entropy_coef,
                                double temperature, int64_t reduction, double grad_scale, bool force) {
  const Placed placed(grad, logits, tokens, old_logprobs, advantages, mask, ref, norm, order, rows, grad_loss);
  const LogitsArgs a(logits, tokens, mask);
  policy_inputs_ok(old_logprobs, advantages, ref, a.n, a.t);
  norm_ok(norm, a.mask, a.n, reduction);
  a.check_kept(order, rows);
  a.check_grad(grad);
  scalar(grad_loss, "grad_loss");
  const Tensor old_lp = f32(old_logprobs), adv = f32(advantages), up = f32(grad_loss);
  const OptT rf = f32(ref);
  const rls_policy_t p = policy_of(clip_low, clip_high, dual_clip, kl_coef, kl, entropy_coef, reduction);
  check(rls_policy_loss_logits_backward(a.x.data_ptr(), a.x.stride(0), a.x.stride(1), a.tokens.data_ptr<int64_t>(),
                                        F(old_lp), F(adv), adv.dim() == 1, F(rf), a.mask.ptr(), a.mask.kind, I(order), &p,
                                        (float)grad_scale, F(up), force, W(norm), W(rows),
                                        grad.data_ptr(), grad.stride(0), grad.stride(1), a.n, a.t, a.v,
                                        temperature, dtype_of(a.x), stream_of(a.x)),
        "rls_policy_loss_logits_backward");
}

// ---- preference loss -------------------------------------------------------------------
// rejected absent: `chosen` holds both halves, [2 pairs, T].
struct Pairs {
  Tensor lp[2];
  const float* p[2];
  const float* ref[2];
  const void* mask[2];
  MaskArg m[2];
  OptT rf[2];
  int kind = RLS_MASK_NONE;
  int64_t b, t[2];
  bool ref_pair = false;
  Pairs(const Tensor& chosen, const OptT& rejected, const OptT& ref_c, const OptT& ref_r, const OptT& mask_c,
        const OptT& mask_r) {
    check_sizes(chosen, rejected, ref_c, ref_r, mask_c, mask_r);
    lp[0] = f32(chosen);
    rf[0] = f32(ref_c);
    m[0] = mask_arg(mask_c);
    if (rejected) {
      lp[1] = f32(*rejected);
      rf[1] = f32(ref_r);
      m[1] = mask_arg(mask_r);
      if (m[0].t && m[1].t && m[0].kind != m[1].kind)
        for (auto& x : m) x = mask_arg(x.t->ne(0));
    }
    const OptT& any = rf[0] ? rf[0] : rf[1];
    ref_pair = any && any->dim() == 1;
    if (rejected) {
      b = lp[0].size(0);
      for (int k = 0; k < 2; ++k) {
        t[k] = lp[k].size(1);
        p[k] = F(lp[k]);
        ref[k] = F(rf[k]);
        mask[k] = m[k].ptr();
        if (m[k].t) kind = m[k].kind;
      }
      return;
    }
    // The second half starts b rows into the first tensor.
    b = lp[0].size(0) / 2;
    t[0] = t[1] = lp[0].size(1);
    const int64_t at = b * t[0];
    p[0] = F(lp[0]);
    p[1] = p[0] + at;
    ref[0] = F(rf[0]);
    ref[1] = rf[0] ? ref[0] + (ref_pair ? b : at) : nullptr;
    mask[0] = m[0].ptr();
    kind = m[0].kind;
    const int64_t esz = m[0].t ? m[0].t->element_size() : 0;
    mask[1] = m[0].t ? static_cast<const char*>(mask[0]) + at * esz : nullptr;
  }
  static void check_sizes(const Tensor& chosen, const OptT& rejected, const OptT& ref_c, const OptT& ref_r,
                          const OptT& mask_c, const OptT& mask_r) {
    TORCH_CHECK(chosen.dim() == 2, "chosen: expected shape [pairs, len], got ", chosen.sizes());
    TORCH_CHECK(rejected || (!ref_r && !mask_r), "rejected: its reference and mask go with it");
    TORCH_CHECK(rejected || chosen.size(0) % 2 == 0, "chosen: expected shape [2 * pairs, len], got ", chosen.sizes());
    TORCH_CHECK(!rejected || (rejected->dim() == 2 && rejected->size(0) == chosen.size(0)),
                "rejected: expected as many responses as chosen");
    TORCH_CHECK(!rejected || ((bool)ref_c == (bool)ref_r && (!ref_c || ref_c->dim() == ref_r->dim())),
                "ref_rejected: expected alike with ref_chosen");
    one(chosen, ref_c, mask_c, "chosen", "ref_chosen", "chosen_mask");
    if (rejected) one(*rejected, ref_r, mask_r, "rejected", "ref_rejected", "rejected_mask");
  }
  static void one(const Tensor& lp, const OptT& ref, const OptT& mask, const char* name, const char* ref_name,
                  const char* mask_name) {
    real(lp, lp.sizes(), name);
    if (ref) real(ref, ref->dim() == 1 ? lp.sizes().slice(0, 1) : lp.sizes(), ref_name);
    masks(mask, lp.sizes(), mask_name);
  }
};

// (loss, rewards of the chosen, of the rejected, coefficients [2, pairs])
std::tuple<Tensor, Tensor, Tensor, Tensor> op_preference(const Tensor& chosen, const OptT& rejected, const OptT& ref_chosen,
                                                 const OptT& ref_rejected, const OptT& chosen_mask,
                                                 const OptT& rejected_mask, double beta, double smoothing,
                                                 int64_t kind, bool normalized) {
  const Placed placed(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask);
  const Pairs q(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask);
  Tensor loss = like(q.lp[0], {}), good = like(q.lp[0], {q.b}), bad = like(q.lp[0], {q.b});
  Tensor coef = like(q.lp[0], {2, q.b});
  const int64_t want = 64 * q.b < (1 << 20) ? (1 << 20) : 64 * q.b;
  Tensor ws = workspace_for(q.lp[0].device(), stream_of(q.lp[0]), want);
  check(rls_preference_loss(q.p[0], q.p[1], q.ref[0], q.ref[1], q.ref_pair, q.mask[0], q.mask[1], q.kind, q.b, q.t[0],
                            q.t[1], (float)beta, (float)smoothing, (int)kind, normalized, loss.data_ptr<float>(),
                            W(good), W(bad), W(coef), ws.data_ptr(), (size_t)ws.numel(), stream_of(q.lp[0])),
        "rls_preference_loss");
  return {loss, good, bad, coef};
}

// The gradients by (chosen, rejected); where `halves`, one gradient over both
// halves and an empty tensor.
std::tuple<Tensor, Tensor> op_preference_backward(const Tensor& coef, const Tensor& grad_loss,
                                                  const OptT& chosen_mask, const OptT& rejected_mask,
                                                  int64_t chosen_len, int64_t rejected_len, bool halves) {
  const Placed placed(coef, grad_loss, chosen_mask, rejected_mask);
  TORCH_CHECK(coef.dim() == 2 && chosen_len >= 0 && rejected_len >= 0, "coef: expected shape [2, pairs], and lengths");
  const int64_t b = coef.size(1);
  kept(coef, {2, b}, at::kFloat, "coef");
  scalar(grad_loss, "grad_loss");
  masks(chosen_mask, {halves ? 2 * b : b, chosen_len}, "chosen_mask");
  masks(rejected_mask, {b, rejected_len}, "rejected_mask");
  const Tensor g = f32(grad_loss);
  MaskArg m[2] = {mask_arg(chosen_mask), mask_arg(rejected_mask)};
  if (m[0].t && m[1].t && m[0].kind != m[1].kind)
    for (auto& x : m) x = mask_arg(x.t->ne(0));
  const int kind = m[0].t ? m[0].kind : m[1].kind;
  Tensor gc, gr;
  if (halves) {
    // coefficients [2, b] are those of 2b rows one below the other
    gc = like(coef, {2 * b, chosen_len});
    gr = none(coef, kGradient);
    check(rls_preference_loss_backward(W(coef), F(g), m[0].ptr(), nullptr, kind, W(gc), nullptr, 2 * b, chosen_len, 0,
                                       stream_of(coef)),
          "rls_preference_loss_backward");
  } else {
    gc = like(coef, {b, chosen_len});
    gr = like(coef, {b, rejected_len});
    check(rls_preference_loss_backward(W(coef), F(g), m[0].ptr(), m[1].ptr(), kind, W(gc), W(gr), b, chosen_len,
                                       rejected_len, stream_of(coef)),
          "rls_preference_loss_backward");
  }
  return {gc, gr};
}

// ---- autograd ------------------------------------------------------------------------
// Calls an operator of this file through the dispatcher where something has to see
// the call (fake or functional tensors, a dispatch mode, a profiler), straight otherwise.
template <class Sig>
struct Inner;
template <class R, class... A>
struct Inner<R(A...)> {
  c10::TypedOperatorHandle<R(A...)> handle;
  R (*kernel)(A...);
  template <class... B>
  R call(const Tensor& first, B&&... rest) const {
    const bool seen =
        first.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize})) ||
        !first.is_cuda() || c10::impl::TorchDispatchModeTLS::any_modes_set() || at::hasCallbacks() ||
        // a backward call that is itself to be differentiated: the dispatcher's fallback refuses
        (at::GradMode::is_enabled() && !c10::impl::tls_is_dispatch_key_excluded(c10::DispatchKey::AutogradCUDA));
    return seen ? through(first, std::forward<B>(rest)...) : straight(first, std::forward<B>(rest)...);
  }

 private:
  template <class... B>
  R through(const Tensor& first, B&&... rest) const {
    return handle.call(const_cast<Tensor&>(first), std::forward<B>(rest)...);
  }
  template <class... B>
  R straight(const Tensor& first, B&&... rest) const {
    return kernel(const_cast<Tensor&>(first), std::forward<B>(rest)...);
  }
};
template <class R, class... A>
Inner<R(A...)> inner(const char* name, R (*kernel)(A...)) {
  return {c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<R(A...)>(), kernel};
}

// What a policy loss keeps for its backward call besides tensors: the
// arguments, and the gradient written by the forward call until it is handed out.
struct Kept : public torch::CustomClassHolder {
  double clip_low, clip_high, dual_clip, kl_coef, entropy_coef = 0.0, temperature = 1.0, grad_scale;
  int64_t kl, reduction;
  Tensor grad;
  // The gradient's buffer, once; an undefined tensor after that.
  Tensor take() {
    std::lock_guard<std::mutex> lock(mu);
    return std::exchange(grad, Tensor());
  }
  std::mutex mu;
};
Kept& kept_of(AutogradContext* ctx) {
  return *static_cast<Kept*>(ctx->saved_data.begin()->second.toCapsule().get());
}

// The losses' gradients have no derivative of their own.  Where the backward call is
// itself recorded (create_graph) they get a node that raises once it is reached, on
// the way to `sources`, so that a term that is made of them cannot get lost.
void no_second_derivative(const char* name, torch::autograd::edge_list sources, const variable_list& grads) {
  if (!at::GradMode::is_enabled()) return;
  auto node = std::make_shared<torch::autograd::NotImplemented>(name, std::move(sources));
  for (const Tensor& g : grads)
    if (g.defined()) torch::autograd::set_history(g, node);
}
// The sources of a loss that does not save them.
struct Sources : public torch::CustomClassHolder {
  torch::autograd::edge_list edges;
};

Tensor call_grad_buffer(const Tensor& logits) {
  static auto op = inner("rl_triton::_grad_buffer", &op_grad_buffer);
  return op.call(logits);
}

// Forward-mode tangents would be dropped in silence below autograd.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptT& t) { return t && has_tangent(*t); }
template <class... Ts>
void no_tangents(const char* name, const Ts&... t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(t) || ...), name, ": forward-mode derivatives are not implemented");
}

struct TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, const OptT& mask,
                               double temperature, bool entropy) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = inner("rl_triton::_token_logprobs", &op_logprobs);
    auto [lp, ent, stats, order] = op.call(logits, tokens, mask, temperature, entropy, true);
    ctx->save_for_backward({logits, tokens, plain(mask), order, stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->set_materialize_grads(false);
    if (!entropy) ctx->mark_non_differentiable({ent});
    return {lp, ent};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    static auto op = inner("rl_triton::_token_logprobs_backward", &op_logprobs_backward);
    const auto s = ctx->get_saved_variables();
    Tensor out;
    if (g[0].defined() || g[1].defined())
      out = op.call(s[0], s[1], opt(s[2]), s[3], s[4], opt(g[0]), opt(g[1]), ctx->saved_data["temperature"].toDouble());
    return {out, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> token_logprobs_autograd(const Tensor& logits, const Tensor& tokens, const OptT& mask,
                                                   double temperature, bool entropy) {
  no_tangents("rl_triton::token_logprobs", logits, mask);
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    auto o = TokenLogprobs::apply(logits, tokens, mask, temperature, entropy);
    return {o[0], o[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = inner("rl_triton::_token_logprobs", &op_logprobs);
  auto [lp, ent, stats, order] = op.call(logits, tokens, mask, temperature, entropy, false);
  return {lp, ent};
}

struct PolicyLoss : public torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& lp, const Tensor& old_lp, const Tensor& adv,
                               const OptT& mask, const OptT& ref, double clip_low, double clip_high, double dual_clip,
                               double kl_coef, int64_t kl, int64_t reduction, double grad_scale, bool need_stats) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = inner("rl_triton::_policy_loss", &op_policy);
    auto [loss, stats, norm, grad] = op.call(lp, old_lp, adv, mask, ref, clip_low, clip_high, dual_clip, kl_coef, kl,
                                             reduction, grad_scale, need_stats, true);
    ctx->save_for_backward({lp, old_lp, adv, plain(mask), plain(ref), norm});
    auto k = c10::make_intrusive<Kept>();
    k->clip_low = clip_low; k->clip_high = clip_high; k->dual_clip = dual_clip; k->kl_coef = kl_coef;
    k->grad_scale = grad_scale; k->kl = kl; k->reduction = reduction;
    k->grad = grad;
    ctx->saved_data["kept"] = c10::IValue::make_capsule(std::move(k));
    ctx->mark_non_differentiable({stats});
    ctx->set_materialize_grads(false);
    return {loss, stats};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    static auto op = inner("rl_triton::_policy_loss_backward_", &op_policy_backward_);
    if (!g[0].defined()) return variable_list(13);
    const auto s = ctx->get_saved_variables();
    Kept& k = kept_of(ctx);
    Tensor grad = k.take();
    const bool fresh = !grad.defined();
    if (fresh) grad = at::empty(s[0].sizes(), s[0].options().dtype(at::kFloat));
    op.call(grad, s[0], s[1], s[2], opt(s[3]), opt(s[4]), s[5], g[0], k.clip_low, k.clip_high, k.dual_clip, k.kl_coef,
            k.kl, k.reduction, k.grad_scale, fresh);
    variable_list out(13);
    out[0] = s[0].scalar_type() == at::kFloat ? grad : grad.to(s[0].scalar_type());
    no_second_derivative("the gradient of rl_triton::policy_loss", torch::autograd::collect_next_edges(s[0], g[0]),
                         {out[0]});
    return out;
  }
};

std::tuple<Tensor, Tensor> policy_loss_autograd(const Tensor& lp, const Tensor& old_lp, const Tensor& adv,
                                                const OptT& mask, const OptT& ref, double clip_low, double clip_high,
                                                double dual_clip, double kl_coef, int64_t kl, int64_t reduction,
                                                double grad_scale, bool need_stats) {
  no_tangents("rl_triton::policy_loss", lp, old_lp, adv, mask, ref);
  if (at::GradMode::is_enabled() && lp.requires_grad()) {
    auto o = PolicyLoss::apply(lp, old_lp, adv, mask, ref, clip_low, clip_high, dual_clip, kl_coef, kl, reduction,
                               grad_scale, need_stats);
    return {o[0], o[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = inner("rl_triton::_policy_loss", &op_policy);
  auto [loss, stats, norm, grad] = op.call(lp, old_lp, adv, mask, ref, clip_low, clip_high, dual_clip, kl_coef, kl,
                                           reduction, grad_scale, need_stats, false);
  return {loss, stats};
}

struct PolicyLossLogits : public torch::autograd::Function<PolicyLossLogits> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, const Tensor& old_lp,
                               const Tensor& adv, const OptT& mask, const OptT& ref, double clip_low, double clip_high,
                               double dual_clip, double kl_coef, int64_t kl, double entropy_coef, bool need_stats,
                               double temperature, int64_t reduction, double grad_scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = inner("rl_triton::_policy_loss_logits", &op_policy_logits);
    auto [loss, lp, ent, stats, norm, order, rows, grad] =
        op.call(logits, tokens, old_lp, adv, mask, ref, clip_low, clip_high, dual_clip, kl_coef, kl, entropy_coef,
                need_stats, temperature, reduction, grad_scale, true);
    ctx->save_for_backward({logits, tokens, old_lp, adv, plain(mask), plain(ref), norm, order, rows});
    auto k = c10::make_intrusive<Kept>();
    k->clip_low = clip_low; k->clip_high = clip_high; k->dual_clip = dual_clip; k->kl_coef = kl_coef;
    k->entropy_coef = entropy_coef; k->temperature = temperature; k->grad_scale = grad_scale;
    k->kl = kl; k->reduction = reduction;
    k->grad = grad;
    ctx->saved_data["kept"] = c10::IValue::make_capsule(std::move(k));
    ctx->mark_non_differentiable({lp, ent, stats});
    ctx->set_materialize_grads(false);
    return {loss, lp, ent, stats};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    static auto op = inner("rl_triton::_policy_loss_logits_backward_", &op_policy_logits_backward_);
    if (!g[0].defined()) return variable_list(16);
    const auto s = ctx->get_saved_variables();
    Kept& k = kept_of(ctx);
    Tensor grad = k.take();
    const bool fresh = !grad.defined();
    if (fresh) grad = call_grad_buffer(s[0]);
    op.call(grad, s[0], s[1], s[2], s[3], opt(s[4]), opt(s[5]), s[6], s[7], s[8], g[0], k.clip_low, k.clip_high, k.dual_clip,
            k.kl_coef, k.kl, k.entropy_coef, k.temperature, k.reduction, k.grad_scale, fresh);
    variable_list out(16);
    out[0] = grad;
    no_second_derivative("the gradient of rl_triton::policy_loss_logits",
                         torch::autograd::collect_next_edges(s[0], g[0]), {out[0]});
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss_logits_autograd(
    const Tensor& logits, const Tensor& tokens, const Tensor& old_lp, const Tensor& adv, const OptT& mask,
    const OptT& ref, double clip_low, double clip_high, double dual_clip, double kl_coef, int64_t kl,
    double entropy_coef, bool need_stats, double temperature, int64_t reduction, double grad_scale) {
  no_tangents("rl_triton::policy_loss_logits", logits, old_lp, adv, mask, ref);
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    auto o = PolicyLossLogits::apply(logits, tokens, old_lp, adv, mask, ref, clip_low, clip_high, dual_clip, kl_coef,
                                     kl, entropy_coef, need_stats, temperature, reduction, grad_scale);
    return {o[0], o[1], o[2], o[3]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = inner("rl_triton::_policy_loss_logits", &op_policy_logits);
  auto r = op.call(logits, tokens, old_lp, adv, mask, ref, clip_low, clip_high, dual_clip, kl_coef, kl, entropy_coef,
                   need_stats, temperature, reduction, grad_scale, false);
  return {std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r)};
}

struct PreferenceLoss : public torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& chosen, const OptT& rejected, const OptT& ref_c,
                               const OptT& ref_r, const OptT& mask_c, const OptT& mask_r, double beta,
                               double smoothing, int64_t kind, bool normalized) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = inner("rl_triton::_preference_loss", &op_preference);
    auto [loss, good, bad, coef] = op.call(chosen, rejected, ref_c, ref_r, mask_c, mask_r, beta, smoothing, kind,
                                         normalized);
    ctx->save_for_backward({coef, plain(mask_c), plain(mask_r)});
    ctx->saved_data["len"] = chosen.size(1);
    ctx->saved_data["rejected_len"] = rejected ? rejected->size(1) : (int64_t)-1;
    ctx->saved_data["types"] = std::vector<int64_t>{
        (int64_t)chosen.scalar_type(), (int64_t)(rejected ? rejected->scalar_type() : chosen.scalar_type())};
    auto sources = c10::make_intrusive<Sources>();
    sources->edges = rejected ? torch::autograd::collect_next_edges(chosen, *rejected)
                              : torch::autograd::collect_next_edges(chosen);
    ctx->saved_data["sources"] = c10::IValue::make_capsule(std::move(sources));
    ctx->mark_non_differentiable({good, bad});
    ctx->set_materialize_grads(false);
    return {loss, good, bad};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    static auto op = inner("rl_triton::_preference_loss_backward", &op_preference_backward);
    if (!g[0].defined()) return variable_list(10);
    const auto s = ctx->get_saved_variables();
    const int64_t other = ctx->saved_data["rejected_len"].toInt();
    auto [gc, gr] = op.call(s[0], g[0], opt(s[1]), opt(s[2]), ctx->saved_data["len"].toInt(), other < 0 ? 0 : other,
                            other < 0);
    const auto types = ctx->saved_data["types"].toIntVector();
    variable_list out(10);
    out[0] = gc.to((at::ScalarType)types[0]);
    if (other >= 0) out[1] = gr.to((at::ScalarType)types[1]);
    if (at::GradMode::is_enabled()) {
      auto edges = static_cast<Sources*>(ctx->saved_data["sources"].toCapsule().get())->edges;
      for (auto& e : torch::autograd::collect_next_edges(g[0])) edges.push_back(std::move(e));
      no_second_derivative("the gradient of rl_triton::preference_loss", std::move(edges), out);
    }
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor> preference_loss_autograd(const Tensor& chosen, const OptT& rejected, const OptT& ref_c,
                                                    const OptT& ref_r, const OptT& mask_c, const OptT& mask_r,
                                                    double beta, double smoothing, int64_t kind, bool normalized) {
  no_tangents("rl_triton::preference_loss", chosen, rejected, ref_c, ref_r, mask_c, mask_r);
  if (at::GradMode::is_enabled() && (chosen.requires_grad() || (rejected && rejected->requires_grad()))) {
    auto o = PreferenceLoss::apply(chosen, rejected, ref_c, ref_r, mask_c, mask_r, beta, smoothing, kind, normalized);
    return {o[0], o[1], o[2]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = inner("rl_triton::_preference_loss", &op_preference);
  auto [loss, good, bad, coef] = op.call(chosen, rejected, ref_c, ref_r, mask_c, mask_r, beta, smoothing, kind,
                                       normalized);
  return {loss, good, bad};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(rl_triton, m) {
  m.def("token_logprobs(Tensor logits, Tensor tokens, Tensor? mask, float temperature, bool entropy) "
        "-> (Tensor, Tensor)");
  m.def("policy_loss(Tensor logprobs, Tensor old_logprobs, Tensor advantages, Tensor? mask, Tensor? ref_logprobs, "
        "float clip_low, float clip_high, float dual_clip, float kl_coef, int kl, int reduction, float grad_scale, "
        "bool need_stats) -> (Tensor, Tensor)");
  m.def("policy_loss_logits(Tensor logits, Tensor tokens, Tensor old_logprobs, Tensor advantages, Tensor? mask, "
        "Tensor? ref_logprobs, float clip_low, float clip_high, float dual_clip, float kl_coef, int kl, "
        "float entropy_coef, bool need_stats, float temperature, int reduction, float grad_scale) "
        "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def("preference_loss(Tensor chosen, Tensor? rejected, Tensor? ref_chosen, Tensor? ref_rejected, "
        "Tensor? chosen_mask, Tensor? rejected_mask, float beta, float smoothing, int kind, bool normalized) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("_grad_buffer(Tensor logits) -> Tensor");
  m.def("_token_logprobs(Tensor logits, Tensor tokens, Tensor? mask, float temperature, bool entropy, bool keep) "
        "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def("_token_logprobs_backward(Tensor logits, Tensor tokens, Tensor? mask, Tensor order, Tensor row_stats, Tensor? g_logprobs, "
        "Tensor? g_entropy, float temperature) -> Tensor");
  m.def("_policy_loss(Tensor logprobs, Tensor old_logprobs, Tensor advantages, Tensor? mask, Tensor? ref_logprobs, "
        "float clip_low, float clip_high, float dual_clip, float kl_coef, int kl, int reduction, float grad_scale, "
        "bool need_stats, bool need_grad) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("_policy_loss_backward_(Tensor(a!) grad, Tensor logprobs, Tensor old_logprobs, Tensor advantages, "
        "Tensor? mask, Tensor? ref_logprobs, Tensor norm, Tensor grad_loss, float clip_low, float clip_high, "
        "float dual_clip, float kl_coef, int kl, int reduction, float grad_scale, bool force) -> ()");
  m.def("_policy_loss_logits(Tensor logits, Tensor tokens, Tensor old_logprobs, Tensor advantages, Tensor? mask, "
        "Tensor? ref_logprobs, float clip_low, float clip_high, float dual_clip, float kl_coef, int kl, "
        "float entropy_coef, bool need_stats, float temperature, int reduction, float grad_scale, bool need_grad) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("_policy_loss_logits_backward_(Tensor(a!) grad, Tensor logits, Tensor tokens, Tensor old_logprobs, "
        "Tensor advantages, Tensor? mask, Tensor? ref_logprobs, Tensor norm, Tensor order, Tensor row_stats, "
        "Tensor grad_loss, float clip_low, float clip_high, float dual_clip, float kl_coef, int kl, "
        "float entropy_coef, float temperature, int reduction, float grad_scale, bool force) -> ()");
  m.def("_preference_loss(Tensor chosen, Tensor? rejected, Tensor? ref_chosen, Tensor? ref_rejected, "
        "Tensor? chosen_mask, Tensor? rejected_mask, float beta, float smoothing, int kind, bool normalized) "
        "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def("_preference_loss_backward(Tensor coef, Tensor grad_loss, Tensor? chosen_mask, Tensor? rejected_mask, "
        "int chosen_len, int rejected_len, bool halves) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(rl_triton, CUDA, m) {
  m.impl("_grad_buffer", &op_grad_buffer);
  m.impl("_token_logprobs", &op_logprobs);
  m.impl("_token_logprobs_backward", &op_logprobs_backward);
  m.impl("_policy_loss", &op_policy);
  m.impl("_policy_loss_backward_", &op_policy_backward_);
  m.impl("_policy_loss_logits", &op_policy_logits);
  m.impl("_policy_loss_logits_backward_", &op_policy_logits_backward_);
  m.impl("_preference_loss", &op_preference);
  m.impl("_preference_loss_backward", &op_preference_backward);
}

TORCH_LIBRARY_IMPL(rl_triton, Autograd, m) {
  m.impl("token_logprobs", &token_logprobs_autograd);
  m.impl("policy_loss", &policy_loss_autograd);
  m.impl("policy_loss_logits", &policy_loss_logits_autograd);
  m.impl("preference_loss", &preference_loss_autograd);
  // The kernels proper have no second derivative: differentiating them raises (the
  // losses' gradients by no_second_derivative()).
  for (const char* name : {"_token_logprobs", "_token_logprobs_backward", "_policy_loss", "_policy_loss_logits",
                           "_preference_loss", "_preference_loss_backward"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
