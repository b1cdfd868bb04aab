// lm_torch.cpp -- torch binding of the language-model C ABI (include/lm_sm100.h): argument checks,
// outputs and workspaces from torch's caching allocator, torch's current stream of the operands'
// device, and the autograd nodes.
//
// In C++ because a training step calls these once per layer or per batch and the kernels of an
// ordinary call take 5 to 50 us: the same binding through ctypes and Python autograd functions
// cost 150 to 230 us of host time for a forward and a backward.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cstdlib>
#include <vector>

#include "../../../include/lm_sm100.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ---------------------------------------------------------------------------- shared helpers

void check(int status, const char* what) {
  TORCH_CHECK(status == 0, what, ": ", rbf_sm100_strerror(status), " (", rbf_sm100_last_error_detail(), ")");
}

void* ptr(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
const int64_t* iptr(const Tensor& t) { return static_cast<const int64_t*>(ptr(t)); }

rbf_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<rbf_stream_t>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// Every operand passes here.  There is no forward-mode derivative: a tangent would be dropped, which reads as 0.
// The kernels read an operand's bytes, which in a lazily negated view (the imaginary part of a conjugate) have the other sign.
void check_cuda(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), name, " carries a forward-mode tangent: there is no forward-mode derivative");
  TORCH_CHECK(!t.is_neg(), name, " is a lazily negated view: take its resolve_neg()");
}

void check_with(const Tensor& t, const char* name, const Tensor& first, const char* first_name) {
  check_cuda(t, name);
  TORCH_CHECK(t.device() == first.device(), name, " and ", first_name, " must be on the same device");
}

int type_code(at::ScalarType t) {
  return t == at::kFloat ? LM_F32 : t == at::kBFloat16 ? LM_BF16 : t == at::kHalf ? LM_F16 : -1;
}

int dtype_of(const Tensor& t, const char* name) {
  const int code = type_code(t.scalar_type());
  TORCH_CHECK(code >= 0, name, " must be float32, bfloat16 or float16, not ", t.scalar_type());
  return code;
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

Tensor fp32(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

// A gradient that is not itself differentiable.  Where any of the operands that it depends on requires a
// gradient, differentiating it raises: without a graph it would count as a constant.
Tensor once(const Tensor& grad, at::ArrayRef<Tensor> depends_on, const char* name) {
  bool again = false;
  if (grad.defined() && at::GradMode::is_enabled())
    for (const auto& t : depends_on) again = again || wants_grad(t);
  if (!again) return grad;
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " cannot be differentiated twice", 1);
  return (*error)({grad.detach().requires_grad_(true)})[0];
}

// --------------------------------------------------------------------------------- layer norm

// x [..., D] as [rows, D] with contiguous rows: a view where the strides allow one.
Tensor rows_of(const Tensor& x, int64_t D) {
  int64_t n = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) n *= x.size(d);
  Tensor t = x.dim() == 2 ? x : x.reshape({n, D});
  if ((D > 1 && t.stride(1) != 1) || (n > 1 && t.stride(0) < D)) t = t.contiguous();
  return t;
}

at::ScalarType check_ln(const Tensor& x, const Tensor& weight, const Tensor& bias) {
  check_cuda(x, "x");
  TORCH_CHECK(x.dim() > 0, "x must have at least one dimension");
  dtype_of(x, "x");
  auto one = [&](const Tensor& t, const char* name) {
    if (!t.defined()) return;
    check_with(t, name, x, "x");
    TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(-1), name, " must have shape [", x.size(-1), "], not ", t.sizes());
    TORCH_CHECK(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, name,
                " must have x's type or float32, not ", t.scalar_type());
  };
  one(weight, "weight");
  one(bias, "bias");
  if (weight.defined() && bias.defined())
    TORCH_CHECK(weight.scalar_type() == bias.scalar_type(), "weight and bias must have the same type");
  return weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
}

// (y, stats): stats [2, rows] are the means and the reciprocal deviations, undefined unless kept.
std::pair<Tensor, Tensor> ln_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, bool keep) {
  const at::ScalarType wtype = check_ln(x, weight, bias);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t D = x.size(-1);
  const Tensor rows = rows_of(x, D);
  const int64_t n = rows.size(0);
  const Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
  Tensor y = at::empty(x.sizes(), x.options());
  Tensor stats = keep ? fp32({2, n}, x) : Tensor();
  float* mean = keep ? fptr(stats) : nullptr;
  check(ln_sm100_forward(ptr(rows), rows.stride(0), ptr(w), ptr(b), ptr(y), mean, mean ? mean + n : nullptr, n, D,
                         (float)eps, type_code(x.scalar_type()), type_code(wtype), stream_of(x)),
        "ln_sm100_forward");
  return {y, stats};
}

variable_list ln_backward(const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& stats,
                          const std::array<bool, 3>& need, at::ScalarType wtype) {
  check_ln(x, weight, Tensor());
  check_with(dy, "dy", x, "x");
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type(), "dy must have x's shape and type");
  TORCH_CHECK(!weight.defined() || weight.scalar_type() == wtype, "dweight and dbias have weight's type");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t D = x.size(-1);
  const Tensor rx = rows_of(x, D), rdy = rows_of(dy, D);
  const int64_t n = rx.size(0);
  TORCH_CHECK(stats.numel() == 2 * n && stats.scalar_type() == at::kFloat && stats.is_contiguous() &&
                  stats.device() == x.device(),
              "stats must be ln_forward's, one mean and one reciprocal deviation per row of x");
  const Tensor w = weight.defined() ? weight.contiguous() : weight;
  variable_list out(3);
  if (need[0]) out[0] = at::empty(x.sizes(), x.options());
  if (need[1]) out[1] = at::empty({D}, x.options().dtype(wtype));
  if (need[2]) out[2] = at::empty({D}, x.options().dtype(wtype));
  Tensor ws;
  size_t bytes = 0;
  if (need[1] || need[2]) {
    bytes = ln_sm100_backward_workspace_bytes(n, D);
    ws = workspace(bytes, x);
  }
  const float* mean = fptr(stats);
  check(ln_sm100_backward(ptr(rdy), rdy.stride(0), ptr(rx), rx.stride(0), ptr(w), mean, mean ? mean + n : nullptr,
                          ptr(out[0]), ptr(out[1]), ptr(out[2]), n, D, type_code(x.scalar_type()), type_code(wtype),
                          ptr(ws), bytes, stream_of(x)),
        "ln_sm100_backward");
  return out;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    const Tensor w = given(weight), b = given(bias);
    auto [y, stats] = ln_forward(x, w, b, eps, true);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["has_bias"] = b.defined();
    ctx->saved_data["wtype"] = (int64_t)(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    // Edges are counted over the tensors that were given.
    const bool has_w = saved[1].defined(), has_b = ctx->saved_data["has_bias"].toBool();
    const std::array<bool, 3> need = {ctx->needs_input_grad(0), has_w && ctx->needs_input_grad(1),
                                      has_b && ctx->needs_input_grad(has_w ? 2 : 1)};
    auto out = ln_backward(g[0], saved[0], saved[1], saved[2], need, (at::ScalarType)ctx->saved_data["wtype"].toInt());
    const Tensor &x = saved[0], &w = saved[1], &dy = g[0];
    return {once(out[0], {dy, x, w}, "layer_norm"), once(out[1], {dy, x}, "layer_norm"), once(out[2], {dy}, "layer_norm"), Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(given(weight)) || wants_grad(given(bias))))
    return LayerNorm::apply(x, weight, bias, eps);
  return ln_forward(x, given(weight), given(bias), eps, false).first;
}

// ------------------------------------------------------------- log-probabilities of tokens

struct Logits {
  Tensor x;       // rows r at (r / T) * batch_stride + (r % T) * t_stride
  Tensor labels;  // contiguous
  int64_t batch_stride, t_stride, rows, T, V;
  int dtype;
};

Logits check_logits(const Tensor& logits, const Tensor& labels) {
  check_cuda(logits, "logits");
  check_with(labels, "labels", logits, "logits");
  Logits l;
  l.dtype = dtype_of(logits, "logits");
  TORCH_CHECK(logits.dim() >= 2, "logits must have shape [..., V] with at least one leading dimension");
  TORCH_CHECK(labels.scalar_type() == at::kLong, "labels must be int64, not ", labels.scalar_type());
  TORCH_CHECK(labels.sizes() == logits.sizes().slice(0, logits.dim() - 1), "labels must have shape ",
              logits.sizes().slice(0, logits.dim() - 1), ", not ", labels.sizes());
  l.V = logits.size(-1);
  l.rows = labels.numel();
  l.T = logits.size(-2);
  l.x = logits.dim() == 3 ? logits
        : logits.dim() == 2
            ? logits.unsqueeze(0)
            : logits.reshape({l.T > 0 && l.V > 0 ? logits.numel() / (l.T * l.V) : 0, l.T, l.V});
  if (l.V > 1 && l.x.stride(2) != 1) l.x = l.x.contiguous();
  l.batch_stride = l.x.stride(0);
  l.t_stride = l.x.stride(1);
  l.labels = labels.contiguous();
  return l;
}

void logprob_forward(const Logits& l, float* logprob, float* rest, float* stats, int64_t ignore_index) {
  check(lp_sm100_forward(ptr(l.x), l.batch_stride, l.t_stride, iptr(l.labels), logprob, rest, stats, l.rows, l.T, l.V,
                         ignore_index, l.dtype, stream_of(l.x)),
        "lp_sm100_forward");
}

Tensor logprob_backward(const Tensor& logits, const Tensor& labels, const float* stats, const float* coef,
                        const float* scale0, const float* scale1, int64_t ignore_index) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const Logits l = check_logits(logits, labels);
  Tensor dx = at::empty(logits.sizes(), logits.options());
  check(lp_sm100_backward(ptr(l.x), l.batch_stride, l.t_stride, iptr(l.labels), stats, coef, scale0, scale1, ptr(dx),
                          l.rows, l.T, l.V, ignore_index, l.dtype, stream_of(l.x)),
        "lp_sm100_backward");
  return dx;
}

// (logprob of labels' shape, stats [rows, 2]; undefined unless kept).
std::pair<Tensor, Tensor> token_logprob_forward(const Tensor& logits, const Tensor& labels, int64_t ignore_index, bool keep) {
  const Logits l = check_logits(logits, labels);
  const c10::cuda::CUDAGuard guard(logits.device());
  Tensor lp = fp32(labels.sizes(), logits);
  Tensor stats = keep ? fp32({l.rows, 2}, logits) : Tensor();
  logprob_forward(l, fptr(lp), nullptr, fptr(stats), ignore_index);
  return {lp, stats};
}

Tensor token_logprob_backward(const Tensor& logits, const Tensor& labels, const Tensor& stats, const Tensor& g,
                              int64_t ignore_index) {
  check_with(g, "coef", logits, "logits");
  check_with(stats, "stats", logits, "logits");
  TORCH_CHECK(g.scalar_type() == at::kFloat && g.numel() == labels.numel() && stats.scalar_type() == at::kFloat &&
                  stats.numel() == 2 * labels.numel() && stats.is_contiguous(),
              "coef and stats must be float32, one and two values per row");
  const Tensor coef = g.contiguous();
  return logprob_backward(logits, labels, fptr(stats), fptr(coef), nullptr, nullptr, ignore_index);
}

struct TokenLogprob : torch::autograd::Function<TokenLogprob> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, int64_t ignore_index) {
    auto [lp, stats] = token_logprob_forward(logits, labels, ignore_index, true);
    ctx->save_for_backward({logits, labels, stats});
    ctx->saved_data["ignore"] = ignore_index;
    return lp;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const Tensor dx = token_logprob_backward(s[0], s[1], s[2], g[0], ctx->saved_data["ignore"].toInt());
    return {once(dx, {g[0], s[0]}, "token_logprob"), Tensor(), Tensor()};
  }
};

Tensor token_logprob(const Tensor& logits, const Tensor& labels, int64_t ignore_index) {
  if (at::GradMode::is_enabled() && wants_grad(logits)) return TokenLogprob::apply(logits, labels, ignore_index);
  return token_logprob_forward(logits, labels, ignore_index, false).first;
}

// -------------------------------------------------------------------------------- the losses

// A constant of a loss: float32, of `shape`.
Tensor constant(const Tensor& t, at::IntArrayRef shape, const char* name, const Tensor& labels) {
  check_with(t, name, labels, "labels");
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.sizes() == shape, name, " must be float32 with shape ", shape);
  TORCH_CHECK(!t.requires_grad(), name, " is a constant of the loss: it must not require a gradient");
  return t.contiguous();
}

// What a loss keeps for its backward, in one allocation: a common factor, the log-probabilities (and what
// fp32 drops of them), the coefficients d loss / d logprob, and the rows' statistics.
struct LossState {
  Tensor all;
  float *norm, *stats, *logprob, *rest, *coef;
  static int64_t size(int64_t rows) { return 4 + 5 * rows; }
  explicit LossState(const Tensor& state) : all(state) {
    const int64_t n = (state.numel() - 4) / 5;
    norm = fptr(state);
    stats = norm + 4;  // pairs, 8-byte aligned
    logprob = stats + 2 * n;
    rest = logprob + n;
    coef = rest + n;
  }
};

struct LossOut {
  Tensor loss, second, state;
};

LossOut preference_forward(const Tensor& logits, const Tensor& labels, const Tensor& ref_logprob, double beta,
                           double smoothing, int64_t ignore_index) {
  const Logits l = check_logits(logits, labels);
  TORCH_CHECK(logits.dim() == 3, "logits must have shape [B, T, V]");
  TORCH_CHECK(logits.size(0) % 2 == 0, "logits must hold pairs: B is odd");
  const Tensor ref = constant(ref_logprob, labels.sizes(), "ref_logprob", labels);
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t B = logits.size(0), T = logits.size(1);
  LossOut o{fp32({}, logits), fp32({B}, logits), fp32({LossState::size(l.rows)}, logits)};
  const LossState s(o.state);
  const size_t bytes = loss_sm100_workspace_bytes(B, T);
  const Tensor ws = workspace(bytes, logits);
  logprob_forward(l, s.logprob, s.rest, s.stats, ignore_index);
  check(pref_sm100_loss(s.logprob, s.rest, fptr(ref), iptr(l.labels), fptr(o.loss), fptr(o.second), s.coef, B, T, (float)beta,
                        (float)smoothing, ignore_index, ptr(ws), bytes, stream_of(logits)),
        "pref_sm100_loss");
  return o;
}

LossOut policy_forward(const Tensor& logits, const Tensor& labels, const Tensor& old_logprob, const Tensor& ref_logprob,
                       const Tensor& advantage, double clip_low, double clip_high, double kl_coef, int64_t ignore_index) {
  const Logits l = check_logits(logits, labels);
  TORCH_CHECK(logits.dim() == 3, "logits must have shape [B, T, V]");
  const Tensor old = constant(old_logprob, labels.sizes(), "old_logprob", labels);
  const Tensor ref = constant(ref_logprob, labels.sizes(), "ref_logprob", labels);
  TORCH_CHECK(advantage.dim() == 1 || advantage.dim() == 2, "advantage must have shape [B] or [B, T]");
  const Tensor adv = constant(advantage, labels.sizes().slice(0, advantage.dim()), "advantage", labels);
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t B = logits.size(0), T = logits.size(1);
  LossOut o{fp32({}, logits), fp32({}, logits), fp32({LossState::size(l.rows)}, logits)};
  const LossState s(o.state);
  const size_t bytes = loss_sm100_workspace_bytes(B, T);
  const Tensor ws = workspace(bytes, logits);
  logprob_forward(l, s.logprob, s.rest, s.stats, ignore_index);
  check(policy_sm100_loss(s.logprob, s.rest, fptr(old), fptr(ref), fptr(adv), advantage.dim() == 2, iptr(l.labels), fptr(o.loss),
                          fptr(o.second), s.coef, s.norm, B, T, (float)clip_low, (float)clip_high, (float)kl_coef,
                          ignore_index, ptr(ws), bytes, stream_of(logits)),
        "policy_sm100_loss");
  return o;
}

// The gradient of a loss for the upstream gradient g of its scalar.
Tensor loss_backward(const Tensor& logits, const Tensor& labels, const Tensor& state, const Tensor& g, bool normed,
                     int64_t ignore_index) {
  check_with(state, "state", logits, "logits");
  TORCH_CHECK(state.numel() == LossState::size(labels.numel()) && state.scalar_type() == at::kFloat && state.is_contiguous(),
              "state must be the loss's forward's");
  if (g.defined())
    TORCH_CHECK(g.numel() == 1 && g.scalar_type() == at::kFloat && g.device() == logits.device(),
                "the upstream gradient must be one float32 on the logits' device");
  const LossState s(state);
  return logprob_backward(logits, labels, s.stats, s.coef, g.defined() ? fptr(g) : nullptr, normed ? s.norm : nullptr,
                          ignore_index);
}

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, const Tensor& ref_logprob,
                               double beta, double smoothing, int64_t ignore_index) {
    LossOut o = preference_forward(logits, labels, ref_logprob, beta, smoothing, ignore_index);
    ctx->save_for_backward({logits, labels, o.state});
    ctx->saved_data["ignore"] = ignore_index;
    ctx->mark_non_differentiable({o.second});
    return {o.loss, o.second};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    variable_list out(6);
    const Tensor dx = loss_backward(s[0], s[1], s[2], g[0], false, ctx->saved_data["ignore"].toInt());
    out[0] = once(dx, {g[0], s[0]}, "preference_loss");
    return out;
  }
};

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, const Tensor& old_logprob,
                               const Tensor& ref_logprob, const Tensor& advantage, double clip_low, double clip_high,
                               double kl_coef, int64_t ignore_index) {
    LossOut o = policy_forward(logits, labels, old_logprob, ref_logprob, advantage, clip_low, clip_high, kl_coef, ignore_index);
    ctx->save_for_backward({logits, labels, o.state});
    ctx->saved_data["ignore"] = ignore_index;
    ctx->mark_non_differentiable({o.second});
    return {o.loss, o.second};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    variable_list out(9);
    const Tensor dx = loss_backward(s[0], s[1], s[2], g[0], true, ctx->saved_data["ignore"].toInt());
    out[0] = once(dx, {g[0], s[0]}, "policy_loss");
    return out;
  }
};

std::pair<Tensor, Tensor> preference_loss(const Tensor& logits, const Tensor& labels, const Tensor& ref_logprob, double beta,
                                          double smoothing, int64_t ignore_index) {
  if (at::GradMode::is_enabled() && wants_grad(logits)) {
    auto o = PreferenceLoss::apply(logits, labels, ref_logprob, beta, smoothing, ignore_index);
    return {o[0], o[1]};
  }
  LossOut o = preference_forward(logits, labels, ref_logprob, beta, smoothing, ignore_index);
  return {o.loss, o.second};
}

std::pair<Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& labels, const Tensor& old_logprob,
                                      const Tensor& ref_logprob, const Tensor& advantage, double clip_low, double clip_high,
                                      double kl_coef, int64_t ignore_index) {
  if (at::GradMode::is_enabled() && wants_grad(logits)) {
    auto o = PolicyLoss::apply(logits, labels, old_logprob, ref_logprob, advantage, clip_low, clip_high, kl_coef, ignore_index);
    return {o[0], o[1]};
  }
  LossOut o = policy_forward(logits, labels, old_logprob, ref_logprob, advantage, clip_low, clip_high, kl_coef, ignore_index);
  return {o.loss, o.second};
}

// ---------------------------------------------------------------------------- orthogonalise

Tensor orthogonalize(const Tensor& update, const std::vector<float>& coefficients, double eps) {
  check_cuda(update, "update");
  const int dtype = dtype_of(update, "update");
  TORCH_CHECK(update.dim() >= 2, "update must have at least two dimensions");
  TORCH_CHECK(!(at::GradMode::is_enabled() && update.requires_grad()),
              "orthogonalize has no gradient: pass a detached update, or call it under torch.no_grad()");
  TORCH_CHECK(coefficients.size() % 3 == 0, "coefficients must hold (a, b, c) for every step");
  const int steps = (int)(coefficients.size() / 3);
  const int64_t m = update.size(-2), n = update.size(-1);
  const c10::cuda::CUDAGuard guard(update.device());
  Tensor out = at::empty(update.sizes(), update.options());
  const int64_t batch = m > 0 && n > 0 ? update.numel() / (m * n) : 0;
  Tensor g = update.dim() == 3 ? update : update.reshape({batch, m, n});
  if ((n > 1 && g.stride(2) != 1) || (m > 1 && g.stride(1) < n)) g = g.contiguous();
  const size_t bytes = ortho_sm100_workspace_bytes(batch, m, n, steps);
  const Tensor ws = workspace(bytes, update);
  check(ortho_sm100(ptr(g), g.stride(1), g.stride(0), ptr(out), batch, m, n, coefficients.data(), steps, (float)eps, dtype,
                    ptr(ws), bytes, stream_of(update)),
        "ortho_sm100");
  const char* env = std::getenv("RBF_CHECK_STATUS");
  // Not while the stream is captured: there is nothing to read yet, and waiting would end the capture.
  if (env != nullptr && *env != '\0' && std::string(env) != "0" && out.numel() > 0 &&
      c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) {
    int status = 0;
    check(rbf_sm100_read_status(ptr(ws), stream_of(update), &status), "rbf_sm100_read_status");
    TORCH_CHECK(status == 0, "orthogonalize: device status ", status, " (a bounded device-side wait timed out)");
  }
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("layer_norm", &layer_norm);
  m.def("ln_forward", [](const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, bool keep) {
    auto [y, stats] = ln_forward(x, given(w), given(b), eps, keep);
    return std::make_pair(y, keep ? OptTensor(stats) : OptTensor());
  });
  m.def("ln_backward", [](const Tensor& dy, const Tensor& x, const OptTensor& w, const Tensor& stats,
                          const std::array<bool, 3>& need, const OptTensor& like) {
    const Tensor weight = given(w);
    const at::ScalarType type = weight.defined() ? weight.scalar_type() : like.has_value() ? like->scalar_type() : x.scalar_type();
    auto out = ln_backward(dy, x, weight, stats, need, type);
    std::vector<OptTensor> r;
    for (auto& t : out) r.push_back(t.defined() ? OptTensor(t) : OptTensor());
    return r;
  });
  m.def("token_logprob", &token_logprob);
  m.def("logprob_forward", [](const Tensor& logits, const Tensor& labels, int64_t ignore, bool keep) {
    auto [lp, stats] = token_logprob_forward(logits, labels, ignore, keep);
    return std::make_pair(lp, keep ? OptTensor(stats) : OptTensor());
  });
  m.def("logprob_backward", &token_logprob_backward);
  m.def("preference_loss", &preference_loss);
  m.def("preference_forward", [](const Tensor& logits, const Tensor& labels, const Tensor& ref, double beta, double s, int64_t ignore) {
    LossOut o = preference_forward(logits, labels, ref, beta, s, ignore);
    return std::make_tuple(o.loss, o.second, o.state);
  });
  m.def("policy_loss", &policy_loss);
  m.def("policy_forward", [](const Tensor& logits, const Tensor& labels, const Tensor& old, const Tensor& ref, const Tensor& adv,
                             double lo, double hi, double k, int64_t ignore) {
    LossOut o = policy_forward(logits, labels, old, ref, adv, lo, hi, k, ignore);
    return std::make_tuple(o.loss, o.second, o.state);
  });
  m.def("loss_backward", [](const Tensor& logits, const Tensor& labels, const Tensor& state, const OptTensor& g, bool normed, int64_t ignore) {
    return loss_backward(logits, labels, state, given(g), normed, ignore);
  });
  m.def("orthogonalize", &orthogonalize);
}
