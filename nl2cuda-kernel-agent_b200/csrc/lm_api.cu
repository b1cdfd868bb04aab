// lm_api.cu -- the C ABI of include/lm_sm100.h: argument checks and dispatch.  Every check that can
// fail on bad arguments runs on the host before any CUDA call, as in rbf_api.cu.
#include <cmath>
#include <cstdio>

#include "lm_common.cuh"
#include "lm_kernels.cuh"

namespace rbf {
namespace lm {
namespace {

constexpr int64_t kMaxRows = int64_t(1) << 31;

int refuse(int status, const char* what) { return set_detail(status, what); }

// A pointer that has `elems` elements must be there, on a boundary of `align` bytes.
int need(const void* p, int64_t elems, size_t align, const char* name) {
  if (elems == 0) return RBF_OK;
  char b[96];
  if (p == nullptr) {
    std::snprintf(b, sizeof(b), "%s is NULL but has %lld elements", name, (long long)elems);
    return set_detail(RBF_ERR_INVALID_ARGUMENT, b);
  }
  if (reinterpret_cast<uintptr_t>(p) % align != 0) {
    std::snprintf(b, sizeof(b), "%s is not aligned to %d bytes", name, (int)align);
    return set_detail(RBF_ERR_MISALIGNED, b);
  }
  return RBF_OK;
}

int check_workspace(const void* ws, size_t have, size_t want) {
  if (want == 0) return RBF_OK;
  if (ws == nullptr || have < want) return refuse(RBF_ERR_WORKSPACE, "workspace too small");
  if (reinterpret_cast<uintptr_t>(ws) % 16 != 0)
    return refuse(RBF_ERR_MISALIGNED, "workspace is not 16-byte aligned");
  return RBF_OK;
}

int check_ln(int64_t rows, int64_t D, int64_t stride, int dtype, int wdtype) {
  if (rows < 0 || D < 0) return refuse(RBF_ERR_INVALID_ARGUMENT, "negative size");
  if (rows >= kMaxRows || D >= kMaxRows) return refuse(RBF_ERR_UNSUPPORTED, "rows or D >= 2^31");
  if (!dtype_ok(dtype) || !dtype_ok(wdtype)) return refuse(RBF_ERR_INVALID_ARGUMENT, "unknown element type");
  if (rows > 1 && stride < D) return refuse(RBF_ERR_INVALID_ARGUMENT, "row stride smaller than D");
  return RBF_OK;
}

int check_logits(int64_t batch_stride, int64_t t_stride, int64_t rows, int64_t T, int64_t V, int dtype) {
  if (rows < 0 || T < 0 || V < 0) return refuse(RBF_ERR_INVALID_ARGUMENT, "negative size");
  if (rows >= kMaxRows / 8 || V >= kMaxRows) return refuse(RBF_ERR_UNSUPPORTED, "rows >= 2^28 or V >= 2^31");
  if (rows > 0 && (T == 0 || rows % T != 0))
    return refuse(RBF_ERR_INVALID_ARGUMENT, "rows must be a multiple of T");
  if (rows > 0 && V == 0) return refuse(RBF_ERR_INVALID_ARGUMENT, "empty vocabulary");
  if (!dtype_ok(dtype)) return refuse(RBF_ERR_INVALID_ARGUMENT, "unknown element type");
  if (batch_stride < 0 || t_stride < 0) return refuse(RBF_ERR_INVALID_ARGUMENT, "negative stride");
  return RBF_OK;
}

int check_loss(int64_t B, int64_t T) {
  if (B < 0 || T < 0) return refuse(RBF_ERR_INVALID_ARGUMENT, "negative size");
  if (B >= kMaxRows || T >= kMaxRows || (T > 0 && B >= (int64_t(1) << 40) / T))
    return refuse(RBF_ERR_UNSUPPORTED, "B or T too large");
  return RBF_OK;
}

cudaStream_t as_stream(rbf_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace
}  // namespace lm
}  // namespace rbf

using namespace rbf;
using namespace rbf::lm;

extern "C" {

int ln_sm100_forward(const void* x, int64_t x_stride, const void* weight, const void* bias, void* y,
                     float* mean, float* rstd, int64_t rows, int64_t D, float eps, int dtype,
                     int wdtype, rbf_stream_t stream) {
  int st = check_ln(rows, D, x_stride, dtype, wdtype);
  if (st) return st;
  if (!std::isfinite(eps) || eps < 0.f) return refuse(RBF_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  const size_t e = elem_bytes(dtype), we = elem_bytes(wdtype);
  if ((st = need(x, rows * D, e, "x"))) return st;
  if ((st = need(y, rows * D, e, "y"))) return st;
  if (weight != nullptr && (st = need(weight, D, we, "weight"))) return st;
  if (bias != nullptr && (st = need(bias, D, we, "bias"))) return st;
  if ((mean == nullptr) != (rstd == nullptr))
    return refuse(RBF_ERR_INVALID_ARGUMENT, "mean and rstd go together");
  if ((st = check_device())) return st;
  LnArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.weight = weight;
  a.bias = bias;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.rows = rows;
  a.D = D;
  a.eps = eps;
  a.dtype = dtype;
  a.wdtype = wdtype;
  return cuda_status(launch_ln_forward(a, as_stream(stream)), "layer norm launch");
}

size_t ln_sm100_backward_workspace_bytes(int64_t rows, int64_t D) {
  if (rows < 0 || D < 0) return 0;
  return sizeof(float) * 2 * (size_t)ln_backward_parts(rows, D) * (size_t)D;
}

int ln_sm100_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                      const void* weight, const float* mean, const float* rstd, void* dx,
                      void* dweight, void* dbias, int64_t rows, int64_t D, int dtype, int wdtype,
                      void* workspace, size_t workspace_bytes, rbf_stream_t stream) {
  int st = check_ln(rows, D, x_stride < dy_stride ? x_stride : dy_stride, dtype, wdtype);
  if (st) return st;
  const size_t e = elem_bytes(dtype), we = elem_bytes(wdtype);
  if ((st = need(dy, rows * D, e, "dy"))) return st;
  if ((st = need(x, rows * D, e, "x"))) return st;
  if (weight != nullptr && (st = need(weight, D, we, "weight"))) return st;
  if ((st = need(mean, rows, 4, "mean"))) return st;
  if ((st = need(rstd, rows, 4, "rstd"))) return st;
  if (dx != nullptr && (st = need(dx, rows * D, e, "dx"))) return st;
  if (dweight != nullptr && (st = need(dweight, D, we, "dweight"))) return st;
  if (dbias != nullptr && (st = need(dbias, D, we, "dbias"))) return st;
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (sums && (st = check_workspace(workspace, workspace_bytes, ln_sm100_backward_workspace_bytes(rows, D))))
    return st;
  if (dx == nullptr && !sums) return RBF_OK;
  if ((st = check_device())) return st;
  LnArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.dy = dy;
  a.dy_stride = dy_stride;
  a.weight = weight;
  a.y = dx;
  a.dw = dweight;
  a.db = dbias;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.part = static_cast<float*>(workspace);
  a.rows = rows;
  a.D = D;
  a.dtype = dtype;
  a.wdtype = wdtype;
  return cuda_status(launch_ln_backward(a, as_stream(stream)), "layer norm backward launch");
}

int lp_sm100_forward(const void* logits, int64_t batch_stride, int64_t t_stride,
                     const int64_t* labels, float* logprob, float* rest, float* stats, int64_t rows,
                     int64_t T, int64_t V, int64_t ignore_index, int dtype, rbf_stream_t stream) {
  int st = check_logits(batch_stride, t_stride, rows, T, V, dtype);
  if (st) return st;
  if ((st = need(logits, rows * V, elem_bytes(dtype), "logits"))) return st;
  if ((st = need(labels, rows, 8, "labels"))) return st;
  if ((st = need(logprob, rows, 4, "logprob"))) return st;
  if (rest != nullptr && (st = need(rest, rows, 4, "rest"))) return st;
  if (stats != nullptr && (st = need(stats, rows, 8, "stats"))) return st;
  if ((st = check_device())) return st;
  LogitArgs a{};
  a.logits = logits;
  a.batch_stride = batch_stride;
  a.t_stride = t_stride;
  a.labels = labels;
  a.rows = rows;
  a.T = T;
  a.V = V;
  a.ignore_index = ignore_index;
  a.dtype = dtype;
  a.logprob = logprob;
  a.rest = rest;
  a.stats = stats;
  return cuda_status(launch_logprob_forward(a, as_stream(stream)), "log-probability launch");
}

int lp_sm100_backward(const void* logits, int64_t batch_stride, int64_t t_stride,
                      const int64_t* labels, const float* stats, const float* coef,
                      const float* scale0, const float* scale1, void* dlogits, int64_t rows,
                      int64_t T, int64_t V, int64_t ignore_index, int dtype, rbf_stream_t stream) {
  int st = check_logits(batch_stride, t_stride, rows, T, V, dtype);
  if (st) return st;
  const size_t e = elem_bytes(dtype);
  if ((st = need(logits, rows * V, e, "logits"))) return st;
  if ((st = need(labels, rows, 8, "labels"))) return st;
  if ((st = need(stats, rows, 8, "stats"))) return st;
  if ((st = need(coef, rows, 4, "coef"))) return st;
  if ((st = need(dlogits, rows * V, e, "dlogits"))) return st;
  if (scale0 != nullptr && (st = need(scale0, 1, 4, "scale0"))) return st;
  if (scale1 != nullptr && (st = need(scale1, 1, 4, "scale1"))) return st;
  if ((st = check_device())) return st;
  LogitArgs a{};
  a.logits = logits;
  a.batch_stride = batch_stride;
  a.t_stride = t_stride;
  a.labels = labels;
  a.rows = rows;
  a.T = T;
  a.V = V;
  a.ignore_index = ignore_index;
  a.dtype = dtype;
  a.stats = const_cast<float*>(stats);
  a.coef = coef;
  a.scale0 = scale0;
  a.scale1 = scale1;
  a.dlogits = dlogits;
  return cuda_status(launch_logprob_backward(a, as_stream(stream)), "log-probability backward launch");
}

size_t loss_sm100_workspace_bytes(int64_t B, int64_t T) {
  if (B < 0 || T < 0) return 0;
  return loss_workspace_bytes(B, T);
}

int pref_sm100_loss(const float* logprob, const float* rest, const float* ref_logprob, const int64_t* labels,
                    float* loss, float* reward, float* coef, int64_t B, int64_t T, float beta,
                    float label_smoothing, int64_t ignore_index, void* workspace,
                    size_t workspace_bytes, rbf_stream_t stream) {
  int st = check_loss(B, T);
  if (st) return st;
  if (B % 2 != 0) return refuse(RBF_ERR_INVALID_ARGUMENT, "B must be even (pairs)");
  if (!std::isfinite(beta)) return refuse(RBF_ERR_INVALID_ARGUMENT, "beta is not finite");
  if (!(label_smoothing >= 0.f && label_smoothing <= 1.f))
    return refuse(RBF_ERR_INVALID_ARGUMENT, "label_smoothing must be in [0, 1]");
  if ((st = need(logprob, B * T, 4, "logprob"))) return st;
  if (rest != nullptr && (st = need(rest, B * T, 4, "rest"))) return st;
  if ((st = need(ref_logprob, B * T, 4, "ref_logprob"))) return st;
  if ((st = need(labels, B * T, 8, "labels"))) return st;
  if ((st = need(loss, 1, 4, "loss"))) return st;
  if ((st = need(reward, B, 4, "reward"))) return st;
  if ((st = need(coef, B * T, 4, "coef"))) return st;
  if ((st = check_workspace(workspace, workspace_bytes, loss_workspace_bytes(B, T)))) return st;
  if ((st = check_device())) return st;
  LossArgs a{};
  a.logprob = logprob;
  a.rest = rest;
  a.ref_logprob = ref_logprob;
  a.labels = labels;
  a.loss = loss;
  a.second = reward;
  a.coef = coef;
  a.part = static_cast<double*>(workspace);
  a.B = B;
  a.T = T;
  a.ignore_index = ignore_index;
  a.beta = beta;
  a.smoothing = label_smoothing;
  return cuda_status(launch_loss(a, true, as_stream(stream)), "preference loss launch");
}

int policy_sm100_loss(const float* logprob, const float* rest, const float* old_logprob, const float* ref_logprob,
                      const float* advantage, int per_token, const int64_t* labels, float* loss,
                      float* kl, float* coef, float* norm, int64_t B, int64_t T, float clip_low,
                      float clip_high, float kl_coef, int64_t ignore_index, void* workspace,
                      size_t workspace_bytes, rbf_stream_t stream) {
  int st = check_loss(B, T);
  if (st) return st;
  if (!(clip_low >= 0.f) || !(clip_high >= 0.f))
    return refuse(RBF_ERR_INVALID_ARGUMENT, "clip_low and clip_high must be >= 0");
  if (!std::isfinite(kl_coef)) return refuse(RBF_ERR_INVALID_ARGUMENT, "kl_coef is not finite");
  if ((st = need(logprob, B * T, 4, "logprob"))) return st;
  if (rest != nullptr && (st = need(rest, B * T, 4, "rest"))) return st;
  if ((st = need(old_logprob, B * T, 4, "old_logprob"))) return st;
  if ((st = need(ref_logprob, B * T, 4, "ref_logprob"))) return st;
  if ((st = need(advantage, per_token ? B * T : B, 4, "advantage"))) return st;
  if ((st = need(labels, B * T, 8, "labels"))) return st;
  if ((st = need(loss, 1, 4, "loss"))) return st;
  if ((st = need(kl, 1, 4, "kl"))) return st;
  if ((st = need(norm, 1, 4, "norm"))) return st;
  if ((st = need(coef, B * T, 4, "coef"))) return st;
  if ((st = check_workspace(workspace, workspace_bytes, loss_workspace_bytes(B, T)))) return st;
  if ((st = check_device())) return st;
  LossArgs a{};
  a.logprob = logprob;
  a.rest = rest;
  a.old_logprob = old_logprob;
  a.ref_logprob = ref_logprob;
  a.advantage = advantage;
  a.per_token = per_token != 0;
  a.labels = labels;
  a.loss = loss;
  a.second = kl;
  a.coef = coef;
  a.norm = norm;
  a.part = static_cast<double*>(workspace);
  a.B = B;
  a.T = T;
  a.ignore_index = ignore_index;
  a.clip_low = clip_low;
  a.clip_high = clip_high;
  a.kl_coef = kl_coef;
  return cuda_status(launch_loss(a, false, as_stream(stream)), "policy loss launch");
}

size_t ortho_sm100_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int steps) {
  if (batch < 0 || rows < 0 || cols < 0 || steps < 1 || steps > ortho_max_steps()) return 0;
  return ortho_workspace_bytes(batch, rows, cols, steps);
}

int ortho_sm100(const void* update, int64_t row_stride, int64_t matrix_stride, void* out,
                int64_t batch, int64_t rows, int64_t cols, const float* coefficients, int steps,
                float eps, int dtype, void* workspace, size_t workspace_bytes,
                rbf_stream_t stream) {
  if (batch < 0 || rows < 0 || cols < 0) return refuse(RBF_ERR_INVALID_ARGUMENT, "negative size");
  if (rows > (1 << 20) || cols > (1 << 20) || batch > 65535)
    return refuse(RBF_ERR_UNSUPPORTED, "rows or cols > 2^20, or batch > 65535");
  if (steps < 1 || steps > ortho_max_steps())
    return refuse(RBF_ERR_INVALID_ARGUMENT, "steps must be in [1, 32]");
  if (!dtype_ok(dtype)) return refuse(RBF_ERR_INVALID_ARGUMENT, "unknown element type");
  if (!std::isfinite(eps) || eps < 0.f) return refuse(RBF_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  if ((rows > 1 && row_stride < cols) || (batch > 1 && matrix_stride < 0))
    return refuse(RBF_ERR_INVALID_ARGUMENT, "row stride smaller than cols, or negative matrix stride");
  if (coefficients == nullptr) return refuse(RBF_ERR_INVALID_ARGUMENT, "coefficients is NULL");
  for (int i = 0; i < 3 * steps; ++i)
    if (!std::isfinite(coefficients[i])) return refuse(RBF_ERR_INVALID_ARGUMENT, "a coefficient is not finite");
  int st;
  const size_t e = elem_bytes(dtype);
  const int64_t n = batch * rows * cols;
  if ((st = need(update, n, e, "update"))) return st;
  if ((st = need(out, n, e, "out"))) return st;
  if ((st = check_workspace(workspace, workspace_bytes, ortho_workspace_bytes(batch, rows, cols, steps)))) return st;
  if ((st = check_device())) return st;
  OrthoArgs a{};
  a.update = update;
  a.out = out;
  a.batch = batch;
  a.rows = rows;
  a.cols = cols;
  a.row_stride = row_stride;
  a.matrix_stride = matrix_stride;
  a.dtype = dtype;
  a.steps = steps;
  a.coefficients = coefficients;
  a.eps = eps;
  a.workspace = workspace;
  return cuda_status(launch_orthogonalize(a, wait_config_from_env(), as_stream(stream)), "orthogonalisation launch");
}

}  // extern "C"
