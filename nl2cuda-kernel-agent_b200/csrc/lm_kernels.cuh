// lm_kernels.cuh -- host-side launchers of the language-model kernels (internal to the library;
// the public C ABI is include/lm_sm100.h).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "rbf_kernels.cuh"

namespace rbf {
namespace lm {

// ln.cu
struct LnArgs {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* y;    // forward output, or dx
  void* dw;
  void* db;
  float* mean;
  float* rstd;
  float* part;  // backward partial sums [2][parts][D]
  int64_t x_stride, dy_stride, rows, D;
  float eps;
  int dtype, wdtype;
};
cudaError_t launch_ln_forward(const LnArgs& a, cudaStream_t stream);
cudaError_t launch_ln_backward(const LnArgs& a, cudaStream_t stream);
int64_t ln_backward_parts(int64_t rows, int64_t D);

// token_loss.cu
struct LogitArgs {
  const void* logits;
  int64_t batch_stride, t_stride;
  const int64_t* labels;
  int64_t rows, T, V, ignore_index;
  int dtype;
  float* logprob;       // forward
  float* rest;          // what fp32 drops of it, or NULL
  float* stats;         // [rows][2]: maximum, 1 / sum
  const float* coef;    // backward
  const float* scale0;
  const float* scale1;
  void* dlogits;
};
cudaError_t launch_logprob_forward(const LogitArgs& a, cudaStream_t stream);
cudaError_t launch_logprob_backward(const LogitArgs& a, cudaStream_t stream);

struct LossArgs {
  const float* logprob;
  const float* rest;
  const float* old_logprob;
  const float* ref_logprob;
  const float* advantage;
  const int64_t* labels;
  float* loss;
  float* second;  // reward [B] of the preference loss, kl [1] of the policy loss
  float* coef;
  float* norm;
  double* part;   // workspace
  int64_t B, T, ignore_index;
  int per_token;
  float beta, smoothing;              // preference
  float clip_low, clip_high, kl_coef; // policy
};
size_t loss_workspace_bytes(int64_t B, int64_t T);
cudaError_t launch_loss(const LossArgs& a, bool preference, cudaStream_t stream);

// ortho.cu
struct OrthoArgs {
  const void* update;
  void* out;
  int64_t batch, rows, cols, row_stride, matrix_stride;
  int dtype, steps;
  const float* coefficients;  // host, [steps][3]
  float eps;
  void* workspace;
};
size_t ortho_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int steps);
int ortho_max_steps();
cudaError_t launch_orthogonalize(const OrthoArgs& a, const WaitConfig& wc, cudaStream_t stream);

}  // namespace lm
}  // namespace rbf
