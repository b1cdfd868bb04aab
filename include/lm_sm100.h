/*
 * lm_sm100.h -- C ABI of the language-model operators in librbf_sm100.so (B200, sm_100a): layer
 * norm, the log-probability of a chosen token, the preference loss and the clipped policy loss
 * on it, and the Newton-Schulz orthogonalisation of an update.
 *
 * Conventions are those of rbf_sm100.h: int64 sizes; caller-owned outputs and workspace; calls
 * are stream-ordered, never allocate and never block; an rbf_status code is returned, with
 * rbf_sm100_last_error_detail() for the reason; nothing aborts.  Two calls may share a workspace
 * only if they are ordered on one stream.  A workspace and the per-row arrays are 16-byte aligned;
 * the large operands (x, dy, logits, ...) need the alignment of their element type only, and
 * their rows may lie apart (a row stride in elements; the elements of a row are contiguous).
 * Kernels compute in fp32 or more, whatever the element type, and round once.
 */
#ifndef LM_SM100_H_
#define LM_SM100_H_

#include "rbf_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum { LM_F32 = 0, LM_BF16 = 1, LM_F16 = 2 };

/* ---- layer norm --------------------------------------------------------------------------
 *   y = (x - mean) * rstd * weight + bias,  rstd = 1 / sqrt(var + eps)      over rows of length D
 * x [rows, D] (type dtype), weight and bias [D] (type wdtype; NULL: 1 and 0), y [rows, D]
 * (type dtype), which must not overlap x.  mean and rstd [rows] fp32 are written for the backward; both
 * NULL: not kept.
 * var is the mean of (x - mean)^2 (two passes over the row on chip, no cancellation). */
RBF_API int ln_sm100_forward(const void* x, int64_t x_stride, const void* weight,
                             const void* bias, void* y, float* mean, float* rstd, int64_t rows,
                             int64_t D, float eps, int dtype, int wdtype, rbf_stream_t stream);

/* Bytes of the backward's workspace (partial sums of dweight and dbias). */
RBF_API size_t ln_sm100_backward_workspace_bytes(int64_t rows, int64_t D);

/*   g = dy * weight,  xh = (x - mean) * rstd
 *   dx = rstd * (g - mean(g) - xh * mean(g * xh)),  dweight = sum_rows dy * xh,
 *   dbias = sum_rows dy
 * dx [rows, D] contiguous (type dtype); dweight and dbias [D] (type wdtype).  Any of the three
 * may be NULL: not computed.  dx must overlap neither x nor dy.  The sums run in a fixed order: equal
 * calls give equal bits. */
RBF_API int ln_sm100_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                              const void* weight, const float* mean, const float* rstd, void* dx,
                              void* dweight, void* dbias, int64_t rows, int64_t D, int dtype,
                              int wdtype, void* workspace, size_t workspace_bytes,
                              rbf_stream_t stream);

/* ---- log-probability of a chosen token -----------------------------------------------------
 * logits [rows, V] (type dtype), row r at logits + (r / T) * batch_stride + (r % T) * t_stride
 * elements: T positions of each sequence.  labels [rows] int64: a vocabulary index, or
 * ignore_index for a row that is not scored (its logits are not read).
 *   logprob[r] = x[label] - log sum_j exp(x[j])     (0 for a row that is not scored)
 * rest [rows] receives what fp32 drops of logprob, for the losses (NULL: not kept).
 * stats [rows, 2] fp32 receives the row's maximum and 1 / sum_j exp(x[j] - maximum) (NULL: not
 * kept).  A label that is neither ignore_index nor in [0, V) gives NaN. */
RBF_API int lp_sm100_forward(const void* logits, int64_t batch_stride, int64_t t_stride,
                             const int64_t* labels, float* logprob, float* rest, float* stats,
                             int64_t rows, int64_t T, int64_t V, int64_t ignore_index, int dtype,
                             rbf_stream_t stream);

/* dlogits[r, j] = c_r * ((j == label_r) - exp(x[j] - max_r) * inv_r),
 * c_r = coef[r] * scale
 * dlogits [rows, V] contiguous (type dtype), which must not overlap the logits; rows that are not scored are zeroed.  scale: the
 * product of the device scalars scale0 and scale1 (either may be NULL: 1). */
RBF_API int lp_sm100_backward(const void* logits, int64_t batch_stride, int64_t t_stride,
                              const int64_t* labels, const float* stats, const float* coef,
                              const float* scale0, const float* scale1, void* dlogits,
                              int64_t rows, int64_t T, int64_t V, int64_t ignore_index, int dtype,
                              rbf_stream_t stream);

/* ---- losses on log-probabilities [B, T] ----------------------------------------------------
 * Sums over tokens and over the batch are taken in 64 bits in a fixed order.  The log-probabilities
 * are logprob + rest, as lp_sm100_forward leaves them (rest may be NULL: 0). */

/* Bytes of the workspace of either loss. */
RBF_API size_t loss_sm100_workspace_bytes(int64_t B, int64_t T);

/* Preference loss of B / 2 pairs: sequence p is preferred to sequence B / 2 + p.
 *   reward_b = beta * sum_t (logprob - ref_logprob)       over scored positions
 *   z_p = reward_p - reward_{B/2+p}
 *   loss = mean_p [ -(1 - s) log sigmoid(z_p) - s log sigmoid(-z_p) ],   s = label_smoothing
 * reward [B], loss [1]; coef [B, T] receives d loss / d logprob for lp_sm100_backward. */
RBF_API int pref_sm100_loss(const float* logprob, const float* rest, const float* ref_logprob,
                            const int64_t* labels, float* loss, float* reward, float* coef,
                            int64_t B, int64_t T, float beta, float label_smoothing,
                            int64_t ignore_index, void* workspace, size_t workspace_bytes, rbf_stream_t stream);

/* Clipped policy loss, a mean over all scored positions (count of them; 1 if there are none):
 *   ratio = exp(logprob - old_logprob),  d = ref_logprob - logprob,  kl = exp(d) - d - 1
 *   loss = mean [ kl_coef * kl - min(ratio * A, clip(ratio, 1 - clip_low, 1 + clip_high) * A) ]
 * A = advantage[b] ([B], per_token = 0) or advantage[b, t] ([B, T], per_token = 1).
 * loss [1] and kl [1] (the mean of kl); coef [B, T] receives count * d loss / d logprob and norm
 * [1] receives 1 / count (pass it to lp_sm100_backward as a scale). */
RBF_API int policy_sm100_loss(const float* logprob, const float* rest, const float* old_logprob,
                              const float* ref_logprob, const float* advantage, int per_token,
                              const int64_t* labels, float* loss, float* kl, float* coef,
                              float* norm, int64_t B, int64_t T, float clip_low, float clip_high,
                              float kl_coef, int64_t ignore_index, void* workspace,
                              size_t workspace_bytes, rbf_stream_t stream);

/* ---- orthogonalisation of an update ---------------------------------------------------------
 * Newton-Schulz products on each of `batch` matrices G [rows, cols] (type dtype; rows contiguous,
 * row_stride and matrix_stride elements apart):
 *   X = G / (|G|_F + eps);  `steps` times:  A = X X^T,  X <- a X + (b A + c A^2) X
 * (with X transposed where rows > cols; the result is the same), (a, b, c) = coefficients[step]
 * (host memory, 3 * steps floats, read during the call).  out [batch, rows, cols] contiguous,
 * type dtype; it must not overlap the update.  Products keep 22 bits of each operand and
 * accumulate in fp32.  1 <= steps <= 32.  The workspace's first int is the device status word
 * (rbf_sm100_read_status): 0, or 7 if a bounded device wait ran out and out is incomplete. */
RBF_API size_t ortho_sm100_workspace_bytes(int64_t batch, int64_t rows, int64_t cols, int steps);
RBF_API int ortho_sm100(const void* update, int64_t row_stride, int64_t matrix_stride, void* out,
                        int64_t batch, int64_t rows, int64_t cols, const float* coefficients,
                        int steps, float eps, int dtype, void* workspace, size_t workspace_bytes,
                        rbf_stream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* LM_SM100_H_ */
