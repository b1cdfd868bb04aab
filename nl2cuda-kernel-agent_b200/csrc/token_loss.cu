// token_loss.cu -- log-probabilities of chosen tokens and the losses on them.
//
//   m = max_j x_j,  s = sum_j exp(x_j - m),  lp = (x_label - m) - log s
//   dx_j = c * ((j == label) - exp(x_j - m) / s)
//
// The logits are the only large operand: the forward reads each scored row once (running maximum
// and sum, in fp32), the backward reads it once more and writes the gradient, and nothing of the
// size of the logits is kept in between.  Both are bound by HBM.  A row that is not scored is
// never read; its gradient is written as zeros.
//
// exp(x - m) = 2^((x - m) log2 e): the difference is taken first, so the largest term is 1 exactly
// and stays 1 in every join of partial sums.  (One fma, x log2(e) - m log2(e), would save an
// operation, but leaves the rounding of m log2(e) in each of the ten joins: 7e-6 of a
// log-probability at m = 15; and it overflows for logits masked with the type's lowest value.)
// lp is formed from x_label - m and log s, both small where the label leads, so no digits are lost
// against a large maximum.  The MUFU ex2 adds 2 ulp.
#include <algorithm>

#include "lm_common.cuh"
#include "lm_kernels.cuh"

namespace rbf {
namespace lm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eRest = (float)(1.4426950408889634 - (double)kLog2e);
constexpr int kFwdWarps = 48, kBwdWarps = 32;   // that an SM holds at least
constexpr int kPacks = 4;                       // 16-byte loads in flight per thread
constexpr int kMaxSplit = 8;     // CTAs (one cluster) of a forward row

struct MaxSum {
  float m, s;
};

// For a term of the gradient: three roundings (the difference, log2 e, the product) leave it off by 1.3e-7 |x - m|
// of itself at most, 1.3e-6 of a term that is e^-10 of the row's largest.  A single term, unlike the sum below, gains
// nothing from more.
__device__ __forceinline__ float exp_diff(float x, float m) { return exp2_approx((x - m) * kLog2e); }

// For the sum: with what log2 e loses in fp32 (1.3e-8 of it), which makes every term of a given size
// come out high alike, 1e-7 at x - m = -8: the rewards of long answers add that up.
__device__ __forceinline__ float exp_diff_exact(float x, float m) {
  const float d = x - m;
  return exp2_approx(fmaf(d, kLog2e, d * kLog2eRest));
}

// For partial sums that move to a larger maximum: ex2.approx comes out low by some 2^-25 on average, and
// a term passes through up to ten of these on its way, all in the same direction.  expf does not.
__device__ __forceinline__ float rescale(float m, float to) { return expf(m - to); }

// The maximum to subtract: any finite value while every term so far is exp(-inf).
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  const float ref = reference(m);
  return {m, a.s * rescale(a.m, ref) + b.s * rescale(b.m, ref)};
}

__device__ __forceinline__ MaxSum warp_merge(MaxSum v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v = merge(v, {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o)});
  return v;
}

template <int N>
__device__ __forceinline__ void accumulate(MaxSum& v, const float (&x)[N]) {
  float m = v.m;
#pragma unroll
  for (int e = 0; e < N; ++e) m = fmaxf(m, x[e]);
  const float ref = reference(m);
  float s = v.s * rescale(v.m, ref);
#pragma unroll
  for (int e = 0; e < N; ++e) s += exp_diff_exact(x[e], ref);
  v.m = m;
  v.s = s;
}

template <typename T>
__device__ __forceinline__ const T* row_of(const LogitArgs& a, int64_t r) {
  const int64_t b = r / a.T;
  return static_cast<const T*>(a.logits) + b * a.batch_stride + (r - b * a.T) * a.t_stride;
}

// Elements before the first 16-byte boundary at or after p (at most n).
template <typename T>
__device__ __forceinline__ int64_t head_of(const T* p, int64_t n) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t h = (VEC - (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % VEC)) % VEC;
  return h < n ? h : n;
}

// The elements of a row outside its whole packs: fewer than a pack at either end.
template <typename T>
__device__ __forceinline__ void accumulate_ends(MaxSum& v, const T* x, int64_t head, int64_t tail, int64_t V) {
  if (threadIdx.x < head) {
    const float f[1] = {to_f32(x[threadIdx.x])};
    accumulate(v, f);
  }
  if (tail + threadIdx.x < V) {
    const float f[1] = {to_f32(x[tail + threadIdx.x])};
    accumulate(v, f);
  }
}

template <typename T, int VEC, int N>
__device__ __forceinline__ void accumulate_packs(MaxSum& v, const Pack<T, VEC> (&p)[N]) {
  float m = v.m;
#pragma unroll
  for (int u = 0; u < N; ++u) m = fmaxf(m, pack_max(p[u]));
  const float ref = reference(m);
  const F2 shift = f2(-ref, -ref), hi = f2(kLog2e, kLog2e), lo = f2(kLog2eRest, kLog2eRest);
  F2 s = f2(v.s * rescale(v.m, ref), 0.f);
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) {
      const F2 d = add2(pair_of(p[u], k), shift);
      float a, b;
      unpack(fma2(d, hi, mul2(d, lo)), a, b);  // exp_diff_exact of both
      s = add2(s, f2(exp2_approx(a), exp2_approx(b)));
    }
  float a, b;
  unpack(s, a, b);
  v.m = m;
  v.s = a + b;
}

template <typename T>
__device__ __forceinline__ void write_row(const LogitArgs& a, int64_t r, int64_t label, bool scored, const T* x, MaxSum t) {
  // In 64 bits, and what fp32 drops of it kept for the losses: a reward is the difference of long sums of
  // these, and the rounding of each (3e-7 at -10) is several times the error of s.
  double lp = 0.0;
  if (scored) lp = label >= 0 && label < a.V ? ((double)to_f32(x[label]) - (double)t.m) - log((double)t.s) : (double)NAN;
  const float rounded = (float)lp;
  a.logprob[r] = rounded;
  if (a.rest != nullptr) a.rest[r] = isfinite(rounded) ? (float)(lp - (double)rounded) : 0.f;
  if (a.stats != nullptr) {
    a.stats[2 * r] = t.m;
    a.stats[2 * r + 1] = 1.f / t.s;
  }
}

// One row per CTA; or a cluster of `split` CTAs per row: with few rows there are more SMs than rows, and
// a row of 128 K elements read by one SM alone takes longer than the rest of the pass.  The shares
// meet in the first CTA's shared memory.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, kFwdWarps * 32 / THREADS) logprob_forward_kernel(const LogitArgs a, int split) {
  constexpr int VEC = 16 / sizeof(T);
  __shared__ MaxSum part[kMaxSplit][THREADS / 32];
  if (split > 1) ptx::cluster_sync();  // every CTA of the cluster runs before one writes to another
  ptx::griddep_wait();
  const int64_t r = blockIdx.x / split;
  const int share = blockIdx.x % split;
  const int64_t label = a.labels[r];
  const bool scored = label != a.ignore_index;  // the same for every CTA of a cluster
  const T* x = row_of<T>(a, r);
  MaxSum v{-INFINITY, 0.f};
  if (scored) {
    const int64_t head = head_of(x, a.V);
    const int64_t packs = (a.V - head) / VEC;
    const T* body = x + head;
    const int64_t begin = packs * share / split, end = packs * (share + 1) / split;
    int64_t i = begin + threadIdx.x;
    for (; i + (kPacks - 1) * THREADS < end; i += kPacks * THREADS) {
      Pack<T, VEC> p[kPacks];
#pragma unroll
      for (int u = 0; u < kPacks; ++u) p[u] = load_stream<T, VEC>(body + (i + u * THREADS) * VEC);
      accumulate_packs(v, p);
    }
    for (; i < end; i += THREADS) {
      const Pack<T, VEC> p[1] = {load_stream<T, VEC>(body + i * VEC)};
      accumulate_packs(v, p);
    }
    if (share == 0) accumulate_ends(v, x, head, head + packs * VEC, a.V);
    v = warp_merge(v);
  }
  if ((threadIdx.x & 31) == 0) {
    MaxSum* dst = &part[share][threadIdx.x >> 5];
    if (split > 1) {
      const uint32_t at = ptx::map_to_rank(dst, 0);
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(v.m), "f"(v.s) : "memory");
    } else {
      *dst = v;
    }
  }
  ptx::griddep_launch_dependents();
  if (split > 1) ptx::cluster_sync();
  else __syncthreads();
  if (share != 0 || threadIdx.x >= 32) return;
  constexpr int W = THREADS / 32;
  MaxSum t{-INFINITY, 0.f};
  for (int i = threadIdx.x; i < split * W; i += 32) t = merge(t, part[i / W][i % W]);
  t = warp_merge(t);
  if (threadIdx.x == 0) write_row(a, r, label, scored, x, t);
}

// `slices` CTAs per row, each a share of its packs.  Registers for four CTAs an SM and no second set of
// packs in flight: 98% of the copy rate at 16384 x 131072 bf16; a software pipeline over two packs in
// the same registers was at 78%, one over single packs with six CTAs at 88%.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, kBwdWarps * 32 / THREADS) logprob_backward_kernel(const LogitArgs a, int slices) {
  constexpr int VEC = 16 / sizeof(T);
  constexpr int STEP = kPacks * THREADS;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  // Last rows first: what the forward read last is still in L2.
  const int64_t block = (int64_t)gridDim.x - 1 - blockIdx.x;
  const int64_t r = block / slices;
  const int64_t slice = block - r * slices;
  const int64_t label = a.labels[r];
  const T* x = row_of<T>(a, r);
  T* dx = static_cast<T*>(a.dlogits) + r * a.V;
  const int64_t head = head_of(dx, a.V);
  const int64_t packs = (a.V - head) / VEC;
  const int64_t tail = head + packs * VEC;
  const int64_t end = packs * (slice + 1) / slices;
  int64_t i = packs * slice / slices + threadIdx.x;
  if (label == a.ignore_index) {
    Pack<T, VEC> zero;
#pragma unroll
    for (int e = 0; e < VEC; ++e) zero.v[e] = from_f32<T>(0.f);
    for (; i < end; i += THREADS) store_pack<T, VEC>(dx + head + i * VEC, zero);
    if (slice == 0) {
      if (threadIdx.x < head) dx[threadIdx.x] = from_f32<T>(0.f);
      if (tail + threadIdx.x < a.V) dx[tail + threadIdx.x] = from_f32<T>(0.f);
    }
    return;
  }
  const bool same = head_of(x, a.V) == head;  // both move in packs
  Pack<T, VEC> p[kPacks];
  auto fetch = [&]() {
#pragma unroll
    for (int u = 0; u < kPacks; ++u) {
      const int64_t k = i + u * THREADS;
      if (k >= end) break;
      const T* q = x + head + k * VEC;
      if (same) {
        p[u] = load_stream<T, VEC>(q);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) p[u].v[e] = q[e];
      }
    }
  };
  fetch();  // next to the row's scalars
  float c = a.coef[r];
  if (a.scale0 != nullptr) c *= *a.scale0;
  if (a.scale1 != nullptr) c *= *a.scale1;
  const float m = a.stats[2 * r];
  const float neg = -c * a.stats[2 * r + 1];
  auto grad = [&](float v, bool chosen) {
    const float g = neg * exp_diff(v, m);
    return chosen ? c + g : g;
  };
  const F2 shift = f2(-m, -m), log2e = f2(kLog2e, kLog2e), factor = f2(neg, neg);
  while (i < end) {
#pragma unroll
    for (int u = 0; u < kPacks; ++u) {
      const int64_t k = i + u * THREADS;
      if (k >= end) break;
      const int64_t j = head + k * VEC;
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) {
        float x0, x1;
        unpack(mul2(add2(pair_of(p[u], e), shift), log2e), x0, x1);
        set_pair(o, e, mul2(f2(exp2_approx(x0), exp2_approx(x1)), factor));
      }
      if (label >= j && label < j + VEC) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (j + e == label) o.v[e] = from_f32<T>(grad(to_f32(p[u].v[e]), true));
      }
      store_pack<T, VEC>(dx + j, o);
    }
    i += STEP;
    fetch();
  }
  if (slice == 0) {
    const int64_t j = threadIdx.x, k = tail + threadIdx.x;
    if (j < head) dx[j] = from_f32<T>(grad(to_f32(x[j]), j == label));
    if (k < a.V) dx[k] = from_f32<T>(grad(to_f32(x[k]), k == label));
  }
}

// ---- the losses: one cluster of kLossCtas CTAs --------------------------------------------------
// A warp takes one part of one sequence at a time (parts(B) parts per sequence, so that the
// cluster's 256 warps have work at any batch size), leaves its sums in the workspace, and after
// one cluster barrier every warp has what it needs of the others.  The work is 20 bytes a token,
// nothing against the logits, so what counts is that it is one launch.  Sums are in 64 bits: a
// reward is a small difference of sums over a long answer.
constexpr int kLossCtas = 8;
constexpr int kLossThreads = 1024;
constexpr int kLossWarps = kLossCtas * kLossThreads / 32;

__host__ __device__ inline int64_t loss_parts(int64_t B, int64_t T) {
  int64_t p = B > 0 ? kLossWarps / B : 1;
  const int64_t most = (T + 31) / 32;
  if (p > most) p = most;
  return p > 0 ? p : 1;
}

__device__ __forceinline__ double sum_parts(const double* part, int64_t b, int64_t parts) {
  double s = 0.0;
  for (int64_t i = 0; i < parts; ++i) s += part[b * parts + i];
  return s;
}

// Sum over the CTA in a fixed order; the result is in thread 0.
__device__ double block_sum(double v, double* smem) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = threadIdx.x < kLossThreads / 32 ? smem[threadIdx.x] : 0.0;
  if (threadIdx.x < 32) t = warp_sum(t);
  return t;
}

__device__ __forceinline__ double logprob_at(const LossArgs& a, int64_t i) {
  return a.rest != nullptr ? (double)a.logprob[i] + (double)a.rest[i] : (double)a.logprob[i];
}

template <bool PREF>
__global__ void __launch_bounds__(kLossThreads) loss_kernel(const LossArgs a) {
  __shared__ double smem[32];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t warp = ((int64_t)blockIdx.x * kLossThreads + threadIdx.x) >> 5;
  const int64_t parts = loss_parts(a.B, a.T);
  const int64_t items = a.B * parts;
  double* p0 = a.part;                 // reward parts, or loss parts
  double* p1 = a.part + items;         // policy: kl parts
  double* p2 = a.part + 2 * items;     // policy: scored positions
  for (int64_t it = warp; it < items; it += kLossWarps) {
    const int64_t b = it / parts, k = it - b * parts;
    const int64_t t0 = a.T * k / parts, t1 = a.T * (k + 1) / parts;
    double s0 = 0.0, s1 = 0.0, n = 0.0;
    for (int64_t t = t0 + lane; t < t1; t += 32) {
      const int64_t i = b * a.T + t;
      const bool scored = a.labels[i] != a.ignore_index;
      if (PREF) {
        if (scored) s0 += logprob_at(a, i) - (double)a.ref_logprob[i];
      } else {
        float c = 0.f;
        if (scored) {
          const double lp = logprob_at(a, i);
          const double adv = a.advantage[a.per_token ? i : b];
          const double ratio = exp(lp - (double)a.old_logprob[i]);
          // NaN passes through both (fmin / fmax would drop it).
          double clipped = ratio;
          if (ratio < 1.0 - (double)a.clip_low) clipped = 1.0 - (double)a.clip_low;
          if (ratio > 1.0 + (double)a.clip_high) clipped = 1.0 + (double)a.clip_high;
          const double d = (double)a.ref_logprob[i] - lp;
          const double ed = exp(d);
          const double free = ratio * adv, held = clipped * adv;
          const bool held_wins = held < free;
          s0 += (double)a.kl_coef * (ed - d - 1.0) - (held_wins ? held : free);
          s1 += ed - d - 1.0;
          n += 1.0;
          c = (float)((held_wins ? 0.0 : -free) + (double)a.kl_coef * (1.0 - ed));
        }
        a.coef[i] = c;
      }
    }
    s0 = warp_sum(s0);
    if (!PREF) {
      s1 = warp_sum(s1);
      n = warp_sum(n);
    }
    if (lane == 0) {
      p0[it] = s0;
      if (!PREF) {
        p1[it] = s1;
        p2[it] = n;
      }
    }
  }
  __threadfence();
  ptx::cluster_sync();
  if (PREF) {
    const int64_t pairs = a.B / 2;
    const double beta = a.beta, sm = a.smoothing;
    for (int64_t it = warp; it < items; it += kLossWarps) {
      const int64_t b = it / parts, k = it - b * parts;
      const int64_t p = b < pairs ? b : b - pairs;
      const double z = beta * (sum_parts(p0, p, parts) - sum_parts(p0, p + pairs, parts));
      // d loss / d z = s sigmoid(z) - (1 - s) sigmoid(-z), over the pairs
      const double up = 1.0 / (1.0 + exp(z)), down = 1.0 / (1.0 + exp(-z));
      const double dz = (sm * down - (1.0 - sm) * up) / (double)pairs;
      const float c = (float)(b < pairs ? dz * beta : -dz * beta);
      for (int64_t t = a.T * k / parts + lane; t < a.T * (k + 1) / parts; t += 32) {
        const int64_t i = b * a.T + t;
        a.coef[i] = a.labels[i] != a.ignore_index ? c : 0.f;
      }
    }
    if (blockIdx.x != 0) return;
    double loss = 0.0;
    for (int64_t p = threadIdx.x; p < pairs; p += kLossThreads) {
      const double rc = beta * sum_parts(p0, p, parts), rr = beta * sum_parts(p0, p + pairs, parts);
      a.second[p] = (float)rc;
      a.second[p + pairs] = (float)rr;
      const double z = rc - rr;
      // -log sigmoid(z) = max(-z, 0) + log(1 + exp(-|z|)), and -log sigmoid(-z) is z more
      const double l = log1p(exp(-fabs(z)));
      loss += (1.0 - sm) * ((z < 0.0 ? -z : 0.0) + l) + sm * ((z > 0.0 ? z : 0.0) + l);
    }
    loss = block_sum(loss, smem);
    if (threadIdx.x == 0) *a.loss = (float)(loss / (double)pairs);
  } else {
    if (blockIdx.x != 0) return;
    double s0 = 0.0, s1 = 0.0, n = 0.0;
    for (int64_t it = threadIdx.x; it < items; it += kLossThreads) {
      s0 += p0[it];
      s1 += p1[it];
      n += p2[it];
    }
    s0 = block_sum(s0, smem);
    s1 = block_sum(s1, smem);
    n = block_sum(n, smem);
    if (threadIdx.x == 0) {
      const double count = n > 0.0 ? n : 1.0;
      *a.loss = (float)(s0 / count);
      *a.second = (float)(s1 / count);
      *a.norm = (float)(1.0 / count);
    }
  }
}

template <typename F>
cudaError_t by_type(int dtype, F f) {
  if (dtype == LM_F32) return f(float{});
  if (dtype == LM_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

}  // namespace

cudaError_t launch_logprob_forward(const LogitArgs& a, cudaStream_t stream) {
  if (a.rows == 0) return cudaSuccess;
  constexpr int kMost = 256;  // threads of a CTA
  // With few rows, enough CTAs for every SM to have two, as long as each keeps a few rounds of loads.
  int split = 1;
  while (split < kMaxSplit && a.rows * split * 2 <= 2 * device_sm_count() && a.V / (split * 2) >= 2 * kMost * 8)
    split *= 2;
  // Rows for all the CTAs of 128 threads that the SMs hold: these, since half as many threads wait for each
  // other at a row's end.  16384 x 32768 bf16 132 us (256 threads: 148), 4096 x 5034 14 (20); but
  // 1024 x 32768 15.5 (14.6) and 4 x 131071 fp32, in clusters, 10.5 (7.9).
  const bool many = a.rows >= kFwdWarps / 4 * (int64_t)device_sm_count();
  cudaError_t e = by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid((unsigned)(a.rows * split));
    if (split > 1)
      return launch_kernel_cluster(logprob_forward_kernel<T, kMost>, grid, dim3(kMost), 0, split, stream, a, split);
    if (many) return launch_kernel(logprob_forward_kernel<T, 128>, grid, dim3(128), 0, stream, a, 1);
    return launch_kernel(logprob_forward_kernel<T, kMost>, grid, dim3(kMost), 0, stream, a, 1);
  });
  if (e != cudaSuccess) return e;
  note_launches(1);
  return cudaGetLastError();
}

cudaError_t launch_logprob_backward(const LogitArgs& a, cudaStream_t stream) {
  if (a.rows == 0 || a.V == 0) return cudaSuccess;
  // Long rows take CTAs of 256 threads: 16384 x 32768 bf16 289 us (128 threads: 296), 2000 x 50001 fp32 115
  // (121).  Rows of up to 32 KB and small calls take 128: 8192 x 1001 bf16 17 us (256: 28), 4096 x 5034 15 (20),
  // 128 x 50257 8.8 (11.4).
  const int64_t row = a.V * (int64_t)elem_bytes(a.dtype);
  const int threads = row <= 32768 || row * a.rows <= (int64_t(64) << 20) ? 128 : 256;
  // CTAs per row: at least four steps each, and no more than give every SM 32 in all.
  const int64_t steps = ceil_div(row, (int64_t)kPacks * threads * 16);
  const int64_t want = ceil_div(32 * (int64_t)device_sm_count(), a.rows);
  const int64_t slices = std::min(want, std::max<int64_t>(1, steps / 4));
  cudaError_t e = by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    auto k = threads == 128 ? logprob_backward_kernel<T, 128> : logprob_backward_kernel<T, 256>;
    return launch_kernel(k, dim3((unsigned)(a.rows * slices)), dim3(threads), 0, stream, a, (int)slices);
  });
  if (e != cudaSuccess) return e;
  note_launches(1);
  return cudaGetLastError();
}

size_t loss_workspace_bytes(int64_t B, int64_t T) {
  return sizeof(double) * 3 * (size_t)(B * loss_parts(B, T));
}

cudaError_t launch_loss(const LossArgs& a, bool preference, cudaStream_t stream) {
  auto k = preference ? loss_kernel<true> : loss_kernel<false>;
  const cudaError_t e = launch_kernel_cluster(k, dim3(kLossCtas), dim3(kLossThreads), 0, kLossCtas, stream, a);
  if (e != cudaSuccess) return e;
  note_launches(1);
  return cudaGetLastError();
}

}  // namespace lm
}  // namespace rbf
