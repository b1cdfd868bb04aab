// ln.cu -- layer norm: forward, and backward with the reduction of the weight's gradient.
//
//   y  = xh * w + b,   xh = (x - mean) * rstd,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g  = dy * w,       dx = rstd * (g - mean(g) - xh * mean(g * xh))
//   dw = sum_rows dy * xh,   db = sum_rows dy
//
// Both passes are bound by HBM: the forward moves 2 elements and the backward 3 per value, at
// some 10 flops each.  A row sits in the registers of a group of `W` warps, 16 values a lane, so
// it is read once; the variance is a second pass over registers, not over memory, and has no
// cancellation.  Groups walk over rows (a persistent grid) and load their next row before they
// work on the present one, so that loads are in flight all the time.
//
// In the backward a lane keeps the sums of its 16 columns' dy * xh and dy in registers over all
// its rows; each CTA writes one row of partial sums at its end and a second, short kernel adds
// those in a fixed order.  No atomics: equal calls give equal bits.
//
// Statistics, sums and partial sums are fp32; every output is rounded once.
#include <type_traits>

#include "lm_common.cuh"
#include "lm_kernels.cuh"

namespace rbf {
namespace lm {
namespace {

constexpr int kLaneElems = 16;                   // values of a row per lane
constexpr int kWarpElems = 32 * kLaneElems;
constexpr int64_t kMaxRegD = 32 * kWarpElems;    // longest row held in the registers of one CTA
constexpr int kWideThreads = 1024;
constexpr int kSumRows = 16;                     // partial rows a thread column of ln_sum adds at a time

// Sum of (a, b) over the warps of a group.  red: two slots of 32 float2 for this group, used in
// turn, so that one barrier per reduction is enough.
__device__ __forceinline__ float2 group_sum(float2 v, int W, int warp_in_group, int bar, float2* red,
                                            int& turn) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  if (W == 1) return v;
  float2* slot = red + turn * 32;
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) slot[warp_in_group] = v;
  named_sync(bar, W * 32);
  const int lane = threadIdx.x & 31;
  float2 t = lane < W ? slot[lane] : make_float2(0.f, 0.f);
  t.x = warp_sum(t.x);
  t.y = warp_sum(t.y);
  return t;
}

// The lanes of a group hold a row as NV packs of VEC values each: pack i of lane l of warp w covers
// columns ((i * W + w) * 32 + l) * VEC ...
template <typename T, int VEC, int NV>
struct Row {
  Pack<T, VEC> p[NV];
  __device__ __forceinline__ void load(const T* row, int D, int W, int w, int lane) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((i * W + w) * 32 + lane) * VEC;
      if (c < D) {
        p[i] = load_stream<T, VEC>(row + c);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) p[i].v[e] = from_f32<T>(0.f);
      }
    }
  }
};

// CTAs of `groups` groups of W warps; each group takes one row at a time.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(1024) ln_forward_kernel(const LnArgs a, int W, int groups) {
  __shared__ float2 red[32 * 2 * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = warp / W, w = warp - g * W;
  float2* slots = red + g * 64;
  int turn = 0;
  const int D = (int)a.D;
  const int64_t step = (int64_t)gridDim.x * groups;
  int64_t r = (int64_t)blockIdx.x * groups + g;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  Row<T, VEC, NV> next;
  if (r < a.rows) next.load(x + r * a.x_stride, D, W, w, lane);
  const float inv_d = 1.f / (float)a.D;
  for (; r < a.rows; r += step) {
    float v[NV * VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i * VEC + e] = to_f32(next.p[i].v[e]);
    if (r + step < a.rows) next.load(x + (r + step) * a.x_stride, D, W, w, lane);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NV * VEC; ++k) s += v[k];
    const float mean = group_sum(make_float2(s, 0.f), W, w, 1 + g, slots, turn).x * inv_d;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool in = ((i * W + w) * 32 + lane) * VEC < D;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = v[i * VEC + e] - mean;
        if (in) q = fmaf(d, d, q);
        v[i * VEC + e] = d;
      }
    }
    const float var = group_sum(make_float2(q, 0.f), W, w, 1 + g, slots, turn).x * inv_d;
    const float rstd = 1.f / sqrtf(var + a.eps);
    if (w == 0 && lane == 0 && a.mean != nullptr) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((i * W + w) * 32 + lane) * VEC;
      if (c >= D) break;
      float wv[VEC], bv[VEC];
      load_param<VEC>(a.weight, c, a.wdtype, 1.f, wv);
      load_param<VEC>(a.bias, c, a.wdtype, 0.f, bv);
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.v[e] = from_f32<T>(fmaf(v[i * VEC + e] * rstd, wv[e], bv[e]));
      store_pack<T, VEC>(y + r * a.D + c, o);
    }
  }
}

template <typename T, int VEC, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) ln_backward_kernel(const LnArgs a, int W, int groups) {
  extern __shared__ float sums[];  // groups > 1: [groups][D] column sums at the end
  __shared__ float2 red[32 * 2 * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = warp / W, w = warp - g * W;
  float2* slots = red + g * 64;
  int turn = 0;
  const int D = (int)a.D;
  const int64_t step = (int64_t)gridDim.x * groups;
  int64_t r = (int64_t)blockIdx.x * groups + g;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.y);
  float wv[NV * VEC], dw[NV * VEC], db[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = ((i * W + w) * 32 + lane) * VEC;
    float t[VEC];
    if (c < D) load_param<VEC>(a.weight, c, a.wdtype, 1.f, t);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      wv[i * VEC + e] = c < D ? t[e] : 0.f;
      dw[i * VEC + e] = db[i * VEC + e] = 0.f;
    }
  }
  Row<T, VEC, NV> nx, ny;
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](int64_t row) {
    nx.load(x + row * a.x_stride, D, W, w, lane);
    ny.load(dy + row * a.dy_stride, D, W, w, lane);
    nmean = a.mean[row];
    nrstd = a.rstd[row];
  };
  if (r < a.rows) fetch(r);
  const float inv_d = 1.f / (float)a.D;
  for (; r < a.rows; r += step) {
    const Row<T, VEC, NV> px = nx, py = ny;
    const float mean = nmean, rstd = nrstd;
    if (r + step < a.rows) fetch(r + step);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int k = i * VEC + e;
        const float h = (to_f32(px.p[i].v[e]) - mean) * rstd;  // columns past D: dy = 0, w = 0
        const float d = to_f32(py.p[i].v[e]);
        const float gw = d * wv[k];
        s.x += gw;
        s.y = fmaf(gw, h, s.y);
        dw[k] = fmaf(d, h, dw[k]);
        db[k] += d;
      }
    if (a.y == nullptr) continue;
    s = group_sum(s, W, w, 1 + g, slots, turn);
    const float m1 = s.x * inv_d, m2 = s.y * inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((i * W + w) * 32 + lane) * VEC;
      if (c >= D) break;
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float h = (to_f32(px.p[i].v[e]) - mean) * rstd;
        const float gw = to_f32(py.p[i].v[e]) * wv[i * VEC + e];
        o.v[e] = from_f32<T>(rstd * (gw - m1 - h * m2));
      }
      store_pack<T, VEC>(dx + r * a.D + c, o);
    }
  }
  if (a.part == nullptr) return;
  // This CTA's column sums: one partial row of dw and one of db.
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float* acc = which == 0 ? dw : db;
    float* out = a.part + ((int64_t)which * gridDim.x + blockIdx.x) * a.D;
    if (groups == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = ((i * W + w) * 32 + lane) * VEC;
        if (c >= D) break;
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[c + e] = acc[i * VEC + e];
      }
      continue;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((i * W + w) * 32 + lane) * VEC;
      if (c >= D) break;
#pragma unroll
      for (int e = 0; e < VEC; ++e) sums[g * D + c + e] = acc[i * VEC + e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      float t = 0.f;
      for (int k = 0; k < groups; ++k) t += sums[k * D + c];
      out[c] = t;
    }
  }
}

// dw[c] = sum_p part[0][p][c], db[c] = sum_p part[1][p][c]: 32 columns per CTA, 16 thread rows
// that each add every 16th partial.
__global__ void __launch_bounds__(32 * kSumRows) ln_sum_kernel(const LnArgs a, int parts) {
  __shared__ float s[kSumRows][33];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  void* out = blockIdx.y == 0 ? a.dw : a.db;
  if (out == nullptr) return;
  const float* p = a.part + (int64_t)blockIdx.y * parts * a.D;
  float t = 0.f;
  if (c < a.D) {
#pragma unroll 8
    for (int k = threadIdx.y; k < parts; k += kSumRows) t += p[(int64_t)k * a.D + c];
  }
  s[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y != 0 || c >= a.D) return;
#pragma unroll
  for (int k = 1; k < kSumRows; ++k) t += s[k][threadIdx.x];
  store_as(out, c, a.wdtype, t);
}

// ---- rows longer than kMaxRegD: one CTA per row, which reads it once per pass (from L2) ----------
// HAS_W, HAS_B: the parameter is given.  An absent one has no load in the code at all: with a test
// for NULL around the load, a row with weight but no bias faulted (an access to address 0).

__device__ __forceinline__ float2 block_sum2(float2 v, float2* red) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float2 t = red[threadIdx.x & 31];
  t.x = warp_sum(t.x);
  t.y = warp_sum(t.y);
  return t;
}

template <typename T, bool HAS_W, bool HAS_B>
__global__ void __launch_bounds__(kWideThreads) ln_wide_forward_kernel(const LnArgs a) {
  __shared__ float2 red[32];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
    T* y = static_cast<T*>(a.y) + r * a.D;
    float s = 0.f, q = 0.f;
    for (int64_t c = threadIdx.x; c < a.D; c += kWideThreads) s += to_f32(x[c]);
    const float mean = block_sum2(make_float2(s, 0.f), red).x / (float)a.D;
    for (int64_t c = threadIdx.x; c < a.D; c += kWideThreads) {
      const float d = to_f32(x[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(block_sum2(make_float2(q, 0.f), red).x / (float)a.D + a.eps);
    if (threadIdx.x == 0 && a.mean != nullptr) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
    for (int64_t c = threadIdx.x; c < a.D; c += kWideThreads) {
      float w[1] = {1.f};
      if constexpr (HAS_W) load_param<1>(a.weight, c, a.wdtype, 1.f, w);
      float b[1] = {0.f};
      if constexpr (HAS_B) load_param<1>(a.bias, c, a.wdtype, 0.f, b);
      y[c] = from_f32<T>(fmaf((to_f32(x[c]) - mean) * rstd, w[0], b[0]));
    }
  }
}

template <typename T, bool HAS_W>
__global__ void __launch_bounds__(kWideThreads) ln_wide_backward_kernel(const LnArgs a) {
  __shared__ float2 red[32];
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + r * a.dy_stride;
    T* dx = static_cast<T*>(a.y) + r * a.D;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float2 s = make_float2(0.f, 0.f);
    for (int64_t c = threadIdx.x; c < a.D; c += kWideThreads) {
      float w[1] = {1.f};
      if constexpr (HAS_W) load_param<1>(a.weight, c, a.wdtype, 1.f, w);
      const float g = to_f32(dy[c]) * w[0];
      s.x += g;
      s.y = fmaf(g, (to_f32(x[c]) - mean) * rstd, s.y);
    }
    s = block_sum2(s, red);
    const float m1 = s.x / (float)a.D, m2 = s.y / (float)a.D;
    for (int64_t c = threadIdx.x; c < a.D; c += kWideThreads) {
      float w[1] = {1.f};
      if constexpr (HAS_W) load_param<1>(a.weight, c, a.wdtype, 1.f, w);
      const float h = (to_f32(x[c]) - mean) * rstd;
      dx[c] = from_f32<T>(rstd * (to_f32(dy[c]) * w[0] - m1 - h * m2));
    }
  }
}

// Column sums of rows [rows * p / parts, rows * (p + 1) / parts), p = blockIdx.y.
template <typename T>
__global__ void __launch_bounds__(256) ln_wide_columns_kernel(const LnArgs a) {
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.D) return;
  const int64_t p = blockIdx.y, parts = gridDim.y;
  float dw = 0.f, db = 0.f;
  for (int64_t r = a.rows * p / parts; r < a.rows * (p + 1) / parts; ++r) {
    const float d = to_f32(static_cast<const T*>(a.dy)[r * a.dy_stride + c]);
    const float h = (to_f32(static_cast<const T*>(a.x)[r * a.x_stride + c]) - a.mean[r]) * a.rstd[r];
    dw = fmaf(d, h, dw);
    db += d;
  }
  a.part[p * a.D + c] = dw;
  a.part[(parts + p) * a.D + c] = db;
}

// ---- host side ----------------------------------------------------------------------------

// Widest pack (in elements) that every row start and the row length allow.
int pack_elems(const LnArgs& a, bool backward) {
  const int64_t eb = (int64_t)elem_bytes(a.dtype), we = (int64_t)elem_bytes(a.wdtype);
  auto fits = [&](int64_t vec) {
    auto ok = [&](const void* p, int64_t stride, int64_t e) {
      return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (vec * e) == 0 && stride % vec == 0);
    };
    // A parameter is read in packs of at most 16 bytes.
    auto okw = [&](const void* p) {
      const int64_t bytes = vec * we < 16 ? vec * we : 16;
      return reinterpret_cast<uintptr_t>(p) % bytes == 0;
    };
    return a.D % vec == 0 && ok(a.x, a.x_stride, eb) && ok(a.y, a.D, eb) && okw(a.weight) &&
           (backward ? ok(a.dy, a.dy_stride, eb) : okw(a.bias));
  };
  const int64_t most = 16 / eb;
  if (fits(most)) return (int)most;
  if (eb == 2 && fits(2)) return 2;
  return 1;
}

struct Shape {
  int vec, nv, W, groups, threads;
};

// A row takes the fewest warps (a power of two) that hold it; short rows share a CTA of 8 warps.
Shape shape_of(const LnArgs& a, bool backward) {
  Shape s;
  s.vec = pack_elems(a, backward);
  const int few = s.vec * 32 >= 256 ? s.vec : 4;  // values a lane when one warp can hold the row so
  const bool small = a.D <= 32 * few;
  s.nv = (small ? few : kLaneElems) / s.vec;
  s.W = 1;
  while ((int64_t)s.W * 32 * s.nv * s.vec < a.D) s.W *= 2;
  s.groups = s.W < 8 ? 8 / s.W : 1;
  s.threads = s.W * s.groups * 32;
  return s;
}

// Calls f(T{}, vec, nv) with the instantiation of the shape.
template <typename T, typename F>
cudaError_t by_shape(const Shape& s, F f) {
  constexpr int MAXV = 16 / sizeof(T);
  using std::integral_constant;
  if (s.vec == MAXV) {
    if (s.nv * s.vec == kLaneElems) return f(T{}, integral_constant<int, MAXV>{}, integral_constant<int, kLaneElems / MAXV>{});
    return f(T{}, integral_constant<int, MAXV>{}, integral_constant<int, 1>{});
  }
  if constexpr (sizeof(T) == 2) {
    if (s.vec == 2) {
      if (s.nv * s.vec == kLaneElems) return f(T{}, integral_constant<int, 2>{}, integral_constant<int, kLaneElems / 2>{});
      return f(T{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
    }
  }
  if (s.nv == kLaneElems) return f(T{}, integral_constant<int, 1>{}, integral_constant<int, kLaneElems>{});
  return f(T{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
}

template <typename F>
cudaError_t by_type(int dtype, F f) {
  if (dtype == LM_F32) return f(float{});
  if (dtype == LM_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

// CTAs of the persistent backward grid, and so rows of partial sums: at most two per SM.
int64_t reg_parts(int64_t rows, int64_t D) {
  const int64_t most = 2 * kSmCount;
  return rows < most ? (rows > 0 ? rows : 1) : most;
}

}  // namespace

int64_t ln_backward_parts(int64_t rows, int64_t D) { return reg_parts(rows, D); }

cudaError_t launch_ln_forward(const LnArgs& a, cudaStream_t stream) {
  if (a.rows == 0 || a.D == 0) return cudaSuccess;
  cudaError_t e;
  if (a.D > kMaxRegD) {
    const unsigned grid = (unsigned)(a.rows < 4 * kSmCount ? a.rows : 4 * kSmCount);
    e = by_type(a.dtype, [&](auto t) {
      using E = decltype(t);
      auto k = a.weight != nullptr
                   ? (a.bias != nullptr ? ln_wide_forward_kernel<E, true, true> : ln_wide_forward_kernel<E, true, false>)
                   : (a.bias != nullptr ? ln_wide_forward_kernel<E, false, true> : ln_wide_forward_kernel<E, false, false>);
      return launch_kernel(k, dim3(grid), dim3(kWideThreads), 0, stream, a);
    });
  } else {
    const Shape s = shape_of(a, false);
    e = by_type(a.dtype, [&](auto t) {
      return by_shape<decltype(t)>(s, [&](auto tt, auto vec, auto nv) {
        auto k = ln_forward_kernel<decltype(tt), decltype(vec)::value, decltype(nv)::value>;
        const int64_t ctas = ceil_div(a.rows, s.groups);
        int per_sm = 1536 / s.threads;
        if (per_sm < 1) per_sm = 1;
        const int64_t most = (int64_t)per_sm * device_sm_count();
        return launch_kernel(k, dim3((unsigned)(ctas < most ? ctas : most)), dim3(s.threads), 0, stream, a, s.W, s.groups);
      });
    });
  }
  if (e != cudaSuccess) return e;
  note_launches(1);
  return cudaGetLastError();
}

cudaError_t launch_ln_backward(const LnArgs& a, cudaStream_t stream) {
  if (a.D == 0) return cudaSuccess;
  const bool sums = a.dw != nullptr || a.db != nullptr;
  const bool dx = a.y != nullptr;
  if (a.rows == 0 && !sums) return cudaSuccess;
  LnArgs b = a;
  if (!sums) b.part = nullptr;
  const int parts = (int)reg_parts(a.rows, a.D);
  cudaError_t e = cudaSuccess;
  int launches = 0;
  if (a.D > kMaxRegD) {
    if (dx && a.rows > 0) {
      const unsigned grid = (unsigned)(a.rows < 4 * kSmCount ? a.rows : 4 * kSmCount);
      e = by_type(a.dtype, [&](auto t) {
        using E = decltype(t);
        auto k = a.weight != nullptr ? ln_wide_backward_kernel<E, true> : ln_wide_backward_kernel<E, false>;
        return launch_kernel(k, dim3(grid), dim3(kWideThreads), 0, stream, b);
      });
      ++launches;
    }
    if (e == cudaSuccess && sums) {
      e = by_type(a.dtype, [&](auto t) {
        return launch_kernel(ln_wide_columns_kernel<decltype(t)>, dim3((unsigned)ceil_div(a.D, 256), parts), dim3(256), 0, stream, b);
      });
      ++launches;
    }
  } else {
    const Shape s = shape_of(a, true);
    e = by_type(a.dtype, [&](auto t) {
      return by_shape<decltype(t)>(s, [&](auto tt, auto vec, auto nv) {
        const size_t smem = s.groups > 1 && sums ? sizeof(float) * s.groups * a.D : 0;
        auto go = [&](auto k) {
          return launch_kernel(k, dim3(parts), dim3(s.threads), smem, stream, b, s.W, s.groups);
        };
        using E = decltype(tt);
        constexpr int V = decltype(vec)::value, N = decltype(nv)::value;
        if (s.threads <= 256) return go(ln_backward_kernel<E, V, N, 256>);
        if constexpr (V * N == kLaneElems) {
          if (s.threads == 512) return go(ln_backward_kernel<E, V, N, 512>);
          return go(ln_backward_kernel<E, V, N, 1024>);
        }
        return cudaErrorInvalidConfiguration;  // unreachable: short rows take 256 threads
      });
    });
    ++launches;
  }
  if (e != cudaSuccess) return e;
  if (sums) {
    e = launch_kernel(ln_sum_kernel, dim3((unsigned)ceil_div(a.D, 32), 2), dim3(32, kSumRows), 0, stream, b, parts);
    if (e != cudaSuccess) return e;
    ++launches;
  }
  note_launches(launches);
  return cudaGetLastError();
}

}  // namespace lm
}  // namespace rbf
