// ln.cu -- layer norm: forward, and backward with the reduction of the weight's gradient.
//
//   y  = xh * w + b,   xh = (x - mean) * rstd,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   g  = dy * w,       dx = rstd * (g - mean(g) - xh * mean(g * xh))
//   dw = sum_rows dy * xh,   db = sum_rows dy
//
// Both passes are bound by HBM: the forward moves 2 elements and the backward 3 per value, at
// some 10 flops each.  Every row is read once and held on chip; the variance is a second pass over
// registers, not over memory, and has no cancellation.
//
// In the backward a thread keeps the sums of its columns' dy * xh and dy in registers (long rows: in
// shared memory) over all its rows; each CTA writes one row of partial sums at its end and a second, short kernel adds
// those in a fixed order.  No atomics: equal calls give equal bits.
//
// Statistics, sums and partial sums are fp32; every output is rounded once.
#include <algorithm>
#include <type_traits>

#include "lm_common.cuh"
#include "lm_kernels.cuh"

namespace rbf {
namespace lm {
namespace {

constexpr int kLaneElems = 16;                   // values of a row per lane
constexpr int kWarpElems = 32 * kLaneElems;
constexpr int64_t kMaxRegD = 32 * kWarpElems;    // longest row held in the registers of one CTA
constexpr int64_t kLongMin = 8 * kWarpElems;     // longest row of ln_backward_kernel, with 256 threads
constexpr int kWideThreads = 1024;
constexpr int kSumRows = 32;                     // partial rows that ln_sum adds side by side

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

// A group of W warps takes a row, `groups` rows a CTA.  The row is read once, all its loads at a time,
// and stays in registers as it came; mean, variance and result are three passes over those.
template <typename T, int VEC, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) ln_forward_kernel(const LnArgs a, int W, int groups) {
  __shared__ float2 red[32 * 2 * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = warp / W, w = warp - g * W;
  float2* slots = red + g * 64;
  int turn = 0;
  const int D = (int)a.D;
  const int64_t r = (int64_t)blockIdx.x * groups + g;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  if (r >= a.rows) return;
  T* y = static_cast<T*>(a.y) + r * D;
  Row<T, VEC, NV> x;
  x.load(static_cast<const T*>(a.x) + r * a.x_stride, D, W, w, lane);
  const float inv_d = 1.f / (float)D;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += to_f32(x.p[i].v[e]);  // columns past D are 0
  const float mean = group_sum(make_float2(s, 0.f), W, w, 1 + g, slots, turn).x * inv_d;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (((i * W + w) * 32 + lane) * VEC < D) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = to_f32(x.p[i].v[e]) - mean;
        q = fmaf(d, d, q);
      }
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
    if (c < D) {
      float wv[VEC], bv[VEC];
      load_param<VEC>(a.weight, c, a.wdtype, 1.f, wv);
      load_param<VEC>(a.bias, c, a.wdtype, 0.f, bv);
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.v[e] = from_f32<T>(fmaf((to_f32(x.p[i].v[e]) - mean) * rstd, wv[e], bv[e]));
      store_pack<T, VEC>(y + c, o);
    }
  }
}

// ---- rows of whole 16-byte packs, and enough of them: one CTA per SM
// `TW` threads (a group, whole warps) take ROWS rows at a time, each thread NV packs of a row; threads that no
// group has room for only wait for the end.  A thread copies
// what it will read itself into shared memory (cp.async), a ring of blocks ahead: 160 to 190 KB
// an SM are on their way at any time, no registers wait for them, and no thread waits for another's
// copy.  The rows of a block share each reduction and its barrier.  Arithmetic is on pairs: a value of
// 16 bits has some 20 issue slots at the rate that HBM delivers them.
//
// SHIFT: rows that do not start on 16 bytes.  Of VEC rows one after another each starts at another place in
// its first 16 bytes, but every VEC-th row at the same, so a CTA takes the rows of one such class: its packs
// are aligned, and a thread's columns (all `shift` less than its place) stay the same.  What the first and the
// last pack hold of other rows is set to 0 and not stored.  8192 x 1023 bf16, forward and backward: 20 and 26 us, 49 and
// 41 with loads of single values; 4-byte and 8-byte packs were slower from 64 rows on as well (8192 x 4084 bf16: 56 and
// 60 us, 68 and 75).
constexpr int kRingThreads = 512;
constexpr size_t kRingBytes = 196608;

__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The first `bytes` of 16, and zeros.
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// OPS operands (x; or x and dy) of ROWS rows a block.  Pointers move from block to block: addresses made
// anew from row and stride took more instructions than the arithmetic.
template <typename T, int NV, int ROWS, int OPS, bool SHIFT>
struct Ring {
  static constexpr int VEC = 16 / sizeof(T);
  static constexpr int kPieces = ROWS * NV * OPS;  // 16-byte pieces of a thread and block
  static constexpr int kFit = (int)(kRingBytes / (kPieces * 16 * kRingThreads));
  static constexpr int STAGES = kFit > 8 ? 8 : kFit;
  static constexpr uint32_t kPiece = 16 * kRingThreads, kStage = kPieces * kPiece;
  static constexpr int CLASSES = SHIFT ? VEC : 1;
  static_assert(STAGES >= 3, "ring");
  int g, in, D, pitch;      // pitch: elements between a thread's packs
  int cls, shift;           // of this CTA's rows, which are every CLASSES-th from `cls` on
  unsigned columns, edge;   // bit i: pack i has elements of the row; and others
  int64_t rows;             // of the class
  int64_t row, step;        // first row of this group's present block, rows from one block to the next
  uint32_t base;            // this thread's slots
  const T* next[OPS];       // this thread's first pack of the next block to copy
  int64_t stride[OPS], hop[OPS];
  int64_t next_row;
  int in_stage, out_stage;

  __device__ __forceinline__ Ring(void* smem, const LnArgs& a, int TW, const T* const (&op)[OPS], const int64_t (&st)[OPS]) {
    const int groups = kRingThreads / TW;
    g = threadIdx.x / TW;
    in = threadIdx.x - g * TW;
    D = (int)a.D;
    pitch = TW * VEC;
    cls = SHIFT ? blockIdx.x % CLASSES : 0;
    shift = SHIFT ? (int)(cls * (a.D % VEC) % VEC) : 0;
    columns = edge = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      columns |= (place(i) < shift + D ? 1u : 0u) << i;
      if (SHIFT) edge |= (place(i) < shift || place(i) + VEC > shift + D ? 1u : 0u) << i;
    }
    rows = (a.rows - cls + CLASSES - 1) / CLASSES;
    step = (int64_t)((gridDim.x - cls + CLASSES - 1) / CLASSES) * groups * ROWS;
    row = next_row = ((int64_t)(blockIdx.x / CLASSES) * groups + g) * ROWS;
    if (g >= groups) {
      columns = 0;
      row = next_row = rows;
    }
    base = ptx::smem_u32(smem) + threadIdx.x * 16;
#pragma unroll
    for (int o = 0; o < OPS; ++o) {
      stride[o] = CLASSES * st[o];
      hop[o] = step * stride[o];
      next[o] = op[o] + cls * st[o] + row * stride[o] - shift + in * VEC;
    }
    in_stage = out_stage = 0;
  }
  // Where pack i of this thread begins, counted from the row's first pack; whether its element e is the row's.
  __device__ __forceinline__ int place(int i) const { return i * pitch + in * VEC; }
  __device__ __forceinline__ bool inside(int i, int e) const { return place(i) + e >= shift && place(i) + e < shift + D; }
  // Row r of the class in the matrix, and this thread's first element of it in an output.
  __device__ __forceinline__ int64_t index(int64_t r) const { return cls + r * CLASSES; }
  __device__ __forceinline__ int64_t out(int64_t r) const { return index(r) * D - shift + in * VEC; }
  // How many of this group's ROWS rows from r on there are.
  __device__ __forceinline__ int left(int64_t r) const {
    const int64_t n = rows - r;
    return n >= ROWS ? ROWS : n > 0 ? (int)n : 0;
  }
  __device__ __forceinline__ void issue() {
    const int n = left(next_row);
    const uint32_t at = base + in_stage * kStage;
#pragma unroll
    for (int o = 0; o < OPS; ++o) {
      const T* p = next[o];
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        if (k < n) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (columns >> i & 1u) {
              const uint32_t to = at + ((k * NV + i) * OPS + o) * kPiece;
              if (SHIFT) copy_async16(to, p + i * pitch, min(16, (shift + D - place(i)) * (int)sizeof(T)));
              else copy_async16(to, p + i * pitch);
            }
        }
        p += stride[o];
      }
      next[o] += hop[o];
    }
    next_row += step;
    if (++in_stage == STAGES) in_stage = 0;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Piece (row k, pack i, operand o) of the present block; zeros outside the matrix.
  __device__ __forceinline__ Pack<T, VEC> read(int n, int k, int i, int o) const {
    Pack<T, VEC> p;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (k < n && (columns >> i & 1u))
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                   : "r"(base + out_stage * kStage + ((k * NV + i) * OPS + o) * kPiece));
    *reinterpret_cast<uint4*>(&p) = u;
    if (SHIFT && (edge >> i & 1u)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (!inside(i, e)) p.v[e] = from_f32<T>(0.f);
    }
    return p;
  }
  // Pack i of an output row, and of a parameter (as pairs).
  __device__ __forceinline__ void store(T* p, int i, const Pack<T, VEC>& v) const {
    if (SHIFT && (edge >> i & 1u)) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (inside(i, e)) p[e] = v.v[e];
    } else {
      store_pack<T, VEC>(p, v);
    }
  }
  __device__ __forceinline__ void param(const void* w, int i, int dtype, float absent, F2 (&v)[VEC / 2]) const {
    if constexpr (!SHIFT) {
      load_param<VEC>(w, place(i), dtype, absent, v);
    } else {
      float f[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float one[1] = {0.f};
        if (inside(i, e)) load_param<1>(w, place(i) + e - shift, dtype, absent, one);
        f[e] = one[0];
      }
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) v[e] = f2(f[2 * e], f[2 * e + 1]);
    }
  }
  __device__ __forceinline__ void advance() {
    row += step;
    if (++out_stage == STAGES) out_stage = 0;
  }
};

// Sums of N values (a power of two) over a group's W warps.  In a warp each step hands half of the
// values to the other half of the lanes, so that N values take N + 5 - log2 N exchanges in place of
// 5 N.  slots: this group's 2^k >= W of [2][kRingSlots][N], used in turn, so that one barrier is enough; those
// past W hold zeros.
constexpr int kRingSlots = 2 * kRingThreads / 32;
template <int N>
__device__ __forceinline__ void ring_sum(float (&s)[N], int W, int wide, int g, float (*red)[kRingSlots][N], int& turn) {
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - g * W;  // of the group
  int v = 0;
#pragma unroll
  for (int n = N / 2, o = 1; o < 32; n >>= 1, o <<= 1) {
    if (n > 0) {
      const bool up = lane & o;
      v = 2 * v + (up ? 1 : 0);
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float send = up ? s[i] : s[i + n], keep = up ? s[i + n] : s[i];
        s[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
      }
    } else {
      s[0] += __shfl_xor_sync(0xffffffffu, s[0], o);
    }
  }
  // This lane holds the warp's sum of value v.
  if (lane < N) red[turn][g * wide + warp][v] = s[0];
  if (W == 1) __syncwarp();
  else named_sync(1 + g, W * 32);
  const float* r = red[turn][g * wide + (lane & (wide - 1))];
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = r[i];
  for (int o = 1; o < wide; o <<= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
  }
  turn ^= 1;
}

// Zeros in the slots; the power of two that a group has of them.
template <int N>
__device__ __forceinline__ int ring_clear(int W, float (*red)[kRingSlots][N]) {
  for (int i = threadIdx.x; i < 2 * kRingSlots * N; i += kRingThreads) (&red[0][0][0])[i] = 0.f;
  __syncthreads();
  return W == 1 ? 1 : 2 << (31 - __clz(W - 1));
}

__device__ __forceinline__ float total(F2 x) {
  float a, b;
  unpack(x, a, b);
  return a + b;
}
__device__ __forceinline__ F2 twice(float x) { return f2(x, x); }

template <typename T, int NV, int ROWS, bool SHIFT>
__global__ void __launch_bounds__(kRingThreads, 1) ln_ring_forward_kernel(const LnArgs a, int TW) {
  using R = Ring<T, NV, ROWS, 1, SHIFT>;
  constexpr int VEC = R::VEC, H = VEC / 2;
  extern __shared__ uint4 smem[];
  __shared__ float red[2][kRingSlots][ROWS];
  const T* const op[1] = {static_cast<const T*>(a.x)};
  const int64_t stride[1] = {a.x_stride};
  R ring(smem, a, TW, op, stride);
  const int W = TW / 32, wide = ring_clear(W, red);
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
#pragma unroll
  for (int s = 0; s < R::STAGES - 1; ++s) ring.issue();
  // Weight and bias of a thread's columns: in registers where they suffice, else read again (from L1).
  constexpr bool KEEP = NV * VEC <= 8;
  F2 wv[KEEP ? NV : 1][H], bv[KEEP ? NV : 1][H];
  auto params = [&](int i) {
    if (ring.columns >> i & 1u) {
      ring.param(a.weight, i, a.wdtype, 1.f, wv[KEEP ? i : 0]);
      ring.param(a.bias, i, a.wdtype, 0.f, bv[KEEP ? i : 0]);
    }
  };
  if (KEEP) {
#pragma unroll
    for (int i = 0; i < NV; ++i) params(i);
  }
  const float inv_d = 1.f / (float)ring.D;
  T* y = static_cast<T*>(a.y) + ring.out(ring.row);
  const int64_t y_row = (int64_t)R::CLASSES * ring.D, y_hop = ring.step * y_row;
  int turn = 0;
  // Values as they came (16 bits), or converted once where a thread holds few enough of them.
  constexpr bool WIDE = NV * ROWS * VEC <= 32;
  for (; ring.row < ring.rows; ring.advance(), y += y_hop) {
    asm volatile("cp.async.wait_group %0;" ::"n"(R::STAGES - 2) : "memory");
    const int n = ring.left(ring.row);
    Pack<T, VEC> x[ROWS][NV];
    F2 xw[WIDE ? ROWS : 1][WIDE ? NV : 1][H] = {};
    float s[ROWS], q[ROWS];
    auto value = [&](int k, int i, int e) { return WIDE ? xw[WIDE ? k : 0][WIDE ? i : 0][e] : pair_of(x[k][i], e); };
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      F2 t = twice(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        x[k][i] = ring.read(n, k, i, 0);
#pragma unroll
        for (int e = 0; e < H; ++e) {
          if (WIDE) xw[WIDE ? k : 0][WIDE ? i : 0][e] = pair_of(x[k][i], e);
          t = add2(t, value(k, i, e));
        }
      }
      s[k] = total(t);
    }
    ring.issue();
    ring_sum(s, W, wide, ring.g, red, turn);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      s[k] *= inv_d;  // the mean
      const F2 m = twice(-s[k]);
      F2 t = twice(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (ring.columns >> i & 1u) {
#pragma unroll
          for (int e = 0; e < H; ++e) {
            F2 d = add2(value(k, i, e), m);
            if (SHIFT && (ring.edge >> i & 1u)) {
              float d0, d1;
              unpack(d, d0, d1);
              d = f2(ring.inside(i, 2 * e) ? d0 : 0.f, ring.inside(i, 2 * e + 1) ? d1 : 0.f);
            }
            if (WIDE) xw[WIDE ? k : 0][WIDE ? i : 0][e] = d;
            t = fma2(d, d, t);
          }
        }
      q[k] = total(t);
    }
    ring_sum(q, W, wide, ring.g, red, turn);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      q[k] = 1.f / sqrtf(q[k] * inv_d + a.eps);  // the reciprocal deviation
      if (ring.in == 0 && k < n && a.mean != nullptr) {
        a.mean[ring.index(ring.row + k)] = s[k];
        a.rstd[ring.index(ring.row + k)] = q[k];
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!(ring.columns >> i & 1u)) break;
      if (!KEEP) params(i);
      T* out = y + i * ring.pitch;
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        const F2 m = twice(-s[k]), rs = twice(q[k]);
        Pack<T, VEC> o;
#pragma unroll
        for (int e = 0; e < H; ++e) {
          const F2 d = WIDE ? value(k, i, e) : add2(value(k, i, e), m);
          set_pair(o, e, fma2(mul2(d, rs), wv[KEEP ? i : 0][e], bv[KEEP ? i : 0][e]));
        }
        if (k < n) ring.store(out, i, o);
        out += y_row;
      }
    }
  }
}

template <typename T, int NV, int ROWS, bool SHIFT>
__global__ void __launch_bounds__(kRingThreads, 1) ln_ring_backward_kernel(const LnArgs a, int TW) {
  using R = Ring<T, NV, ROWS, 2, SHIFT>;
  constexpr int VEC = R::VEC, H = VEC / 2;
  extern __shared__ uint4 smem[];
  __shared__ float red[2][kRingSlots][2 * ROWS];
  const T* const op[2] = {static_cast<const T*>(a.x), static_cast<const T*>(a.dy)};
  const int64_t stride[2] = {a.x_stride, a.dy_stride};
  R ring(smem, a, TW, op, stride);
  const int W = TW / 32, wide = ring_clear(W, red), D = ring.D;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
#pragma unroll
  for (int s = 0; s < R::STAGES - 1; ++s) ring.issue();
  constexpr bool KEEP = NV * VEC <= 8;
  F2 wv[KEEP ? NV : 1][H], dw[NV][H], db[NV][H];
  auto weight = [&](int i) {
    if (ring.columns >> i & 1u) {
      ring.param(a.weight, i, a.wdtype, 1.f, wv[KEEP ? i : 0]);
    } else {
#pragma unroll
      for (int e = 0; e < H; ++e) wv[KEEP ? i : 0][e] = twice(0.f);
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (KEEP) weight(i);
#pragma unroll
    for (int e = 0; e < H; ++e) dw[i][e] = db[i][e] = twice(0.f);
  }
  float mean[ROWS], rstd[ROWS];
  auto stats = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      mean[k] = r + k < ring.rows ? a.mean[ring.index(r + k)] : 0.f;
      rstd[k] = r + k < ring.rows ? a.rstd[ring.index(r + k)] : 0.f;
    }
  };
  stats(ring.row);
  // x and dy are read from shared memory again for dx where they and the column sums take more registers than
  // there are.
  constexpr bool AGAIN = NV * VEC * ROWS > 16;
  const float inv_d = 1.f / (float)D;
  T* dx = static_cast<T*>(a.y) + ring.out(ring.row);
  const int64_t dx_row = (int64_t)R::CLASSES * D, dx_hop = ring.step * dx_row;
  int turn = 0;
  for (; ring.row < ring.rows; ring.advance(), dx += dx_hop) {
    asm volatile("cp.async.wait_group %0;" ::"n"(R::STAGES - 2) : "memory");
    const int n = ring.left(ring.row);
    Pack<T, VEC> x[AGAIN ? 1 : ROWS][AGAIN ? 1 : NV], dy[AGAIN ? 1 : ROWS][AGAIN ? 1 : NV];
    auto fetch = [&](int k, int i) {
      x[AGAIN ? 0 : k][AGAIN ? 0 : i] = ring.read(n, k, i, 0);
      dy[AGAIN ? 0 : k][AGAIN ? 0 : i] = ring.read(n, k, i, 1);
    };
    auto x_of = [&](int k, int i, int e) { return pair_of(x[AGAIN ? 0 : k][AGAIN ? 0 : i], e); };
    auto dy_of = [&](int k, int i, int e) { return pair_of(dy[AGAIN ? 0 : k][AGAIN ? 0 : i], e); };
    float s[2 * ROWS];
    F2 shift[ROWS], rs[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      rs[k] = twice(rstd[k]);
      shift[k] = twice(-mean[k]);
      if (!AGAIN) {
#pragma unroll
        for (int i = 0; i < NV; ++i) fetch(k, i);
      }
    }
    ring.issue();
    stats(ring.row + ring.step);
    F2 t0[ROWS], t1[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) t0[k] = t1[k] = twice(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!KEEP) weight(i);
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        if (AGAIN) fetch(k, i);
#pragma unroll
        for (int e = 0; e < H; ++e) {
          const F2 h = mul2(add2(x_of(k, i, e), shift[k]), rs[k]);
          const F2 d = dy_of(k, i, e);  // 0 past D and past the last row
          const F2 gw = mul2(d, wv[KEEP ? i : 0][e]);
          t0[k] = add2(t0[k], gw);
          t1[k] = fma2(gw, h, t1[k]);
          dw[i][e] = fma2(d, h, dw[i][e]);
          db[i][e] = add2(db[i][e], d);
        }
      }
    }
    if (a.y == nullptr) continue;
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      s[2 * k] = total(t0[k]);
      s[2 * k + 1] = total(t1[k]);
    }
    ring_sum(s, W, wide, ring.g, red, turn);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!(ring.columns >> i & 1u)) break;
      if (!KEEP) weight(i);
      T* out = dx + i * ring.pitch;
#pragma unroll
      for (int k = 0; k < ROWS; ++k) {
        const F2 m1 = twice(-s[2 * k] * inv_d), m2 = twice(-s[2 * k + 1] * inv_d);
        Pack<T, VEC> o;
        if (AGAIN) fetch(k, i);
#pragma unroll
        for (int e = 0; e < H; ++e) {
          const F2 h = mul2(add2(x_of(k, i, e), shift[k]), rs[k]);
          const F2 gw = fma2(dy_of(k, i, e), wv[KEEP ? i : 0][e], m1);
          set_pair(o, e, mul2(fma2(h, m2, gw), rs[k]));
        }
        if (k < n) ring.store(out, i, o);
        out += dx_row;
      }
    }
  }
  if (a.part == nullptr) return;
  // This CTA's column sums; groups add theirs up in shared memory (the ring's, whose copies are done).
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  const int groups = kRingThreads / TW;
  F2* sums = reinterpret_cast<F2*>(smem);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    auto& acc = which == 0 ? dw : db;
    float* out = a.part + ((int64_t)which * gridDim.x + blockIdx.x) * D;
    __syncthreads();
    if (SHIFT) {
      float* all = reinterpret_cast<float*>(smem);  // [groups][D]
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < H; ++e) {
          float v[2];
          unpack(acc[i][e], v[0], v[1]);
#pragma unroll
          for (int o = 0; o < 2; ++o)
            if ((ring.columns >> i & 1u) && ring.inside(i, 2 * e + o)) all[ring.g * D + ring.place(i) + 2 * e + o - ring.shift] = v[o];
        }
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += kRingThreads) {
        float t = all[c];
        for (int k = 1; k < groups; ++k) t += all[k * D + c];
        out[c] = t;
      }
      continue;
    }
    if (ring.g > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!(ring.columns >> i & 1u)) break;
#pragma unroll
        for (int e = 0; e < H; ++e) sums[((ring.g - 1) * D + ring.place(i)) / 2 + e] = acc[i][e];
      }
    }
    __syncthreads();
    if (ring.g == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!(ring.columns >> i & 1u)) break;
        const int c = ring.place(i);
#pragma unroll
        for (int e = 0; e < H; ++e) {
          F2 t = acc[i][e];
          for (int k = 1; k < groups; ++k) t = add2(t, sums[((k - 1) * D + c) / 2 + e]);
          *reinterpret_cast<F2*>(out + c + 2 * e) = t;
        }
      }
    }
  }
}

// ---- backward, any rows
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(256) ln_backward_kernel(const LnArgs a, int W, int groups) {
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

// ---- backward, long rows that the ring does not take
// A CTA takes a row, 16 values a thread; the sums of a thread's own columns are in shared memory (64 or
// 128 KB), at a quarter of the time that the row takes from HBM.  In registers, of which 1024 threads have
// 64 each, they spilled: 4096 x 12288 fp32 in 132 us in place of 400, 4096 x 9001 bf16 in 137 in place of 1118.
// Rows of up to 8192 values take two CTAs of 512 threads an SM, one of which loads while the other waits for its sums:
// 8192 x 4101 fp32 in 117 us, 164 with one of 1024 (230 with 512 threads and registers).
template <typename T, int VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) ln_long_backward_kernel(const LnArgs a) {
  constexpr int NV = kLaneElems / VEC, W = THREADS / 32;
  extern __shared__ float sums[];  // [dw, db][value of the thread][thread]
  __shared__ float2 red[2 * 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* const dw = sums + threadIdx.x;
  float* const db = dw + kLaneElems * THREADS;
  int turn = 0;
  const int D = (int)a.D;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
#pragma unroll
  for (int k = 0; k < kLaneElems; ++k) dw[k * THREADS] = db[k * THREADS] = 0.f;
  const float inv_d = 1.f / (float)D;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    Row<T, VEC, NV> x, dy;
    x.load(static_cast<const T*>(a.x) + r * a.x_stride, D, W, warp, lane);
    dy.load(static_cast<const T*>(a.dy) + r * a.dy_stride, D, W, warp, lane);
    const float mean = a.mean[r], rstd = a.rstd[r];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((i * W + warp) * 32 + lane) * VEC;
      if (c >= D) break;
      float w[VEC];
      load_param<VEC>(a.weight, c, a.wdtype, 1.f, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int k = (i * VEC + e) * THREADS;
        const float h = (to_f32(x.p[i].v[e]) - mean) * rstd, d = to_f32(dy.p[i].v[e]);
        const float gw = d * w[e];
        s.x += gw;
        s.y = fmaf(gw, h, s.y);
        if (a.part != nullptr) {
          dw[k] = fmaf(d, h, dw[k]);
          db[k] += d;
        }
      }
    }
    if (a.y == nullptr) continue;
    s = group_sum(s, W, warp, 1, red, turn);
    const float m1 = s.x * inv_d, m2 = s.y * inv_d;
    T* dx = static_cast<T*>(a.y) + r * D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ((i * W + warp) * 32 + lane) * VEC;
      if (c >= D) break;
      float w[VEC];
      load_param<VEC>(a.weight, c, a.wdtype, 1.f, w);
      Pack<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float h = (to_f32(x.p[i].v[e]) - mean) * rstd;
        o.v[e] = from_f32<T>(rstd * (to_f32(dy.p[i].v[e]) * w[e] - m1 - h * m2));
      }
      store_pack<T, VEC>(dx + c, o);
    }
  }
  if (a.part == nullptr) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = ((i * W + warp) * 32 + lane) * VEC;
    if (c >= D) break;
    constexpr int N = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int e = 0; e < VEC; e += N) {
      Pack<float, N> v, u;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        v.v[k] = dw[(i * VEC + e + k) * THREADS];
        u.v[k] = db[(i * VEC + e + k) * THREADS];
      }
      store_pack<float, N>(a.part + (int64_t)blockIdx.x * D + c + e, v);
      store_pack<float, N>(a.part + ((int64_t)gridDim.x + blockIdx.x) * D + c + e, u);
    }
  }
}

// dw[c] = sum_p part[0][p][c], db[c] = sum_p part[1][p][c]: 32 columns per CTA, 32 thread rows
// that each add every 32nd partial.
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
// HAS_W, HAS_B: the parameter is given.  An absent one has neither a load nor a test for NULL in the loops
// over the row.  (The test alone is safe too, as in the other kernels, while the load behind it is a plain one: a
// read-only load, __ldg, had been lifted above the test and read address 0.)

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
  for (int64_t vec = 16 / eb; vec > 1; vec /= 2)
    if (fits(vec)) return (int)vec;
  return 1;
}

struct Shape {
  int vec, nv, W, groups, threads;
};

// Backward of any rows: a row takes the fewest warps (a power of two) that hold it 16 values a lane;
// short rows share a CTA of 8 warps.
Shape backward_shape(const LnArgs& a, int vec) {
  Shape s;
  s.vec = vec;
  const int few = s.vec * 32 >= 256 ? s.vec : 4;  // values a lane when one warp can hold the row so
  const bool small = a.D <= 32 * few;
  s.nv = (small ? few : kLaneElems) / s.vec;
  s.W = 1;
  while ((int64_t)s.W * 32 * s.nv * s.vec < a.D) s.W *= 2;
  s.groups = s.W < 8 ? 8 / s.W : 1;
  s.threads = s.W * s.groups * 32;
  return s;
}

// Packs that a lane of the forward holds at most: 64 bytes of single values, 128 of wider ones.
constexpr int most_packs(int vec, int elem_bytes) { return vec == 1 ? 32 : vec * elem_bytes == 4 ? 16 : 128 / (vec * elem_bytes); }

// Forward: a row takes the fewest warps that hold it in up to 8 packs of 16 bytes (16 pairs, 32 single
// values) a lane, so that few warps wait for one another; more of them while the rows alone do not fill the SMs.
Shape forward_shape(const LnArgs& a) {
  Shape s;
  s.vec = pack_elems(a, false);
  const int most = most_packs(s.vec, (int)elem_bytes(a.dtype));
  const int64_t packs = ceil_div(a.D, 32 * s.vec);  // of a lane, with one warp
  s.W = 1;
  while (s.W * most < packs || (s.W < packs && s.W < 8 && a.rows * s.W < 8 * (int64_t)kSmCount)) s.W *= 2;
  s.nv = 1;
  while ((int64_t)s.nv * s.W < packs) s.nv *= 2;
  s.groups = s.W < 4 ? 4 / s.W : 1;
  s.threads = s.W * s.groups * 32;
  return s;
}

// Calls f(T{}, vec, nv) with the instantiation of the shape.
template <typename T, typename F>
cudaError_t by_backward_shape(const Shape& s, F f) {
  constexpr int MAXV = 16 / sizeof(T);
  using std::integral_constant;
  if (s.vec == MAXV) {
    if (s.nv * s.vec == kLaneElems) return f(T{}, integral_constant<int, MAXV>{}, integral_constant<int, kLaneElems / MAXV>{});
    return f(T{}, integral_constant<int, MAXV>{}, integral_constant<int, 1>{});
  }
  if (s.vec == 2) {
    if (s.nv * s.vec == kLaneElems) return f(T{}, integral_constant<int, 2>{}, integral_constant<int, kLaneElems / 2>{});
    return f(T{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
  }
  if constexpr (MAXV == 8) {
    if (s.vec == 4) {
      if (s.nv * s.vec == kLaneElems) return f(T{}, integral_constant<int, 4>{}, integral_constant<int, kLaneElems / 4>{});
      return f(T{}, integral_constant<int, 4>{}, integral_constant<int, 1>{});
    }
  }
  if (s.nv == kLaneElems) return f(T{}, integral_constant<int, 1>{}, integral_constant<int, kLaneElems>{});
  return f(T{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
}

template <typename T, int VEC, int NV, typename F>
cudaError_t by_forward_count(const Shape& s, F f) {
  constexpr int most = most_packs(VEC, sizeof(T));
  if (s.nv <= NV) {
    if (s.threads <= 256) return f(ln_forward_kernel<T, VEC, NV, 256>);
    if constexpr (NV == most) return f(ln_forward_kernel<T, VEC, NV, 512>);  // only the longest rows
  }
  if constexpr (NV < most) return by_forward_count<T, VEC, NV * 2>(s, f);
  return cudaErrorInvalidConfiguration;
}

template <typename T, typename F>
cudaError_t by_forward_shape(const Shape& s, F f) {
  constexpr int MAXV = 16 / sizeof(T);
  if (s.vec == MAXV) return by_forward_count<T, MAXV, 1>(s, f);
  if (s.vec == 2) return by_forward_count<T, 2, 2>(s, f);
  if constexpr (MAXV == 8) {
    if (s.vec == 4) return by_forward_count<T, 4, 1>(s, f);
  }
  return by_forward_count<T, 1, 4>(s, f);
}

template <typename T, int THREADS>
auto long_backward(int vec) {
  constexpr int V = 16 / sizeof(T);
  if (V == 8 && vec == 4) return ln_long_backward_kernel<T, 4, THREADS>;
  return vec == V ? ln_long_backward_kernel<T, V, THREADS> : vec == 2 ? ln_long_backward_kernel<T, 2, THREADS> : ln_long_backward_kernel<T, 1, THREADS>;
}

template <typename F>
cudaError_t by_type(int dtype, F f) {
  if (dtype == LM_F32) return f(float{});
  if (dtype == LM_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

// CTAs of the persistent backward grids, and so rows of partial sums, at most.
int64_t reg_parts(int64_t rows) {
  const int64_t most = 2 * kSmCount;
  return rows < most ? (rows > 0 ? rows : 1) : most;
}

// Rows of whole 16-byte packs go through the ring: up to 32 KB each in the forward, 16 KB in the backward, whose column
// sums leave no registers for four packs a thread (4096 x 8192 fp32: 101 us, ln_long_backward_kernel 81;
// 4096 x 16384 bf16: 155, 138).
// The forward below so many values goes a row at a time: its CTAs then have a block or two each.
constexpr int64_t kRingForwardMin = 2 * 1024 * 1024;
bool ring_fits(const LnArgs& a, bool backward) {
  const int64_t eb = (int64_t)elem_bytes(a.dtype);
  return pack_elems(a, backward) * eb == 16 && a.D * eb <= (backward ? 16384 : 32768);
}

// Other rows, where the matrices start on 16 bytes and their rows shift alike: up to four packs a thread in the
// forward, 4096 x 9001 bf16 in 96 us (212 with loads of single values); up to two in the backward, 8192 x 8175 bf16
// in 171 us (ln_long_backward_kernel: 212), while with four 4096 x 9001 takes 266 (137).  With two packs of which
// many lie past the row it is the slower one: 8192 rows of 4500 bf16 values 138 us (97), 5001 143 (133), 5700 142 (109),
// 6100 148 (113).  Odd lengths near the upper end are about even: 8192 x 5801 145 (149), 8192 x 6001 149 (158), 1000 x 6001
// 31.4 (30.7).
constexpr int64_t kShiftMinRows = 64;  // eight classes of a few rows (no slower than the other path from there on)
bool shift_fits(const LnArgs& a, bool backward) {
  const int64_t vec = 16 / (int64_t)elem_bytes(a.dtype);
  auto ok = [&](const void* p, int64_t stride) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride - a.D) % vec == 0);
  };
  if (backward && a.D > kLongMin && a.D < kLongMin * 3 / 2) return false;
  return a.rows >= kShiftMinRows && a.D + vec - 1 <= (backward ? 2 : 4) * vec * kRingThreads && ok(a.x, a.x_stride) && ok(a.y, a.D) &&
         (!backward || ok(a.dy, a.dy_stride));
}

// `nv` packs a thread or as many more as 512 threads need, and the threads of a row.
template <typename T, bool SHIFT>
void ring_shape(const LnArgs& a, int* nv, int* TW) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t D = SHIFT ? a.D + VEC - 1 : a.D;
  while ((int64_t)*nv * VEC * kRingThreads < D) *nv *= 2;
  *TW = (int)(32 * ceil_div(D, (int64_t)32 * *nv * VEC));
}

template <typename K>
cudaError_t launch_ring(K k, const LnArgs& a, int classes, int TW, int rows, int* parts, cudaStream_t stream) {
  const int64_t blocks = classes * ceil_div(ceil_div(a.rows, classes), (int64_t)(kRingThreads / TW) * rows);
  *parts = (int)std::max<int64_t>(1, std::min<int64_t>(blocks, kSmCount));
  const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kRingBytes);
  if (e != cudaSuccess) return e;
  return launch_kernel(k, dim3(*parts), dim3(kRingThreads), kRingBytes, stream, a, TW);
}

// Four rows a block, since each block costs two reductions and their barriers: 8192 x 4096 bf16 in 33 us
// with two packs a thread and four rows, 54 us with one row, 38 us with one pack (and 512 threads that
// wait for each other) and four rows.
template <typename T, bool SHIFT>
cudaError_t launch_ring_forward(const LnArgs& a, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T), classes = SHIFT ? VEC : 1;
  int nv = a.D > 32 * VEC && !(SHIFT && VEC == 8) ? 2 : 1, TW, parts;
  ring_shape<T, SHIFT>(a, &nv, &TW);
  if (nv == 1) return launch_ring(ln_ring_forward_kernel<T, 1, 4, SHIFT>, a, classes, TW, 4, &parts, stream);
  if (nv == 2) return launch_ring(ln_ring_forward_kernel<T, 2, 4, SHIFT>, a, classes, TW, 4, &parts, stream);
  return launch_ring(ln_ring_forward_kernel<T, 4, 2, SHIFT>, a, classes, TW, 2, &parts, stream);
}

// As few packs a thread as hold the row, since its column sums take 2 registers a value; two rows a block,
// four where that leaves 16 values a thread.  8192 x 4096 bf16: 48 us, 57 with one row, 50 with four; fp32: 67 us,
// 74 with two rows.  8192 x 8192 bf16: 108 us, 139 with one row.
template <typename T, bool SHIFT>
cudaError_t launch_ring_backward(const LnArgs& a, int* parts, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T), classes = SHIFT ? VEC : 1, R = sizeof(T) == 4 ? 4 : 2;
  int nv = 1, TW;
  ring_shape<T, SHIFT>(a, &nv, &TW);
  if (nv == 1) return launch_ring(ln_ring_backward_kernel<T, 1, R, SHIFT>, a, classes, TW, R, parts, stream);
  return launch_ring(ln_ring_backward_kernel<T, 2, 2, SHIFT>, a, classes, TW, 2, parts, stream);
}

}  // namespace

int64_t ln_backward_parts(int64_t rows, int64_t D) { return reg_parts(rows); }

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
  } else if (ring_fits(a, false) && a.rows * a.D >= kRingForwardMin) {
    e = by_type(a.dtype, [&](auto t) { return launch_ring_forward<decltype(t), false>(a, stream); });
  } else if (shift_fits(a, false) && a.rows * a.D >= kRingForwardMin) {
    e = by_type(a.dtype, [&](auto t) { return launch_ring_forward<decltype(t), true>(a, stream); });
  } else {
    const Shape s = forward_shape(a);
    const unsigned grid = (unsigned)ceil_div(a.rows, s.groups);
    e = by_type(a.dtype, [&](auto t) {
      return by_forward_shape<decltype(t)>(s, [&](auto k) {
        return launch_kernel(k, dim3(grid), dim3(s.threads), 0, stream, a, s.W, s.groups);
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
  int parts = (int)reg_parts(a.rows);
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
  } else if (ring_fits(a, true)) {
    e = by_type(a.dtype, [&](auto t) { return launch_ring_backward<decltype(t), false>(b, &parts, stream); });
    ++launches;
  } else if (shift_fits(a, true)) {
    e = by_type(a.dtype, [&](auto t) { return launch_ring_backward<decltype(t), true>(b, &parts, stream); });
    ++launches;
  } else if (a.D > kLongMin) {
    const bool half = a.D <= 512 * kLaneElems;
    parts = (int)std::min<int64_t>(parts, (half ? 2 : 1) * kSmCount);
    e = by_type(a.dtype, [&](auto t) {
      const int threads = half ? 512 : 1024;
      auto k = half ? long_backward<decltype(t), 512>(pack_elems(a, true)) : long_backward<decltype(t), 1024>(pack_elems(a, true));
      const int smem = (int)sizeof(float) * 2 * kLaneElems * threads;
      const cudaError_t set = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      return set != cudaSuccess ? set : launch_kernel(k, dim3(parts), dim3(threads), smem, stream, b);
    });
    ++launches;
  } else {
    const Shape s = backward_shape(a, pack_elems(a, true));
    e = by_type(a.dtype, [&](auto t) {
      return by_backward_shape<decltype(t)>(s, [&](auto tt, auto vec, auto nv) {
        const size_t smem = s.groups > 1 && sums ? sizeof(float) * s.groups * a.D : 0;
        return launch_kernel(ln_backward_kernel<decltype(tt), decltype(vec)::value, decltype(nv)::value>, dim3(parts),
                             dim3(s.threads), smem, stream, b, s.W, s.groups);
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
