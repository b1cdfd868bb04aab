// lm_common.cuh -- element types, vector access and reductions shared by the language-model
// kernels (ln.cu, token_loss.cu, ortho.cu) and the host helpers of their C entries.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/lm_sm100.h"
#include "rbf_common.cuh"
#include "rbf_kernels.cuh"
#include "rbf_ptx.cuh"

namespace rbf {

// ---- host side (rbf_api.cu): the status detail and the device check of every C entry
int set_detail(int status, const char* what, cudaError_t e = cudaSuccess);
int cuda_status(cudaError_t e, const char* what);
int check_device();

namespace lm {

inline size_t elem_bytes(int dtype) { return dtype == LM_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == LM_F32 || dtype == LM_BF16 || dtype == LM_F16; }

// ---- element conversion: everything is computed in fp32 and rounded once, to nearest even
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements as one access of VEC * sizeof(T) bytes (naturally aligned).
template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
  T v[VEC];
};

// ---- two fp32 values in one register pair: sm_100 adds and multiplies both in one instruction
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Elements 2 k and 2 k + 1 of a pack, and back (one rounding each).
template <typename T, int VEC>
__device__ __forceinline__ F2 pair_of(const Pack<T, VEC>& p, int k) {
  if constexpr (sizeof(T) == 4) {
    return f2(p.v[2 * k], p.v[2 * k + 1]);
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t w = reinterpret_cast<const uint32_t*>(&p)[k];
    return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    const float2 x = __half22float2(reinterpret_cast<const __half2*>(&p)[k]);
    return f2(x.x, x.y);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void set_pair(Pack<T, VEC>& p, int k, F2 x) {
  float a, b;
  unpack(x, a, b);
  if constexpr (sizeof(T) == 4) {
    p.v[2 * k] = a;
    p.v[2 * k + 1] = b;
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    reinterpret_cast<__nv_bfloat162*>(&p)[k] = __floats2bfloat162_rn(a, b);
  } else {
    reinterpret_cast<__half2*>(&p)[k] = __floats2half2_rn(a, b);
  }
}

// The largest element of a pack (NaN is passed over), 16-bit types two at a time.
template <typename T, int VEC>
__device__ __forceinline__ float pack_max(const Pack<T, VEC>& p) {
  if constexpr (sizeof(T) == 4) {
    float m = p.v[0];
#pragma unroll
    for (int e = 1; e < VEC; ++e) m = fmaxf(m, p.v[e]);
    return m;
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162* q = reinterpret_cast<const __nv_bfloat162*>(&p);
    __nv_bfloat162 m = q[0];
#pragma unroll
    for (int e = 1; e < VEC / 2; ++e) m = __hmax2(m, q[e]);
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    const __half2* q = reinterpret_cast<const __half2*>(&p);
    __half2 m = q[0];
#pragma unroll
    for (int e = 1; e < VEC / 2; ++e) m = __hmax2(m, q[e]);
    return fmaxf(__low2float(m), __high2float(m));
  }
}

// Streaming read: data that this kernel reads once bypasses L1 (the operands that CTAs share,
// such as a weight vector, keep it).
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_stream(const T* p) {
  Pack<T, VEC> r;
  if constexpr (sizeof(r) == 16) {
    uint4 u;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
    *reinterpret_cast<uint4*>(&r) = u;
  } else {
    r = *reinterpret_cast<const Pack<T, VEC>*>(p);
  }
  return r;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& r) {
  if constexpr (sizeof(r) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
  else *reinterpret_cast<Pack<T, VEC>*>(p) = r;
}

// An element of a vector whose type is known at run time only (a parameter's gradient).
__device__ __forceinline__ void store_as(void* p, int64_t i, int dtype, float v) {
  if (dtype == LM_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == LM_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// VEC consecutive elements of a parameter vector (NULL: `absent`), in loads of at most 16 bytes.
// Plain loads behind the test for NULL: a read-only (__ldg) load may be hoisted above it.
template <int VEC, typename T>
__device__ __forceinline__ void load_param_as(const T* p, float (&out)[VEC]) {
  constexpr int N = VEC * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : VEC;
#pragma unroll
  for (int i = 0; i < VEC; i += N) {
    const Pack<T, N> q = *reinterpret_cast<const Pack<T, N>*>(p + i);
#pragma unroll
    for (int e = 0; e < N; ++e) out[i + e] = to_f32(q.v[e]);
  }
}
template <int VEC>
__device__ __forceinline__ void load_param(const void* p, int64_t i, int dtype, float absent,
                                           float (&out)[VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) out[e] = absent;
  } else if (dtype == LM_F32) {
    load_param_as<VEC>(static_cast<const float*>(p) + i, out);
  } else if (dtype == LM_BF16) {
    load_param_as<VEC>(static_cast<const __nv_bfloat16*>(p) + i, out);
  } else {
    load_param_as<VEC>(static_cast<const __half*>(p) + i, out);
  }
}

// The same as pairs.
template <int VEC>
__device__ __forceinline__ void load_param(const void* p, int64_t i, int dtype, float absent, F2 (&out)[VEC / 2]) {
  float t[VEC];
  load_param<VEC>(p, i, dtype, absent, t);
#pragma unroll
  for (int e = 0; e < VEC / 2; ++e) out[e] = f2(t[2 * e], t[2 * e + 1]);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Barrier `id` (1..15) among `threads` threads of the CTA (whole warps).
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

}  // namespace lm
}  // namespace rbf
