// pb2_epilogue.cuh -- the activations and 16-bit conversions the linear and
// expert kernels share.
//
// All in f32, on values that are rounded to 16 or 8 bits afterwards, so the
// approximate exponential and reciprocal (a few f32 ulps, denormals flushed)
// do not show in a result; each is one instruction beside its multiply.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "pb2_common.cuh"

namespace pb2 {

__device__ __forceinline__ float exp_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 1 / (1 + e^-x): e^-x overflows to inf for x < -88 and the quotient is then 0.
__device__ __forceinline__ float sigmoid_fast(float x) { return rcp_fast(1.0f + exp_fast(-x)); }

// The normal distribution function by Abramowitz & Stegun 7.1.26:
// erfc(z) = (a1 t + ... + a5 t^5) e^(-z^2) + eps, t = 1 / (1 + p z), z >= 0,
// |eps| < 1.5e-7.  Taking the tail on the side of x keeps gelu's small
// negative values free of cancellation.
__device__ __forceinline__ float normal_cdf(float x) {
  const float z = fabsf(x) * 0.70710678f;
  const float t = rcp_fast(fmaf(0.3275911f, z, 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float tail = 0.5f * p * t * exp_fast(-z * z);
  return x < 0.0f ? tail : 1.0f - tail;
}

// The larger, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int kAct>
__device__ __forceinline__ float activate(float x) {
  if constexpr (kAct == PB2_ACT_RELU) return max_nan(x, 0.0f);  // a NaN stays one, as in the other activations
  if constexpr (kAct == PB2_ACT_SILU) return x * sigmoid_fast(x);
  if constexpr (kAct == PB2_ACT_GELU) return x * normal_cdf(x);
  // 0.5 (1 + tanh u) = sigmoid(2 u)
  if constexpr (kAct == PB2_ACT_GELU_TANH)
    return x * sigmoid_fast(1.5957691216f * fmaf(0.044715f * x * x, x, x));
  return x;
}

__device__ __forceinline__ uint32_t pack_half2(float x, float y, bool f16) {
  if (f16) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t w, bool f16) {
  if (f16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float half_at(const void* p, int64_t i, bool f16) {
  return f16 ? __half2float(static_cast<const __half*>(p)[i]) : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ uint16_t half_bits(float x, bool f16) {
  return f16 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

// A launch with programmatic stream serialization (see griddep_wait).
template <typename K, typename... Args>
int launch_programmatic(K kernel, dim3 grid, int threads, int smem, cudaStream_t s, int cluster, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads), 1, 1);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return launch_status();
}

}  // namespace pb2
