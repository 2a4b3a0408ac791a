// pb2_epilogue.cuh -- the activations and 16-bit conversions the linear and
// expert kernels share.
//
// All in f32, on values that are rounded to 16 or 8 bits afterwards.  The
// approximate exponential and reciprocal are one instruction each beside a
// multiply; the exponential's relative error grows with its argument, whose
// rounding it takes along: 2^-22 at 0, 2^-17 at e^-80.  An activation is within
// 2^-15 of its value (in f32's normal numbers; smaller ones are flushed to 0),
// a sixteenth of a unit of f16 at most.
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

// The normal distribution function by its tail on the side of x:
//   Phi(-|x|) = e^(-x^2 / 2) (c1 t + ... + c6 t^6), t = 1 / (1 + p |x|),
// the form of Abramowitz & Stegun 7.1.26 with coefficients of its own, fitted
// for the least relative error: 5e-6 of the tail for all |x| <= 14, beyond
// which f32 has no tail.  (7.1.26 bounds the absolute error, which was 0.1%
// of the tail at -5 and 0.65% at -7, 1.5 units of an f16 result.)
__device__ __forceinline__ float normal_cdf(float x) {
  const float t = rcp_fast(fmaf(0.31f, fabsf(x), 1.0f));
  float p = fmaf(-0.0739291534f, t, 0.1804503947f);
  p = fmaf(p, t, 0.0157446619f);
  p = fmaf(p, t, 0.1334298104f);
  p = fmaf(p, t, 0.1204412729f);
  p = fmaf(p, t, 0.1238607019f);
  const float tail = p * t * exp_fast(-0.5f * x * x);
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
