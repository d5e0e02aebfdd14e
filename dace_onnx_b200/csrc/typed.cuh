// Typed vector access, e4m3 conversion and the activations shared by the 8-bit linear path
// (rows_quant.cu, gemm_scaled.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200 {

constexpr float kE4M3Max = 448.f;
constexpr float kTinyRowMax = 7.888609052210118e-31f;  // 2^-100: keeps 448 / max finite for rows of zeros

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two values to 16-bit types, packed lo | hi << 16, round to nearest even
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t u, float &lo, float &hi);
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t u, float &lo, float &hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u));
  lo = f.x; hi = f.y;
}
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t u, float &lo, float &hi) {
  lo = __uint_as_float(u << 16);
  hi = __uint_as_float(u & 0xffff0000u);
}

// Two values to e4m3 (nearest even, saturating at 448, NaN stays NaN), lo in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Activations in fp32. exp and the division in their fast forms (each within a few ulp, ~3e-7 relative): the
// results are rounded to 8 or 16 bits, or to fp32 next to an fp32 sum whose own error is of that size.
__device__ __forceinline__ float sigmoid_times(float x, float z) { return __fdividef(x, 1.f + __expf(-z)); }
template <int ACT>
__device__ __forceinline__ float activate_t(float x) {
  if (ACT == B200_ACT_RELU) return x > 0.f ? x : (x != x ? x : 0.f);
  if (ACT == B200_ACT_GELU) return gelu_erf(x);
  // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u))
  if (ACT == B200_ACT_GELU_TANH) return sigmoid_times(x, 1.5957691216057308f * x * fmaf(0.044715f * x, x, 1.f));
  if (ACT == B200_ACT_SILU) return sigmoid_times(x, x);
  return x;
}

}  // namespace b200
