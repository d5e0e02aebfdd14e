// Typed vector access, e4m3 conversion and the activations shared by the 8-bit linear path
// (rows_quant.cu, gemm_scaled.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200 {

// ---- overlapped launches ----------------------------------------------------------------------
// The kernels of the 8-bit path follow one another in a stream and many last a few microseconds. Each is launched so that it may
// start while the one before it drains (programmatic stream serialisation): it sets itself up, then waits in wait_previous(),
// which returns when everything before it in the stream is complete and visible; only after that does it touch
// global memory. let_next_start() allows the next kernel the same. A kernel with TMEM calls it after its own allocation: a waiting
// successor could otherwise hold the columns its predecessor still needs.
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename Kernel, typename... Args>
int launch_overlapped(const char *what, Kernel kern, unsigned grid, unsigned block, size_t smem, cudaStream_t st, unsigned cluster,
                      const Args &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kern, args...);
  return check_launch(what);
}

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

// ---- pairs of fp32 values: one instruction for two (sm_100) ----------------------------------
struct Pair {
  uint64_t u;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(u) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ void get(float &lo, float &hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(u)); }
};
__device__ __forceinline__ Pair operator*(const Pair &a, const Pair &b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ Pair operator+(const Pair &a, const Pair &b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ Pair fma2(const Pair &a, const Pair &b, const Pair &c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(a.u), "l"(b.u), "l"(c.u));
  return r;
}

// x / (1 + 2^e), the two special-function operations in their fast forms (within 2^-22 and 2^-23 relative)
__device__ __forceinline__ Pair over_one_plus_exp2(const Pair &x, const Pair &e) {
  float e0, e1;
  e.get(e0, e1);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e0));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e1));
  float d0, d1;
  (Pair(e0, e1) + Pair(1.f, 1.f)).get(d0, d1);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d1));
  return x * Pair(d0, d1);
}
__device__ __forceinline__ Pair both(float v) { return Pair(v, v); }

// Activations of two fp32 values. All three smooth ones have the form x / (1 + 2^e(x)):
//   silu       e = -log2(e) x
//   gelu_tanh  0.5 (1 + tanh u) = 1 / (1 + exp(-2u)), so e = -2 log2(e) sqrt(2/pi) (x + 0.044715 x^3)
//   gelu       Phi(x) = 1 / (1 + exp(-logit Phi(x))), and logit Phi(x) / x is an even, smooth function of x: a polynomial of
//              degree 6 in x^2, fitted on |x| <= 6 by weighted least squares so that the error of x Phi(x) is at most 7.4e-8
//              (and below 3e-4 of the value down to x = -4); past 6, where Phi is 0 or 1 to 1e-9, x^2 stays at 36.
// Relative error otherwise that of an fp32 exponential, about (4 + |e|) 2^-24.
template <int ACT>
__device__ __forceinline__ Pair activate2_t(const Pair &x) {
  if (ACT == B200_ACT_RELU) {
    float a, b;
    x.get(a, b);
    return Pair(a > 0.f || a != a ? a : 0.f, b > 0.f || b != b ? b : 0.f);
  }
  if (ACT == B200_ACT_SILU) return over_one_plus_exp2(x, x * both(-1.4426950408889634f));
  if (ACT == B200_ACT_GELU_TANH)
    return over_one_plus_exp2(x, x * fma2(x * x, both(-0.10294324f), both(-2.3022082f)));
  if (ACT == B200_ACT_GELU) {
    float a, b;
    (x * x).get(a, b);
    const Pair q(fminf(a, 36.f), fminf(b, 36.f));
    constexpr float c[7] = {-2.3022067f, -0.104839917f, 9.66251724e-05f, 0.000159056584f, -1.14027313e-05f, 3.81676884e-07f, -5.12706323e-09f};
    Pair poly = both(c[6]);
#pragma unroll
    for (int i = 5; i >= 0; --i) poly = fma2(poly, q, both(c[i]));
    return over_one_plus_exp2(x, x * poly);
  }
  return x;
}
template <int ACT>
__device__ __forceinline__ float activate_t(float x) {
  float lo, hi;
  activate2_t<ACT>(Pair(x, x)).get(lo, hi);
  return lo;
}

}  // namespace b200
