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

// Activations of two fp32 values.
//   silu       x / (1 + 2^e), e = -log2(e) x
//   gelu_tanh  the same with 0.5 (1 + tanh u) = 1 / (1 + exp(-2u)): e = -2 log2(e) sqrt(2/pi) (x + 0.044715 x^3)
//   gelu       x Phi(x) = max(x, 0) - |x| Phi(-|x|), and Phi(-w) = P(t) exp(-w^2 / 2) with t = 1 / (1 + 0.35 w): a polynomial without
//              constant term of degree 9, fitted to erfcx(w / sqrt 2) / 2 on w <= 16 by reweighted least squares so that its relative
//              error is at most 3.3e-8. The tail keeps its relative accuracy, which the scale of a row of negative gates needs.
// Relative error: silu and gelu_tanh that of an fp32 exponential, about (4 + |e|) 2^-24; gelu below (16 + 1.25 x^2) 2^-24 for x < 0
// and 4e-7 for x > 0 (2.4e-7 absolute anywhere). Values below 2^-126 come out as 0. NaN and gelu(-inf) give NaN.
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
    float a, b, t0, t1, e0, e1;
    x.get(a, b);
    const Pair positive(fmaxf(a, 0.f), fmaxf(b, 0.f));
    // +inf - 16 * 0, not inf * 0; -inf and NaN stay
    asm("min.NaN.f32 %0, %0, 0f41800000;" : "+f"(a));
    asm("min.NaN.f32 %0, %0, 0f41800000;" : "+f"(b));
    const Pair w(fabsf(a), fabsf(b));
    fma2(w, both(0.35f), both(1.f)).get(t0, t1);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(t0));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(t1));
    (w * both(-0.7213475204444817f) * w).get(e0, e1);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e0));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e1));
    constexpr float c[9] = {-0.139621243f, -0.139864519f, -0.119814187f, -0.105579816f, 0.0232753269f, -0.15940915f, 0.255915701f,
                            -0.144067347f, 0.02916524f};  // of -P(t) / t
    const Pair t(t0, t1);
    Pair poly = both(c[8]);
#pragma unroll
    for (int i = 7; i >= 0; --i) poly = fma2(poly, t, both(c[i]));
    return fma2(w, poly * t * Pair(e0, e1), positive);
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
