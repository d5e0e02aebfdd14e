// RMS norm with the residual's addition and 8-bit output, and the row quantiser.
//
//   norm      h = x + r,  y = h * rho * gamma,  rho = 1 / sqrt(mean(h^2) + eps)
//   quantise  y = x  or  y = act(gate) * x
//   8 bits    scale = max(max|y|, 2^-100) / 448,  code = e4m3(y / scale)
//
// Both are bound by memory: each input is read once, each output written once. A row stays in the registers of the
// threads that loaded it (up to 32 values a thread). The norm needs two reductions over the row, sum(h^2) and max|y|;
// because rho is a positive factor common to the row, max|y| = rho * max|h * gamma|, so both are taken in ONE pass
// over the registers and joined in one exchange between warps. The maximum keeps a NaN, so that it reaches the scale; between threads it
// runs on bit patterns as unsigned integers, which order like the values, with a NaN's above infinity's.
//
// Measured over three sets of data in rotation, sustained (bytes read and written once / time; boards differ by up to 6 %): 8192 x 8192 bf16
// norm with residual to e4m3 81 us, 5.8 TB/s; 16384 x 1024 fp32 the same 36 us, 6.1 TB/s; 8192 x 14336 bf16 silu(gate) * x 105 us, 5.6
// TB/s; 16384 x 4096 fp32 59 us, 5.7 TB/s. A copy runs at 6.5 TB/s.
#include <math.h>

#include "typed.cuh"

namespace b200 {
namespace {

constexpr int kRowsPerCta = 8;         // rows of a CTA of the warp-per-row form
constexpr int kMaxBlock = 1024;
constexpr int kShiftedBlock = 576;      // of a row with ends
constexpr int kLongBlock = 1024;

struct RowParams {
  int64_t rows;
  int64_t x_stride, z_stride, h_stride, y_stride;  // z: residual or gate
  const void *x, *z, *gamma;
  void *h, *y;
  float *scale;
  int len;
  float eps;
  int activation;
  bool gamma_f32;  // gamma is fp32 although x is not
};

// VEC adjacent values: one 16-byte access (VEC * sizeof(T) == 16), or one value. They are kept as loaded until they are
// used: two inputs of 16 bits then take no more registers than one row of fp32.
template <typename T, int VEC>
struct Raw {
  uint32_t w[4];
  __device__ __forceinline__ void load(const T *p) {
    // plain (not .nc): an output may be the same rows, written later by the thread that read them
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(p)
                 : "memory");
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
      else unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    }
  }
};
template <typename T>
struct Raw<T, 1> {
  T w;
  __device__ __forceinline__ void load(const T *p) { w = *p; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = to_f32<T>(w); }
};
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint4 *>(p) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}
template <int VEC>
__device__ __forceinline__ void store_codes(uint8_t *p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) *p = (uint8_t)e4m3x2(v[0], 0.f);
  else if constexpr (VEC == 4) *reinterpret_cast<uint32_t *>(p) = e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16;
  else
    *reinterpret_cast<uint2 *>(p) = make_uint2(e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16,
                                               e4m3x2(v[4], v[5]) | e4m3x2(v[6], v[7]) << 16);
}
// gamma, read by every row: cached loads, but not those of the read-only path (__ldg). That path asks for data that nobody
// writes while the kernel exists, and the kernel before this one, which may write gamma, still runs when this one starts; the loads
// of 16-bit floats among its functions are also assembly without side effects to the compiler, which may move it in front of
// the checks that guard it.
template <typename T, int VEC>
__device__ __forceinline__ void load_gamma(const RowParams &p, int c, float (&g)[VEC]) {
  if (p.gamma_f32) {
    const float *q = static_cast<const float *>(p.gamma) + c;
    if constexpr (VEC == 1) {
      g[0] = *q;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 f = *reinterpret_cast<const float4 *>(q + i);
        g[i] = f.x; g[i + 1] = f.y; g[i + 2] = f.z; g[i + 3] = f.w;
      }
    }
  } else {
    const T *q = static_cast<const T *>(p.gamma) + c;
    if constexpr (VEC == 1) {
      g[0] = to_f32<T>(*q);
    } else {
      const uint4 u = *reinterpret_cast<const uint4 *>(q);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) g[i] = __uint_as_float(w[i]);
        else unpack2<T>(w[i], g[2 * i], g[2 * i + 1]);
      }
    }
  }
}

__device__ __forceinline__ float activate(int act, float x) {
  switch (act) {
    case B200_ACT_RELU: return activate_t<B200_ACT_RELU>(x);
    case B200_ACT_GELU: return activate_t<B200_ACT_GELU>(x);
    case B200_ACT_GELU_TANH: return activate_t<B200_ACT_GELU_TANH>(x);
    case B200_ACT_SILU: return activate_t<B200_ACT_SILU>(x);
    default: return x;
  }
}
template <int ACT, int VEC>
__device__ __forceinline__ void gate_vec(float (&v)[VEC], const float (&z)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] *= activate_t<ACT>(z[0]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) (Pair(v[i], v[i + 1]) * activate2_t<ACT>(Pair(z[i], z[i + 1]))).get(v[i], v[i + 1]);
  }
}

// The largest |v|, or NaN: one instruction for two values.
template <int VEC>
__device__ __forceinline__ void largest(float &top, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v[0])));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(fabsf(v[i])), "f"(fabsf(v[i + 1])));
  }
}

__device__ __forceinline__ uint32_t warp_umax(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// Sum and maximum over the threads of a row. WARP: a warp is a row. Otherwise the CTA is; `red` holds 2 x 32 words.
template <bool WARP>
__device__ __forceinline__ void join(float &sum, float &largest, float *red) {
  sum = warp_sum(sum);
  uint32_t top = warp_umax(__float_as_uint(largest));
  if (!WARP) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
    if (lane == 0) {
      red[warp] = sum;
      red[32 + warp] = __uint_as_float(top);
    }
    __syncthreads();
    // every warp joins the partial results itself, in the same order
    sum = warp_sum(lane < nwarp ? red[lane] : 0.f);
    top = warp_umax(lane < nwarp ? __float_as_uint(red[32 + lane]) : 0u);
  }
  largest = __uint_as_float(top);
}

// `top` is the pattern of max|y|: the floor keeps 448 / max finite; a NaN fails the comparison and stays.
__device__ __forceinline__ float row_max(float top) { return top < kTinyRowMax ? kTinyRowMax : top; }

// What both in-register kernels do with the values of one access. NORM: w is the residual; otherwise w is the gate.
template <typename T, bool NORM, int VEC>
__device__ __forceinline__ void combine(const RowParams &p, float (&v)[VEC], const float (&w)[VEC]) {
  if (NORM) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] += w[i];
  } else {
    switch (p.activation) {  // uniform
      case B200_ACT_RELU: gate_vec<B200_ACT_RELU, VEC>(v, w); break;
      case B200_ACT_GELU: gate_vec<B200_ACT_GELU, VEC>(v, w); break;
      case B200_ACT_GELU_TANH: gate_vec<B200_ACT_GELU_TANH, VEC>(v, w); break;
      case B200_ACT_SILU: gate_vec<B200_ACT_SILU, VEC>(v, w); break;
      default: gate_vec<B200_ACT_NONE, VEC>(v, w);
    }
  }
}

// What turns h * gamma (or y itself) into the output: y = v * rho, and code = y / scale. The two are not one factor: 448 / max alone
// is up to 5.7e32 (rows of zeros), which times rho overflows once eps is below 3e-12; and the product y * (448 / max) is not
// the quotient y / scale where that lies at a tie of e4m3, which for 16-bit inputs it often does.
//
// The quotient takes one reciprocal a row: q = y * inv, corrected once by its remainder, q + (y - q * scale) * inv (Markstein, IBM J.
// Res. Dev. 34, 1990). The remainder is exact but for its last bit, so the sum is y / scale to within 2^-45 before its one
// rounding. (A division for every value: 8192 x 14336 gate 108 -> 140 us.)
struct RowFactor {
  float rho, inv, minus_scale;
};
// From the row's sum of squares and largest pattern; the first thread of the row stores its scale.
template <bool NORM, bool CODES>
__device__ __forceinline__ RowFactor row_factor(const RowParams &p, int64_t row, float sum, float top, bool first) {
  const float rho = NORM ? 1.f / sqrtf(sum / (float)p.len + p.eps) : 1.f;
  if (!CODES) return RowFactor{rho, 1.f, 0.f};
  const float scale = row_max(top * rho) / kE4M3Max;
  if (first) p.scale[row] = scale;
  // an infinite scale makes quotients of finite values 0, which need no correction (and 0 * inf would be none)
  return RowFactor{rho, 1.f / scale, scale == INFINITY ? 0.f : -scale};
}
template <bool NORM, bool CODES, int VEC>
__device__ __forceinline__ void finish(const RowFactor &f, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    if (NORM) v[0] *= f.rho;
    if (CODES) {
      const float q = v[0] * f.inv;
      v[0] = fmaf(fmaf(q, f.minus_scale, v[0]), f.inv, q);
    }
  } else {
    const Pair rho = both(f.rho), inv = both(f.inv), minus_scale = both(f.minus_scale);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      Pair y(v[i], v[i + 1]);
      if (NORM) y = y * rho;
      if (CODES) {
        const Pair q = y * inv;
        y = fma2(fma2(q, minus_scale, y), inv, q);
      }
      y.get(v[i], v[i + 1]);
    }
  }
}

// Registers of a thread. A CTA that holds a row has up to 1024 threads: those of at most 8 values share an SM with another such CTA,
// and 16 values in two accesses, which run as CTAs of up to 512 threads, leave room for three of them (8192 x 8192 bf16 norm with
// 45 registers, two CTAs 87 us, with 40 77). 16 values read one by one take up to 128 and 512 threads.
constexpr int row_block(int vec, int accesses) { return vec == 1 && accesses > 4 ? kMaxBlock / 2 : kMaxBlock; }
constexpr int row_registers(int vec, int accesses, bool warp) {
  return warp || row_block(vec, accesses) < kMaxBlock ? 128 : vec * accesses <= 8 ? 32 : accesses == 2 ? 40 : 64;
}

// The row in registers, NV accesses of VEC values a thread. (CTAs that take several rows and load the next while they store
// were slower, their second set of registers halves the rows in flight: 8192 x 8192 norm 73 -> 84 us, 16384 x 4096 fp32
// rows 55 -> 77 us.)
template <typename T, bool NORM, bool CODES, int VEC, int NV, bool WARP>
__global__ void __maxnreg__(row_registers(VEC, NV, WARP))
rows_kernel(const RowParams p) {
  __shared__ float red[64];
  let_next_start();
  wait_previous();
  const int lanes = WARP ? 32 : blockDim.x;
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * kRowsPerCta + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (WARP && row >= p.rows) return;
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
  const T *z = static_cast<const T *>(p.z) + (p.z ? row * p.z_stride : 0);
  T *h = static_cast<T *>(p.h) + (p.h ? row * p.h_stride : 0);
  Raw<T, VEC> xr[NV], zr[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * lanes + t) * VEC;
    if (c < p.len) {
      xr[n].load(x + c);
      if (p.z) zr[n].load(z + c);
    }
  }
  float v[NV][VEC];
  float sum = 0.f;
  float top = 0.f;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * lanes + t) * VEC;
    if (c >= p.len) continue;
    xr[n].get(v[n]);
    if (p.z) {
      float w[VEC];
      zr[n].get(w);
      combine<T, NORM, VEC>(p, v[n], w);
    }
    if (NORM) {
      float g[VEC];
      if (p.gamma) load_gamma<T, VEC>(p, c, g);
      if (p.z) store_vec<T, VEC>(h + c, v[n]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum = fmaf(v[n][i], v[n][i], sum);
      if (p.gamma) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[n][i] *= g[i];
      }
    }
    if (CODES) largest<VEC>(top, v[n]);
  }
  join<WARP>(sum, top, red);
  const RowFactor factor = row_factor<NORM, CODES>(p, row, sum, top, t == 0);
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = (n * lanes + t) * VEC;
    if (c < p.len) {
      finish<NORM, CODES, VEC>(factor, v[n]);
      if (CODES) store_codes<VEC>(static_cast<uint8_t *>(p.y) + row * p.y_stride + c, v[n]);
      else store_vec<T, VEC>(static_cast<T *>(p.y) + row * p.y_stride + c, v[n]);
    }
  }
}

// Rows that do not start at multiples of 16 bytes, but all tensors of the operands' type at the same distance `off` (in values)
// behind one, as contiguous tensors of an odd width have. Accesses are the aligned 16 bytes around the row; only its two
// ends are read and written value by value. The codes' rows start elsewhere: they are put together in shared memory, at
// the accesses' positions, and leave shifted by `off` bytes, sixteen at a time. A CTA is a row.
template <typename T, bool NORM, bool CODES, int NV>
__global__ void __launch_bounds__(kShiftedBlock)
shifted_rows_kernel(const RowParams p) {
  constexpr int V = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) uint32_t packed[];
  __shared__ float red[64];
  let_next_start();
  wait_previous();
  const int lanes = blockDim.x, t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
  const T *z = static_cast<const T *>(p.z) + (p.z ? row * p.z_stride : 0);
  T *h = static_cast<T *>(p.h) + (p.h ? row * p.h_stride : 0);
  const int off = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  auto first = [&](int n) { return (n * lanes + t) * V - off; };  // column of access n's first value
  auto whole = [&](int c) { return c >= 0 && c + V <= p.len; };
  auto read = [&](const T *q, int c, float (&v)[V]) {  // an end of the row
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = c + i >= 0 && c + i < p.len ? to_f32<T>(q[c + i]) : 0.f;
  };
  auto write = [&](T *q, int c, const float (&v)[V]) {
    if (whole(c)) {
      store_vec<T, V>(q + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i >= 0 && c + i < p.len) q[c + i] = from_f32<T>(v[i]);
    }
  };
  Raw<T, V> xr[NV], zr[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = first(n);
    if (whole(c)) {
      xr[n].load(x + c);
      if (p.z) zr[n].load(z + c);
    }
  }
  float v[NV][V];
  float sum = 0.f;
  float top = 0.f;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = first(n);
    if (c >= p.len) continue;
    float w[V];
    if (whole(c)) {
      xr[n].get(v[n]);
      if (p.z) zr[n].get(w);
    } else {
      read(x, c, v[n]);
      if (p.z) read(z, c, w);
    }
    if (p.z) combine<T, NORM, V>(p, v[n], w);
    if (NORM) {
      if (p.z) write(h, c, v[n]);
#pragma unroll
      for (int i = 0; i < V; ++i) sum = fmaf(v[n][i], v[n][i], sum);
      if (p.gamma) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float g[1] = {0.f};
          if (c + i >= 0 && c + i < p.len) load_gamma<T, 1>(p, c + i, g);
          v[n][i] *= g[0];
        }
      }
    }
    if (CODES) largest<V>(top, v[n]);
  }
  join<false>(sum, top, red);
  const RowFactor factor = row_factor<NORM, CODES>(p, row, sum, top, t == 0);
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int c = first(n);
    if (c >= p.len) continue;
    finish<NORM, CODES, V>(factor, v[n]);
    if (CODES) store_codes<V>(reinterpret_cast<uint8_t *>(packed) + (c + off), v[n]);
    else write(static_cast<T *>(p.y) + row * p.y_stride, c, v[n]);
  }
  if (CODES) {
    __syncthreads();
    uint8_t *q = static_cast<uint8_t *>(p.y) + row * p.y_stride;
    const uint32_t *word = packed + off / 4;
    const int shift = off % 4 * 8;
    for (int c = 16 * t; c < p.len; c += 16 * lanes) {
      uint32_t w[5];
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = word[c / 4 + i];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], shift);
      if (c + 16 <= p.len) {
        *reinterpret_cast<uint4 *>(q + c) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + i < p.len) q[c + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
      }
    }
  }
}

// Rows longer than the registers of a CTA: the same arithmetic, the inputs read a second time instead of kept (the
// second read of a row of that length comes from L2). Each thread writes only where it has read, and h only in the
// second pass, so an output may be the same rows as an input.
template <typename T, bool NORM, bool CODES>
__global__ void __launch_bounds__(kLongBlock)
long_rows_kernel(const RowParams p) {
  __shared__ float red[64];
  let_next_start();
  wait_previous();
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
  const T *z = static_cast<const T *>(p.z) + (p.z ? row * p.z_stride : 0);
  T *h = static_cast<T *>(p.h) + (p.h ? row * p.h_stride : 0);
  auto value = [&](int c) {
    float v = to_f32<T>(x[c]);
    if (p.z) v = NORM ? v + to_f32<T>(z[c]) : v * activate(p.activation, to_f32<T>(z[c]));
    return v;
  };
  auto times_gamma = [&](float v, int c) {
    if (!NORM || !p.gamma) return v;
    return v * (p.gamma_f32 ? static_cast<const float *>(p.gamma)[c] : to_f32<T>(static_cast<const T *>(p.gamma)[c]));
  };
  float sum = 0.f;
  float top = 0.f;
  for (int c = threadIdx.x; c < p.len; c += blockDim.x) {
    const float v = value(c);
    if (NORM) sum = fmaf(v, v, sum);
    const float g[1] = {times_gamma(v, c)};
    if (CODES) largest<1>(top, g);
  }
  join<false>(sum, top, red);
  const RowFactor factor = row_factor<NORM, CODES>(p, row, sum, top, threadIdx.x == 0);
  for (int c = threadIdx.x; c < p.len; c += blockDim.x) {
    const float v = value(c);
    float o[1] = {times_gamma(v, c)};
    finish<NORM, CODES, 1>(factor, o);
    if (NORM && p.z) h[c] = from_f32<T>(v);
    if (CODES) static_cast<uint8_t *>(p.y)[row * p.y_stride + c] = (uint8_t)e4m3x2(o[0], 0.f);
    else static_cast<T *>(p.y)[row * p.y_stride + c] = from_f32<T>(o[0]);
  }
}

template <typename T, bool NORM, bool CODES, int VEC, int NV>
int launch_rows(cudaStream_t st, const RowParams &p, bool warp, int threads) {
  if (warp) {
    const int64_t ctas = (p.rows + kRowsPerCta - 1) / kRowsPerCta;
    return launch_overlapped("rows", rows_kernel<T, NORM, CODES, VEC, NV, true>, (unsigned)ctas, kRowsPerCta * 32, 0, st, 1, p);
  }
  return launch_overlapped("rows", rows_kernel<T, NORM, CODES, VEC, NV, false>, (unsigned)p.rows, threads, 0, st, 1, p);
}

template <typename T, bool NORM, bool CODES, int NV>
int launch_shifted(cudaStream_t st, const RowParams &p, int units) {
  const int threads = ((units + NV - 1) / NV + 31) / 32 * 32;
  // a row's codes from the first access on, and what the last sixteen read behind them
  const size_t smem = CODES ? ((size_t)units * (16 / sizeof(T)) + 16 + 32) / 16 * 16 : 0;
  return launch_overlapped("rows(shifted)", shifted_rows_kernel<T, NORM, CODES, NV>, (unsigned)p.rows, threads, smem, st, 1, p);
}

// How the rows of the operands lie: at multiples of 16 bytes, all equally far behind one, or neither.
enum class Rows { kAligned, kShifted, kAny };

template <typename T, bool NORM, bool CODES>
int dispatch(cudaStream_t st, const RowParams &p, Rows rows) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool vec = rows == Rows::kAligned;
  const bool few = p.rows <= 2 * kNumSMs;
  // Shorter rows, and few that a CTA of scalar accesses covers, are not worth the two ends (bf16 gate: 40000 x 511 scalar
  // 33 us, this 64; 30000 x 701 45 and 41; 8192 x 4097 192 and 45; 100 x 1001 1.9 and 3.1; 100 x 4095 3.2 and 3.4).
  if (rows == Rows::kShifted && p.len > (few ? 4096 : 512)) {
    const int units = (p.len + 2 * V - 2) / V;  // aligned accesses that an unaligned row touches at most
    if (units <= (V == 8 ? 2 * kShiftedBlock : 1024)) return launch_shifted<T, NORM, CODES, 2>(st, p, units);
    if (units <= 4 * kShiftedBlock) return launch_shifted<T, NORM, CODES, 4>(st, p, units);
    if (units <= 32 / V * kShiftedBlock) return launch_shifted<T, NORM, CODES, 32 / V>(st, p, units);
  }
  const int per = vec ? V : 1;                     // values of one access
  const int units = (p.len + per - 1) / per;       // accesses of a row (len is a multiple of V when vec)
  // Many rows: about one CTA starts per nanosecond, so short rows are put eight to a CTA, a warp each (131072 x 256 bf16 norm
  // 42 us, a CTA each 70; 60000 x 333 value by value 60 and 69; these and the times below before codes were quotients). A longer row is a CTA's: two accesses a thread, four where
  // one 16-bit input leaves few bytes on the way (8192 x 8192 bf16 quantise 48 -> 36 us, norm 73 either way), and more until the
  // CTA has at most 512 threads (norm with 1024 threads 84 us), but for the spills of eight (8192 x 14336 fp32 norm 272 us, 896
  // threads with four 235). Few rows leave SMs idle: one access each, the shortest way through a row.
  const bool warp = units <= (!vec ? 512 : V == 4 && !p.z ? 256 : 128) && p.rows >= kRowsPerCta * kNumSMs;
  int nv = 1;
  if (warp) {
    while (nv * 32 < units) nv *= 2;
  } else if (vec) {
    if (!few) nv = NORM || V == 4 ? 2 : 4;
    while (nv < 4 && nv * (few ? kMaxBlock : 512) < units) nv *= 2;
    if (V == 4 && nv * kMaxBlock < units) nv = 8;
  } else {
    nv = 4 * kMaxBlock < units ? 16 : 4;
  }
  if (!warp && nv * row_block(per, nv) < units)
    return launch_overlapped("rows(long)", long_rows_kernel<T, NORM, CODES>, (unsigned)p.rows, kLongBlock, 0, st, 1, p);
  const int threads = ((units + nv - 1) / nv + 31) / 32 * 32;
  if (vec) {
    switch (nv) {
      case 1: return launch_rows<T, NORM, CODES, V, 1>(st, p, warp, threads);
      case 2: return launch_rows<T, NORM, CODES, V, 2>(st, p, warp, threads);
      case 4: return launch_rows<T, NORM, CODES, V, 4>(st, p, warp, threads);
      default: return launch_rows<T, NORM, CODES, V, 32 / V>(st, p, warp, threads);
    }
  }
  if (nv <= 4) return launch_rows<T, NORM, CODES, 1, 4>(st, p, warp, threads);
  return launch_rows<T, NORM, CODES, 1, 16>(st, p, warp, threads);
}

bool rows16(const void *p, int64_t rows, int64_t stride, int64_t elem) {
  return aligned16(p) && (rows <= 1 || (stride * elem) % 16 == 0);
}
// The distance of every row behind a multiple of 16 bytes follows from the base's and the stride's.
bool same_distance(const void *p, const void *q, int64_t rows, int64_t p_stride, int64_t q_stride, int64_t elem) {
  return (reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(q)) % 16 == 0 &&
         (rows <= 1 || (p_stride - q_stride) * elem % 16 == 0);
}
bool stride_ok(int64_t stride, int64_t len, int64_t rows, bool input) {
  return stride >= (input ? 0 : len) || rows <= 1;
}

int type_bytes(int type) { return type == B200_TYPE_F32 ? 4 : 2; }
bool float_type(int type) { return type == B200_TYPE_F32 || type == B200_TYPE_F16 || type == B200_TYPE_BF16; }

template <bool NORM, bool CODES>
int by_type(cudaStream_t st, int type, const RowParams &p, Rows rows) {
  switch (type) {
    case B200_TYPE_F32: return dispatch<float, NORM, CODES>(st, p, rows);
    case B200_TYPE_F16: return dispatch<__half, NORM, CODES>(st, p, rows);
    default: return dispatch<__nv_bfloat16, NORM, CODES>(st, p, rows);
  }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" B200_API int b200_rmsnorm(void *stream, const b200_rmsnorm_desc *desc, const void *x, const void *residual,
                                     const void *gamma, void *h, void *y, float *scale) {
  if (!desc) return fail(B200_EINVAL, "rmsnorm: null descriptor");
  const b200_rmsnorm_desc &d = *desc;
  if (d.rows < 0) return fail(B200_EINVAL, "rmsnorm: negative number of rows");
  if (d.len < 1) return fail(B200_EINVAL, "rmsnorm: rows need at least one value");
  if (!float_type(d.type)) return fail(B200_EINVAL, "rmsnorm: unknown type %d", d.type);
  if (gamma && d.gamma_type != d.type && d.gamma_type != B200_TYPE_F32)
    return fail(B200_EINVAL, "rmsnorm: gamma must have the type of x or be fp32");
  const bool codes = d.y_type == B200_TYPE_E4M3;
  if (!codes && d.y_type != d.type) return fail(B200_EINVAL, "rmsnorm: the output has the type of x, or is e4m3");
  if (!(d.eps >= 0.f)) return fail(B200_EINVAL, "rmsnorm: eps must not be negative");
  if (d.rows == 0) return B200_OK;
  if (d.rows > 0x7fffffffLL || d.len > 0x7fffffffLL - kLongBlock)
    return fail(B200_EUNSUPPORTED, "rmsnorm: more than 2^31 rows or values a row");
  if (!x || !y || (codes && !scale)) return fail(B200_EINVAL, "rmsnorm: null pointer");
  if (!residual != !h) return fail(B200_EINVAL, "rmsnorm: residual and h come together");
  if (!stride_ok(d.x_stride, d.len, d.rows, true) || (residual && !stride_ok(d.residual_stride, d.len, d.rows, true)) ||
      (h && !stride_ok(d.h_stride, d.len, d.rows, false)) || !stride_ok(d.y_stride, d.len, d.rows, false))
    return fail(B200_EINVAL, "rmsnorm: an input's row stride is negative, or an output's smaller than the row");
  const int b = type_bytes(d.type);
  const bool vec = d.len % (16 / b) == 0 && rows16(x, d.rows, d.x_stride, b) &&
                   (!residual || (rows16(residual, d.rows, d.residual_stride, b) && rows16(h, d.rows, d.h_stride, b))) &&
                   (!gamma || aligned16(gamma)) && rows16(y, d.rows, d.y_stride, codes ? 1 : b);
  auto like_x = [&](const void *q, int64_t stride) { return same_distance(q, x, d.rows, stride, d.x_stride, b); };
  const bool shifted = (!residual || (like_x(residual, d.residual_stride) && like_x(h, d.h_stride))) &&
                       (codes ? rows16(y, d.rows, d.y_stride, 1) : like_x(y, d.y_stride));
  const Rows rows = vec ? Rows::kAligned : shifted ? Rows::kShifted : Rows::kAny;
  RowParams p = {d.rows, d.x_stride, d.residual_stride, d.h_stride, d.y_stride, x, residual, gamma, h, y, scale,
                 (int)d.len, d.eps, B200_ACT_NONE, gamma && d.gamma_type == B200_TYPE_F32 && d.type != B200_TYPE_F32};
  return codes ? by_type<true, true>((cudaStream_t)stream, d.type, p, rows)
               : by_type<true, false>((cudaStream_t)stream, d.type, p, rows);
}

extern "C" B200_API int b200_quantize_rows(void *stream, const b200_quantize_desc *desc, const void *x,
                                           const void *gate, void *q, float *scale) {
  if (!desc) return fail(B200_EINVAL, "quantize_rows: null descriptor");
  const b200_quantize_desc &d = *desc;
  if (d.rows < 0) return fail(B200_EINVAL, "quantize_rows: negative number of rows");
  if (d.len < 1) return fail(B200_EINVAL, "quantize_rows: rows need at least one value");
  if (!float_type(d.type)) return fail(B200_EINVAL, "quantize_rows: unknown type %d", d.type);
  if (d.activation < B200_ACT_NONE || d.activation > B200_ACT_SILU)
    return fail(B200_EINVAL, "quantize_rows: unknown activation %d", d.activation);
  if (!gate && d.activation != B200_ACT_NONE)
    return fail(B200_EINVAL, "quantize_rows: an activation belongs to a gate");
  if (d.rows == 0) return B200_OK;
  if (d.rows > 0x7fffffffLL || d.len > 0x7fffffffLL - kLongBlock)
    return fail(B200_EUNSUPPORTED, "quantize_rows: more than 2^31 rows or values a row");
  if (!x || !q || !scale) return fail(B200_EINVAL, "quantize_rows: null pointer");
  if (!stride_ok(d.x_stride, d.len, d.rows, true) || (gate && !stride_ok(d.gate_stride, d.len, d.rows, true)) ||
      !stride_ok(d.q_stride, d.len, d.rows, false))
    return fail(B200_EINVAL, "quantize_rows: an input's row stride is negative, or the output's smaller than the row");
  const int b = type_bytes(d.type);
  const bool vec = d.len % (16 / b) == 0 && rows16(x, d.rows, d.x_stride, b) && (!gate || rows16(gate, d.rows, d.gate_stride, b)) &&
                   rows16(q, d.rows, d.q_stride, 1);
  const bool shifted = (!gate || same_distance(gate, x, d.rows, d.gate_stride, d.x_stride, b)) && rows16(q, d.rows, d.q_stride, 1);
  const Rows rows = vec ? Rows::kAligned : shifted ? Rows::kShifted : Rows::kAny;
  RowParams p = {d.rows, d.x_stride, d.gate_stride, 0, d.q_stride, x, gate, nullptr, nullptr, q, scale,
                 (int)d.len, 0.f, d.activation, false};
  return by_type<false, true>((cudaStream_t)stream, d.type, p, rows);
}
