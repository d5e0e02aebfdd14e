// Matrix product on e4m3 / fp16 / bf16 operands with scales, bias, activation and residual in its epilogue:
//   Y[m, n] = act(sa[m] * sw[n] * sum_k A[m, k] W[n, k] + bias[n]) + residual[m, n]
//
// Row scales are constant along K, so they leave the sum: the tensor cores multiply the codes as they are (an e4m3
// product is exact in fp32) and the epilogue multiplies once per output.
//
// Two kernels, both TMA -> shared memory -> tcgen05.mma -> TMEM -> registers, warp-specialised (one loading thread, one
// issuing thread, epilogue warps), K-blocks of 128 bytes with the 128-byte swizzle:
//
//   pair   many rows of A. A cluster of two CTAs computes 256 x BN outputs (rows of A are TMEM lanes), persistent, several
//          accumulators so that the epilogue of a tile runs under the MMAs of the next. Outputs leave through shared memory and
//          TMA stores: 32-byte stores of each thread's own row took a third of the epilogue. Bound by the power limit: 8192 x
//          14336, K 4096, e4m3 with bias and silu 387 to 406 us (2.4 to 2.5 PFLOP/s) at 1000 W and 1.1 to 1.2 GHz.
//   split  few rows of A, where the weights' bytes bound the product and there are fewer tiles than SMs. Operands
//          change places: 128 rows of W are the TMEM lanes and NT rows of A the columns, so that a single token fills
//          the tensor core's wide side with weights. K is split over the CTAs of a cluster (at most 8), whose partial
//          sums meet in distributed shared memory in a fixed order (the same bits every time, no workspace). Lanes of
//          a warp write neighbouring columns of Y, so its stores are dense at any alignment: it also takes outputs
//          whose rows the pair kernel's vector accesses cannot address. Bound by memory and by its start and end: 32 x 28672,
//          K 4096, e4m3 23 us (5.2 TB/s); one row, 4096 x 4096, 6 us.
//
// The tensor core adds into its fp32 accumulator with truncation, an error that grows with the number of additions: up to 2^-24 of the
// result for each when the terms have one sign. 16-bit outputs take all of K in one accumulator: 1792 additions for K = 28672 of
// 16-bit operands, up to 1.1e-4 beside the output's own rounding of up to 4.9e-4 (fp16) or 3.9e-3 (bf16). For fp32 outputs the sum is
// cut into chunks of kChunkKb K-blocks whose accumulators the epilogue warps add in registers, rounding to nearest. The shorter the
// chunks, the sooner the issuing warp runs out of accumulators while the epilogue stores (16384 x 4096 x 1024 to fp32, 16 and 32
// additions: bf16 221K and 183K cycles, e4m3 143K and 127K). Products of codes are short and lose little: with 32 additions the outputs
// are within 1.0e-7 of 64 bits in the 2-norm up to K = 16384, 1.7e-7 with terms of one sign. 16-bit operands lose more (32 additions: fp16
// 6.5e-7, terms of one sign 2.5e-6) and keep 16: fp16 3.6e-7 and 1.2e-6, bf16 2.5e-7 and 3.8e-7. The sums of 256 columns are 64 a thread,
// more than its 96 registers hold beside the rest: the fp32 pair kernel spills (96 bytes stored, 528 loaded), part of its
// distance to the 16-bit one (bf16 139K, e4m3 102K cycles).
//
// Every mbarrier wait is bounded by a cycle budget, as in gemm_tcgen05.cu.
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "tc_common.cuh"
#include "typed.cuh"

namespace b200 {
using namespace tc;
namespace {

constexpr int kRowBytes = 128;                    // bytes of K of one K-block
constexpr int kTileBytes = 128 * kRowBytes;       // 128 rows of a K-block
constexpr int kMmasPerKb = 4;                     // 32 bytes of K per instruction
template <bool F8>
constexpr int kChunkKb = F8 ? 8 : 4;              // K-blocks of one in-core sum of fp32 outputs: 32 or 16 additions

struct ScaledParams {
  int64_t M, N;
  int num_kb;
  int num_m_tiles, num_n_tiles;
  uint32_t idesc;
  int a_scale_step, w_scale_step;
  int bias_type, activation;
  int vec;                                        // widest access to rows of Y and residual: 32, 16, 8 or 0 bytes
  int64_t ldy, ldr;
  const float *a_scale, *w_scale;
  const void *bias, *residual;
  void *Y;
  unsigned *status;
};

// Scales and bias may be what the kernel before this one in the stream has just written, and that kernel was still running when
// this one started: plain loads behind wait_previous(). The read-only path (__ldg) asks for data that nobody writes while the
// kernel exists; neither its cache nor the compiler is bound by the wait.
__device__ __forceinline__ float bias_at(const ScaledParams &p, int64_t n) {
  if (!p.bias) return 0.f;
  switch (p.bias_type) {
    case B200_TYPE_F32: return static_cast<const float *>(p.bias)[n];
    case B200_TYPE_F16: return __half2float(static_cast<const __half *>(p.bias)[n]);
    default: return __bfloat162float(static_cast<const __nv_bfloat16 *>(p.bias)[n]);
  }
}
__device__ __forceinline__ float w_scale_at(const ScaledParams &p, int64_t n) {
  return p.w_scale ? p.w_scale[n * p.w_scale_step] : 1.f;
}
__device__ __forceinline__ float a_scale_at(const ScaledParams &p, int64_t m) {
  return p.a_scale ? p.a_scale[m * p.a_scale_step] : 1.f;
}

// 32 bytes of a row of the residual, in one access or two
__device__ __forceinline__ void load32(const void *p, int vec, uint32_t *w) {
  if (vec == 32) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
  } else {
    const uint4 a = static_cast<const uint4 *>(p)[0], b = static_cast<const uint4 *>(p)[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
}

// Pair kernel: 64 bytes of outputs of one row, held by one thread (32 of a 16-bit type, 16 of fp32), to shared memory. sw,
// bs: scales and biases of these columns in shared memory (broadcast reads). r: the row's residual (RES) or null; cols: how
// many of the outputs exist (the others are computed from zeros and cut off by the store). row: the row's 64 bytes; flip: the
// exchange of its 16-byte pieces.
template <typename OUT>
constexpr int kBlockCols = 64 / (int)sizeof(OUT);
template <typename OUT, int ACT, bool RES>
__device__ __forceinline__ void finish_block_t(const ScaledParams &p, const float *v, float sa, const float *sw,
                                               const float *bs, const OUT *r, int cols, uint32_t row, uint32_t flip) {
  constexpr int B = kBlockCols<OUT>, C = 16 / (int)sizeof(OUT);  // outputs of the block, of 16 bytes
  const Pair sa2 = both(sa);
  uint32_t add[RES ? 16 : 1];
  if (RES) {
    if (r && cols >= B) {
      load32(r, p.vec, add);
      load32(r + B / 2, p.vec, add + 8);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if constexpr (sizeof(OUT) == 4) {
          add[i] = r && i < cols ? __float_as_uint(to_f32<OUT>(r[i])) : 0u;
        } else {
          add[i] = pack2<OUT>(r && 2 * i < cols ? to_f32<OUT>(r[2 * i]) : 0.f,
                              r && 2 * i + 1 < cols ? to_f32<OUT>(r[2 * i + 1]) : 0.f);
        }
      }
    }
  }
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < C; i += 4) {
      const int j = g * C + i;
      const float4 s = *reinterpret_cast<const float4 *>(sw + j), b = *reinterpret_cast<const float4 *>(bs + j);
      Pair lo = activate2_t<ACT>(fma2(Pair(v[j], v[j + 1]) * sa2, Pair(s.x, s.y), Pair(b.x, b.y)));
      Pair hi = activate2_t<ACT>(fma2(Pair(v[j + 2], v[j + 3]) * sa2, Pair(s.z, s.w), Pair(b.z, b.w)));
      float o[4];
      if (RES) {
        if constexpr (sizeof(OUT) == 4) {
          lo = lo + Pair(__uint_as_float(add[j]), __uint_as_float(add[j + 1]));
          hi = hi + Pair(__uint_as_float(add[j + 2]), __uint_as_float(add[j + 3]));
        } else {
          float x, y;
          unpack2<OUT>(add[j / 2], x, y);
          lo = lo + Pair(x, y);
          unpack2<OUT>(add[j / 2 + 1], x, y);
          hi = hi + Pair(x, y);
        }
      }
      lo.get(o[0], o[1]);
      hi.get(o[2], o[3]);
      if constexpr (sizeof(OUT) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __float_as_uint(o[k]);
      } else {
        w[i / 2] = pack2<OUT>(o[0], o[1]);
        w[i / 2 + 1] = pack2<OUT>(o[2], o[3]);
      }
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row + ((g ^ flip) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3])
                 : "memory");
  }
}
template <typename OUT, bool RES>
__device__ __forceinline__ void finish_block(const ScaledParams &p, const float *v, float sa, const float *sw,
                                             const float *bs, const OUT *r, int cols, uint32_t row, uint32_t flip) {
  switch (p.activation) {  // uniform for the launch
    case B200_ACT_RELU: finish_block_t<OUT, B200_ACT_RELU, RES>(p, v, sa, sw, bs, r, cols, row, flip); break;
    case B200_ACT_GELU: finish_block_t<OUT, B200_ACT_GELU, RES>(p, v, sa, sw, bs, r, cols, row, flip); break;
    case B200_ACT_GELU_TANH: finish_block_t<OUT, B200_ACT_GELU_TANH, RES>(p, v, sa, sw, bs, r, cols, row, flip); break;
    case B200_ACT_SILU: finish_block_t<OUT, B200_ACT_SILU, RES>(p, v, sa, sw, bs, r, cols, row, flip); break;
    default: finish_block_t<OUT, B200_ACT_NONE, RES>(p, v, sa, sw, bs, r, cols, row, flip);
  }
}

template <typename OUT>
__device__ __forceinline__ OUT ld_shared(uint32_t addr) {
  if constexpr (sizeof(OUT) == 4) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
  } else {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
    return *reinterpret_cast<const OUT *>(&v);
  }
}

// The loading and the issuing warp run converged, with one elected lane issuing: loop variables, addresses and
// descriptors then live in uniform registers. (With a single lane in a branch of its own each of them had to be moved there for
// every instruction: 170 clk per TMA load and 85 per MMA, against 128 clk that an MMA takes.)
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}
// mbar_wait by a converged warp; the answer is the same in all lanes.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int *abort_flag, unsigned *status,
                                               unsigned code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const long long t0 = clock64();
  for (uint32_t it = 1;; ++it) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((it & 0xffu) == 0) {
      const bool late = clock64() - t0 > kWaitCycleBudget;
      if (__any_sync(0xffffffffu, late || *abort_flag)) {
        if (late) {
          *abort_flag = 1;
          atomicOr(status, code);
        }
        return false;
      }
    }
  }
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }

__device__ __forceinline__ void teardown_after_abort(int aborted) {
  // copies may still be in flight after a wait gave up: leave them time before the shared memory goes
  if (aborted) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) __nanosleep(1000);
  }
}

// ---------------------------------------------------------------------------------------------
// pair
// ---------------------------------------------------------------------------------------------
template <int BN, typename OUT>
struct PairCfg {
  static constexpr bool kChunked = std::is_same<OUT, float>::value;
  static constexpr int kStageBytes = kTileBytes + BN / 2 * kRowBytes;  // 128 rows of A, half of the tile's rows of W
  // fp32 outputs leave in twice as many blocks: two under way take the place of the fifth stage
  static constexpr int kBlocks = kChunked || BN == 128 ? 2 : 1;
  static constexpr int kStages = BN == 128 ? 6 : kChunked ? 4 : 5;
  static constexpr int kAccs = kChunked ? 512 / BN : 2;    // accumulators
  static constexpr int kTmemCols = kAccs * BN;
  static constexpr int kColsPerWarp = BN / 4;              // four warps on each quarter of the lanes
  static constexpr int kEpilogueWarps = 16;
  static constexpr int kThreads = 32 * (2 + kEpilogueWarps);
  static constexpr int kStoreBytes = 32 * 64;              // a warp's block of outputs: 32 rows of 64 bytes
  static constexpr int kVectorBytes = kColsPerWarp * 2 * 4;  // a warp's scales and biases
  static constexpr int kSmemBytes =
      kStages * kStageBytes + kEpilogueWarps * (kBlocks * kStoreBytes + kVectorBytes) + 1024 + 256;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory of an SM");
};

// Tiles in groups of eight row tiles, column tiles across a group: the ~74 tiles in flight then share about 8 + 9 tile
// edges of operands in L2 instead of 1 + 74.
constexpr int kGroupM = 8;
__device__ __forceinline__ void tile_at(const ScaledParams &p, int64_t tile, int &m_t, int &n_t) {
  const int64_t per_group = (int64_t)kGroupM * p.num_n_tiles;
  const int g = (int)(tile / per_group);
  const int64_t in = tile - g * per_group;
  const int first = g * kGroupM, rows = min(kGroupM, p.num_m_tiles - first);
  n_t = (int)(in / rows);
  m_t = first + (int)(in - (int64_t)n_t * rows);
}

// RAGGED: rows of Y end inside 16 bytes (they are further apart than they are long). A TMA store is cut off at the tensor's edge in
// pieces of 16 bytes, so it would write behind such an end: there each thread stores the last block of its row itself, value
// by value. (A variant of its own: with the branch in every instance 16384 x 4096 x 1024 e4m3 took 76 us, without 68.)
template <bool F8, typename OUT, int BN, bool RAGGED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg<BN, OUT>::kThreads, 1)
scaled_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                   const __grid_constant__ CUtensorMap map_y, const ScaledParams p) {
  using C = PairCfg<BN, OUT>;
  constexpr bool kChunked = C::kChunked;
  constexpr int kStages = C::kStages;
  constexpr int kKbElems = F8 ? 128 : 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *store_smem = smem + kStages * C::kStageBytes;
  uint8_t *vector_smem = store_smem + C::kEpilogueWarps * C::kBlocks * C::kStoreBytes;
  uint64_t *bars = reinterpret_cast<uint64_t *>(vector_smem + C::kEpilogueWarps * C::kVectorBytes);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_tfull = bar_empty + 8 * kStages;
  const uint32_t bar_tempty = bar_tfull + 8 * C::kAccs;
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t rank = cluster_ctarank();
  const int64_t pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int64_t num_tiles = (int64_t)p.num_m_tiles * p.num_n_tiles;

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_w);
    prefetch_map(&map_y);
    s_abort = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);   // even CTA: its expect_tx for the bytes of both
      mbar_init(bar_empty + 8 * s, 1);  // each CTA: the issuer commits to both
    }
    for (int a = 0; a < C::kAccs; ++a) {
      mbar_init(bar_tfull + 8 * a, 1);                       // each CTA: the issuer commits to both
      mbar_init(bar_tempty + 8 * a, 2 * C::kEpilogueWarps);  // even CTA: one arrival per epilogue warp of both
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&s_tmem_base), C::kTmemCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  let_next_start();
  wait_previous();
  const uint32_t tmem_base = s_tmem_base;
  volatile int *abort_flag = &s_abort;

  if (warp == 0) {
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    const uint32_t full_pair0 = map_to_cta(bar_full, 0);
    for (int64_t tile = pair; tile < num_tiles && ok; tile += num_pairs) {
      int m_t, n_t;
      tile_at(p, tile, m_t, n_t);
      const int row_a = m_t * 256 + (int)rank * 128;
      const int row_w = n_t * BN + (int)rank * (BN / 2);
      for (int kb = 0; kb < p.num_kb; ++kb) {
        if (!(ok = mbar_wait_warp(bar_empty + 8 * s, ph ^ 1, abort_flag, p.status, 1u))) break;
        // one expect_tx, by the even CTA, for the bytes of both: its partner's can arrive only after the stage's previous
        // phase is complete, because they too wait for the commit that follows it
        const uint32_t a_dst = smem_base + s * C::kStageBytes, w_dst = a_dst + kTileBytes;
        if (elect_one()) {
          if (rank == 0) {
            mbar_expect_tx(bar_full + 8 * s, 2 * C::kStageBytes);
            tma_load_2d(a_dst, &map_a, bar_full + 8 * s, kb * kKbElems, row_a);
            tma_load_2d(w_dst, &map_w, bar_full + 8 * s, kb * kKbElems, row_w);
          } else {
            tma_load_2d_pair(a_dst, &map_a, full_pair0 + 8 * s, kb * kKbElems, row_a);
            tma_load_2d_pair(w_dst, &map_w, full_pair0 + 8 * s, kb * kKbElems, row_w);
          }
        }
        __syncwarp();
        if (++s == kStages) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint64_t a_desc0 = make_smem_desc(smem_base, 16, 1024, kLayoutSw128);
      const uint64_t w_desc0 = make_smem_desc(smem_base + kTileBytes, 16, 1024, kLayoutSw128);
      const uint32_t idesc = p.idesc;
      const int chunk = kChunked ? kChunkKb<F8> : p.num_kb;
      int s = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int64_t tile = pair; tile < num_tiles && ok; tile += num_pairs) {
        for (int kb0 = 0; kb0 < p.num_kb && ok; kb0 += chunk) {
          if (!(ok = mbar_wait_warp(bar_tempty + 8 * acc, acc_ph ^ 1, abort_flag, p.status, 2u))) break;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
          const int kb_end = min(kb0 + chunk, p.num_kb);
          for (int kb = kb0; kb < kb_end; ++kb) {
            if (!(ok = mbar_wait_warp(bar_full + 8 * s, ph, abort_flag, p.status, 4u))) break;
            tc_fence_after();
            const uint64_t a_d = a_desc0 + (uint32_t)s * (C::kStageBytes >> 4);
            const uint64_t w_d = w_desc0 + (uint32_t)s * (C::kStageBytes >> 4);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kMmasPerKb; ++k) {
                const uint32_t accumulate = (k > 0 || kb > kb0) ? 1u : 0u;
                if (F8) umma_f8_pair(d_tmem, a_d + 2 * k, w_d + 2 * k, idesc, accumulate);
                else umma_bf16_pair(d_tmem, a_d + 2 * k, w_d + 2 * k, idesc, accumulate);
              }
              umma_commit_pair_both(bar_empty + 8 * s, 3);
              if (kb + 1 == kb_end) umma_commit_pair_both(bar_tfull + 8 * acc, 3);
            }
            __syncwarp();
            if (++s == kStages) { s = 0; ph ^= 1; }
          }
          if (++acc == C::kAccs) { acc = 0; acc_ph ^= 1; }
        }
      }
    }
  } else {
    const int ew = warp - 2, quarter = warp & 3;
    const int col0 = (ew >> 2) * C::kColsPerWarp;
    float *sw = reinterpret_cast<float *>(vector_smem + ew * C::kVectorBytes), *bs = sw + C::kColsPerWarp;
    // the block of outputs on its way to memory: rows of 64 bytes whose 16-byte pieces are exchanged as the 64-byte
    // swizzle of map_y has them, so that a warp's 16-byte accesses meet no bank twice
    const uint32_t blocks = smem_u32(store_smem + ew * C::kBlocks * C::kStoreBytes);
    const uint32_t flip = (lane >> 1) & 3;
    int turn = 0;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + col0;
    const int chunks = kChunked ? (p.num_kb + kChunkKb<F8> - 1) / kChunkKb<F8> : 1;
    constexpr int B = kBlockCols<OUT>;
    int acc = 0;
    uint32_t acc_ph = 0;
    bool ok = true;
    for (int64_t tile = pair; tile < num_tiles && ok; tile += num_pairs) {
      int m_t, n_t;
      tile_at(p, tile, m_t, n_t);
      const int64_t m0 = (int64_t)m_t * 256 + (int)rank * 128 + quarter * 32, m = m0 + lane;
      const int64_t n0 = (int64_t)n_t * BN + col0;
      // this warp's columns: scales and biases to shared memory, while the MMAs run
      __syncwarp();
      for (int c = lane; c < C::kColsPerWarp; c += 32) {
        const bool in = n0 + c < p.N;
        sw[c] = in ? w_scale_at(p, n0 + c) : 0.f;
        bs[c] = in ? bias_at(p, n0 + c) : 0.f;
      }
      __syncwarp();
      const bool row_in = m < p.M;
      const float sa = row_in ? a_scale_at(p, m) : 0.f;
      const OUT *r = p.residual && row_in ? static_cast<const OUT *>(p.residual) + m * p.ldr + n0 : nullptr;
      // 64 bytes of each of the warp's rows, from the accumulators v of columns c..c+B-1
      auto emit = [&](const float *v, int c) {
        const int64_t left = p.N - n0 - c;
        if (left <= 0 || m0 >= p.M) return;  // uniform
        const int cols = left < B ? (int)left : B;
        const uint32_t block = blocks + turn * C::kStoreBytes, my_row = block + lane * 64;
        if (C::kBlocks > 1) turn ^= 1;
        if (lane == 0) bulk_wait_read<C::kBlocks - 1>();  // what was in this block has left
        __syncwarp();
        if (p.residual) finish_block<OUT, true>(p, v, sa, sw + c, bs + c, r ? r + c : nullptr, cols, my_row, flip);
        else finish_block<OUT, false>(p, v, sa, sw + c, bs + c, nullptr, cols, my_row, flip);
        if (RAGGED && cols < B) {  // uniform
          if (m0 + lane < p.M) {
            OUT *y = static_cast<OUT *>(p.Y) + (m0 + lane) * p.ldy + n0 + c;
#pragma unroll 1
            for (int i = 0; i < cols; ++i) {
              const uint32_t piece = (uint32_t)i * sizeof(OUT) / 16, in = (uint32_t)i * sizeof(OUT) % 16;
              y[i] = ld_shared<OUT>(my_row + ((piece ^ flip) << 4) + in);
            }
          }
          if (lane == 0) bulk_commit();  // an empty group: the wait above counts one for each block
          __syncwarp();
          return;
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&map_y, block, (int)(n0 + c), (int)m0);
          bulk_commit();
        }
      };
      if (kChunked) {
        float sum[C::kColsPerWarp] = {};
        for (int ch = 0; ch < chunks; ++ch) {
          if (!(ok = mbar_wait_warp(bar_tfull + 8 * acc, acc_ph, abort_flag, p.status, 8u))) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < C::kColsPerWarp; c += 16) {
            uint32_t t[16];
            tmem_ld16(lane_addr + (uint32_t)(acc * BN + c), t);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) sum[c + j] += __uint_as_float(t[j]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(bar_tempty + 8 * acc, 0));
          if (++acc == C::kAccs) { acc = 0; acc_ph ^= 1; }
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < C::kColsPerWarp; c += B) emit(sum + c, c);
      } else {
        if (!(ok = mbar_wait_warp(bar_tfull + 8 * acc, acc_ph, abort_flag, p.status, 8u))) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < C::kColsPerWarp; c += 32) {
          uint32_t t[32];
          float v[32];
          tmem_ld32(lane_addr + (uint32_t)(acc * BN + c), t);
          tmem_ld_wait();
          if (c + 32 >= C::kColsPerWarp) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(bar_tempty + 8 * acc, 0));
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(t[j]);
          emit(v, c);
        }
        if (++acc == C::kAccs) { acc = 0; acc_ph ^= 1; }
      }
    }
    if (lane == 0) bulk_wait();
  }

  // neither CTA may leave while its partner can still signal its barriers or read its shared memory
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  teardown_after_abort(s_abort);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, C::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------
// split
// ---------------------------------------------------------------------------------------------
template <int NT, bool CHUNKED>
struct SplitCfg {
  static constexpr int kStageBytes = kTileBytes + NT * kRowBytes;
  // two CTAs on an SM (one for NT = 256), so that one's start and end run under the other's loads
  static constexpr int kStages = NT == 256 ? 4 : NT == 128 ? 3 : NT == 64 ? 4 : NT == 32 ? 5 : 6;
  static constexpr int kCtasPerSm = NT == 256 ? 1 : 2;
  static constexpr int kWarpsPerQuarter = NT <= 64 ? 1 : NT / 64;
  static constexpr int kColsPerWarp = NT / kWarpsPerQuarter;   // at most 64 sums in a thread's registers
  static constexpr int kEpilogueWarps = 4 * kWarpsPerQuarter;
  static constexpr int kThreads = 32 * (2 + kEpilogueWarps);
  static constexpr int kAccCols = NT < 32 ? 32 : NT;
  static constexpr int kTmemCols = CHUNKED ? 2 * kAccCols : kAccCols;
  static constexpr int kSmemBytes = kStages * kStageBytes + 1024 + 256;
  static_assert(NT * 128 * 4 <= kStages * kStageBytes, "partial sums take the place of the stages");
};

// Loads from the shared memory of a CTA of the cluster, after a cluster barrier. Not ordered against global accesses, so
// that those of several rows are in flight together.
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// Four neighbouring outputs in one access (8 bytes of a 16-bit type, 16 of fp32).
template <typename OUT>
__device__ __forceinline__ void load4(const OUT *p, float (&v)[4]) {
  if constexpr (sizeof(OUT) == 4) {
    const float4 f = *reinterpret_cast<const float4 *>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    unpack2<OUT>(u.x, v[0], v[1]);
    unpack2<OUT>(u.y, v[2], v[3]);
  }
}
template <typename OUT>
__device__ __forceinline__ void store4(OUT *p, const float (&v)[4]) {
  if constexpr (sizeof(OUT) == 4) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3]));
}

template <typename OUT, int ACT>
__device__ __forceinline__ void epilogue4_t(const float4 &v, float sa, const float (&sw)[4], const float (&bs)[4],
                                            const float (&add)[4], float (&o)[4]) {
  const Pair sa2 = both(sa);
  const Pair lo = activate2_t<ACT>(fma2(Pair(v.x, v.y) * sa2, Pair(sw[0], sw[1]), Pair(bs[0], bs[1])));
  const Pair hi = activate2_t<ACT>(fma2(Pair(v.z, v.w) * sa2, Pair(sw[2], sw[3]), Pair(bs[2], bs[3])));
  (lo + Pair(add[0], add[1])).get(o[0], o[1]);
  (hi + Pair(add[2], add[3])).get(o[2], o[3]);
}

// Outputs of this CTA: its share of the tile's rows of A (rank, rank + RANKS, ...). A warp takes a row of A at a time and
// the tile's 128 columns of Y: VEC: lane l has columns 4l..4l+3 and one access; otherwise columns l, l+32, l+64, l+96
// and dense scalar accesses. Eight partial sums (4 to 1 rows) are in flight together.
template <typename OUT, bool VEC, int RANKS>
__device__ __forceinline__ void finish_split_t(const ScaledParams &p, uint32_t partial, int rank, int warp, int warps,
                                               int lane, int64_t m0, int rows, int64_t n0, const float (&sw)[4],
                                               const float (&bs)[4]) {
  constexpr int R = RANKS == 8 ? 1 : RANKS == 4 ? 2 : 4;
  const int64_t left = p.N - n0;
  auto col = [&](int k) { return VEC ? 4 * lane + k : lane + 32 * k; };
  OUT *y = static_cast<OUT *>(p.Y) + m0 * p.ldy + n0;
  const OUT *r = p.residual ? static_cast<const OUT *>(p.residual) + m0 * p.ldr + n0 : nullptr;
  const bool whole = VEC && col(3) < left;
  uint32_t base[RANKS];
#pragma unroll
  for (int s = 0; s < RANKS; ++s) base[s] = map_to_cta(partial, s);
  for (int j0 = warp; rank + RANKS * j0 < rows; j0 += R * warps) {
    float4 part[R][RANKS];
    float add[R][4], sa[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int t = rank + RANKS * (j0 + i * warps);
      if (t >= rows) break;
#pragma unroll
      for (int s = 0; s < RANKS; ++s) {
        if (VEC) {
          part[i][s] = ld_cluster4(base[s] + t * 512 + lane * 16);
        } else {
          const uint32_t q = base[s] + t * 512 + lane * 4;
          part[i][s] = make_float4(ld_cluster(q), ld_cluster(q + 128), ld_cluster(q + 256), ld_cluster(q + 384));
        }
      }
      sa[i] = a_scale_at(p, m0 + t);
#pragma unroll
      for (int k = 0; k < 4; ++k) add[i][k] = 0.f;
      if (r) {
        if (whole) {
          load4<OUT>(r + t * p.ldr + 4 * lane, add[i]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (col(k) < left) add[i][k] = to_f32<OUT>(r[t * p.ldr + col(k)]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int t = rank + RANKS * (j0 + i * warps);
      if (t >= rows) break;
      float4 v = part[i][0];
#pragma unroll
      for (int s = 1; s < RANKS; ++s) {
        v.x += part[i][s].x; v.y += part[i][s].y; v.z += part[i][s].z; v.w += part[i][s].w;
      }
      float o[4];
      switch (p.activation) {  // uniform for the launch
        case B200_ACT_RELU: epilogue4_t<OUT, B200_ACT_RELU>(v, sa[i], sw, bs, add[i], o); break;
        case B200_ACT_GELU: epilogue4_t<OUT, B200_ACT_GELU>(v, sa[i], sw, bs, add[i], o); break;
        case B200_ACT_GELU_TANH: epilogue4_t<OUT, B200_ACT_GELU_TANH>(v, sa[i], sw, bs, add[i], o); break;
        case B200_ACT_SILU: epilogue4_t<OUT, B200_ACT_SILU>(v, sa[i], sw, bs, add[i], o); break;
        default: epilogue4_t<OUT, B200_ACT_NONE>(v, sa[i], sw, bs, add[i], o);
      }
      if (whole) {
        store4<OUT>(y + t * p.ldy + 4 * lane, o);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (col(k) < left) y[t * p.ldy + col(k)] = from_f32<OUT>(o[k]);
      }
    }
  }
}
template <typename OUT, bool VEC>
__device__ __forceinline__ void finish_split(const ScaledParams &p, uint32_t partial, int ranks, int rank, int warp,
                                             int warps, int lane, int64_t m0, int rows, int64_t n0, const float (&sw)[4],
                                             const float (&bs)[4]) {
  switch (ranks) {  // uniform for the launch
    case 1: finish_split_t<OUT, VEC, 1>(p, partial, rank, warp, warps, lane, m0, rows, n0, sw, bs); break;
    case 2: finish_split_t<OUT, VEC, 2>(p, partial, rank, warp, warps, lane, m0, rows, n0, sw, bs); break;
    case 4: finish_split_t<OUT, VEC, 4>(p, partial, rank, warp, warps, lane, m0, rows, n0, sw, bs); break;
    default: finish_split_t<OUT, VEC, 8>(p, partial, rank, warp, warps, lane, m0, rows, n0, sw, bs);
  }
}

template <bool F8, typename OUT, int NT>
__global__ void __launch_bounds__(SplitCfg<NT, std::is_same<OUT, float>::value>::kThreads,
                                  SplitCfg<NT, std::is_same<OUT, float>::value>::kCtasPerSm)
scaled_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                    const ScaledParams p, const int ranks) {
  constexpr bool kChunked = std::is_same<OUT, float>::value;
  using C = SplitCfg<NT, kChunked>;
  constexpr int kStages = C::kStages;
  constexpr int kKbElems = F8 ? 128 : 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kStages * C::kStageBytes);
  const uint32_t bar_full = smem_u32(bars);
  const uint32_t bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_tfull = bar_empty + 8 * kStages;
  const uint32_t bar_tempty = bar_tfull + 16;
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t smem_base = smem_u32(smem);
  const int rank = (int)cluster_ctarank();
  const int64_t tile = blockIdx.x / ranks;
  const int n_t = (int)(tile / p.num_m_tiles), m_t = (int)(tile - (int64_t)n_t * p.num_m_tiles);
  const int kb_begin = (int)((int64_t)p.num_kb * rank / ranks), kb_end = (int)((int64_t)p.num_kb * (rank + 1) / ranks);

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_w);
    s_abort = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_tfull + 8 * a, 1);
      mbar_init(bar_tempty + 8 * a, C::kEpilogueWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&s_tmem_base), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_next_start();
  wait_previous();
  const uint32_t tmem_base = s_tmem_base;
  volatile int *abort_flag = &s_abort;
  const int64_t m0 = (int64_t)m_t * NT, n0 = (int64_t)n_t * 128;
  const bool vec = p.vec >= 4 * (int)sizeof(OUT);
  float sw[4], bs[4];  // scales and biases of this lane's columns of Y, loaded while the operands arrive

  if (warp == 0) {
    int s = 0;
    uint32_t ph = 0;
    for (int kb = kb_begin; kb < kb_end; ++kb) {
      if (!mbar_wait_warp(bar_empty + 8 * s, ph ^ 1, abort_flag, p.status, 1u)) break;
      const uint32_t stage = smem_base + s * C::kStageBytes;
      if (elect_one()) {
        mbar_expect_tx(bar_full + 8 * s, C::kStageBytes);
        tma_load_2d(stage, &map_w, bar_full + 8 * s, kb * kKbElems, n_t * 128);
        tma_load_2d(stage + kTileBytes, &map_a, bar_full + 8 * s, kb * kKbElems, m_t * NT);
      }
      __syncwarp();
      if (++s == kStages) { s = 0; ph ^= 1; }
    }
  } else if (warp == 1) {
    const uint64_t w_desc0 = make_smem_desc(smem_base, 16, 1024, kLayoutSw128);
    const uint64_t a_desc0 = make_smem_desc(smem_base + kTileBytes, 16, 1024, kLayoutSw128);
    const uint32_t idesc = p.idesc;
    const int chunk = kChunked ? kChunkKb<F8> : p.num_kb;
    int s = 0, acc = 0;
    uint32_t ph = 0, acc_ph = 0;
    bool ok = true;
    for (int kb0 = kb_begin; kb0 < kb_end && ok; kb0 += chunk) {
      if (!(ok = mbar_wait_warp(bar_tempty + 8 * acc, acc_ph ^ 1, abort_flag, p.status, 2u))) break;
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + (uint32_t)(acc * C::kAccCols);
      const int end = min(kb0 + chunk, kb_end);
      for (int kb = kb0; kb < end; ++kb) {
        if (!(ok = mbar_wait_warp(bar_full + 8 * s, ph, abort_flag, p.status, 4u))) break;
        tc_fence_after();
        const uint64_t w_d = w_desc0 + (uint32_t)s * (C::kStageBytes >> 4);
        const uint64_t a_d = a_desc0 + (uint32_t)s * (C::kStageBytes >> 4);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kMmasPerKb; ++k) {
            const uint32_t accumulate = (k > 0 || kb > kb0) ? 1u : 0u;
            if (F8) umma_f8(d_tmem, w_d + 2 * k, a_d + 2 * k, idesc, accumulate);
            else umma_bf16(d_tmem, w_d + 2 * k, a_d + 2 * k, idesc, accumulate);
          }
          umma_commit(bar_empty + 8 * s);
          if (kb + 1 == end) umma_commit(bar_tfull + 8 * acc);
        }
        __syncwarp();
        if (++s == kStages) { s = 0; ph ^= 1; }
      }
      if (kChunked && ++acc == 2) { acc = 0; acc_ph ^= 1; }
    }
  } else {
    const int ew = warp - 2, quarter = warp & 3;
    const int col0 = (ew >> 2) * C::kColsPerWarp;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + col0;
    const int chunks = kChunked ? (kb_end - kb_begin + kChunkKb<F8> - 1) / kChunkKb<F8> : 1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t n = n0 + (vec ? 4 * lane + k : lane + 32 * k);
      sw[k] = n < p.N ? w_scale_at(p, n) : 0.f;
      bs[k] = n < p.N ? bias_at(p, n) : 0.f;
    }
    float sum[C::kColsPerWarp] = {};
    int acc = 0;
    uint32_t acc_ph = 0;
    bool ok = true;
    for (int ch = 0; ch < chunks; ++ch) {
      if (!(ok = mbar_wait_warp(bar_tfull + 8 * acc, acc_ph, abort_flag, p.status, 8u))) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < C::kColsPerWarp; c += 16) {
        uint32_t t[16];
        tmem_ld16(lane_addr + (uint32_t)(acc * C::kAccCols + c), t);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[c + j] += __uint_as_float(t[j]);
      }
      if (kChunked) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_tempty + 8 * acc);
        if (++acc == 2) { acc = 0; acc_ph ^= 1; }
      }
    }
    if (ok) {
      // the last accumulator is complete, so every load has landed and every MMA has read its stage: the
      // stages' memory now takes the partial sums, [row of A][row of W]
      float *partial = reinterpret_cast<float *>(smem) + quarter * 32 + lane;
#pragma unroll
      for (int j = 0; j < C::kColsPerWarp; ++j) partial[(col0 + j) * 128] = sum[j];
    }
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync_all();  // every CTA's partial sums are in place
  if (warp >= 2) {
    const int rows = (int)min((int64_t)NT, p.M - m0);
    if (vec) finish_split<OUT, true>(p, smem_base, ranks, rank, warp - 2, C::kEpilogueWarps, lane, m0, rows, n0, sw, bs);
    else finish_split<OUT, false>(p, smem_base, ranks, rank, warp - 2, C::kEpilogueWarps, lane, m0, rows, n0, sw, bs);
  }
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while another reads its partial sums
  teardown_after_abort(s_abort);
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
template <typename Kernel>
int raise_smem(Kernel kern, int bytes, std::atomic<uint64_t> &done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(B200_ECUDA, "gemm_scaled: bad device");
  if (done.load(std::memory_order_relaxed) >> dev & 1) return B200_OK;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return fail(B200_ECUDA, "gemm_scaled: cannot set dynamic shared memory to %d", bytes);
  done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return B200_OK;
}

struct Plan {
  bool pair;
  int cols;   // pair: BN; split: NT
  int ranks;  // split: CTAs over which K is split
};

struct Operands {
  const void *A, *W;
  int64_t K, a_pitch, w_pitch;
  int type, y_type;
};

template <bool F8, typename OUT, int BN, bool RAGGED>
int launch_pair(cudaStream_t st, const Operands &o, ScaledParams &p) {
  using C = PairCfg<BN, OUT>;
  auto kern = scaled_pair_kernel<F8, OUT, BN, RAGGED>;
  static std::atomic<uint64_t> smem_set{0};
  if (int rc = raise_smem(kern, C::kSmemBytes, smem_set)) return rc;
  // the clusters the device holds at once: a persistent grid must not exceed them (per device, never changes)
  static std::atomic<int> max_pairs[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(B200_ECUDA, "gemm_scaled: bad device");
  if (max_pairs[dev].load(std::memory_order_relaxed) == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kNumSMs, 1, 1);
    cfg.blockDim = dim3(C::kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1)
      return fail(B200_ECUDA, "gemm_scaled: cudaOccupancyMaxActiveClusters failed");
    max_pairs[dev].store(n, std::memory_order_relaxed);
  }
  CUtensorMap ma, mw, my;
  if (int rc = encode_map_2d(&ma, o.A, o.type, o.K, p.M, o.a_pitch, F8 ? 128 : 64, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = encode_map_2d(&mw, o.W, o.type, o.K, p.N, o.w_pitch, F8 ? 128 : 64, BN / 2, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  const int64_t y_pitch = p.M > 1 ? p.ldy * (int64_t)sizeof(OUT) : (p.N * (int64_t)sizeof(OUT) + 15) / 16 * 16;
  if (int rc = encode_map_2d(&my, p.Y, o.y_type, p.N, p.M, y_pitch, kBlockCols<OUT>, 32, CU_TENSOR_MAP_SWIZZLE_64B)) return rc;
  p.num_m_tiles = (int)((p.M + 255) / 256);
  p.num_n_tiles = (int)((p.N + BN - 1) / BN);
  p.idesc |= (uint32_t)(BN >> 3) << 17 | (uint32_t)(256 >> 4) << 24;
  const int64_t tiles = (int64_t)p.num_m_tiles * p.num_n_tiles, cap = max_pairs[dev].load(std::memory_order_relaxed);
  return launch_overlapped("gemm_scaled(pair)", kern, (unsigned)(2 * (tiles < cap ? tiles : cap)), C::kThreads, C::kSmemBytes, st, 1,
                           ma, mw, my, p);
}

template <bool F8, typename OUT, int NT>
int launch_split(cudaStream_t st, const Operands &o, ScaledParams &p, int ranks) {
  using C = SplitCfg<NT, std::is_same<OUT, float>::value>;
  auto kern = scaled_split_kernel<F8, OUT, NT>;
  static std::atomic<uint64_t> smem_set{0};
  if (int rc = raise_smem(kern, C::kSmemBytes, smem_set)) return rc;
  CUtensorMap ma, mw;
  if (int rc = encode_map_2d(&ma, o.A, o.type, o.K, p.M, o.a_pitch, F8 ? 128 : 64, NT, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = encode_map_2d(&mw, o.W, o.type, o.K, p.N, o.w_pitch, F8 ? 128 : 64, 128, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  p.num_m_tiles = (int)((p.M + NT - 1) / NT);
  p.num_n_tiles = (int)((p.N + 127) / 128);
  p.idesc |= (uint32_t)(NT >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
  const int64_t ctas = (int64_t)p.num_m_tiles * p.num_n_tiles * ranks;
  if (ctas > 0x7fffffffLL) return fail(B200_EUNSUPPORTED, "gemm_scaled: too many tiles");
  return launch_overlapped("gemm_scaled(split)", kern, (unsigned)ctas, C::kThreads, C::kSmemBytes, st, (unsigned)ranks, ma, mw, p,
                           ranks);
}

template <bool F8, typename OUT>
int launch_plan(cudaStream_t st, const Operands &o, ScaledParams &p, const Plan &plan) {
  if (plan.pair) {
    if (p.N * (int64_t)sizeof(OUT) % 16 == 0)
      return plan.cols == 256 ? launch_pair<F8, OUT, 256, false>(st, o, p) : launch_pair<F8, OUT, 128, false>(st, o, p);
    return plan.cols == 256 ? launch_pair<F8, OUT, 256, true>(st, o, p) : launch_pair<F8, OUT, 128, true>(st, o, p);
  }
  switch (plan.cols) {
    case 16: return launch_split<F8, OUT, 16>(st, o, p, plan.ranks);
    case 32: return launch_split<F8, OUT, 32>(st, o, p, plan.ranks);
    case 64: return launch_split<F8, OUT, 64>(st, o, p, plan.ranks);
    case 128: return launch_split<F8, OUT, 128>(st, o, p, plan.ranks);
    default: return launch_split<F8, OUT, 256>(st, o, p, plan.ranks);
  }
}

int type_bytes(int type) { return type == B200_TYPE_F32 ? 4 : type == B200_TYPE_E4M3 ? 1 : 2; }

// Which kernel, tile and split: the one with the smallest estimated time. The estimates (in microseconds) have the form that
// the kernels have: a start, K-blocks one after the other at a rate set by the tensor core or by the bytes that an SM
// takes in, an epilogue. Their constants are fitted to 660 timings over 59 products (1 to 16384 rows, 64 to 28672
// columns, K 64 to 14336, e4m3 and bf16); the plan taken is on average 3 % slower than the best of all plans, at worst 26 %.
//   pair   tiles of 256 x cols on 74 pairs. 4096 columns, K 4096, e4m3: 128 rows 10.7 us (split: 9.3), 256 rows 10.6 (11.8),
//          512 rows 12.3 (15.1), 1024 rows 18.2 (22.7).
//   split  tiles of 128 columns of Y and cols rows of A, each on `ranks` CTAs; two CTAs share an SM. One row, 4096 x 4096:
//          4 ranks 5.9 us, 1 rank 9.1; 28672 columns (224 tiles): 1 rank 22, 4 ranks 30.
double pair_us(int64_t M, int64_t N, int64_t kb, int cols) {
  const int64_t tiles = (M + 255) / 256 * ((N + cols - 1) / cols);
  const double waves = (double)((tiles + kNumSMs / 2 - 1) / (kNumSMs / 2));
  const double block = cols == 256 ? 0.30 : 0.227, epilogue = 5.3 * cols / 256;
  const double mmas = waves * (double)kb * block + epilogue, epilogues = waves * epilogue;
  return 2.4 + (mmas > epilogues ? mmas : epilogues);
}
double split_us(int64_t M, int64_t N, int64_t kb, int cols, int ranks) {
  const int64_t ctas = (M + cols - 1) / cols * ((N + 127) / 128) * ranks, sms = cols == 256 ? kNumSMs : 2 * kNumSMs;
  const double waves = (double)((ctas + kNumSMs - 1) / kNumSMs), rounds = (double)((ctas + sms - 1) / sms);
  const double bytes = (16 + cols / 8) * 0.0086, mmas = cols * 0.0017;  // of one K-block
  return 0.3 + waves * (double)((kb + ranks - 1) / ranks) * (bytes > mmas ? bytes : mmas) + rounds * (4.3 + 0.026 * cols / ranks) +
         (ranks == 8 ? 2.5 : ranks == 4 ? 1.6 : ranks == 2 ? 0.8 : 0.0);
}

Plan choose(const b200_gemm_scaled_desc &d, bool vector_rows) {
  const int64_t kb = (d.K * type_bytes(d.type) + kRowBytes - 1) / kRowBytes;
  Plan best = {false, 16, 1};
  double best_us = 1e30;
  for (int cols = 16; cols <= 256; cols *= 2) {
    if (cols > 16 && cols >= 2 * d.M) break;
    for (int ranks = 1; ranks <= (cols == 256 ? 4 : 8) && (ranks == 1 || 2 * ranks <= kb); ranks *= 2) {
      const double us = split_us(d.M, d.N, kb, cols, ranks);
      if (us < best_us) { best_us = us; best = Plan{false, cols, ranks}; }
    }
  }
  for (int cols = 128; vector_rows && d.M > 32 && cols <= 256; cols *= 2) {
    const double us = pair_us(d.M, d.N, kb, cols);
    if (us < best_us) { best_us = us; best = Plan{true, cols, 1}; }
  }
  return best;
}

int run_plan(cudaStream_t st, const b200_gemm_scaled_desc &d, const Plan &plan, int vec, const void *A, const void *W,
             const float *a_scale, const float *w_scale, const void *bias, const void *residual, void *Y) {
  const int b = type_bytes(d.type);
  ScaledParams p = {};
  p.M = d.M;
  p.N = d.N;
  p.num_kb = (int)((d.K * b + kRowBytes - 1) / kRowBytes);
  p.idesc = d.type == B200_TYPE_BF16 ? make_idesc_bf16(0, 0) : make_idesc_fp16_or_e4m3(0, 0);
  p.a_scale_step = d.a_scale_step;
  p.w_scale_step = d.w_scale_step;
  p.bias_type = d.bias_type;
  p.activation = d.activation;
  p.vec = vec;
  p.ldy = d.ldy;
  p.ldr = d.ldr;
  p.a_scale = a_scale;
  p.w_scale = w_scale;
  p.bias = bias;
  p.residual = residual;
  p.Y = Y;
  p.status = device_status_ptr();
  if (!p.status) return fail(B200_ECUDA, "gemm_scaled: device status word unavailable");
  const Operands o = {A, W, d.K, d.lda * b, d.ldw * b, d.type, d.y_type};
  const bool f8 = d.type == B200_TYPE_E4M3;
  switch (d.y_type) {
    case B200_TYPE_F32: return f8 ? launch_plan<true, float>(st, o, p, plan) : launch_plan<false, float>(st, o, p, plan);
    case B200_TYPE_F16: return f8 ? launch_plan<true, __half>(st, o, p, plan) : launch_plan<false, __half>(st, o, p, plan);
    default:
      return f8 ? launch_plan<true, __nv_bfloat16>(st, o, p, plan) : launch_plan<false, __nv_bfloat16>(st, o, p, plan);
  }
}

// Widest access with which every row of `q` can be read or written: 32, 16, 8 or fewer (0) bytes.
int row_access(const void *q, int64_t rows, int64_t ld, int bytes) {
  const uint64_t bits = reinterpret_cast<uintptr_t>(q) | (rows > 1 ? (uint64_t)(ld * bytes) : 0);
  return bits % 32 == 0 ? 32 : bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : 0;
}

// The same for a call's outputs and residual together.
int output_access(const b200_gemm_scaled_desc &d, const void *residual, const void *Y) {
  const int vec = row_access(Y, d.M, d.ldy, type_bytes(d.y_type));
  return residual ? min(vec, row_access(residual, d.M, d.ldr, type_bytes(d.y_type))) : vec;
}

bool is_float(int type) { return type == B200_TYPE_F32 || type == B200_TYPE_F16 || type == B200_TYPE_BF16; }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" B200_API int b200_gemm_scaled(void *stream, const b200_gemm_scaled_desc *desc, const void *A, const void *W,
                                         const float *a_scale, const float *w_scale, const void *bias,
                                         const void *residual, void *Y) {
  if (!desc) return fail(B200_EINVAL, "gemm_scaled: null descriptor");
  const b200_gemm_scaled_desc &d = *desc;
  if (d.M < 0 || d.N < 0) return fail(B200_EINVAL, "gemm_scaled: negative extent");
  if (d.K < 1) return fail(B200_EINVAL, "gemm_scaled: K must be at least 1");
  if (d.type != B200_TYPE_E4M3 && d.type != B200_TYPE_F16 && d.type != B200_TYPE_BF16)
    return fail(B200_EINVAL, "gemm_scaled: operands are e4m3, fp16 or bf16, not type %d", d.type);
  if (!is_float(d.y_type)) return fail(B200_EINVAL, "gemm_scaled: unknown output type %d", d.y_type);
  if (bias && !is_float(d.bias_type)) return fail(B200_EINVAL, "gemm_scaled: unknown bias type %d", d.bias_type);
  if (d.activation < B200_ACT_NONE || d.activation > B200_ACT_SILU)
    return fail(B200_EINVAL, "gemm_scaled: unknown activation %d", d.activation);
  if ((a_scale && (d.a_scale_step < 0 || d.a_scale_step > 1)) || (w_scale && (d.w_scale_step < 0 || d.w_scale_step > 1)))
    return fail(B200_EINVAL, "gemm_scaled: scale steps are 0 or 1");
  if (d.M == 0 || d.N == 0) return B200_OK;
  if (!A || !W || !Y) return fail(B200_EINVAL, "gemm_scaled: null pointer");
  if ((d.lda < d.K && d.M > 1) || (d.ldw < d.K && d.N > 1) || (d.ldy < d.N && d.M > 1) ||
      (residual && d.ldr < d.N && d.M > 1))
    return fail(B200_EINVAL, "gemm_scaled: leading dimension smaller than the row length");
  if (d.M > 0x7fffff00LL || d.N > 0x7fffff00LL || d.K > 0x7fffff00LL)
    return fail(B200_EUNSUPPORTED, "gemm_scaled: an extent is too large");
  const int b = type_bytes(d.type);
  b200_gemm_scaled_desc e = d;
  // one row: its stride is never used, any valid one will do for the tensor map
  const int64_t pitch = (d.K * b + 15) / 16 * 16 / b;
  if (e.M == 1) e.lda = pitch;
  if (e.N == 1) e.ldw = pitch;
  if (!aligned16(A) || !aligned16(W) || e.lda * b % 16 || e.ldw * b % 16)
    return fail(B200_EUNSUPPORTED, "gemm_scaled: A and W need 16-byte aligned bases and row strides of multiples of 16 bytes");
  if (e.lda * b >= (1LL << 40) || e.ldw * b >= (1LL << 40)) return fail(B200_EUNSUPPORTED, "gemm_scaled: a row stride is too large");
  const int vec = output_access(e, residual, Y);
  return run_plan((cudaStream_t)stream, e, choose(e, vec >= 16), vec, A, W, a_scale, w_scale, bias, residual, Y);
}

extern "C" B200_API int b200_gemm_scaled_plan(const b200_gemm_scaled_desc *desc, const void *residual, const void *Y,
                                              int32_t plan[3]) {
  if (!desc || !plan) return fail(B200_EINVAL, "gemm_scaled_plan: null pointer");
  if (desc->M < 1 || desc->N < 1 || desc->K < 1) return fail(B200_EINVAL, "gemm_scaled_plan: a product without outputs");
  if ((desc->type != B200_TYPE_E4M3 && desc->type != B200_TYPE_F16 && desc->type != B200_TYPE_BF16) || !is_float(desc->y_type))
    return fail(B200_EINVAL, "gemm_scaled_plan: unknown type");
  const Plan p = choose(*desc, output_access(*desc, residual, Y) >= 16);
  plan[0] = p.pair;
  plan[1] = p.cols;
  plan[2] = p.ranks;
  return B200_OK;
}
