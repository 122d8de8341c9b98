// Products of int8 rows that carry a scale each with int8 weights that carry one per output channel:
//   y[m, n] = xscale[m] wscale[n] sum_k x[m, k] w[n, k] + bias[n] + residual[m, n],      gated: silu(gate) up
// where a gated product has 2 N weight rows, the gate's first.  The sums are exact (int32: K below 2^17); they are scaled in
// fp32 and rounded once to the output's type.
//
// Two kernels on tcgen05 (kind::i8, int32 accumulators in tensor memory), operands brought by TMA in 128-byte slices of K.
//
// Few rows (linear_i8_few_kernel).  The floor is the weights' bytes, so the weights are the M side of the MMA (128 of them per
// tile) and up to MT tokens its N side: no tensor time goes into empty rows, a lane of tensor memory is an output channel, and
// a token's outputs leave in whole lines.  Where the tiles are fewer than the SMs, a cluster of up to 8 CTAs shares a tile's K
// and adds its parts through distributed shared memory; whole numbers, so the order does not matter.  64 x 49280 x 960 to fp32:
// 13.7 us, 4.4 TB/s (385 tiles in one round of three CTAs per SM; 27 us with 4 epilogue warps and two CTAs); one row by 1600 x 960:
// 3.9 us, of which the launch is 2.
//
// Many rows (linear_i8_many_kernel).  Bound by the tensor pipe: CTA pairs compute 256 tokens x 256 weights (cta_group::2), which
// halves the weights' way into each SM: an MMA of 128 x 256 x 32 per SM takes 128 cycles and 8 KB of shared memory, its operands
// arrive at 64 bytes a cycle.  Persistent, accumulators double-buffered (all 512 columns), 8 epilogue warps for each.  Outputs leave through
// shared memory and TMA stores: written by the threads that own a row each, every warp's store touches 32 lines, and the stores'
// way through L1 took 8000 cycles per tile.
// 8192 x 4096 x 11008: 220 us, 3.3 POPS; in fp16 with a residual 241, called again and again, under the power cap, 286.
// 11328 x 2560 x 960, gated: 47 us, 2.4 POPS, 31.5 with K = 128: a tile has 8 slices of K only, and its epilogue holds the accumulator
// longer than they take.  No pipe is at its limit there (tensor 54%, issue slots 49%, exponentials and reciprocals 32%): a warp waits
// for its columns, works, waits for its box to be read.  Not gated, where outputs are twice as many per tile: 11328 x 960 x 960 16.8 us,
// 1600 columns 24.4, 2560 31.5 (2.43, 4.26 and 6.08 tiles per pair, in 3, 5 and 7 rounds).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"
#include "serving_common.cuh"

namespace svla {

struct LinearI8Args {
  CUtensorMap tx, tw;  // 2-D (k, row), 128-byte swizzle
  CUtensorMap to;      // many rows, staged: 2-D (n, row) of the output, a warp's box
  const float *xscale, *wscale, *bias;
  const void* residual;
  void* out;
  long long residual_rs, out_rs;
  int m, n, k;
  int tiles_m, tiles_n;
  int splits;  // few rows: CTAs of a cluster that share a tile's K
  int staged;  // many rows: outputs leave by TMA, which writes whole 16 bytes (and residual rows come 16 bytes at a time)
  int* err;
};

namespace li8 {
constexpr int kSlice = 128;  // bytes of K per stage

template <typename T>
__device__ __forceinline__ void put(T* p, float v);
template <>
__device__ __forceinline__ void put<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void put<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ void put<__half>(__half* p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ float scaled(uint32_t acc, float a, float b) {
  return __fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(acc)), a), b);
}

// the same for pairs, through the packed fp32 pipe: each half rounds as the scalar operation does
__device__ __forceinline__ float2 scaled2(uint32_t a0, uint32_t a1, float a, float2 b) {
  const float2 v = make_float2(static_cast<float>(static_cast<int>(a0)), static_cast<float>(static_cast<int>(a1)));
  return __fmul2_rn(__fmul2_rn(v, make_float2(a, a)), b);
}

// x sigmoid(x) with the hardware's 2^z and reciprocal (2^-22 and 2^-23 relative).  z = -x log2(e) is rounded, which puts the
// exponential off by 2^-24 |x|; outputs of 16 bits hide that.  For fp32 ones what z lacks, -x - z ln 2, comes in to first order
// (11328 x 2560 x 960: 56.7 us, 55 without; 68 with expf and a division).  A sigmoid below 2^-126, x < -87.3, is 0.
template <typename T>
__device__ __forceinline__ float2 silu2(float2 x) {
  if constexpr (sizeof(T) == 4) {
    auto clamp = [](float v) { return fminf(fmaxf(v, -88.f), 128.f); };  // 2^z and what z lacks stay finite; beyond, 2^z is 0 or the sigmoid is
    const float2 c = make_float2(clamp(x.x), clamp(x.y));                // (x itself carries a NaN on)
    const float2 z = __fmul2_rn(c, make_float2(-serving::kLog2e, -serving::kLog2e));
    float2 t = __ffma2_rn(z, make_float2(-0.6931471824645996f, -0.6931471824645996f), make_float2(-c.x, -c.y));
    t = __ffma2_rn(z, make_float2(1.9046542121259336e-09f, 1.9046542121259336e-09f), t);
    const float2 e = make_float2(ex2_approx(z.x), ex2_approx(z.y));
    const float2 d = __fadd2_rn(make_float2(1.f, 1.f), __ffma2_rn(e, t, e));
    return __fmul2_rn(x, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
  } else {
    const float2 z = __fmul2_rn(x, make_float2(-serving::kLog2e, -serving::kLog2e));
    const float2 d = __fadd2_rn(make_float2(1.f, 1.f), make_float2(ex2_approx(z.x), ex2_approx(z.y)));
    return __fmul2_rn(x, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
  }
}
template <typename T>
__device__ __forceinline__ float silu(float x) {
  if constexpr (sizeof(T) == 4) {
    const float c = fminf(fmaxf(x, -88.f), 128.f), z = __fmul_rn(c, -serving::kLog2e);
    const float t = __fmaf_rn(z, 1.9046542121259336e-09f, __fmaf_rn(z, -0.6931471824645996f, -c)), e = ex2_approx(z);
    return __fmul_rn(x, rcp_approx(__fadd_rn(1.f, __fmaf_rn(e, t, e))));
  } else {
    return __fmul_rn(x, rcp_approx(__fadd_rn(1.f, ex2_approx(__fmul_rn(x, -serving::kLog2e)))));
  }
}

template <int MT, bool GATED>
struct Few {
  static constexpr int kP = GATED ? 2 : 1;
  static constexpr int kW = 128 * kSlice, kX = MT * kSlice;
  static constexpr int kStage = kP * kW + kX;
  // three CTAs per SM (a tile's start and end beside the others' streams) where three stages of each fit, or two, or one
  static constexpr int kStages = (kStage <= 24576 ? 73728 : kStage <= 32768 ? 98304 : 196608) / kStage;
  static constexpr int kBar = kStages * kStage;
  static constexpr int kScales = kBar + 256;              // of the tokens
  static constexpr int kBytes = kScales + MT * 4 + 1024;  // + alignment slack
  static constexpr int kCols = kP * MT < 32 ? 32 : kP * MT;
  static_assert(kStages * kStage >= kP * MT * 512, "a tile's parts lie where its operands were");
  static_assert(kCols <= 512 && kBytes <= 232448);
};
constexpr int kFewThreads = 256;

// 32 lanes x 32 bit, 8 consecutive columns -> 8 registers per thread
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
}  // namespace li8

// One tile of 128 output channels x MT tokens per CTA, or per cluster of `splits` CTAs
template <typename T, int MT, bool GATED>
__global__ void __launch_bounds__(li8::kFewThreads) linear_i8_few_kernel(const __grid_constant__ LinearI8Args a) {
  using namespace li8;
  using C = Few<MT, GATED>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBar);
  uint64_t* empty = full + C::kStages;
  uint64_t* done = empty + C::kStages;
  uint32_t* slot = reinterpret_cast<uint32_t*>(done + 1);
  const int warp = threadIdx.x >> 5;
  const int split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits;
  const int m0 = (tile / a.tiles_n) * MT, n0 = (tile % a.tiles_n) * 128;
  const int slices = (a.k + kSlice - 1) / kSlice;
  const int per = (slices + a.splits - 1) / a.splits;
  const int kb = min(split * per, slices), ke = min(kb + per, slices);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(slot, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  pdl_wait();
  pdl_trigger();

  bool ok = true;
  float* scales = reinterpret_cast<float*>(smem + C::kScales);
  if (warp >= 2)
    for (int c = threadIdx.x - 64; c < MT; c += kFewThreads - 64) scales[c] = m0 + c < a.m ? __ldg(a.xscale + m0 + c) : 0.f;
  if (warp == 0) {
    for (int i = 0; i < ke - kb && ok; ++i) {
      const int s = i % C::kStages;
      ok = serving::wait_warp(&empty[s], ((i / C::kStages) & 1) ^ 1, a.err);
      if (ok && serving::elect_one()) {
        uint8_t* st = smem + s * C::kStage;
        mbar_arrive_expect_tx(&full[s], C::kStage);
#pragma unroll
        for (int p = 0; p < C::kP; ++p) tma_load_2d(st + p * C::kW, &a.tw, &full[s], (kb + i) * kSlice, p * a.n + n0);
        tma_load_2d(st + C::kP * C::kW, &a.tx, &full[s], (kb + i) * kSlice, m0);
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    for (int i = 0; i < ke - kb && ok; ++i) {
      const int s = i % C::kStages;
      ok = serving::wait_warp(&full[s], (i / C::kStages) & 1, a.err);
      tc_fence_after();
      if (ok && serving::elect_one()) {
        const uint32_t st = smem_u32(smem + s * C::kStage);
        const uint64_t x = smem_desc_sw128(st + C::kP * C::kW);
#pragma unroll
        for (int p = 0; p < C::kP; ++p) {
          const uint64_t w = smem_desc_sw128(st + p * C::kW);
#pragma unroll
          for (int kk = 0; kk < kSlice / 32; ++kk)  // 32 bytes are 2 units of a descriptor's address
            mma_i8(tmem + p * MT, w + 2 * kk, x + 2 * kk, idesc_i8(128, MT), i > 0 || kk > 0);
        }
        mma_commit(&empty[s]);
        if (i + 1 == ke - kb) mma_commit(done);
      }
      __syncwarp();
    }
  }
  __syncthreads();  // the tokens' scales are there
  // (a producer or issuer that gave up leaves `done` alone, and this wait gives up too)
  ok = ke > kb ? serving::wait_warp(done, 0, a.err) : true;
  __syncwarp();
  tc_fence_after();

  // warps w and w + 4 share the lanes 32 (w % 4) .. and take every other 8 tokens
  const int lane_n = threadIdx.x & 127, part = threadIdx.x >> 7, n = n0 + lane_n;
  const uint32_t t_row = tmem + (static_cast<uint32_t>(warp & 3) << 21);
  const int cols = min(MT, a.m - m0);
  const bool in = n < a.n;
  const float ws = in ? __ldg(a.wscale + n) : 0.f, wu = GATED && in ? __ldg(a.wscale + a.n + n) : 0.f;
  const float bias = a.bias && in ? __ldg(a.bias + n) : -0.f;
  auto value = [&](uint32_t acc, uint32_t acc2, float xs) {
    float v = scaled(acc, xs, ws);
    if constexpr (GATED) v = __fmul_rn(silu<T>(v), scaled(acc2, xs, wu));
    return __fadd_rn(v, bias);
  };
  if (a.splits == 1) {
    for (int c = part * 8; c < cols; c += 16) {
      uint32_t r[8], r2[GATED ? 8 : 1];
      if (ok) {
        tmem_ld8(t_row + c, r);
        if constexpr (GATED) tmem_ld8(t_row + MT + c, reinterpret_cast<uint32_t(&)[8]>(r2));
        tmem_ld_wait();
      }
      if (ok && in) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = value(r[j], r2[GATED ? j : 0], scales[c + j]);
        const int some = min(8, cols - c);
        if (a.residual) {
          const T* res = static_cast<const T*>(a.residual) + (m0 + c) * a.residual_rs + n;
#pragma unroll
          for (int j = 0; j < 8; ++j, res += a.residual_rs)
            if (j < some) v[j] = __fadd_rn(v[j], static_cast<float>(*res));
        }
        T* out = static_cast<T*>(a.out) + (m0 + c) * a.out_rs + n;
#pragma unroll
        for (int j = 0; j < 8; ++j, out += a.out_rs)
          if (j < some) put<T>(out, v[j]);
      }
      __syncwarp();
    }
  } else {
    uint32_t* parts = reinterpret_cast<uint32_t*>(smem);  // [P][MT][128]; every operand has been read
    for (int c = part * 8; c < cols; c += 16) {
      uint32_t r[8], r2[GATED ? 8 : 1];
      if (ok && ke > kb) {
        tmem_ld8(t_row + c, r);
        if constexpr (GATED) tmem_ld8(t_row + MT + c, reinterpret_cast<uint32_t(&)[8]>(r2));
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = 0u, r2[GATED ? j : 0] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        parts[(c + j) * 128 + lane_n] = r[j];
        if constexpr (GATED) parts[(MT + c + j) * 128 + lane_n] = r2[j];
      }
    }
    __syncwarp();
    cluster_sync();
    // a warp adds up a token's 128 outputs, four a lane: the parts of all CTAs are on their way at once
    if (ok) {
      const int n4 = n0 + (threadIdx.x & 31) * 4;
      float w4[4], u4[4], b4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool there = n4 + e < a.n;
        w4[e] = there ? __ldg(a.wscale + n4 + e) : 0.f;
        u4[e] = GATED && there ? __ldg(a.wscale + a.n + n4 + e) : 0.f;
        b4[e] = a.bias && there ? __ldg(a.bias + n4 + e) : -0.f;
      }
      const uint32_t base = smem_u32(parts) + (threadIdx.x & 31) * 16;
      for (int c = split + warp * a.splits; c < cols; c += (kFewThreads / 32) * a.splits) {
        uint32_t sum[4] = {0u, 0u, 0u, 0u}, sum2[4] = {0u, 0u, 0u, 0u};
        auto add = [&](uint32_t (&to)[4], uint32_t from) {
          uint32_t v[4];
          asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(from));
#pragma unroll
          for (int e = 0; e < 4; ++e) to[e] += v[e];
        };
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          if (s >= a.splits) break;
          const uint32_t from = mapa_shared(base + c * 512, s);
          add(sum, from);
          if constexpr (GATED) add(sum2, from + MT * 512);
        }
        T* out = static_cast<T*>(a.out) + (m0 + c) * a.out_rs + n4;
        const T* res = static_cast<const T*>(a.residual) + (m0 + c) * a.residual_rs + n4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (n4 + e >= a.n) break;
          float v = scaled(sum[e], scales[c], w4[e]);
          if constexpr (GATED) v = __fmul_rn(silu<T>(v), scaled(sum2[e], scales[c], u4[e]));
          v = __fadd_rn(v, b4[e]);
          if (a.residual) v = __fadd_rn(v, static_cast<float>(res[e]));
          put<T>(out + e, v);
        }
      }
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while its parts are read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kCols);
  }
}

namespace li8 {
struct Many {
  // A CTA's rows of x and its half of w.  A stage more is worth more than a second box per warp (4 stages and two boxes
  // took 8% longer with K = 11008, as long with K = 960, gated)
  static constexpr int kStages = 5, kTile = 128 * kSlice, kStage = 2 * kTile;
  static constexpr int kOut = kStages * kStage, kBoxBytes = 2048;  // each epilogue warp's box of 32 rows x 64 bytes
  static constexpr int kBar = kOut + 16 * kBoxBytes;
  static constexpr int kConst = kBar + 256;                    // each epilogue warp's 2 x 128 column constants
  static constexpr int kBytes = kConst + 16 * 256 * 4 + 1024;  // + alignment slack
  static_assert(kBytes <= 232448);
};
constexpr int kManyThreads = 576;  // TMA, MMA, 2 x 8 warps of epilogue
template <typename T>
constexpr int kBoxCols = 64 / static_cast<int>(sizeof(T));
// 16-byte chunk j of a box's row r: rows of 64 bytes, spread over the banks as TMA's swizzle of them does
__device__ __forceinline__ uint8_t* chunk_of(uint8_t* box, int r, int j) { return box + r * 64 + ((j ^ ((r >> 1) & 3)) << 4); }
}  // namespace li8

// Tiles of 256 tokens x 256 weights (gated: 128 gates and their 128 ups) per CTA pair
template <typename T, bool GATED>
__global__ void __launch_bounds__(li8::kManyThreads, 1) linear_i8_many_kernel(const __grid_constant__ LinearI8Args a) {
  using namespace li8;
  using C = Many;
  constexpr int kOutCols = GATED ? 128 : 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBar);  // the leader's: both CTAs' operands are there
  uint64_t* empty = full + C::kStages;                           // each CTA's own: its operands have been read
  uint64_t* tfull = empty + C::kStages;                          // [2] each CTA's own: an accumulator is complete
  uint64_t* tempty = tfull + 2;                                  // [2] the leader's: both CTAs' epilogues have read it
  uint32_t* slot = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
  const int slices = (a.k + kSlice - 1) / kSlice, tiles = a.tiles_m * a.tiles_n;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 16);
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are initialised before either uses the other's
  tc_fence_after();
  const uint32_t tmem = *slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    uint32_t s = 0, ph = 1;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int m0 = (t / a.tiles_n) * 256 + static_cast<int>(rank) * 128;
      const int n0 = (t % a.tiles_n) * kOutCols + static_cast<int>(rank) * (GATED ? a.n : 128);
      for (int i = 0; i < slices && ok; ++i) {
        ok = serving::wait_warp(&empty[s], ph, a.err);
        if (ok && serving::elect_one()) {
          uint8_t* st = smem + s * C::kStage;
          const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::kStage);
          tma_load_2d_pair(st, &a.tx, bar, i * kSlice, m0);
          tma_load_2d_pair(st + C::kTile, &a.tw, bar, i * kSlice, n0);
        }
        __syncwarp();
        if (++s == C::kStages) s = 0, ph ^= 1;
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      uint32_t s = 0, ph = 0, lt = 0;
      bool ok = true;
      auto commit = [&](uint64_t* bar) {
        mma_commit_pair(mapa_shared(smem_u32(bar), 0));
        mma_commit_pair(mapa_shared(smem_u32(bar), 1));
      };
      for (int t = pair; t < tiles && ok; t += pairs, ++lt) {
        const uint32_t ab = lt & 1;
        ok = serving::wait_warp(&tempty[ab], ((lt >> 1) & 1) ^ 1, a.err);
        tc_fence_after();
        for (int i = 0; i < slices && ok; ++i) {
          ok = serving::wait_warp(&full[s], ph, a.err);
          tc_fence_after();
          if (ok && serving::elect_one()) {
            const uint32_t st = smem_u32(smem + s * C::kStage);
            const uint64_t x = smem_desc_sw128(st), w = smem_desc_sw128(st + C::kTile);
#pragma unroll
            for (int kk = 0; kk < kSlice / 32; ++kk)
              mma_i8_pair(tmem + ab * 256, x + 2 * kk, w + 2 * kk, idesc_i8(256, 256), i > 0 || kk > 0);
            commit(&empty[s]);
            if (i + 1 == slices) commit(&tfull[ab]);
          }
          __syncwarp();
          if (++s == C::kStages) s = 0, ph ^= 1;
        }
      }
    }
  } else {
    // Warps 2-9 take the even tiles and 10-17 the odd ones, so that one half's exponentials run beside the other's stores; of a
    // tile, two warps per lane quarter have half of the columns each.  (Gated products gain by it, 68 us to 49 when it was
    // brought in; plain ones of short K lose: 11328 x 5120 x 128 took 37.7 us with all 16 warps on a tile and takes 40.7.)
    const int q = warp & 3, part = ((warp - 2) / 4) & 1, half = (warp - 2) / 8;
    constexpr int kCols = kOutCols / 2, kChunk = GATED ? 16 : 32, kBox = kBoxCols<T>, kPer = 16 / static_cast<int>(sizeof(T));
    float* consts = reinterpret_cast<float*>(smem + C::kConst) + (warp - 2) * 256;  // scales, then biases or ups' scales
    uint8_t* box = smem + C::kOut + (warp - 2) * C::kBoxBytes;
    const uint32_t tempty_leader = mapa_shared(smem_u32(&tempty[half]), 0);
    // a tile's constants: fetched one tile ahead
    float next[2 * kCols / 32], next_xs;
    auto row0_of = [&](int t) { return (t / a.tiles_n) * 256 + static_cast<int>(rank) * 128 + q * 32; };
    auto fetch = [&](int t) {
      if (t >= tiles) return;
      const int n = (t % a.tiles_n) * kOutCols + part * kCols + lane, m = row0_of(t) + lane;
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) {
        const bool in = n + i * 32 < a.n;
        next[2 * i] = in ? __ldg(a.wscale + n + i * 32) : 0.f;
        next[2 * i + 1] = GATED ? (in ? __ldg(a.wscale + a.n + n + i * 32) : 0.f) : (a.bias && in ? __ldg(a.bias + n + i * 32) : -0.f);
      }
      next_xs = m < a.m ? __ldg(a.xscale + m) : 0.f;
    };
    fetch(pair + half * pairs);
    bool ok = true;
    uint32_t use = 0;
    for (int t = pair + half * pairs; t < tiles; t += 2 * pairs, ++use) {
      const int m0 = row0_of(t), n0 = (t % a.tiles_n) * kOutCols + part * kCols;
      const int cols = m0 < a.m ? max(0, min(kCols, a.n - n0)) : 0, rows = min(32, a.m - m0);
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) consts[i * 32 + lane] = next[2 * i], consts[128 + i * 32 + lane] = next[2 * i + 1];
      const float xs = next_xs;
      fetch(t + 2 * pairs);
      // the box is free once its last store has read it; then the residual is brought there, whole lines at a time
      auto take_box = [&](int c) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
        if (!a.residual) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + lane / 4, from = c + (lane % 4) * kPer;
          const int bytes = r < rows ? max(0, min(16, (cols - from) * static_cast<int>(sizeof(T)))) : 0;
          const T* res = static_cast<const T*>(a.residual);
          serving::copy16(chunk_of(box, r, lane % 4), bytes ? res + (m0 + r) * a.residual_rs + n0 + from : res, bytes);
        }
        serving::copy_commit();
      };
      if (a.staged && cols > 0) take_box(0);
      __syncwarp();
      ok = ok && serving::wait_warp(&tfull[half], use & 1, a.err);
      tc_fence_after();
      const uint32_t t_row = tmem + half * 256 + (static_cast<uint32_t>(q * 32) << 16) + part * kCols;
      // the accumulator is free once its last columns are in registers; the arrival releases nothing beyond that (a release at
      // cluster scope would wait for the stores)
      auto give_back = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(tempty_leader) : "memory");
      };
      if (cols == 0) give_back();
#pragma unroll 1
      for (int c = 0; c < cols; c += kChunk) {
        uint32_t r[kChunk], r2[GATED ? kChunk : 1];
        if (ok) {
          if constexpr (GATED) {
            tmem_ld16(t_row + c, r);
            tmem_ld16(t_row + 128 + c, r2);
          } else {
            tmem_ld32(t_row + c, r);
          }
          tmem_ld_wait();
        }
        if (c + kChunk >= cols) give_back();
        float v[kChunk];
#pragma unroll
        for (int j = 0; j < kChunk; j += 4) {
          const float4 w4 = *reinterpret_cast<const float4*>(consts + c + j);
          const float4 b4 = *reinterpret_cast<const float4*>(consts + 128 + c + j);
          const float2 w[2] = {make_float2(w4.x, w4.y), make_float2(w4.z, w4.w)}, b[2] = {make_float2(b4.x, b4.y), make_float2(b4.z, b4.w)};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float2 y = scaled2(r[j + 2 * e], r[j + 2 * e + 1], xs, w[e]);
            if constexpr (GATED) y = __fmul2_rn(silu2<T>(y), scaled2(r2[GATED ? j + 2 * e : 0], r2[GATED ? j + 2 * e + 1 : 0], xs, b[e]));
            else y = __fadd2_rn(y, b[e]);
            v[j + 2 * e] = y.x, v[j + 2 * e + 1] = y.y;
          }
        }
        if (a.staged) {
          constexpr int kSub = kChunk < kBox ? kChunk : kBox;  // columns that go to one box at once
#pragma unroll
          for (int u = 0; u < kChunk; u += kSub) {
            if (c + u >= cols) break;
            const int first = (c + u) % kBox;
            if (a.residual && first == 0) {
              serving::copy_wait<0>();
              __syncwarp();
            }
#pragma unroll
            for (int j = u; j < u + kSub; j += kPer) {
              uint4* place = reinterpret_cast<uint4*>(chunk_of(box, lane, (first + j - u) / kPer));
              if (!GATED && a.residual) {
                const uint4 w = *place;
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if constexpr (sizeof(T) == 4) {
                    v[j + e] = __fadd_rn(v[j + e], __uint_as_float(x[e]));
                  } else {
                    const float2 f = serving::unpack2<T>(x[e]);
                    v[j + 2 * e] = __fadd_rn(v[j + 2 * e], f.x);
                    v[j + 2 * e + 1] = __fadd_rn(v[j + 2 * e + 1], f.y);
                  }
                }
              }
              uint32_t p[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 4) p[e] = __float_as_uint(v[j + e]);
                else p[e] = serving::pack2<T>(v[j + 2 * e], v[j + 2 * e + 1]);
              }
              *place = make_uint4(p[0], p[1], p[2], p[3]);
            }
            if (first + kSub == kBox || c + u + kSub >= cols) {  // the box is complete (what is behind the last column TMA leaves out)
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                if (ok)
                  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                                   reinterpret_cast<uint64_t>(&a.to)),
                               "r"(n0 + c + u - first), "r"(m0), "r"(smem_u32(box))
                               : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
              }
              __syncwarp();
              if (c + u + kSub < cols) take_box(c + u + kSub);
            }
          }
        } else {  // through the box as well, 16 columns in fp32 at a time, and on from there two rows of them at a time
#pragma unroll
          for (int u = 0; u < kChunk; u += 16) {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<float4*>(chunk_of(box, lane, j / 4)) = make_float4(v[u + j], v[u + j + 1], v[u + j + 2], v[u + j + 3]);
            __syncwarp();
            const int col = lane % 16, n = n0 + c + u + col;
            if (ok && c + u + col < cols) {
              T* out = static_cast<T*>(a.out) + m0 * a.out_rs + n;
              const T* res = static_cast<const T*>(a.residual) + m0 * a.residual_rs + n;
#pragma unroll 8
              for (int i = lane / 16; i < rows; i += 2) {
                float y = *reinterpret_cast<const float*>(chunk_of(box, i, col / 4) + (col % 4) * 4);
                if (a.residual) y = __fadd_rn(y, static_cast<float>(res[i * a.residual_rs]));
                put<T>(out + i * a.out_rs, y);
              }
            }
            __syncwarp();
          }
        }
        __syncwarp();
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the box is read before the CTA ends
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still arrive on its barriers
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

}  // namespace svla
