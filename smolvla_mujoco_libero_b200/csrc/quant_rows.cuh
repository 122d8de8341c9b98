// Rows quantised to int8 with a scale each, behind an optional sum, norm and smoothing:
//   h = x + residual,  y = h | h rstd w | (h - mean) rstd w + b,  y /= smooth,
//   scale = max |y| / 127,  code = round(y / scale)      (ties to even, as torch rounds)
// and, where asked for, h and the values code * scale in the input's type.
//
// The floor is memory: x and residual once in, h, codes and values once out.  A row is held in registers from its load to its
// codes, so every statistic (mean, centred squares, largest magnitude) is a pass over registers: 2 rounds of shuffles with
// RMSNorm, 3 with LayerNorm, 1 without a norm.  Rows of up to 1024 elements belong to one warp, which needs no shared memory
// and no barrier; longer ones, and rows that are too few to fill the GPU, to a block of 4 to 32 warps.
//
// Sums and statistics in fp32, of the unrounded h.  Quotients are correctly rounded (quotient() below), so without a norm the
// codes are those of the definition bit for bit.  A row that holds no finite maximum (an infinity, a NaN) has scale NaN and codes 0:
// it stays visible in every product.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"
#include "serving_common.cuh"

namespace svla {

struct QuantRowsArgs {
  const void *x, *residual, *weight, *bias;
  const float* smooth;
  int8_t* codes;
  float* scale;
  void *sum, *values;
  long long x_rs, residual_rs, codes_rs, sum_rs, values_rs;
  int m, k;
  float eps;
};

namespace qrows {
constexpr int kMaxChunks = 4;  // of 8 elements per lane

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// d / s correctly rounded, r = 1 / s correctly rounded: P. Markstein's correction of a quotient (Computation of elementary
// functions on the IBM RISC System/6000 processor, 1990); the caller keeps s within 2^+-60 and |d| below 2^8 s
__device__ __forceinline__ float quotient(float d, float s, float r) {
  const float q = __fmul_rn(d, r);
  return __fmaf_rn(__fmaf_rn(-q, s, d), r, q);
}

// 8 elements from column c; VEC: whole 16-byte chunks, otherwise element by element up to k
template <typename T, bool VEC>
__device__ __forceinline__ void load8(float (&v)[8], const T* row, int c, int k) {
  if constexpr (VEC) {
    const uint4 w = *reinterpret_cast<const uint4*>(row + c);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = serving::unpack2<T>(u[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < k ? static_cast<float>(row[c + e]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ T rounded(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half rounded<__half>(float x) { return __float2half_rn(x); }

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, const float (&v)[8], int c, int k) {
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(row + c) = make_uint4(serving::pack2<T>(v[0], v[1]), serving::pack2<T>(v[2], v[3]),
                                                    serving::pack2<T>(v[4], v[5]), serving::pack2<T>(v[6], v[7]));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < k) row[c + e] = rounded<T>(v[e]);
  }
}

enum class Join { Add, Max };
template <Join J>
__device__ __forceinline__ float join(float a, float b) {
  if constexpr (J == Join::Add) return __fadd_rn(a, b);
  else return max_nan(a, b);
}
// over the lanes of a row: one warp, or W warps through shared memory (`part` is used by one reduction only)
template <Join J, int W>
__device__ __forceinline__ float reduce_row(float v, float* part) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = join<J>(v, __shfl_xor_sync(0xffffffffu, v, d));
  if constexpr (W > 1) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v = join<J>(v, part[i]);  // the same order in every thread
  }
  return v;
}
}  // namespace qrows

// W warps per row (1: four rows per block), CH chunks of 8 elements per lane
template <typename T, bool VEC, int W, int CH>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) quant_rows_kernel(const QuantRowsArgs a) {
  using namespace qrows;
  __shared__ float part[3][W];
  const int lane = W == 1 ? threadIdx.x & 31 : threadIdx.x;
  const long long row = W == 1 ? static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  pdl_wait();
  pdl_trigger();
  if (row >= a.m) return;
  const int k = a.k;
  float y[CH][8];
  auto column = [&](int i) { return (i * W * 32 + lane) * 8; };
  {
    const T* x = static_cast<const T*>(a.x) + row * a.x_rs;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[i][e] = 0.f;
      if (column(i) < k) load8<T, VEC>(y[i], x, column(i), k);
    }
  }
  if (a.residual) {
    const T* r = static_cast<const T*>(a.residual) + row * a.residual_rs;
    float v[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (column(i) < k) load8<T, VEC>(v[i], r, column(i), k);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (column(i) >= k) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[i][e] = __fadd_rn(y[i][e], v[i][e]);
    }
  }
  if (a.sum) {
    T* s = static_cast<T*>(a.sum) + row * a.sum_rs;
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (column(i) < k) store8<T, VEC>(s, y[i], column(i), k);
  }
  if (a.weight) {
    const float inv = __fdiv_rn(1.f, static_cast<float>(k));
    float mean = 0.f, squares = 0.f, eps = a.eps;
    // Squares beyond fp32's range (components above 1e17 or so) are seen in their sum; the row is then scaled by 2^-80, which
    // a norm does not notice, and its statistics are taken again.  The choice is the row's, so its threads agree.
    for (int pass = 0; pass < 2; ++pass) {
      if (a.bias) {
        mean = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) mean = __fadd_rn(mean, y[i][e]);
        mean = __fmul_rn(reduce_row<Join::Add, W>(mean, part[0]), inv);
      }
      squares = 0.f;
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float d = VEC ? (column(i) < k ? __fsub_rn(y[i][e], mean) : 0.f)
                              : (column(i) + e < k ? __fsub_rn(y[i][e], mean) : 0.f);
          squares = __fmaf_rn(d, d, squares);
        }
      squares = reduce_row<Join::Add, W>(squares, part[1]);
      if (pass == 1 || squares < __int_as_float(0x7f800000)) break;
      constexpr float kDown = 8.271806125530277e-25f;  // 2^-80
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = __fmul_rn(y[i][e], kDown);
      eps = 0.f;
      if constexpr (W > 1) __syncthreads();  // the partial sums are read before they are written again
    }
    const float rstd = __frsqrt_rn(__fmaf_rn(squares, inv, eps));
    const T* w = static_cast<const T*>(a.weight);
    const T* b = static_cast<const T*>(a.bias);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (column(i) >= k) continue;
      float g[8];
      load8<T, VEC>(g, w, column(i), k);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[i][e] = __fmul_rn(__fmul_rn(__fsub_rn(y[i][e], mean), rstd), g[e]);
      if (a.bias) {
        load8<T, VEC>(g, b, column(i), k);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = __fadd_rn(y[i][e], g[e]);
      }
    }
  }
  if (a.smooth) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (column(i) >= k) continue;
      if constexpr (VEC) {
        const float4* s = reinterpret_cast<const float4*>(a.smooth + column(i));
        const float4 s0 = __ldg(s), s1 = __ldg(s + 1);
        const float d[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = __fdiv_rn(y[i][e], d[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (column(i) + e < k) y[i][e] = __fdiv_rn(y[i][e], __ldg(a.smooth + column(i) + e));
      }
    }
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (column(i) >= k) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (!VEC)
        if (column(i) + e >= k) continue;
      top = max_nan(top, fabsf(y[i][e]));
    }
  }
  top = reduce_row<Join::Max, W>(top, part[2]);
  const bool finite = top < __int_as_float(0x7f800000);
  const float scale = finite ? __fdiv_rn(top, 127.f) : __int_as_float(0x7fc00000);
  if (lane == 0) a.scale[row] = scale;
  const bool plain = scale > 8.6e-19f && scale < 1.2e18f;  // 2^+-60
  const float r = plain ? __frcp_rn(scale) : 0.f;
  int8_t* codes = a.codes + row * a.codes_rs;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (column(i) >= k) continue;
    uint32_t packed[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float q;
      if (plain) {
        q = quotient(y[i][e], scale, r);
      } else {
        q = scale > 0.f ? __fdiv_rn(y[i][e], scale) : 0.f;  // NaN: no
      }
      q = fminf(fmaxf(q, -127.f), 127.f);
      const float t = __fadd_rn(q, 12582912.f);  // 1.5 * 2^23: rounds to an integer (ties to even) in the low bits
      packed[e / 4] |= (__float_as_uint(t) & 0xFFu) << (8 * (e % 4));
      y[i][e] = __fmul_rn(__fsub_rn(t, 12582912.f), scale);
    }
    if constexpr (VEC) {
      *reinterpret_cast<uint2*>(codes + column(i)) = make_uint2(packed[0], packed[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (column(i) + e < k) codes[column(i) + e] = static_cast<int8_t>(packed[e / 4] >> (8 * (e % 4)));
    }
    if (a.values) store8<T, VEC>(static_cast<T*>(a.values) + row * a.values_rs, y[i], column(i), k);
  }
}

}  // namespace svla
