// Rows quantised to int8 with a scale each, behind an optional sum, norm and smoothing:
//   h = x + residual,  y = h | h rstd w | (h - mean) rstd w + b,  y /= smooth,
//   scale = max |y| / 127,  code = round(y / scale)      (ties to even, as torch rounds)
// and, where asked for, h and the values code * scale in the input's type.
//
// The floor is memory: x and residual once in, h, codes and values once out.  A row is held in registers from its load to its
// codes, so every statistic (mean, centred squares, largest magnitude) is a pass over registers and a round of shuffles (and one
// of shared memory, where a row has several warps).  A block owns a row at a time, two chunks of 8 elements per thread, and asks
// for its next row before it works on this one.
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

// 8 elements from column c as they are stored; VEC: 16 bytes at once, otherwise element by element up to k (zeros behind it)
template <typename T, bool VEC>
__device__ __forceinline__ uint4 raw8(const T* row, int c, int k) {
  if constexpr (VEC) {
    return *reinterpret_cast<const uint4*>(row + c);
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = (c + 2 * i < k ? p[c + 2 * i] : 0u) | (c + 2 * i + 1 < k ? static_cast<uint32_t>(p[c + 2 * i + 1]) << 16 : 0u);
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
}
template <typename T>
__device__ __forceinline__ void unpack8(float (&v)[8], const uint4& w) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = serving::unpack2<T>(u[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
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
// over the block's threads; `part` is used by one reduction of every other row only
template <Join J>
__device__ __forceinline__ float reduce_block(float v, float* part) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = join<J>(v, __shfl_xor_sync(0xffffffffu, v, d));
  const int warps = blockDim.x >> 5;
  if (warps > 1) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < warps; ++i) v = join<J>(v, part[i]);  // the same order in every thread
  }
  return v;
}

// y / s: by the hardware's reciprocal (2^-22 or so) and Markstein's correction where s is within 2^+-100 (off by half a step and
// 2^-43), by the division itself elsewhere
__device__ __forceinline__ void divide8(float (&y)[8], const float (&s)[8]) {
  float least = fabsf(s[0]), most = least;
#pragma unroll
  for (int e = 1; e < 8; ++e) least = fminf(least, fabsf(s[e])), most = fmaxf(most, fabsf(s[e]));
  if (least > 7.9e-31f && most < 1.2e30f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = quotient(y[e], s[e], rcp_approx(s[e]));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __fdiv_rn(y[e], s[e]);
  }
}
constexpr int kMaxWarps = 32;
}  // namespace qrows

// CH chunks of 8 elements per thread; the block's threads hold a row
template <typename T, bool VEC, int CH>
__global__ void __launch_bounds__(1024) quant_rows_kernel(const QuantRowsArgs a) {
  using namespace qrows;
  __shared__ float part[2][3][kMaxWarps];
  pdl_wait();
  pdl_trigger();
  const int k = a.k;
  auto column = [&](int i) { return (i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8; };
  uint4 rx[CH], rr[CH];
  auto fetch = [&](long long row) {
    if (row >= a.m) return;
    const T* x = static_cast<const T*>(a.x) + row * a.x_rs;
    const T* r = static_cast<const T*>(a.residual) + row * a.residual_rs;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      rx[i] = column(i) < k ? raw8<T, VEC>(x, column(i), k) : make_uint4(0u, 0u, 0u, 0u);
      if (a.residual) rr[i] = column(i) < k ? raw8<T, VEC>(r, column(i), k) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  // whether element e of chunk i is one of the row's (whole chunks are, where they are read at once)
  auto in = [&](int i, int e) { return VEC ? column(i) < k : column(i) + e < k; };
  fetch(blockIdx.x);
  int turn = 0;
  for (long long row = blockIdx.x; row < a.m; row += gridDim.x, turn ^= 1) {
    float y[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i) unpack8<T>(y[i], rx[i]);
    if (a.residual) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float v[8];
        unpack8<T>(v, rr[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = __fadd_rn(y[i][e], v[e]);
      }
    }
    fetch(row + gridDim.x);
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
          mean = __fmul_rn(reduce_block<Join::Add>(mean, part[turn][0]), inv);
        }
        squares = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float d = in(i, e) ? __fsub_rn(y[i][e], mean) : 0.f;
            squares = __fmaf_rn(d, d, squares);
          }
        squares = reduce_block<Join::Add>(squares, part[turn][1]);
        if (pass == 1 || squares < __int_as_float(0x7f800000)) break;
        constexpr float kDown = 8.271806125530277e-25f;  // 2^-80
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) y[i][e] = __fmul_rn(y[i][e], kDown);
        eps = 0.f;
        __syncthreads();  // the partial sums are read before they are written again
      }
      const float rstd = __frsqrt_rn(__fmaf_rn(squares, inv, eps));
      const T* w = static_cast<const T*>(a.weight);
      const T* b = static_cast<const T*>(a.bias);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (column(i) >= k) continue;
        float g[8];
        unpack8<T>(g, raw8<T, VEC>(w, column(i), k));
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = __fmul_rn(__fmul_rn(__fsub_rn(y[i][e], mean), rstd), g[e]);
        if (a.bias) {
          unpack8<T>(g, raw8<T, VEC>(b, column(i), k));
#pragma unroll
          for (int e = 0; e < 8; ++e) y[i][e] = __fadd_rn(y[i][e], g[e]);
        }
      }
    }
    if (a.smooth) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (column(i) >= k) continue;
        float d[8];
        if constexpr (VEC) {
          const float4* s = reinterpret_cast<const float4*>(a.smooth + column(i));
          const float4 s0 = __ldg(s), s1 = __ldg(s + 1);
          d[0] = s0.x, d[1] = s0.y, d[2] = s0.z, d[3] = s0.w, d[4] = s1.x, d[5] = s1.y, d[6] = s1.z, d[7] = s1.w;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = in(i, e) ? __ldg(a.smooth + column(i) + e) : 1.f;
        }
        divide8(y[i], d);
      }
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (in(i, e)) top = max_nan(top, fabsf(y[i][e]));
    top = reduce_block<Join::Max>(top, part[turn][2]);
    const bool finite = top < __int_as_float(0x7f800000);
    const float scale = finite ? __fdiv_rn(top, 127.f) : __int_as_float(0x7fc00000);
    if (threadIdx.x == 0) a.scale[row] = scale;
    const bool plain = scale > 8.6e-19f && scale < 1.2e18f;  // 2^+-60
    const float r = plain ? __frcp_rn(scale) : 0.f;
    int8_t* codes = a.codes + row * a.codes_rs;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (column(i) >= k) continue;
      float t[8];  // the code in the low bits: adding 1.5 * 2^23 rounds to an integer, ties to even
      if (plain) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = __fadd_rn(quotient(y[i][e], scale, r), 12582912.f);  // (at most 127 (1 + 2^-23))
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float q = scale > 0.f ? __fdiv_rn(y[i][e], scale) : 0.f;  // (NaN: no)
          t[e] = __fadd_rn(fminf(fmaxf(q, -127.f), 127.f), 12582912.f);
        }
      }
      uint32_t packed[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t lo = __byte_perm(__float_as_uint(t[4 * h]), __float_as_uint(t[4 * h + 1]), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(t[4 * h + 2]), __float_as_uint(t[4 * h + 3]), 0x0040);
        packed[h] = __byte_perm(lo, hi, 0x5410);
      }
      if constexpr (VEC) {
        *reinterpret_cast<uint2*>(codes + column(i)) = make_uint2(packed[0], packed[1]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (in(i, e)) codes[column(i) + e] = static_cast<int8_t>(packed[e / 4] >> (8 * (e % 4)));
      }
      if (a.values) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = __fmul_rn(__fsub_rn(t[e], 12582912.f), scale);
        store8<T, VEC>(static_cast<T*>(a.values) + row * a.values_rs, t, column(i), k);
      }
    }
  }
}

}  // namespace svla
