// Rows quantised to int8 with a scale each, behind an optional sum, norm and smoothing:
//   h = x + residual,  y = h | h rstd w | (h - mean) rstd w + b,  y /= smooth,
//   scale = max |y| / 127,  code = round(y / scale)      (ties to even, as torch rounds)
// and, where asked for, h and the values code * scale in the input's type.
//
// The floor is memory: x and residual once in, h, codes and values once out.  A row is held in registers from its load to its
// codes, so every statistic (mean, centred squares, largest magnitude) is a pass over registers and a round of shuffles (and one
// of shared memory, where a row has several warps).  A block owns a row at a time, two chunks of 8 elements per thread, and asks
// for its next row before it works on this one.  Instructions come next: pairs of elements go through the packed fp32 pipe (with
// scalar operations 8192 rows of 4096 with everything took 53 instructions an element and 73 us).
//
// Measured: 11328 rows of 960, residual and RMSNorm, 17.7 us (5.5 TB/s); 8192 of 4096, residual and LayerNorm, 53 us (5.7 TB/s,
// issue slots 71%); 11328 of 2560, smoothed, 31.3 us (4.6 TB/s): without the smoothing it takes 25.0, with a product in the
// quotients' place 26.6, and with the divisors held in registers from row to row 38.
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
// max(a, |b|, |c|), NaN where one is; a >= 0
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// d / s correctly rounded, r = 1 / s correctly rounded, minus_s = -s: P. Markstein's correction of a quotient (Computation of
// elementary functions on the IBM RISC System/6000 processor, 1990); the caller keeps s within 2^+-60 and |d| below 2^8 s
__device__ __forceinline__ float2 quotient(float2 d, float2 minus_s, float2 r) {
  const float2 q = __fmul2_rn(d, r);
  return __ffma2_rn(__ffma2_rn(q, minus_s, d), r, q);
}

// 8 elements of a vector of all rows (weight, bias) from column c, zeros behind k.  VEC: 16 bytes at once.  Otherwise what the
// address allows: 16 bytes, or the 4-byte words that hold an element, shifted by one where the vector begins inside a word.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 raw8(const T* row, int c, int k) {
  if constexpr (VEC) return *reinterpret_cast<const uint4*>(row + c);
  const uintptr_t at = reinterpret_cast<uintptr_t>(row + c);
  const int n = k - c;
  if (n >= 8 && at % 16 == 0) return *reinterpret_cast<const uint4*>(at);
  const uint32_t* p = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
  const int ahead = static_cast<int>(at & 2) / 2;  // 1: element 0 is the upper half of word 0
  uint32_t w[5], u[4];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = 2 * i - ahead < n && 2 * i - ahead < 8 ? p[i] : 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u[i] = ahead ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
    if (2 * i + 1 >= n) u[i] = 2 * i < n ? u[i] & 0xFFFFu : 0u;
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
template <typename T>
__device__ __forceinline__ void unpack8(float2 (&v)[4], const uint4& w) {
  v[0] = serving::unpack2<T>(w.x), v[1] = serving::unpack2<T>(w.y), v[2] = serving::unpack2<T>(w.z), v[3] = serving::unpack2<T>(w.w);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float2 (&v)[4]) {
  return make_uint4(serving::pack2<T>(v[0].x, v[0].y), serving::pack2<T>(v[1].x, v[1].y), serving::pack2<T>(v[2].x, v[2].y),
                    serving::pack2<T>(v[3].x, v[3].y));
}

// A warp's 256 elements of a row from column c0 on.  VEC: 16 bytes a lane.  Otherwise (k no multiple of 8, or rows that are
// not 16-byte aligned) the 4-byte words that hold them, a word per lane after the other, and through shared memory to the lanes
// that own them (11328 rows of 2561 with residual and RMSNorm: 116 us; 2560: 47.6; words taken by the lanes that own them took 1.7
// times as long).
template <typename T, bool VEC>
struct Piece;
template <typename T>
struct Piece<T, true> {
  uint4 w;
  __device__ __forceinline__ void fetch(const T* row, int c0, int k, int lane) {
    w = c0 + lane * 8 < k ? *reinterpret_cast<const uint4*>(row + c0 + lane * 8) : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ uint4 take(const T*, int, int, int, uint32_t*) const { return w; }
  static __device__ __forceinline__ void put(T* row, int c0, int k, int lane, const uint4& v, uint32_t*) {
    if (c0 + lane * 8 < k) *reinterpret_cast<uint4*>(row + c0 + lane * 8) = v;
  }
};
template <typename T>
struct Piece<T, false> {
  uint32_t w[4], last;
  // 1: the first element is the upper half of word 0
  static __device__ __forceinline__ int ahead(const T* row, int c0) { return static_cast<int>(reinterpret_cast<uintptr_t>(row + c0) & 2) / 2; }
  static __device__ __forceinline__ uint32_t* words(const T* row, int c0) {
    return reinterpret_cast<uint32_t*>(reinterpret_cast<uintptr_t>(row + c0) & ~uintptr_t(3));
  }
  __device__ __forceinline__ void fetch(const T* row, int c0, int k, int lane) {
    const int off = ahead(row, c0), n = min(256, k - c0);
    const uint32_t* p = words(row, c0);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = 2 * (j * 32 + lane) - off < n ? p[j * 32 + lane] : 0u;
    last = off && n == 256 ? p[128] : 0u;
  }
  __device__ __forceinline__ uint4 take(const T* row, int c0, int k, int lane, uint32_t* stage) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) stage[j * 32 + lane] = w[j];
    if (lane == 0) stage[128] = last;
    __syncwarp();
    const uint4 q = *reinterpret_cast<const uint4*>(stage + 4 * lane);
    const uint32_t u[5] = {q.x, q.y, q.z, q.w, stage[4 * lane + 4]};
    __syncwarp();
    uint32_t v[4];
    const int off = ahead(row, c0), n = k - c0 - lane * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = off ? __funnelshift_r(u[i], u[i + 1], 16) : u[i];
      if (2 * i + 1 >= n) v[i] = 2 * i < n ? v[i] & 0xFFFFu : 0u;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  static __device__ __forceinline__ void put(T* row, int c0, int k, int lane, const uint4& v, uint32_t* stage) {
    *reinterpret_cast<uint4*>(stage + 4 * lane) = v;
    __syncwarp();
    // A piece behind the row's end stores nothing.  (One that begins there would store its word 0 otherwise, which holds element
    // k - 1, another warp's, and what stands behind the row; a return in this place: 11328 rows of 961 50 us, so 46.)
    const int n = min(256, k - c0), off = n > 0 ? ahead(row, c0) : 0;
    uint32_t* p = words(row, c0);
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      const int i = j * 32 + lane, e = 2 * i - off;  // the word's lower element, -1 at least
      if (j == 4 && lane > 0) break;
      if (e >= n) continue;
      const uint32_t lower = off ? (i > 0 ? stage[i - 1] >> 16 : 0u) : stage[i] & 0xFFFFu;
      const uint32_t upper = off ? (i < 128 ? stage[i] << 16 : 0u) : stage[i] & 0xFFFF0000u;
      if (e >= 0 && e + 1 < n) p[i] = lower | upper;
      else if (e >= 0) *reinterpret_cast<uint16_t*>(p + i) = static_cast<uint16_t>(lower);
      else *(reinterpret_cast<uint16_t*>(p + i) + 1) = static_cast<uint16_t>(upper >> 16);
    }
    __syncwarp();
  }
};

// Over the block's threads: a warp's lanes, then the warps through `part`, which holds zeros behind them and is used by one
// reduction of every other row only.
__device__ __forceinline__ float add_block(float v, float* part) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, d));
  const int warps = blockDim.x >> 5;
  if (warps > 1) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < warps; i += 4) {  // the same order in every thread
      const float4 p = *reinterpret_cast<const float4*>(part + i);
      v = __fadd_rn(v, __fadd_rn(__fadd_rn(p.x, p.y), __fadd_rn(p.z, p.w)));
    }
  }
  return v;
}
// the largest of values >= 0, NaN where one is: as integers they compare alike, and a NaN (without its sign) is above infinity
__device__ __forceinline__ float max_block(float v, float* part) {
  unsigned u = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7FFFFFFFu);
  const int warps = blockDim.x >> 5;
  if (warps > 1) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = __uint_as_float(u);
    __syncthreads();
    for (int i = 0; i < warps; i += 4) {
      const uint4 p = *reinterpret_cast<const uint4*>(part + i);
      u = max(max(u, max(p.x, p.y)), max(p.z, p.w));
    }
  }
  return __uint_as_float(u);
}

// y / s: by the hardware's reciprocal (2^-22 or so) and Markstein's correction where s is within 2^+-100 (off by half a step and
// 2^-43), by the division itself elsewhere
__device__ __forceinline__ void divide8(float2 (&y)[4], const float2 (&s)[4]) {
  float least = fabsf(s[0].x), most = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) least = fminf(least, fminf(fabsf(s[e].x), fabsf(s[e].y))), most = max_abs(most, s[e].x, s[e].y);
  if (least > 7.9e-31f && most < 1.2e30f) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      y[e] = quotient(y[e], make_float2(-s[e].x, -s[e].y), make_float2(rcp_approx(s[e].x), rcp_approx(s[e].y)));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = make_float2(__fdiv_rn(y[e].x, s[e].x), __fdiv_rn(y[e].y, s[e].y));
  }
}
constexpr int kMaxWarps = 32;
}  // namespace qrows

// CH chunks of 8 elements per thread; the block's threads hold a row
template <typename T, bool VEC, int CH>
__global__ void __launch_bounds__(1024) quant_rows_kernel(const QuantRowsArgs a) {
  using namespace qrows;
  __shared__ __align__(16) float part[2][3][kMaxWarps];
  for (int i = threadIdx.x; i < 6 * kMaxWarps; i += blockDim.x) (&part[0][0][0])[i] = 0.f;
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int k = a.k;
  __shared__ __align__(16) uint32_t stages[VEC ? 1 : kMaxWarps][VEC ? 4 : 132];
  uint32_t* stage = stages[VEC ? 0 : threadIdx.x >> 5];
  const int lane = threadIdx.x & 31;
  auto column = [&](int i) { return (i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8; };
  auto column0 = [&](int i) { return (i * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x) - lane) * 8; };  // lane 0's
  Piece<T, VEC> rx[CH], rr[CH];
  auto fetch = [&](long long row) {
    if (row >= a.m) return;
    const T* x = static_cast<const T*>(a.x) + row * a.x_rs;
    const T* r = static_cast<const T*>(a.residual) + row * a.residual_rs;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      rx[i].fetch(x, column0(i), k, lane);
      if (a.residual) rr[i].fetch(r, column0(i), k, lane);
    }
  };
  // a chunk's elements behind the row's end set to zero (where chunks are read whole, the chunk is in or out)
  auto clip = [&](float2 (&v)[4], int i) {
    if constexpr (!VEC) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (column(i) + 2 * e >= k) v[e].x = 0.f;
        if (column(i) + 2 * e + 1 >= k) v[e].y = 0.f;
      }
    }
  };
  fetch(blockIdx.x);
  int turn = 0;
  for (long long row = blockIdx.x; row < a.m; row += gridDim.x, turn ^= 1) {
    float2 y[CH][4];
#pragma unroll
    for (int i = 0; i < CH; ++i) unpack8<T>(y[i], rx[i].take(static_cast<const T*>(a.x) + row * a.x_rs, column0(i), k, lane, stage));
    if (a.residual) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float2 v[4];
        unpack8<T>(v, rr[i].take(static_cast<const T*>(a.residual) + row * a.residual_rs, column0(i), k, lane, stage));
#pragma unroll
        for (int e = 0; e < 4; ++e) y[i][e] = __fadd2_rn(y[i][e], v[e]);
      }
    }
    fetch(row + gridDim.x);
    if (a.sum) {
#pragma unroll
      for (int i = 0; i < CH; ++i) Piece<T, VEC>::put(static_cast<T*>(a.sum) + row * a.sum_rs, column0(i), k, lane, pack8<T>(y[i]), stage);
    }
    if (a.weight) {
      const float inv = __fdiv_rn(1.f, static_cast<float>(k));
      float power, eps = a.eps;  // what the root is taken of
      // One round over the row, and another for a few: the choices are the row's, so its threads agree, and each is made once.
      for (bool scaled = false, centred = false;;) {
        float2 sum = both(0.f);
        float mean = 0.f, squares = __int_as_float(0x7f800000);
        if (a.bias) {
#pragma unroll
          for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = __fadd2_rn(sum, y[i][e]);
          mean = __fdiv_rn(add_block(__fadd_rn(sum.x, sum.y), part[turn][0]), static_cast<float>(k));
          sum = both(0.f);
        }
        if (fabsf(mean) < 1.2676506002282294e30f || scaled) {  // (from 2^100 on centring might overflow)
          if (a.bias) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
              if (column(i) >= k) continue;
#pragma unroll
              for (int e = 0; e < 4; ++e) y[i][e] = __fadd2_rn(y[i][e], both(-mean));
              clip(y[i], i);
            }
          }
#pragma unroll
          for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = __ffma2_rn(y[i][e], y[i][e], sum);
          squares = add_block(__fadd_rn(sum.x, sum.y), part[turn][1]);
        }
        const float variance = __fmul_rn(squares, inv);
        power = __fmaf_rn(squares, inv, eps);
        const bool fits = power >= 8.3e-25f && power < __int_as_float(0x7f800000), far = mean != 0.f && 0.0625f * mean * mean >= variance;
        if (fits && !far) break;
        if (!fits && !scaled) {
          // Squares beyond fp32's range (components above 1e17 or so), or below it with an eps as small: the row is scaled by 2^-80
          // or 2^80, which a norm does not notice.  (What is scaled up lies below 2^-32: centred, and not over 2^8 deviations.)
          const float by = power < 1.f ? 1.2089258196146292e24f : 8.271806125530277e-25f;
#pragma unroll
          for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[i][e] = __fmul2_rn(y[i][e], both(by));
          eps = __fmul_rn(__fmul_rn(eps, by), by);
          scaled = true;
        } else if (far && !centred) {
          // A mean of more than 4 deviations: as a sum of large numbers it is off by a step of them or more, so the mean of what is
          // left is taken off as well (8192 rows of 4096 with all, every one such a row: 64 us, none: 53; the sum of what is left
          // taken beside the squares of every row: 62)
          centred = true;
        } else {
          break;
        }
        __syncthreads();  // the partial sums are read before they are written again
      }
      const float2 rstd = both(power == 0.f ? 0.f : __frsqrt_rn(power));  // 0: every y is
      const T* w = static_cast<const T*>(a.weight);
      const T* b = static_cast<const T*>(a.bias);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (column(i) >= k) continue;
        float2 g[4];
        unpack8<T>(g, raw8<T, VEC>(w, column(i), k));
#pragma unroll
        for (int e = 0; e < 4; ++e) y[i][e] = __fmul2_rn(__fmul2_rn(y[i][e], rstd), g[e]);
        if (a.bias) {
          unpack8<T>(g, raw8<T, VEC>(b, column(i), k));
#pragma unroll
          for (int e = 0; e < 4; ++e) y[i][e] = __fadd2_rn(y[i][e], g[e]);
        }
      }
    }
    if (a.smooth) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (column(i) >= k) continue;
        float2 d[4];
        if (VEC || (column(i) + 8 <= k && reinterpret_cast<uintptr_t>(a.smooth) % 16 == 0)) {
          const float4* s = reinterpret_cast<const float4*>(a.smooth + column(i));
          const float4 s0 = __ldg(s), s1 = __ldg(s + 1);
          d[0] = make_float2(s0.x, s0.y), d[1] = make_float2(s0.z, s0.w), d[2] = make_float2(s1.x, s1.y), d[3] = make_float2(s1.z, s1.w);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int c = column(i) + 2 * e;
            d[e] = make_float2(c < k ? __ldg(a.smooth + c) : 1.f, c + 1 < k ? __ldg(a.smooth + c + 1) : 1.f);
          }
        }
        divide8(y[i], d);
      }
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      clip(y[i], i);  // (0 * infinity behind the end is no element's)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max_abs(top, y[i][e].x, y[i][e].y);
    }
    top = max_block(top, part[turn][2]);
    const bool finite = top < __int_as_float(0x7f800000);
    const float scale = finite ? __fdiv_rn(top, 127.f) : __int_as_float(0x7fc00000);
    if (threadIdx.x == 0) a.scale[row] = scale;
    const bool plain = scale > 8.6e-19f && scale < 1.2e18f;  // 2^+-60
    const float2 r = both(plain ? __frcp_rn(scale) : 0.f);
    int8_t* codes = a.codes + row * a.codes_rs;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer in the low bits, ties to even
      float2 t[4];
      if (plain) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = __fadd2_rn(quotient(y[i][e], both(-scale), r), both(kRound));  // (at most 127 (1 + 2^-23))
      } else {
        auto code = [&](float v) {
          const float q = scale > 0.f ? __fdiv_rn(v, scale) : 0.f;  // (NaN: no)
          return __fadd_rn(fminf(fmaxf(q, -127.f), 127.f), kRound);
        };
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = make_float2(code(y[i][e].x), code(y[i][e].y));
      }
      uint32_t packed[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t lo = __byte_perm(__float_as_uint(t[2 * h].x), __float_as_uint(t[2 * h].y), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(t[2 * h + 1].x), __float_as_uint(t[2 * h + 1].y), 0x0040);
        packed[h] = __byte_perm(lo, hi, 0x5410);
      }
      if (column(i) + 8 <= k && (VEC || reinterpret_cast<uintptr_t>(codes) % 8 == 0)) {
        *reinterpret_cast<uint2*>(codes + column(i)) = make_uint2(packed[0], packed[1]);
      } else if (!VEC) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (column(i) + e < k) codes[column(i) + e] = static_cast<int8_t>(packed[e / 4] >> (8 * (e % 4)));
      }
      if (a.values) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = __fmul2_rn(__fadd2_rn(t[e], both(-kRound)), both(scale));
        Piece<T, VEC>::put(static_cast<T*>(a.values) + row * a.values_rs, column0(i), k, lane, pack8<T>(t), stage);
      }
    }
  }
}

}  // namespace svla
