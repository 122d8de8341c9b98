// Appending keys and values to a paged cache, with the position rotation on the way.
//
// Token i of sequence b (packed row t = cu_q[b] + i, of n_b = cu_q[b + 1] - cu_q[b] new ones) goes to cache entry
//   n = kv_len[b] - n_b + i                (kv_len counts the new tokens)
// in page page_table[b, n / page], slot n % page.  Rotate-half at position p = pos[t], or n without positions:
//   o1 = x1 cos - x2 sin,  o2 = x2 cos + x1 sin      (pairs (i, i + D / 2), (cos, sin) = rope_cs[p][i], fp32; both
// products and their sum rounded to fp32, so that the same operations elsewhere give the same bits).
//
// 16-bit pages [kv_heads][2][page][D]: the rotated key and the value, rounded once to the type.
// 4-bit pages, per kv head: key codes [page][D / 2] bytes, value codes, then for keys and for values bf16 (step, low)
// pairs [page][D / 32].  Per group of 32 dimensions
//   low = bf16(min),  step = bf16((max - min) / 15),  code = clamp(rint((x - low) / step), 0, 15)   (0 for step 0)
// and the entry stands for low + step * code.  A linear code with its own offset spends all 16 codes on the group's
// range, and the codes are computed against the rounded pair that the reader sees.  An entry is off by half a step where
// its code is not clamped; rounding the pair to bf16 moves the ends of the range by 2^-8 |low| at the lower and by 2^-8 |low|
// + 15 steps 2^-8 at the upper, and what lies beyond them is clamped.  So a group whose offset is large beside its range
// loses more: 100.2 to 101.2 has step 0.067 and low 100, and its largest value reads back as 101, three steps off.  Both
// quotients are true divisions: bf16 inputs often lie exactly between two codes, and a reciprocal's last bit would then
// decide.  A group with a NaN, an infinity or a range beyond fp32's largest number reads back as NaN.
//
// Work split: a warp takes one token and, when there are few tokens, a share of its heads; D / 16 lanes hold a head's row (8
// dimensions of each half), so a warp's accesses are whole 128- or 256-byte rows, the rotation pairs meet in one lane, the
// token's (cos, sin) are read once for all heads, and a quantisation group is 4 lanes (two shuffles per extremum).  The
// first row is on its way while the token's place is looked up, every other one while the one before is worked on.
// Bound by memory traffic at many tokens (26337 rows of 48 heads into 4 bits, D = 128: 694 MB in 127 us, 5.5 TB/s, in a
// graph, 136 where calls follow each other; with library divisions for the quotients 195 us), by latency at few.  Measured
// for 15579 rows of 25 heads at D = 64 (104 MB in 26 us) and left: four tokens per warp 34 us, two rows ahead 30 us, whole
// blocks of tokens staged in shared memory 29 us.
#pragma once

#include "serving_common.cuh"

namespace svla {

struct KvAppendArgs {
  const void *q, *k, *v;   // [total, heads * D] with row strides; q may be null
  void *qo, *ko, *vo;      // outputs; ko / vo may be null
  uint8_t* cache;
  const int *cu_q, *kv_len, *table, *pos;
  const float2* cs;        // [max_pos][D / 2] or null (no rotation)
  long long q_rs, k_rs, v_rs, qo_rs, ko_rs, vo_rs, table_rs;
  int batch, total, hq, hkv, page, n_pages, max_pages, max_pos;
  int parts;               // warps per token
  int* err;
};

namespace append_detail {
constexpr int kWarps = 4;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// d / s correctly rounded, r = 1 / s correctly rounded: P. Markstein's correction of a quotient (Computation of elementary
// functions on the IBM RISC System/6000 processor, 1990), q + (d - q s) r with two fused operations.  Checked for all
// significands of a bf16 s and an fp32 d; steps beyond 2^+-60 take the division itself.
__device__ __forceinline__ float quotient(float d, float s, float r) {
  const float q = __fmul_rn(d, r);
  return __fmaf_rn(__fmaf_rn(-q, s, d), r, q);
}

// 8 values of a lane, quantised with the 4 lanes of their group; x becomes what the codes stand for
__device__ __forceinline__ void quantise8(float (&x)[8], uint32_t& codes, uint32_t& pair) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = min_nan(lo, x[e]);
    hi = max_nan(hi, x[e]);
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, d));
  }
  pair = pack_bf16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f), lo);
  const float s = __uint_as_float(pair << 16), m = __uint_as_float(pair & 0xFFFF0000u);
  codes = 0u;
  constexpr float kC = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer (ties to even) in the low bits
  if (s > 8.6e-19f && s < 1.2e18f) {
    const float r = __frcp_rn(s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = fminf(fmaxf(quotient(__fsub_rn(x[e], m), s, r), 0.f), 15.f);
      const float t = __fadd_rn(q, kC);
      codes |= (__float_as_uint(t) & 15u) << (4 * e);
      x[e] = __fmaf_rn(__fsub_rn(t, kC), s, m);  // the product is exact
    }
  } else {  // a step of zero, a tiny or a huge one, or none (NaN)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float c = s > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[e], m), s)) : 0.f;
      c = fminf(fmaxf(c, 0.f), 15.f);
      codes |= static_cast<uint32_t>(c) << (4 * e);
      x[e] = __fadd_rn(__fmul_rn(c, s), m);
    }
  }
}

template <typename T>
__device__ __forceinline__ void unpack8(float (&x)[8], const uint4& w) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = serving::unpack2<T>(u[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(serving::pack2<T>(x[0], x[1]), serving::pack2<T>(x[2], x[3]), serving::pack2<T>(x[4], x[5]),
                    serving::pack2<T>(x[6], x[7]));
}
}  // namespace append_detail

// 4 bits: at most 64 registers, 32 warps per SM (26337 rows of 48 heads at D = 128: 127 us, 160 with 86 registers)
template <typename T, int D, int BITS>
__global__ void __launch_bounds__(append_detail::kWarps * 32, BITS == 4 ? 8 : 1) kv_append_kernel(const KvAppendArgs a) {
  using namespace append_detail;
  constexpr int kLanes = D / 16, kSlots = 32 / kLanes;  // lanes of a head's row, rows per warp
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long task = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(task / a.parts), part = static_cast<int>(task % a.parts);
  if (t >= a.total) return;
  const int row = lane / kLanes, c = (lane % kLanes) * 8;  // this lane: dimensions c.. and D / 2 + c..
  const int nq = a.q ? a.hq : 0, heads = nq + 2 * a.hkv;
  // input row of head h: query heads, then key heads, then value heads
  auto source = [&](int h) -> const T* {
    const size_t row_t = static_cast<size_t>(t);
    if (h < nq) return static_cast<const T*>(a.q) + row_t * a.q_rs + h * D;
    h -= nq;
    if (h < a.hkv) return static_cast<const T*>(a.k) + row_t * a.k_rs + h * D;
    return static_cast<const T*>(a.v) + row_t * a.v_rs + (h - a.hkv) * D;
  };
  const int stride = kSlots * a.parts;
  int h0 = part * kSlots;
  // the first row is on its way while the token's place is looked up
  uint4 w1 = make_uint4(0, 0, 0, 0), w2 = w1;
  if (h0 + row < heads) {
    const T* s = source(h0 + row);
    w1 = *reinterpret_cast<const uint4*>(s + c);
    w2 = *reinterpret_cast<const uint4*>(s + D / 2 + c);
  }
  const int b = serving::find_sequence(a.cu_q, a.batch, t, lane);
  if (b < 0) return;  // a row behind the last sequence
  const int first = __ldg(a.cu_q + b), n_new = __ldg(a.cu_q + b + 1) - first;
  const int n = __ldg(a.kv_len + b) - n_new + (t - first);

  // the cache entry's page and slot; -1: there is none
  int page = -1, slot = 0;
  if (n >= 0 && n / a.page < a.max_pages) {
    page = __ldg(a.table + static_cast<size_t>(b) * a.table_rs + n / a.page);
    slot = n % a.page;
  }
  const bool kept = page >= 0 && page < a.n_pages;
  if (!kept && lane == 0) record_error(a.err, serving::kErrBadPage);

  float cs_c[8], cs_s[8];
  if (a.cs) {
    int p = a.pos ? __ldg(a.pos + t) : n;
    p = p < 0 ? 0 : (p >= a.max_pos ? a.max_pos - 1 : p);
    const float4* src = reinterpret_cast<const float4*>(a.cs + static_cast<size_t>(p) * (D / 2) + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = __ldg(src + i);
      cs_c[2 * i] = f.x;
      cs_s[2 * i] = f.y;
      cs_c[2 * i + 1] = f.z;
      cs_s[2 * i + 1] = f.w;
    }
  }
  for (; h0 < heads; h0 += stride) {
    const int h = h0 + row;
    const bool in = h < heads;
    float x1[8], x2[8];
    unpack8<T>(x1, w1);
    unpack8<T>(x2, w2);
    if (h + stride < heads) {  // the next row is on its way while this one is rotated
      const T* s = source(h + stride);
      w1 = *reinterpret_cast<const uint4*>(s + c);
      w2 = *reinterpret_cast<const uint4*>(s + D / 2 + c);
    }
    const int kvh = h < nq ? -1 : (h - nq) % a.hkv;
    const bool is_v = h >= nq + a.hkv;
    if (a.cs && !is_v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float o1 = __fsub_rn(__fmul_rn(x1[e], cs_c[e]), __fmul_rn(x2[e], cs_s[e]));
        const float o2 = __fadd_rn(__fmul_rn(x2[e], cs_c[e]), __fmul_rn(x1[e], cs_s[e]));
        x1[e] = o1;
        x2[e] = o2;
      }
    }
    uint32_t code1, code2, pair1, pair2;
    if constexpr (BITS == 4) {
      if (h0 + kSlots > nq) {  // warp-uniform: some row of the warp is a key or a value
        float y1[8], y2[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y1[e] = x1[e];
          y2[e] = x2[e];
        }
        quantise8(y1, code1, pair1);
        quantise8(y2, code2, pair2);
        if (kvh >= 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x1[e] = y1[e];
            x2[e] = y2[e];
          }
        }
      }
    }
    if (!in) continue;
    const uint4 o1 = pack8<T>(x1), o2 = pack8<T>(x2);
    T* dst = nullptr;
    if (kvh < 0) {
      dst = static_cast<T*>(a.qo) + static_cast<size_t>(t) * a.qo_rs + h * D;
    } else if (is_v) {
      if (a.vo) dst = static_cast<T*>(a.vo) + static_cast<size_t>(t) * a.vo_rs + kvh * D;
    } else if (a.ko) {
      dst = static_cast<T*>(a.ko) + static_cast<size_t>(t) * a.ko_rs + kvh * D;
    }
    if (dst) {
      *reinterpret_cast<uint4*>(dst + c) = o1;
      *reinterpret_cast<uint4*>(dst + D / 2 + c) = o2;
    }
    if (kvh < 0 || !kept) continue;
    const size_t block = static_cast<size_t>(page) * a.hkv + kvh;  // this head's part of the page
    if constexpr (BITS == 16) {
      T* entry = reinterpret_cast<T*>(a.cache) + ((block * 2 + (is_v ? 1 : 0)) * a.page + slot) * D;
      *reinterpret_cast<uint4*>(entry + c) = o1;
      *reinterpret_cast<uint4*>(entry + D / 2 + c) = o2;
    } else {
      uint8_t* base = a.cache + block * (static_cast<size_t>(a.page) * (D + D / 4));
      uint8_t* codes = base + (static_cast<size_t>(is_v ? a.page : 0) + slot) * (D / 2);
      *reinterpret_cast<uint32_t*>(codes + c / 2) = code1;
      *reinterpret_cast<uint32_t*>(codes + D / 4 + c / 2) = code2;
      if ((lane & 3) == 0) {
        uint8_t* pairs = base + static_cast<size_t>(a.page) * D + (static_cast<size_t>(is_v ? a.page : 0) + slot) * (D / 8);
        *reinterpret_cast<uint32_t*>(pairs + (c / 32) * 4) = pair1;
        *reinterpret_cast<uint32_t*>(pairs + ((D / 2 + c) / 32) * 4) = pair2;
      }
    }
  }
}

// cs[p][i] = (cos, sin)(p / max_wavelength^(2 i / D)) with the angle in 64 bits: at position 100000 an fp32 angle is
// off by up to 0.004 radians, more than bf16 rows resolve.
__global__ void rope_table_wide_kernel(float2* cs, int max_pos, int half, double max_wavelength) {
  pdl_wait();
  pdl_trigger();
  const long long idx = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (idx >= static_cast<long long>(max_pos) * half) return;
  const int i = static_cast<int>(idx % half);
  const double angle = static_cast<double>(idx / half) * pow(max_wavelength, -static_cast<double>(i) / half);
  double s, c;
  sincos(angle, &s, &c);
  cs[idx] = make_float2(static_cast<float>(c), static_cast<float>(s));
}

}  // namespace svla
