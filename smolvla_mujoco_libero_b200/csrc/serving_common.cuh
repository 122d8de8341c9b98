// Shared pieces of the serving kernels (packed-prompt attention, paged cache append, paged attention): the two
// 16-bit element types, mma.sync / ldmatrix / cp.async wrappers and the search for a token's sequence.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "ptx.cuh"

namespace svla {
namespace serving {

// device error word: a cache index outside the page table, or a page outside the cache (the row is not written, the
// keys are not read)
constexpr int kErrBadPage = 104;

constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16_rn(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}

// Softmax weights, rounded to the type for the second product, are 2^(score - maximum + lift); the lift cancels in O / l.
// A lazy maximum lets them grow by 2^8, so fp16, which ends at 2^16, has room for 2^7: weights are rounded by 2^-11 of
// themselves down to 2^-21 of the largest, and below by 2^-32 of the largest (half a subnormal step, 2^-25).  bf16 has
// fp32's range.
template <typename T>
constexpr float kWeightLift = 0.f;
template <>
constexpr float kWeightLift<__half> = 7.f;

// bits that are all ones in an infinity or a NaN of the type, for two packed values
template <typename T>
__device__ __forceinline__ bool any_nonfinite(uint32_t w);
template <>
__device__ __forceinline__ bool any_nonfinite<__nv_bfloat16>(uint32_t w) {
  return (((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u) != 0u;
}
template <>
__device__ __forceinline__ bool any_nonfinite<__half>(uint32_t w) {
  return (((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u) != 0u;
}

// D (16 x 8, fp32) += A (16 x 16) B (16 x 8)
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// the first product of an accumulator: D = A B
template <typename T>
__device__ __forceinline__ void mma16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816_first<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p))
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p))
               : "memory");
}
// 8 x 8 matrix of 16-bit elements, transposed across the warp
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// 16-byte asynchronous copy; src_bytes = 0 fills the destination with zeros and reads nothing
__device__ __forceinline__ void copy16(void* dst, const void* src, int src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(src_bytes)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// one lane of a converged warp; the compiler knows that it is one, which `lane == 0` does not tell it
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// Bounded wait of a whole warp.  A phase that is over already, the usual case here, is seen by test_wait in about 40
// cycles; try_wait takes 100 then, and one lane polling for the others 200.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int* err) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  bool ok = done != 0;
  if (!ok) {
    for (uint32_t i = 0; i < kSpinLimit && !ok; ++i) ok = mbar_try_wait(bar, parity);
    if (!ok && (threadIdx.x & 31) == 0) record_error(err, kErrMbarTimeout);
  }
  return __all_sync(0xffffffffu, ok);
}

// The sequence of packed row t: the b with starts[b] <= t < starts[b + 1], or -1.  Every lane of the warp calls it and
// gets the answer; each round reads 32 entries at once and narrows the range 32 times, so 1024 sequences take two
// dependent reads.
__device__ __forceinline__ int find_sequence(const int* starts, int batch, int t, int lane) {
  if (__ldg(starts) > t || __ldg(starts + batch) <= t) return -1;
  int lo = 0, hi = batch;  // starts[lo] <= t < starts[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + (lane + 1) * step;
    const bool below = at < hi && __ldg(starts + at) <= t;
    lo += __popc(__ballot_sync(0xffffffffu, below)) * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

// [begin, end) of sequence b inside a tensor of `total` rows: whatever `starts` holds, no row outside it
struct Span {
  int begin, end;
};
__device__ __forceinline__ Span span_of(const int* starts, int b, int total) {
  const int s = min(max(__ldg(starts + b), 0), total), e = min(max(__ldg(starts + b + 1), s), total);
  return {s, e};
}

}  // namespace serving
}  // namespace svla
