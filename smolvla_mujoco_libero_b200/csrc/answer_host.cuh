// Host-side checks shared by the operators that answer with the text model in 8-bit integers.
#pragma once

#include "host.cuh"

namespace svla {

inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// rows of `width` elements of `size` bytes, `rs` apart
inline int32_t check_rows(const char* who, const char* name, const void* p, int64_t rs, int64_t width, int size) {
  if (!p) return fail(SVLA_ERR_ARG, "%s: %s is null", who, name);
  if (!aligned(p, size)) return fail(SVLA_ERR_ARG, "%s: %s must be aligned to its elements", who, name);
  if (rs < width) return fail(SVLA_ERR_ARG, "%s: %s has a row stride below %lld", who, name, static_cast<long long>(width));
  return SVLA_OK;
}

template <typename Kern>
int32_t allow_smem(Kern kern, int bytes, bool (&configured)[64]) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(SVLA_ERR_ARG, "device index %d out of range", dev);
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return fail(SVLA_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  return SVLA_OK;
}

}  // namespace svla
