// C-ABI entry points of the operators that answer with the text model in 8-bit integers (include/svla.h): rows normalised
// and quantised with a scale each, and products of such rows.  Argument checks, dispatch and launches; nothing allocates memory.
#include <cmath>
#include <cstring>

#include "answer_host.cuh"
#include "linear_i8.cuh"
#include "quant_rows.cuh"

namespace svla {
namespace {

int32_t check_dtype16(const char* who, int32_t dtype) {
  if (dtype != SVLA_DT_BF16 && dtype != SVLA_DT_HALF) return fail(SVLA_ERR_ARG, "%s: dtype must be BF16 or HALF (got %d)", who, dtype);
  return SVLA_OK;
}

// ---------------------------------------------------------------- quantised rows
template <typename T, bool VEC, int CH>
int32_t launch_quant(const QuantRowsArgs& a, cudaStream_t st) {
  static int resident[64][qrows::kMaxWarps + 1] = {{0}};  // blocks that fit an SM
  auto kern = quant_rows_kernel<T, VEC, CH>;
  const int warps = (a.k + CH * 256 - 1) / (CH * 256);
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(SVLA_ERR_ARG, "device index %d out of range", dev);
  if (resident[dev][warps] == 0) {
    int n = 0;
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, warps * 32, 0);
    if (e != cudaSuccess) return fail(SVLA_ERR_CUDA, "cudaOccupancyMaxActiveBlocksPerMultiprocessor: %s", cudaGetErrorString(e));
    resident[dev][warps] = n < 1 ? 1 : n;
  }
  const int blocks = resident[dev][warps] * sm_count();
  return launch(kern, dim3(static_cast<unsigned>(a.m < blocks ? a.m : blocks)), dim3(warps * 32), 0, st, "quant_rows_kernel", a);
}

template <typename T, bool VEC>
int32_t launch_quant_t(const QuantRowsArgs& a, cudaStream_t st) {
  // by k alone, so that a row's sums are the same in any batch (one row of 960 with a chunk per thread: 2.1 us, with two 2.7)
  if (a.k <= 16384) return launch_quant<T, VEC, 2>(a, st);
  return launch_quant<T, VEC, 4>(a, st);
}

// ---------------------------------------------------------------- int8 products
int32_t make_tmap_i8(CUtensorMap* map, const void* base, uint64_t k, uint64_t rows, uint64_t rs, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(SVLA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {k, rows};
  cuuint64_t strides[1] = {rs};
  cuuint32_t box[2] = {li8::kSlice, box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SVLA_ERR_ARG, "cuTensorMapEncodeTiled (int8 rows) failed (%d)", static_cast<int>(r));
  return SVLA_OK;
}

// the output as (column, row) with a warp's box of 32 rows of 64 bytes
int32_t make_tmap_out(CUtensorMap* map, const svla_linear_i8_desc* d, int size) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(SVLA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(d->n), static_cast<cuuint64_t>(d->m)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(d->out_rs) * size};
  cuuint32_t box[2] = {64u / size, 32};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, d->out, dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SVLA_ERR_ARG, "cuTensorMapEncodeTiled (output) failed (%d)", static_cast<int>(r));
  return SVLA_OK;
}

template <typename T, int MT, bool GATED>
int32_t launch_few(LinearI8Args& a, const svla_linear_i8_desc* d, cudaStream_t st) {
  static bool configured[64] = {false};
  auto kern = linear_i8_few_kernel<T, MT, GATED>;
  if (int32_t rc = allow_smem(kern, li8::Few<MT, GATED>::kBytes, configured)) return rc;
  if (int32_t rc = make_tmap_i8(&a.tx, d->x, d->k, d->m, d->x_rs, MT)) return rc;
  if (int32_t rc = make_tmap_i8(&a.tw, d->w, d->k, static_cast<uint64_t>(d->n) * (GATED ? 2 : 1), d->w_rs, 128)) return rc;
  a.tiles_m = (d->m + MT - 1) / MT, a.tiles_n = (d->n + 127) / 128;
  const long long tiles = static_cast<long long>(a.tiles_m) * a.tiles_n;
  const int slices = (d->k + li8::kSlice - 1) / li8::kSlice;
  // K is shared where a tile's parts keep 5 slices at least, within one round over the SMs: adding them up costs half a us with one
  // token and 2 with 128 (K = 4096, N = 4096, 1 token: 6.8 us, alone 11.4; 128 tokens 10.9 and 15.4; K = 960, N = 1600, 1 token:
  // 4.4 us by 8, alone 4.0; 128 tokens 7.5 and 5.8)
  a.splits = 1;
  while (a.splits < 8 && tiles * a.splits * 2 <= sm_count() && a.splits * 10 <= slices) a.splits *= 2;
  if (tiles * a.splits > 0x7fffffffll) return fail(SVLA_ERR_ARG, "svla_linear_i8: too many tiles");
  return launch_cluster(kern, dim3(static_cast<unsigned>(tiles * a.splits)), dim3(li8::kFewThreads), li8::Few<MT, GATED>::kBytes, st,
                        "linear_i8_few_kernel", static_cast<unsigned>(a.splits), a);
}

template <typename T, bool GATED>
int32_t launch_many(LinearI8Args& a, const svla_linear_i8_desc* d, cudaStream_t st) {
  static bool configured[64] = {false};
  auto kern = linear_i8_many_kernel<T, GATED>;
  if (int32_t rc = allow_smem(kern, li8::Many::kBytes, configured)) return rc;
  if (int32_t rc = make_tmap_i8(&a.tx, d->x, d->k, d->m, d->x_rs, 128)) return rc;
  if (int32_t rc = make_tmap_i8(&a.tw, d->w, d->k, static_cast<uint64_t>(d->n) * (GATED ? 2 : 1), d->w_rs, 128)) return rc;
  a.tiles_m = (d->m + 255) / 256, a.tiles_n = (d->n + (GATED ? 127 : 255)) / (GATED ? 128 : 256);
  const long long tiles = static_cast<long long>(a.tiles_m) * a.tiles_n;
  if (tiles > 0x7fffffffll / 2) return fail(SVLA_ERR_ARG, "svla_linear_i8: too many tiles");
  const int size = static_cast<int>(sizeof(T));
  auto by_16 = [&](const void* p, int64_t rs) { return aligned(p, 16) && rs * size % 16 == 0; };
  a.staged = static_cast<int64_t>(d->n) * size % 16 == 0 && by_16(a.out, a.out_rs) && (!a.residual || by_16(a.residual, a.residual_rs));
  if (a.staged) if (int32_t rc = make_tmap_out(&a.to, d, size)) return rc;
  const long long pairs = sm_count() / 2;
  return launch_cluster(kern, dim3(static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs))), dim3(li8::kManyThreads),
                        li8::Many::kBytes, st, "linear_i8_many_kernel", 2, a);
}

template <typename T, bool GATED>
int32_t launch_linear(LinearI8Args& a, const svla_linear_i8_desc* d, cudaStream_t st) {
  // Up to 128 rows the weights are read once by either kernel, and the one for few rows takes 17.8 us for 128 x 49280 x 960 where
  // the other takes 22.4.  Beyond, it moves twice the bytes per product and starts 3 us earlier: it is the faster one while its
  // tiles fit one round over the SMs (few / many, us: 768 x 1600 x 960, 78 tiles, 6.0 / 8.8; 512 x 4096 x 4096, 128 tiles, 15.7 /
  // 16.3; 768 x 4096 x 4096, 192 tiles, 17.2 / 16.8; 177 x 49280 x 960, 770 tiles, 26.1 / 21.8; 49280 columns in fp32)
  const long long tiles = (static_cast<long long>(d->m) + 127) / 128 * ((static_cast<long long>(d->n) + 127) / 128);
  if (d->impl == SVLA_LINEAR_MANY || (d->impl == SVLA_LINEAR_AUTO && d->m > 128 && tiles > sm_count())) return launch_many<T, GATED>(a, d, st);
  if (d->m <= 16) return launch_few<T, 16, GATED>(a, d, st);
  if (d->m <= 32) return launch_few<T, 32, GATED>(a, d, st);
  if (d->m <= 64) return launch_few<T, 64, GATED>(a, d, st);
  return launch_few<T, 128, GATED>(a, d, st);
}

template <typename T>
int32_t launch_linear_t(LinearI8Args& a, const svla_linear_i8_desc* d, cudaStream_t st) {
  return d->gated ? launch_linear<T, true>(a, d, st) : launch_linear<T, false>(a, d, st);
}

}  // namespace
}  // namespace svla

using namespace svla;

extern "C" {

int32_t svla_quant_rows(const svla_quant_rows_desc* d, svla_stream_t stream) {
  const char* who = "svla_quant_rows";
  if (!d) return fail(SVLA_ERR_ARG, "%s: null descriptor", who);
  if (int32_t rc = check_dtype16(who, d->dtype)) return rc;
  if (d->m < 0 || d->k < 1 || d->k > 32768) return fail(SVLA_ERR_ARG, "%s: rows of 1 to 32768 elements (got %d of %d)", who, d->m, d->k);
  if (!(d->eps >= 0.f) || std::isinf(d->eps)) return fail(SVLA_ERR_ARG, "%s: eps must be finite and not negative (got %g)", who, d->eps);
  if (d->bias && !d->weight) return fail(SVLA_ERR_ARG, "%s: bias without weight", who);
  if (d->m == 0) return SVLA_OK;
  if (int32_t rc = check_rows(who, "x", d->x, d->x_rs, d->k, 2)) return rc;
  if (d->residual) if (int32_t rc = check_rows(who, "residual", d->residual, d->residual_rs, d->k, 2)) return rc;
  if (int32_t rc = check_rows(who, "codes", d->codes, d->codes_rs, d->k, 1)) return rc;
  if (!d->scale || !aligned(d->scale, 4)) return fail(SVLA_ERR_ARG, "%s: scale is null or not aligned", who);
  if (d->sum) if (int32_t rc = check_rows(who, "sum", d->sum, d->sum_rs, d->k, 2)) return rc;
  if (d->values) if (int32_t rc = check_rows(who, "values", d->values, d->values_rs, d->k, 2)) return rc;
  if (!aligned(d->weight, 2) || !aligned(d->bias, 2) || !aligned(d->smooth, 4))
    return fail(SVLA_ERR_ARG, "%s: weight, bias or smooth is not aligned to its elements", who);
  QuantRowsArgs a;
  std::memset(&a, 0, sizeof(a));
  a.x = d->x, a.residual = d->residual, a.weight = d->weight, a.bias = d->bias, a.smooth = d->smooth;
  a.codes = d->codes, a.scale = d->scale, a.sum = d->sum, a.values = d->values;
  a.x_rs = d->x_rs, a.residual_rs = d->residual_rs, a.codes_rs = d->codes_rs, a.sum_rs = d->sum_rs, a.values_rs = d->values_rs;
  a.m = d->m, a.k = d->k, a.eps = d->eps;
  auto rows16 = [](const void* p, int64_t rs) { return !p || (aligned(p, 16) && rs % 8 == 0); };
  const bool vec = d->k % 8 == 0 && rows16(d->x, d->x_rs) && rows16(d->residual, d->residual_rs) && rows16(d->sum, d->sum_rs) &&
                   rows16(d->values, d->values_rs) && aligned(d->weight, 16) && aligned(d->bias, 16) && aligned(d->smooth, 16) &&
                   aligned(d->codes, 8) && d->codes_rs % 8 == 0;
  if (d->dtype == SVLA_DT_HALF) return vec ? launch_quant_t<__half, true>(a, cs(stream)) : launch_quant_t<__half, false>(a, cs(stream));
  return vec ? launch_quant_t<__nv_bfloat16, true>(a, cs(stream)) : launch_quant_t<__nv_bfloat16, false>(a, cs(stream));
}

int32_t svla_linear_i8(const svla_linear_i8_desc* d, svla_stream_t stream) {
  const char* who = "svla_linear_i8";
  if (!d) return fail(SVLA_ERR_ARG, "%s: null descriptor", who);
  if (d->dtype != SVLA_DT_BF16 && d->dtype != SVLA_DT_HALF && d->dtype != SVLA_DT_FLOAT)
    return fail(SVLA_ERR_ARG, "%s: dtype must be BF16, HALF or FLOAT (got %d)", who, d->dtype);
  if (d->m < 0 || d->n < 0) return fail(SVLA_ERR_ARG, "%s: negative m or n", who);
  // fewer than 2^17 products of two codes (of -128 too) stay below 2^31
  if (d->k < 1 || d->k >= 131072) return fail(SVLA_ERR_ARG, "%s: k must be 1 to 131071 (got %d)", who, d->k);
  // (tiles' counts and origins, and two weight rows per gated output, in 31 bits)
  if (d->m > 0x3fffffff || d->n > 0x3fffffff) return fail(SVLA_ERR_ARG, "%s: m and n must stay below 2^30 (got %d and %d)", who, d->m, d->n);
  if (d->impl < SVLA_LINEAR_AUTO || d->impl > SVLA_LINEAR_MANY) return fail(SVLA_ERR_ARG, "%s: bad impl %d", who, d->impl);
  if (d->gated && (d->bias || d->residual)) return fail(SVLA_ERR_ARG, "%s: a gated product takes no bias and no residual", who);
  if (d->m == 0 || d->n == 0) return SVLA_OK;
  const int size = d->dtype == SVLA_DT_FLOAT ? 4 : 2;
  if (int32_t rc = check_rows(who, "x", d->x, d->x_rs, d->k, 1)) return rc;
  if (int32_t rc = check_rows(who, "w", d->w, d->w_rs, d->k, 1)) return rc;
  if (!aligned(d->x, 16) || d->x_rs % 16 || !aligned(d->w, 16) || d->w_rs % 16)
    return fail(SVLA_ERR_ARG, "%s: x and w must be 16-byte aligned with row strides that are multiples of 16", who);
  if (!d->xscale || !d->wscale || !aligned(d->xscale, 4) || !aligned(d->wscale, 4) || !aligned(d->bias, 4))
    return fail(SVLA_ERR_ARG, "%s: xscale or wscale is null, or a scale or bias is not aligned", who);
  if (int32_t rc = check_rows(who, "out", d->out, d->out_rs, d->n, size)) return rc;
  if (d->residual) if (int32_t rc = check_rows(who, "residual", d->residual, d->residual_rs, d->n, size)) return rc;
  LinearI8Args a;
  std::memset(&a, 0, sizeof(a));
  a.xscale = d->xscale, a.wscale = d->wscale, a.bias = d->bias, a.residual = d->residual, a.out = d->out;
  a.residual_rs = d->residual_rs, a.out_rs = d->out_rs;
  a.m = d->m, a.n = d->n, a.k = d->k;
  a.err = device_error_ptr();
  if (d->dtype == SVLA_DT_FLOAT) return launch_linear_t<float>(a, d, cs(stream));
  if (d->dtype == SVLA_DT_HALF) return launch_linear_t<__half>(a, d, cs(stream));
  return launch_linear_t<__nv_bfloat16>(a, d, cs(stream));
}

}  // extern "C"
