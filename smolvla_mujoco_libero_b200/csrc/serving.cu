// C-ABI entry points of the serving operators (include/svla.h): attention over packed prompts, appending to a paged
// cache, attention over a paged cache.  Argument checks, template dispatch and launches; nothing allocates memory.
#include <cmath>
#include <cstring>

#include "host.cuh"
#include "kv_append.cuh"
#include "packed_attention.cuh"
#include "packed_attention_tc.cuh"
#include "paged_attention.cuh"

namespace svla {
namespace {

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int32_t check_heads(const char* who, int32_t hq, int32_t hkv, int32_t head_dim, int32_t dtype) {
  if (hq <= 0 || hkv <= 0 || hq % hkv) return fail(SVLA_ERR_ARG, "%s: hq must be a positive multiple of hkv", who);
  if (head_dim != 64 && head_dim != 128) return fail(SVLA_ERR_ARG, "%s: head_dim must be 64 or 128 (got %d)", who, head_dim);
  if (dtype != SVLA_DT_BF16 && dtype != SVLA_DT_HALF) return fail(SVLA_ERR_ARG, "%s: dtype must be BF16 or HALF (got %d)", who, dtype);
  return SVLA_OK;
}

// a packed tensor [rows][heads * head_dim]: 16-byte aligned rows that hold all heads
int32_t check_rows(const char* who, const char* name, const void* p, int64_t rs, int64_t width) {
  if (!p) return fail(SVLA_ERR_ARG, "%s: %s is null", who, name);
  if (!aligned(p, 16) || rs % 8 || rs < width)
    return fail(SVLA_ERR_ARG, "%s: %s must be 16-byte aligned with a row stride that is a multiple of 8 and >= %lld", who,
                name, static_cast<long long>(width));
  return SVLA_OK;
}

int32_t check_cache(const char* who, const void* cache, int32_t bits, int32_t page, int32_t n_pages, const int32_t* table,
                    int64_t table_rs, int32_t max_pages, const int32_t* kv_len) {
  if (!cache || !table || !kv_len) return fail(SVLA_ERR_ARG, "%s: null cache, page_table or kv_len", who);
  if (!aligned(cache, 16)) return fail(SVLA_ERR_ARG, "%s: cache must be 16-byte aligned", who);
  if (bits != 4 && bits != 16) return fail(SVLA_ERR_ARG, "%s: bits must be 4 or 16 (got %d)", who, bits);
  if (page < 16 || page > 256 || page % 16)
    return fail(SVLA_ERR_ARG, "%s: page_size must be a multiple of 16, 16 to 256 (got %d)", who, page);
  if (n_pages <= 0 || max_pages <= 0 || table_rs < max_pages)
    return fail(SVLA_ERR_ARG, "%s: n_pages and max_pages must be positive, page_table rows at least max_pages", who);
  return SVLA_OK;
}

// the scores' factor in log2 units; 0 stands for head_dim^-1/2.  Not negative: the kernels take the maximum of unscaled
// scores
int32_t score_scale(const char* who, float scale, int32_t head_dim, float* log2_scale) {
  if (!(scale >= 0.f) || std::isinf(scale))
    return fail(SVLA_ERR_ARG, "%s: scale must be positive and finite, or 0 for head_dim^-1/2 (got %g)", who, scale);
  *log2_scale = (scale > 0.f ? scale : 1.f / std::sqrt(static_cast<float>(head_dim))) * serving::kLog2e;
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

// ---------------------------------------------------------------- append
template <typename T, int D>
int32_t launch_append(const KvAppendArgs& a, int bits, dim3 grid, cudaStream_t st) {
  const dim3 block(append_detail::kWarps * 32);
  if (bits == 16) return launch(kv_append_kernel<T, D, 16>, grid, block, 0, st, "kv_append_kernel", a);
  return launch(kv_append_kernel<T, D, 4>, grid, block, 0, st, "kv_append_kernel", a);
}

// ---------------------------------------------------------------- packed prompts
template <typename T, int D>
int32_t launch_packed(const PackedAttnArgs& a, long long items, cudaStream_t st) {
  static bool configured[64] = {false};
  auto kern = packed_attention_kernel<T, D>;
  if (int32_t rc = allow_smem(kern, PackedSmem<T, D>::kBytes, configured)) return rc;
  return launch(kern, dim3(static_cast<unsigned>(items)), dim3(packed_detail::kWarps * 32), PackedSmem<T, D>::kBytes, st,
                "packed_attention_kernel", a);
}

// a packed tensor as (dim, head, token) with a box of 64 dimensions, 128-byte swizzle
int32_t make_tmap_packed(CUtensorMap* map, const void* base, int32_t dtype, uint64_t d, uint64_t heads, uint64_t rows,
                         uint64_t rs, uint32_t box_heads, uint32_t box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(SVLA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {d, heads, rows};
  cuuint64_t strides[2] = {d * 2, rs * 2};
  cuuint32_t box[3] = {64, box_heads, box_rows};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, dtype == SVLA_DT_HALF ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                  const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SVLA_ERR_ARG, "cuTensorMapEncodeTiled (packed) failed (%d)", static_cast<int>(r));
  return SVLA_OK;
}

template <typename T, int D>
int32_t launch_packed_tc(const PackedTcArgs& a, long long items, cudaStream_t st) {
  static bool configured[64] = {false};
  auto kern = packed_attention_tc_kernel<T, D>;
  if (int32_t rc = allow_smem(kern, ptc::Cfg<D>::kSmem, configured)) return rc;
  return launch(kern, dim3(static_cast<unsigned>(items)), dim3(ptc::kThreads), ptc::Cfg<D>::kSmem, st,
                "packed_attention_tc_kernel", a);
}

int32_t run_packed_tc(const svla_packed_attn_desc* d, float scale_log2, cudaStream_t st) {
  PackedTcArgs a;
  std::memset(&a, 0, sizeof(a));
  a.g = d->hq / d->hkv, a.qt = 128 / a.g;
  if (int32_t rc = make_tmap_packed(&a.tq, d->q, d->dtype, d->head_dim, d->hq, d->total_q, d->q_rs, a.g, a.qt)) return rc;
  if (int32_t rc = make_tmap_packed(&a.tk, d->k, d->dtype, d->head_dim, d->hkv, d->total_k, d->k_rs, 1, ptc::kKeys)) return rc;
  if (int32_t rc = make_tmap_packed(&a.tv, d->v, d->dtype, d->head_dim, d->hkv, d->total_k, d->v_rs, 1, ptc::kKeys)) return rc;
  a.v = d->v, a.o = d->o, a.cu_q = d->cu_q, a.cu_k = d->cu_k, a.v_rs = d->v_rs, a.o_rs = d->o_rs;
  a.batch = d->batch, a.total_q = d->total_q, a.total_k = d->total_k, a.hq = d->hq, a.hkv = d->hkv;
  a.causal = d->causal != 0;
  a.scale_log2 = scale_log2;
  a.err = device_error_ptr();
  const long long items = (static_cast<long long>(d->total_q) / (2 * a.qt) + d->batch) * d->hkv;
  if (items > 0x7fffffffll) return fail(SVLA_ERR_ARG, "svla_packed_attention: too many query tiles");
  const bool h = d->dtype == SVLA_DT_HALF;
  if (d->head_dim == 64) return h ? launch_packed_tc<__half, 64>(a, items, st) : launch_packed_tc<__nv_bfloat16, 64>(a, items, st);
  return h ? launch_packed_tc<__half, 128>(a, items, st) : launch_packed_tc<__nv_bfloat16, 128>(a, items, st);
}

// The automatic choice between the two kernels, from what the host knows: the average lengths, of which a query sees
// `seen` keys on the average.  An item of the tcgen05 kernel (256 query rows) costs 5 to 6 us beside its key tiles, one of
// the mma.sync kernel (64 rows, several per SM) 1 or 2; a key costs it less.  One round of items (mma.sync against tcgen05,
// us): D = 64, one prompt of 177 tokens 5.9 / 8.4, of 768 14.5 / 14.8, of 1024 21.2 / 18.0, one token after 500 keys
// 8.9 / 8.2; D = 128, 256 tokens 11.1 / 13.2, 384 16.1 / 16.1, 512 21.5 / 18.5.  Many rounds: it is the keys per item that
// count, less what its rows are not filled.  D = 64, 3 heads per group, 64 prompts of 256 tokens 69 / 77, of 320 94 / 87, of
// 384 121 / 109, of 64 after 300 39 / 30, of 16 after 500 20 / 30; D = 128, 4 heads, of 48 37 / 40, of 96 79 / 77, of 192
// 180 / 143, one token after 200 keys 25 / 32, after 2000 144 / 128.  Lengths that differ move the border: 64 prompts with
// lengths spread evenly over the logarithm from 1 to 512 after 0 to 300 keys take 50 / 45 and stay with mma.sync.
bool packed_prefers_tc(const svla_packed_attn_desc* d, int g) {
  const long long q = (static_cast<long long>(d->total_q) + d->batch - 1) / d->batch;
  const long long keys = static_cast<long long>(d->total_k) / d->batch, half = (q < keys ? q : keys) / 2;
  const long long seen = d->causal ? keys - half : keys;
  const long long pair = 2 * (128 / g), per_head = (q + pair - 1) / pair;
  const bool narrow = d->head_dim == 64;
  if (d->batch * per_head * d->hkv <= sm_count()) return seen >= (narrow ? 400 : 192);
  return seen * (q * g / per_head) >= 256 * (narrow ? 145 : 28);
}

// ---------------------------------------------------------------- paged
constexpr int kPagedCtas = 4;  // most CTAs per SM

// rows of a query tile / 8: single tokens of up to 8 grouped heads, or more
int paged_nt(int batch, int total_q, int g) { return static_cast<long long>(total_q) * g <= 8ll * batch ? 1 : 2; }

// items of at most 512 entries are not worth a second launch to join their parts
bool paged_split(long long max_entries) { return max_entries > 512; }

size_t paged_part_bytes(long long ctas, int nt, int d) { return static_cast<size_t>(2 * ctas) * 8 * nt * (d + 2) * 4; }

template <typename T, int D, int BITS, int NT>
int32_t launch_paged_inst(PagedAttnArgs a, cudaStream_t st) {
  using Sm = PagedSmem<T, D, BITS, NT>;
  static bool configured[64] = {false};
  static int ctas[64] = {0};
  auto kern = paged_attention_kernel<T, D, BITS, NT>;
  if (int32_t rc = allow_smem(kern, Sm::kBytes, configured)) return rc;
  int dev = 0;
  cudaGetDevice(&dev);
  if (ctas[dev] == 0) {
    int n = 0;
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, paged_detail::kWarps * 32, Sm::kBytes);
    if (e != cudaSuccess) return fail(SVLA_ERR_CUDA, "cudaOccupancyMaxActiveBlocksPerMultiprocessor: %s", cudaGetErrorString(e));
    ctas[dev] = (n < 1 ? 1 : (n > kPagedCtas ? kPagedCtas : n)) * sm_count();
  }
  const int grid = ctas[dev];
  // a piece is worth at least 256 entries (64 a warp); an item's start and join cost about as much as 512
  a.min_share = a.split ? 256 / paged_detail::Tile<D, BITS>::kKeys : 1;
  a.item_cost = 512 / paged_detail::Tile<D, BITS>::kKeys;
  if (a.split) a.meta = reinterpret_cast<int4*>(reinterpret_cast<uint8_t*>(a.part) + paged_part_bytes(grid, NT, D));
  int32_t rc = launch(kern, dim3(grid), dim3(paged_detail::kWarps * 32), Sm::kBytes, st, "paged_attention_kernel", a);
  if (rc || !a.split) return rc;
  return launch(paged_combine_kernel<T, D, NT>, dim3(grid), dim3(kPagedJoinWarps * 32), 0, st, "paged_combine_kernel", a);
}

template <typename T, int D>
int32_t launch_paged(const PagedAttnArgs& a, int bits, int nt, cudaStream_t st) {
  if (bits == 16) return nt == 1 ? launch_paged_inst<T, D, 16, 1>(a, st) : launch_paged_inst<T, D, 16, 2>(a, st);
  return nt == 1 ? launch_paged_inst<T, D, 4, 1>(a, st) : launch_paged_inst<T, D, 4, 2>(a, st);
}

}  // namespace
}  // namespace svla

using namespace svla;

extern "C" {

int32_t svla_rope_table_wide(float* c, int32_t max_pos, int32_t head_dim, double max_wavelength, svla_stream_t stream) {
  if (!c || !aligned(c, 16) || max_pos <= 0 || head_dim <= 0 || head_dim % 2 || !(max_wavelength > 0))
    return fail(SVLA_ERR_ARG, "svla_rope_table_wide: bad args");
  const long long n = static_cast<long long>(max_pos) * (head_dim / 2);
  return launch(rope_table_wide_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, cs(stream),
                "rope_table_wide_kernel", reinterpret_cast<float2*>(c), max_pos, head_dim / 2, max_wavelength);
}

int32_t svla_kv_append(const svla_kv_append_desc* d, svla_stream_t stream) {
  const char* who = "svla_kv_append";
  if (!d) return fail(SVLA_ERR_ARG, "%s: null descriptor", who);
  if (d->batch < 0 || d->total_q < 0) return fail(SVLA_ERR_ARG, "%s: negative batch or total_q", who);
  const int32_t hq = d->q ? d->hq : d->hkv;  // without queries hq is not read
  if (int32_t rc = check_heads(who, hq, d->hkv, d->head_dim, d->dtype)) return rc;
  if (int32_t rc = check_cache(who, d->cache, d->bits, d->page_size, d->n_pages, d->page_table, d->page_table_rs, d->max_pages, d->kv_len)) return rc;
  if (!d->cu_q) return fail(SVLA_ERR_ARG, "%s: cu_q is null", who);
  const int64_t qw = static_cast<int64_t>(hq) * d->head_dim, kw = static_cast<int64_t>(d->hkv) * d->head_dim;
  if (int32_t rc = check_rows(who, "k", d->k, d->k_rs, kw)) return rc;
  if (int32_t rc = check_rows(who, "v", d->v, d->v_rs, kw)) return rc;
  if (d->q) {
    if (int32_t rc = check_rows(who, "q", d->q, d->q_rs, qw)) return rc;
    if (int32_t rc = check_rows(who, "q_out", d->q_out, d->q_out_rs, qw)) return rc;
  }
  if (d->k_out) if (int32_t rc = check_rows(who, "k_out", d->k_out, d->k_out_rs, kw)) return rc;
  if (d->v_out) if (int32_t rc = check_rows(who, "v_out", d->v_out, d->v_out_rs, kw)) return rc;
  if (d->rope_cs && (!aligned(d->rope_cs, 16) || d->max_pos <= 0))
    return fail(SVLA_ERR_ARG, "%s: rope_cs must be 16-byte aligned with max_pos > 0", who);
  if (d->batch == 0 || d->total_q == 0) return SVLA_OK;
  KvAppendArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = d->q, a.k = d->k, a.v = d->v;
  a.qo = d->q_out, a.ko = d->k_out, a.vo = d->v_out;
  a.cache = static_cast<uint8_t*>(d->cache);
  a.cu_q = d->cu_q, a.kv_len = d->kv_len, a.table = d->page_table, a.pos = d->pos;
  a.cs = reinterpret_cast<const float2*>(d->rope_cs);
  a.q_rs = d->q_rs, a.k_rs = d->k_rs, a.v_rs = d->v_rs;
  a.qo_rs = d->q_out_rs, a.ko_rs = d->k_out_rs, a.vo_rs = d->v_out_rs, a.table_rs = d->page_table_rs;
  a.batch = d->batch, a.total = d->total_q, a.hq = d->hq, a.hkv = d->hkv;
  a.page = d->page_size, a.n_pages = d->n_pages, a.max_pages = d->max_pages, a.max_pos = d->max_pos;
  a.err = device_error_ptr();
  // few tokens: several warps share a token's heads, so that a call fills the GPU and its rows are fetched at once
  const int slots = 32 / (d->head_dim / 16), rounds = ((d->q ? d->hq : 0) + 2 * d->hkv + slots - 1) / slots;
  long long parts = 16ll * sm_count() / d->total_q;
  a.parts = static_cast<int>(parts < 1 ? 1 : (parts > rounds ? rounds : parts));
  const long long warps = static_cast<long long>(d->total_q) * a.parts;
  const dim3 grid(static_cast<unsigned>((warps + append_detail::kWarps - 1) / append_detail::kWarps));
  const bool h = d->dtype == SVLA_DT_HALF;
  if (d->head_dim == 64) return h ? launch_append<__half, 64>(a, d->bits, grid, cs(stream)) : launch_append<__nv_bfloat16, 64>(a, d->bits, grid, cs(stream));
  return h ? launch_append<__half, 128>(a, d->bits, grid, cs(stream)) : launch_append<__nv_bfloat16, 128>(a, d->bits, grid, cs(stream));
}

int32_t svla_packed_attention(const svla_packed_attn_desc* d, svla_stream_t stream) {
  const char* who = "svla_packed_attention";
  if (!d) return fail(SVLA_ERR_ARG, "%s: null descriptor", who);
  if (d->batch < 0 || d->total_q < 0 || d->total_k < 0) return fail(SVLA_ERR_ARG, "%s: negative batch, total_q or total_k", who);
  if (int32_t rc = check_heads(who, d->hq, d->hkv, d->head_dim, d->dtype)) return rc;
  const int g = d->hq / d->hkv;
  if (g > packed_detail::kRows) return fail(SVLA_ERR_ARG, "%s: at most %d query heads per kv head (got %d)", who, packed_detail::kRows, g);
  if (!d->cu_q || !d->cu_k) return fail(SVLA_ERR_ARG, "%s: cu_q or cu_k is null", who);
  float scale_log2 = 0.f;
  if (int32_t rc = score_scale(who, d->scale, d->head_dim, &scale_log2)) return rc;
  if (d->batch == 0 || d->total_q == 0) return SVLA_OK;
  const int64_t qw = static_cast<int64_t>(d->hq) * d->head_dim, kw = static_cast<int64_t>(d->hkv) * d->head_dim;
  if (int32_t rc = check_rows(who, "q", d->q, d->q_rs, qw)) return rc;
  if (int32_t rc = check_rows(who, "o", d->o, d->o_rs, qw)) return rc;
  if (d->total_k > 0) {
    if (int32_t rc = check_rows(who, "k", d->k, d->k_rs, kw)) return rc;
    if (int32_t rc = check_rows(who, "v", d->v, d->v_rs, kw)) return rc;
  }
  PackedAttnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = d->q, a.k = d->k, a.v = d->v, a.o = d->o;
  a.cu_q = d->cu_q, a.cu_k = d->cu_k;
  a.q_rs = d->q_rs, a.k_rs = d->k_rs, a.v_rs = d->v_rs, a.o_rs = d->o_rs;
  a.batch = d->batch, a.total_q = d->total_q, a.total_k = d->total_k, a.hq = d->hq, a.hkv = d->hkv, a.g = g;
  a.causal = d->causal != 0;
  a.scale_log2 = scale_log2;
  if (d->impl < SVLA_ATTN_AUTO || d->impl > SVLA_ATTN_TCGEN05) return fail(SVLA_ERR_ARG, "%s: bad impl %d", who, d->impl);
  if (d->impl == SVLA_ATTN_TCGEN05 && d->total_k == 0) return fail(SVLA_ERR_ARG, "%s: the tcgen05 kernel needs keys", who);
  if (d->impl == SVLA_ATTN_TCGEN05 || (d->impl == SVLA_ATTN_AUTO && d->total_k > 0 && packed_prefers_tc(d, g)))
    return run_packed_tc(d, a.scale_log2, cs(stream));
  a.qt = packed_detail::kRows / g;
  a.g_magic = (65535u + g) / g;
  // the lengths are on the device: as many items as the sequences can have (each one's last tile may be short)
  const long long items = (static_cast<long long>(d->total_q) / a.qt + d->batch) * d->hkv;
  if (items > 0x7fffffffll) return fail(SVLA_ERR_ARG, "%s: too many query tiles", who);
  const bool h = d->dtype == SVLA_DT_HALF;
  if (d->head_dim == 64) return h ? launch_packed<__half, 64>(a, items, cs(stream)) : launch_packed<__nv_bfloat16, 64>(a, items, cs(stream));
  return h ? launch_packed<__half, 128>(a, items, cs(stream)) : launch_packed<__nv_bfloat16, 128>(a, items, cs(stream));
}

size_t svla_paged_attention_workspace_size(int32_t batch, int32_t total_q, int32_t hq, int32_t hkv, int32_t head_dim,
                                           int64_t max_entries) {
  if (batch <= 0 || total_q <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || head_dim <= 0 || !paged_split(max_entries)) return 0;
  const long long ctas = static_cast<long long>(kPagedCtas) * sm_count();
  return paged_part_bytes(ctas, paged_nt(batch, total_q, hq / hkv), head_dim) + static_cast<size_t>(2 * ctas) * sizeof(int4);
}

int32_t svla_paged_attention(const svla_paged_attn_desc* d, svla_stream_t stream) {
  const char* who = "svla_paged_attention";
  if (!d) return fail(SVLA_ERR_ARG, "%s: null descriptor", who);
  if (d->batch < 0 || d->total_q < 0) return fail(SVLA_ERR_ARG, "%s: negative batch or total_q", who);
  if (int32_t rc = check_heads(who, d->hq, d->hkv, d->head_dim, d->dtype)) return rc;
  if (int32_t rc = check_cache(who, d->cache, d->bits, d->page_size, d->n_pages, d->page_table, d->page_table_rs, d->max_pages, d->kv_len)) return rc;
  if (!d->cu_q) return fail(SVLA_ERR_ARG, "%s: cu_q is null", who);
  float scale_log2 = 0.f;
  if (int32_t rc = score_scale(who, d->scale, d->head_dim, &scale_log2)) return rc;
  if (d->batch == 0 || d->total_q == 0) return SVLA_OK;
  const int64_t qw = static_cast<int64_t>(d->hq) * d->head_dim;
  if (int32_t rc = check_rows(who, "q", d->q, d->q_rs, qw)) return rc;
  if (int32_t rc = check_rows(who, "o", d->o, d->o_rs, qw)) return rc;
  const long long max_entries = static_cast<long long>(d->max_pages) * d->page_size;
  if (max_entries > 0x7fffffffll - 63)  // entries, up to the end of a sequence's last tile, are numbered in 32 bits
    return fail(SVLA_ERR_ARG, "%s: max_pages * page_size must stay below 2^31 - 63 (got %lld)", who, max_entries);
  const size_t need = svla_paged_attention_workspace_size(d->batch, d->total_q, d->hq, d->hkv, d->head_dim, max_entries);
  if (need && (!d->workspace || !aligned(d->workspace, 256) || d->workspace_bytes < need))
    return fail(SVLA_ERR_ARG, "%s: workspace must be 256-byte aligned with at least %zu bytes (got %zu)", who, need, d->workspace_bytes);
  PagedAttnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = d->q, a.o = d->o, a.cache = static_cast<const uint8_t*>(d->cache);
  a.cu_q = d->cu_q, a.kv_len = d->kv_len, a.table = d->page_table;
  a.part = static_cast<float*>(d->workspace);
  a.q_rs = d->q_rs, a.o_rs = d->o_rs, a.table_rs = d->page_table_rs;
  a.batch = d->batch, a.total = d->total_q, a.hq = d->hq, a.hkv = d->hkv, a.g = d->hq / d->hkv;
  a.page = d->page_size, a.n_pages = d->n_pages, a.max_pages = d->max_pages;
  a.page_magic = ((1ull << 32) + a.page / 16 - 1) / (a.page / 16);
  a.scale_log2 = scale_log2;
  a.err = device_error_ptr();
  a.split = paged_split(max_entries);
  const int nt = paged_nt(d->batch, d->total_q, a.g);
  const bool h = d->dtype == SVLA_DT_HALF;
  if (d->head_dim == 64) return h ? launch_paged<__half, 64>(a, d->bits, nt, cs(stream)) : launch_paged<__nv_bfloat16, 64>(a, d->bits, nt, cs(stream));
  return h ? launch_paged<__half, 128>(a, d->bits, nt, cs(stream)) : launch_paged<__nv_bfloat16, 128>(a, d->bits, nt, cs(stream));
}

}  // extern "C"
