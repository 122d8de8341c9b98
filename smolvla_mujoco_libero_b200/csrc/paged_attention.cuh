// Attention over a paged key / value cache (layouts in kv_append.cuh), 16-bit or 4-bit entries, for a few new tokens
// per sequence: query i of sequence b (of n_b) sees the cache entries n <= kv_len[b] - n_b + i,
//   o_i = sum_n softmax_n(scale q_i . k_n) v_n      (zeros where no entry weighs anything: none to see, none whose page
// is there, or every score -infinity).
//
// The floor is the bytes of the live cache; the work around them has to stay below what an SM issues in the time they
// take (4 bits, D = 64: 1280 bytes, 55 cycles, per 16 entries of one head).
//
// Shape of the products.  Entries are the M side: S^T (16 entries x 8 query rows) = K Q^T, O^T (16 dimensions x 8 query
// rows) += V^T P^T.  A query row is a (token, head) of one kv head, packed token-major, so grouped heads and several
// tokens share every entry that is read; 8 rows fit one MMA column block, and single tokens of up to 8 grouped heads
// waste half of what 16 query rows would (that form, without the transposition of P, takes twice the products and
// registers; of two early versions with one choice each it took 60 us, this one 50).
//
// 4-bit entries are never expanded to 16-bit values.  A nibble c masked out of a word, as it stands, is the fp16
// subnormal c 2^-24 (or 16 c 2^-24 for the second nibble of a byte): tensor cores take subnormals exactly, so one AND
// makes two MMA operands.  With k = low + step c per group of 32 dimensions
//   q . k = sum_g step_g (sum_{d in g} q_d c_d) + low_g (sum_{d in g} q_d)
// needs one accumulator per group and two FMAs per score, and
//   sum_n p_n v_n = sum_n (p_n step_n) c_n + sum_n p_n low_n
// takes p_n step_n as the other operand.  Query rows are scaled by a power of two to the top of fp16's range (exact but
// for components below 2^-25 of the row's largest), so bf16 queries lose nothing.
//
// p_n step_n is rounded to fp16, 2^-11 relative, less than a bf16 result's own rounding (1.75e-3 off instead of 1.67e-3 with
// exact weights).  For fp16 results, which it would move from 2.1e-4 to 5.3e-4, what the rounding left is a second operand of
// the same products: 46.0 and 77.3 us instead of 42.3 and 67.0 for the shapes below.  Every query column and group has a
// power of two of its own that brings the largest p_n step_n so far to 2^2, so that groups of different size, and large
// entries of little weight, leave the others their bits; what is smaller than 2^-16 of the largest is off by 2^-27 of it
// (half a subnormal step).  These factors move with the maximum, or when a step reaches a limit below which nothing can
// leave fp16's range; what a tile costs for them otherwise is a comparison and one product per weight.  Steps that vary by a
// factor of 4.5 (a standard deviation) from entry to entry reach it all the time: 46 and 86 us.  The products with low_n
// stay in fp32.
//
// Every warp works alone: its own tiles of 16 to 64 entries through its own ring of asynchronous copies, its own running
// maximum, sum and O, no barrier in the loop.  The maximum is lazy: it moves (and O is rescaled) only when a score
// passes it by more than 8 in log2 units (or a step the limit), one vote per tile instead of shuffles.  Instruction issue
// is what stands beside the memory system: the two query columns of a thread go through packed fp32 operations, a page's
// address is worked out once by one lane for 16 tiles, and the masks are in a branch that only a sequence's end takes.
//
// Work split.  All tiles of all (sequence, kv head, query tile) items form one line, each item 512 entries longer than it
// is (what its start and its join cost: without that, pieces of many short items come last); every CTA takes an equal
// piece of it, whatever the sequences' lengths are, and finds its place from cu_q and kv_len on the device.  An item that
// lies in one CTA is finished there; one cut by a piece's border leaves partials (maximum, sum, O in fp32) in the
// workspace, which the combine kernel joins in the line's order, so results do not depend on timing.
//
// Measured, both kernels, bf16, 4 bits: 64 single tokens at D = 64 over 255 to 8191 entries (118 MB) 42.3 us, 2.8 TB/s; two
// of D = 128 over 100000 to 131071 (291 MB) 67.0 us, 4.3 TB/s.  16 bits: 24 x 5 tokens over 100 to 4000 (65 MB) 21.5 us,
// 3.0 TB/s; single tokens as above 65 us (376 MB, 5.8 TB/s) and 145 us (930 MB, 6.4 TB/s: what the memory gives).  The first
// shape with 2 or 4 CTAs per SM instead of 3: 46 and 44 us; no cost per item: 55; 384 or 1024 entries per item: 44 and 43.
// What bounds 4 bits is the latency of dependent instructions with two or three warps per scheduler (issue slots 53% busy,
// DRAM 35 and 50%); time stamps gave about 12 us of the first shape to the start of a piece and of its items (place, pages,
// first copies, queries, each from cold code), 3 to the join, the rest to the tiles: 300 cycles per 16 entries and
// scheduler, of which the products take 75.
#pragma once

#include <type_traits>

#include "serving_common.cuh"

namespace svla {

struct PagedAttnArgs {
  const void* q;
  const uint8_t* cache;
  void* o;
  const int *cu_q, *kv_len, *table;
  float* part;             // workspace: 2 slots per CTA
  int4* meta;              // workspace, per CTA: {b, kv head, query tile, CTA of its last tile} of a cut item that starts
                           // there, or {-1, ..}; then per CTA that item's {first slot, first row, new tokens, -}
  long long q_rs, o_rs, table_rs;
  int batch, total, hq, hkv, g, page, n_pages, max_pages;
  unsigned long long page_magic;  // ceil(2^32 / (page / 16)): 16-entry slab -> page
  int split;               // 0: items are not cut
  int min_share;           // tiles a piece has at least
  int item_cost;           // what an item costs beside its tiles, in tiles
  float scale_log2;
  int* err;
};

namespace paged_detail {
constexpr int kWarps = 4;

template <int D, int BITS>
struct Tile {
  // entries per tile, in 16-entry slabs that lie inside one page each: enough independent work per warp to cover the
  // latency of the chain from scores to products, and 5 to 8 KB per copy
  static constexpr int kKeys = BITS == 4 ? (D == 64 ? 64 : 32) : (D == 64 ? 32 : 16);
  static constexpr int kSlabs = kKeys / 16;
  static constexpr int kStages = 3;                        // tiles in a warp's ring
  static constexpr int kRow = BITS == 16 ? D * 2 : D / 2;  // bytes of an entry's key (or value)
  static constexpr int kPairs = BITS == 16 ? 0 : D / 8;    // bytes of its (step, low) pairs
  static constexpr int kK = 0, kV = kKeys * kRow, kKP = 2 * kKeys * kRow, kVP = kKP + kKeys * kPairs;
  static constexpr int kBytes = 2 * kKeys * (kRow + kPairs);
};

// 4 bits, weights p step of the second product in fp16: a factor brings a column's largest weight in a group to 2^2 (below
// 2^3); p grows by 2^8 at most before the maximum moves, so steps below 2^7 / factor keep them below 2^15.  Factors are
// powers of two from 2^-126 to 2^100; a limit is kept as the bits of a step without its sign, times 2.
constexpr int kWeightTop = 2;
constexpr float kWeightFactorTop = 0x1p100f;
__device__ __forceinline__ float power_inverse(float f) { return __uint_as_float(0x7F000000u - __float_as_uint(f)); }
__device__ __forceinline__ uint32_t step_limit(float factor) {
  return 2u * min(0x7F000000u - __float_as_uint(factor) + (7u << 23), 0x7F800000u);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// a / b of two numbers that are not negative; 64 bits only where it has to be (a long division is a long piece of code)
__device__ __forceinline__ long long divide(long long a, long long b) {
  if (((a | b) >> 31) == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

// an entry's (step, low) pairs
__device__ __forceinline__ void load_pairs(uint32_t (&p)[2], const uint8_t* src) {
  const uint2 u = *reinterpret_cast<const uint2*>(src);
  p[0] = u.x, p[1] = u.y;
}
__device__ __forceinline__ void load_pairs(uint32_t (&p)[4], const uint8_t* src) {
  const uint4 u = *reinterpret_cast<const uint4*>(src);
  p[0] = u.x, p[1] = u.y, p[2] = u.z, p[3] = u.w;
}

// rows of a (sequence, kv head) and their tiles
template <int NT>
__device__ __forceinline__ int query_tiles(int n_new, int g) {
  return (n_new * g + 8 * NT - 1) / (8 * NT);
}
}  // namespace paged_detail

template <typename T, int D, int BITS, int NT>
struct PagedSmem {
  static constexpr int kRows = 8 * NT;
  static constexpr int kRing = paged_detail::Tile<D, BITS>::kStages * paged_detail::Tile<D, BITS>::kBytes;  // per warp
  static constexpr int kJoin = kRows * (D + 1 + 2) * 4;  // per warp: O, maximum, sum
  static constexpr int kPerWarp = kRing > kJoin ? kRing : (kJoin + 15) / 16 * 16;
  static constexpr int kBytes = paged_detail::kWarps * kPerWarp;
};

// single tokens at D = 64: three CTAs per SM
template <typename T, int D, int BITS, int NT>
__global__ void __launch_bounds__(paged_detail::kWarps * 32, (D == 64 && NT == 1) ? 3 : 1)
    paged_attention_kernel(const PagedAttnArgs a) {
  using namespace paged_detail;
  using serving::copy16;
  using Tl = Tile<D, BITS>;
  using Sm = PagedSmem<T, D, BITS, NT>;
  using serving::mma16816;
  constexpr int kRows = 8 * NT, kGroups = D / 32, kStages = Tl::kStages, kKeys = Tl::kKeys, kSlabs = Tl::kSlabs;
  constexpr int kBatch = 32 / kSlabs;  // tiles whose pages a warp holds
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int place[1];         // first sequence of this CTA's piece, and ...
  __shared__ long long place64[4]; // its start on the line; the piece; what every piece has
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + warp * Sm::kPerWarp;
  pdl_wait();
  pdl_trigger();

  // entries a sequence really has: its table's reach bounds them
  const long long reach = static_cast<long long>(a.max_pages) * a.page;
  auto entries = [&](int b) { return static_cast<int>(min(static_cast<long long>(max(__ldg(a.kv_len + b), 0)), reach)); };
  auto tiles_of = [&](int len) { return a.split ? (len + kKeys - 1) / kKeys + a.item_cost : 1; };  // on the line, per item
  auto weight = [&](int b) -> long long {
    const serving::Span s = serving::span_of(a.cu_q, b, a.total);
    return static_cast<long long>(tiles_of(entries(b))) * query_tiles<NT>(s.end - s.begin, a.g) * a.hkv;
  };
  // ---- this CTA's piece of the line and the sequence where it starts; the weights of the first 128 sequences are held
  if (warp == 0) {
    constexpr int kHeld = 4;
    long long held[kHeld], sum = 0;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      held[u] = 32 * u + lane < a.batch ? weight(32 * u + lane) : 0;
      sum += held[u];
    }
    for (int i = 32 * kHeld + lane; i < a.batch; i += 32) sum += weight(i);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const long long share = max(divide(sum + gridDim.x - 1, gridDim.x), static_cast<long long>(a.min_share));
    const long long from = share * blockIdx.x, to = min(from + share, sum);
    int b0 = a.batch;
    long long at = 0, base = 0;
    // sequences 32 i .. + 31, of weight w in this lane: does the piece start there?
    auto look = [&](int first, long long w) {
      long long upto = w;  // inclusive prefix
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
      }
      const unsigned past = __ballot_sync(0xffffffffu, base + upto > from);
      if (past) {
        const int l = __ffs(past) - 1;
        b0 = first + l;
        at = base + __shfl_sync(0xffffffffu, upto - w, l);
      } else {
        base += __shfl_sync(0xffffffffu, upto, 31);
      }
    };
    if (from < to) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
        if (b0 == a.batch && 32 * u < a.batch) look(32 * u, held[u]);
      for (int c = 32 * kHeld; c < a.batch && b0 == a.batch; c += 32) look(c, c + lane < a.batch ? weight(c + lane) : 0);
    }
    if (lane == 0) {
      place[0] = b0;
      place64[0] = at;
      place64[1] = from;
      place64[2] = to;
      place64[3] = share;
      if (a.split) a.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
    }
  }
  __syncthreads();
  int b = place[0];
  long long at = place64[0];  // start of sequence b on the line
  long long cur = place64[1];
  const long long from = cur, to = place64[2], full_share = place64[3];
  const long long page_bytes = BITS == 16 ? 4ll * a.page * D : static_cast<long long>(a.page) * (D + D / 4);

  const int slabs_per_page = a.page / 16;
  // 4 bits: the row (one group's codes of an entry) whose address this lane gives to an ldmatrix of a slab's groups 2 u and
  // 2 u + 1: lanes 0-7 entries 0-7 of the first, 8-15 entries 8-15, 16-31 the same of the second (swizzle of `issue`)
  int code_at[kGroups / 2];
#pragma unroll
  for (int u = 0; u < kGroups / 2; ++u) {
    const int r = lane & 15, gr = 2 * u + (lane >> 4);
    code_at[u] = r * Tl::kRow + ((gr ^ (D == 64 ? (r >> 2) & 1 : (r >> 1) & 3)) * 16);
  }
  // 4 bits: this lane's chunk of a slab's (step, low) pairs, first the keys', then the values'
  const int pair_is_v = lane / (D / 8), pair_c = lane % (D / 8);
  const int pair_dst = (pair_is_v ? Tl::kVP : Tl::kKP) + pair_c * 16;
  const int pair_src = a.page * D + (pair_is_v ? a.page * (D / 8) : 0) + pair_c * 16;

  while (cur < to) {
    // ---- the item at `cur`
    const serving::Span sq = serving::span_of(a.cu_q, b, a.total);
    const int n_new = sq.end - sq.begin, len = entries(b), n_tiles = tiles_of(len);
    // entries that token i sees; the causal limit counts from kv_len itself, also where the table ends before it
    const int past = min(max(__ldg(a.kv_len + b), 0) - n_new, len);
    auto seen = [&](int i) { return min(max(past + i + 1, 0), len); };
    const int qt_n = query_tiles<NT>(n_new, a.g);
    const long long w = static_cast<long long>(n_tiles) * qt_n * a.hkv;
    if (cur >= at + w) {
      at += w;
      ++b;
      continue;
    }
    if (threadIdx.x == 0 && __ldg(a.kv_len + b) > reach) record_error(a.err, serving::kErrBadPage);
    const int item = static_cast<int>(divide(cur - at, n_tiles));
    const long long item_at = at + static_cast<long long>(item) * n_tiles;
    const int kh = item % a.hkv, qt = item / a.hkv;
    const long long seg_end = min(item_at + n_tiles, to);
    const bool whole = cur == item_at && seg_end == item_at + n_tiles;
    if (!whole && cur == item_at && threadIdx.x == 0) {
      // the item's last piece: the CTA whose piece holds the item's last tile
      const long long last = divide(item_at + n_tiles - 1, full_share);
      a.meta[blockIdx.x] = make_int4(b, kh, qt, static_cast<int>(last));
      a.meta[gridDim.x + blockIdx.x] = make_int4(2 * blockIdx.x + (cur > from ? 1 : 0), sq.begin, n_new, 0);
    }
    // tiles of the sequence in this segment (an uncut item: all of them)
    const int real_tiles = (len + kKeys - 1) / kKeys;
    const int tile0 = a.split ? max(static_cast<int>(cur - item_at) - a.item_cost, 0) : 0;
    int tile1 = a.split ? min(static_cast<int>(seg_end - item_at) - a.item_cost, real_tiles) : real_tiles;
    const int row0 = qt * kRows, rows = min(kRows, n_new * a.g - row0);
    // entries the last / first row of this query tile sees
    const int sees_last = seen((row0 + rows - 1) / a.g), sees_first = seen(row0 / a.g);
    tile1 = min(tile1, (sees_last + kKeys - 1) / kKeys);

    // ---- this warp's tiles: tile0 + warp, + 4, ...
    const int mine = tile1 - tile0 - warp > 0 ? (tile1 - tile0 - warp + kWarps - 1) / kWarps : 0;
    // Slab s of the warp's i-th tile: lane kSlabs (i % kBatch) + s holds the byte offset of this kv head's part of its
    // page, with slot / 16 in the low four bits (parts are multiples of 16 bytes); -1: there is nothing to read.
    auto load_pages = [&](int i0, unsigned& bad) -> long long {
      const int i = i0 + lane / kSlabs;
      long long off = -1;
      bool wrong = false;
      if (i < mine) {
        const int slab = (tile0 + warp + i * kWarps) * kSlabs + lane % kSlabs;
        if (slab * 16 < sees_last) {
          const int pg = static_cast<int>((static_cast<unsigned long long>(slab) * a.page_magic) >> 32);
          const int id = __ldg(a.table + static_cast<size_t>(b) * a.table_rs + pg);
          wrong = id < 0 || id >= a.n_pages;
          if (!wrong) off = (static_cast<long long>(id) * a.hkv + kh) * page_bytes + (slab - pg * slabs_per_page);
        }
      }
      if (wrong) record_error(a.err, serving::kErrBadPage);
      bad = __ballot_sync(0xffffffffu, wrong);
      return off;
    };
    unsigned bad, bad_next;
    long long pages = load_pages(0, bad), pages_next = -1;
    bad_next = 0u;
    if (mine > kBatch) pages_next = load_pages(kBatch, bad_next);
    // copies tile i of the warp into its ring stage
    auto issue = [&](int i, int stage, long long offs) {
      uint8_t* st = ring + stage * Tl::kBytes;
#pragma unroll
      for (int s = 0; s < kSlabs; ++s) {
        const long long off = __shfl_sync(0xffffffffu, offs, kSlabs * (i % kBatch) + s);
        const bool have = off >= 0;
        const uint8_t* base = a.cache + (have ? off & ~15ll : 0);
        const int slot = (static_cast<int>(off) & 15) * 16;
        if constexpr (BITS == 16) {
          constexpr int kChunks = D / 8;  // 16-byte chunks of a row; chunk c of row r sits at c ^ (r % 8)
          // entries past the sequence are zeros, whatever the page holds there
          const int left = have ? len - ((tile0 + warp + i * kWarps) * kKeys + s * 16) : 0;
          const uint8_t* src = base + slot * (2 * D) + lane * 16;
          const int v_off = a.page * (2 * D);
#pragma unroll
          for (int u = 0; u < kChunks / 2; ++u) {
            const int idx = lane + u * 32, r = idx / kChunks, c = idx % kChunks;
            const int n = r < left ? 16 : 0;
            const int dst = (s * 16 + r) * Tl::kRow + ((c ^ (r & 7)) * 16);
            copy16(st + Tl::kK + dst, src + u * 512, n);
            copy16(st + Tl::kV + dst, src + u * 512 + v_off, n);
          }
        } else {
          constexpr int kChunks = D / 32;  // chunk c (one group's codes) of row r sits at c ^ swizzle(r): no bank conflicts
          const int n = have ? 16 : 0;
          const uint8_t* src = base + slot * (D / 2) + lane * 16;
          const int v_off = a.page * (D / 2);
#pragma unroll
          for (int u = 0; u < kChunks / 2; ++u) {
            const int idx = lane + u * 32, r = idx / kChunks, c = idx % kChunks;
            const int sw = D == 64 ? (r >> 2) & 1 : (r >> 1) & 3;
            const int dst = (s * 16 + r) * Tl::kRow + ((c ^ sw) * 16);
            copy16(st + Tl::kK + dst, src + u * 512, n);
            copy16(st + Tl::kV + dst, src + u * 512 + v_off, n);
          }
          if (lane < D / 4)  // 16 entries' pairs: D / 8 chunks for keys, D / 8 for values
            copy16(st + pair_dst + s * 16 * Tl::kPairs, base + pair_src + slot * (D / 8), n);
        }
      }
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (i < mine) issue(i, i, pages);
      serving::copy_commit();
    }

    // ---- Q^T operands: column g8 of block nt is row row0 + nt * 8 + g8; a missing row is zeros
    constexpr int kQRegs = BITS == 16 ? D / 16 * 2 : kGroups * 4;
    uint32_t qb[NT][kQRegs];
    float qf[NT][2];            // factors of this thread's two score columns (queries 2 t4, 2 t4 + 1)
    float qs[NT][kGroups][2];   // 4 bits: sums of their components, per group, times scale
    // 4 bits: powers of two that bring the weights p step of a column and group into fp16's range; a step of the group from
    // limit on may leave it
    float2 f[NT][kGroups];
    uint32_t limit[kGroups];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + nt * 8 + g8;
      const bool in = nt * 8 + g8 < rows;
      const T* src = static_cast<const T*>(a.q) + static_cast<size_t>(sq.begin + (in ? r / a.g : 0)) * a.q_rs +
                     (kh * a.g + (in ? r % a.g : 0)) * D;
      if constexpr (BITS == 16) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qb[nt][2 * kk] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + kk * 16 + 2 * t4)) : 0u;
          qb[nt][2 * kk + 1] = in ? __ldg(reinterpret_cast<const uint32_t*>(src + kk * 16 + 8 + 2 * t4)) : 0u;
        }
        qf[nt][0] = qf[nt][1] = a.scale_log2;
      } else {
        float x[kGroups][8];
        float top = 0.f, sum[kGroups];
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) {
          const uint4 u = in ? __ldg(reinterpret_cast<const uint4*>(src + gr * 32 + t4 * 8)) : make_uint4(0, 0, 0, 0);
          const uint32_t uu[4] = {u.x, u.y, u.z, u.w};
          sum[gr] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = serving::unpack2<T>(uu[i]);
            x[gr][2 * i] = f.x;
            x[gr][2 * i + 1] = f.y;
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            sum[gr] += f.x + f.y;
          }
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr) sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], d);
        }
        // up = 2^(14 - exponent of the largest component): the row then fills fp16's range (largest in [2^14, 2^15))
        int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
        ex = (top > 0.f && ex < 128) ? max(ex, -100) : 14;
        const float up = __uint_as_float(static_cast<uint32_t>(14 - ex + 127) << 23);
        // undoes 2^-24 of the codes and `up`
        const float down = a.scale_log2 * 1024.f * __uint_as_float(static_cast<uint32_t>(ex + 127) << 23);
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) {
          // step 0 of the group: (n0, n4 | n1, n5), step 1: (n2, n6 | n3, n7); odd nibbles count 16 times
          qb[nt][4 * gr + 0] = serving::pack2<__half>(x[gr][0] * up, x[gr][4] * up);
          qb[nt][4 * gr + 1] = serving::pack2<__half>(x[gr][1] * (up * 0.0625f), x[gr][5] * (up * 0.0625f));
          qb[nt][4 * gr + 2] = serving::pack2<__half>(x[gr][2] * up, x[gr][6] * up);
          qb[nt][4 * gr + 3] = serving::pack2<__half>(x[gr][3] * (up * 0.0625f), x[gr][7] * (up * 0.0625f));
        }
        // the score columns of this thread are queries 2 t4 and 2 t4 + 1: take their factors from lanes 8 t4, 8 t4 + 4
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          qf[nt][u] = __shfl_sync(0xffffffffu, down, 8 * t4 + 4 * u);
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr)
            qs[nt][gr][u] = __shfl_sync(0xffffffffu, sum[gr] * a.scale_log2, 8 * t4 + 4 * u);
        }
      }
    }
    // entries that this thread's two score columns see
    int sees[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = row0 + nt * 8 + 2 * t4 + u;
        sees[nt][u] = seen(r / a.g);
      }

    float o[NT][D / 16][4];     // O^T: see the P.V product for which dimensions a thread holds
    float om[NT][kGroups][2];   // 4 bits: sums of p low
    float m[NT][2], ref[NT][2], l[NT][2];
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr) limit[gr] = step_limit(kWeightFactorTop);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr) {
        om[nt][gr][0] = om[nt][gr][1] = 0.f;
        f[nt][gr] = make_float2(kWeightFactorTop, kWeightFactorTop);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) m[nt][u] = -INFINITY, ref[nt][u] = 0.f, l[nt][u] = 0.f;
    }

    int stage = 0, refill = kStages - 1;  // i % kStages, (i + kStages - 1) % kStages
    for (int i = 0; i < mine; ++i) {
      // refill the stage that tile i - 1 used (every lane has passed the __syncwarp that ends tile i - 1)
      const int ahead = i + kStages - 1;
      if (ahead < mine) issue(ahead, refill, ahead / kBatch == i / kBatch ? pages : pages_next);
      serving::copy_commit();
      serving::copy_wait<kStages - 1>();
      __syncwarp();
      const uint8_t* st = ring + stage * Tl::kBytes;
      refill = stage;
      stage = stage + 1 == kStages ? 0 : stage + 1;
      const int key0 = (tile0 + warp + i * kWarps) * kKeys;
      const unsigned gone = (bad >> (kSlabs * (i % kBatch))) & ((1u << kSlabs) - 1u);  // slabs without a page
      if (i % kBatch == kBatch - 1) {
        pages = pages_next;
        bad = bad_next;
        if (i + 1 + kBatch < mine) pages_next = load_pages(i + 1 + kBatch, bad_next);
      }
      // some entry of the tile is hidden from some row (warp-uniform)
      const bool edge = key0 + kKeys > sees_first || gone != 0u;

      // ---- scores, in log2 units: s[nt][slab][e]: entry slab * 16 + g8 + 8 (e / 2), query column 2 t4 + e % 2
      float s[NT][kSlabs][4];
#pragma unroll
      for (int sl = 0; sl < kSlabs; ++sl) {
        if constexpr (BITS == 16) {
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t ka[4];  // entries (lane & 15), dimensions kk * 16 + 8 (lane >> 4)
            const int r = sl * 16 + (lane & 15), ch = kk * 2 + (lane >> 4);
            serving::ldsm_x4(ka, st + Tl::kK + r * Tl::kRow + ((ch ^ (r & 7)) * 16));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<T>(acc[nt], ka, qb[nt][2 * kk], qb[nt][2 * kk + 1]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) s[nt][sl][x] = acc[nt][x] * qf[nt][x & 1];
        } else {
          float acc[NT][kGroups][4];
          // word t4 of each group's codes, entries g8 and g8 + 8: an ldmatrix of 32-bit words
          uint32_t kw[kGroups][2];
#pragma unroll
          for (int gr = 0; gr < kGroups; gr += 2) {
            uint32_t w[4];
            serving::ldsm_x4(w, st + Tl::kK + sl * 16 * Tl::kRow + code_at[gr / 2]);
            kw[gr][0] = w[0], kw[gr][1] = w[1], kw[gr + 1][0] = w[2], kw[gr + 1][1] = w[3];
          }
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr) {
            const uint32_t w0 = kw[gr][0], w1 = kw[gr][1];
            const uint32_t x0 = w0 >> 8, x1 = w1 >> 8;
            const uint32_t a0[4] = {w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u};
            const uint32_t a1[4] = {x0 & 0x000F000Fu, x1 & 0x000F000Fu, x0 & 0x00F000F0u, x1 & 0x00F000F0u};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              serving::mma16816_first<__half>(acc[nt][gr], a0, qb[nt][4 * gr], qb[nt][4 * gr + 1]);
              mma16816<__half>(acc[nt][gr], a1, qb[nt][4 * gr + 2], qb[nt][4 * gr + 3]);
            }
          }
#pragma unroll
          for (int hr = 0; hr < 2; ++hr) {
            uint32_t kp[kGroups];
            load_pairs(kp, st + Tl::kKP + (sl * 16 + g8 + 8 * hr) * Tl::kPairs);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float2 dot = make_float2(0.f, 0.f), add = dot;
#pragma unroll
              for (int gr = 0; gr < kGroups; ++gr) {
                const float step = __uint_as_float(kp[gr] << 16), low = __uint_as_float(kp[gr] & 0xFFFF0000u);
                dot = __ffma2_rn(make_float2(step, step), make_float2(acc[nt][gr][2 * hr], acc[nt][gr][2 * hr + 1]), dot);
                add = __ffma2_rn(make_float2(low, low), make_float2(qs[nt][gr][0], qs[nt][gr][1]), add);
              }
              const float2 x = __ffma2_rn(dot, make_float2(qf[nt][0], qf[nt][1]), add);
              s[nt][sl][2 * hr] = x.x, s[nt][sl][2 * hr + 1] = x.y;
            }
          }
        }
      }
      // 4 bits: does a step of the tile's values, a lane's share of the pairs at a time, reach its group's limit?
      bool large = false;
      if constexpr (BITS == 4) {
        constexpr int kWords = kKeys * kGroups / 32;  // 4
        static_assert(kWords == 4, "a lane takes 16 bytes of the pairs");
        const uint4 v = *reinterpret_cast<const uint4*>(st + Tl::kVP + lane * 16);
        const uint32_t vv[4] = {v.x, v.y, v.z, v.w};
        auto reaches = [&](int w) { return vv[w] << 17 >= limit[w % kGroups]; };  // (or is no number)
        large = reaches(0) || reaches(1) || reaches(2) || reaches(3);
        if (edge) {  // whatever stands in entries that nobody sees does not count
          large = false;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int n = (lane * 4 + w) / kGroups;
            if (key0 + n < sees_last && !((gone >> (n / 16)) & 1u)) large |= reaches(w);
          }
        }
      }
      if (edge) {
#pragma unroll
        for (int sl = 0; sl < kSlabs; ++sl)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int n = (gone >> sl) & 1u ? 0x7fffffff : key0 + sl * 16 + g8 + 8 * (x >> 1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              if (n >= sees[nt][x & 1]) s[nt][sl][x] = -INFINITY;
          }
      }
      // ---- lazy running maximum
      float top[NT][2];
      bool pass = large;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float t = fmaxf(s[nt][0][u], s[nt][0][2 + u]);
#pragma unroll
          for (int sl = 1; sl < kSlabs; ++sl) t = max3(t, s[nt][sl][u], s[nt][sl][2 + u]);
          top[nt][u] = t;
          pass |= t > m[nt][u] + 8.f;
        }
      const bool moves = __any_sync(0xffffffffu, pass);
      if (moves) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float t = fmaxf(top[nt][u], m[nt][u]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
            float alpha;
            if constexpr (BITS == 4) {  // a power of two, 0 from 2^-127 on and where nothing has been seen
              t = ceilf(t);
              alpha = __uint_as_float(static_cast<uint32_t>(127 - static_cast<int>(fminf(t - m[nt][u], 127.f))) << 23);
            } else {  // nothing seen so far: O and the sums are zeros, any factor will do
              alpha = m[nt][u] == -INFINITY ? 1.f : ex2_approx(m[nt][u] - t);
            }
            m[nt][u] = t;
            ref[nt][u] = t == -INFINITY ? 0.f : t - (BITS == 16 ? serving::kWeightLift<T> : 0.f);
            l[nt][u] *= alpha;
            if constexpr (BITS == 4) {
              top[nt][u] = alpha;  // O follows below, with its factors
#pragma unroll
              for (int gr = 0; gr < kGroups; ++gr) om[nt][gr][u] *= alpha;
            } else {
#pragma unroll
              for (int i2 = 0; i2 < D / 16; ++i2) {
                o[nt][i2][u] *= alpha;
                o[nt][i2][2 + u] *= alpha;
              }
            }
          }
      }
      // ---- probabilities
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 shift = make_float2(-ref[nt][0], -ref[nt][1]);
        float2 sum = make_float2(l[nt][0], l[nt][1]);
#pragma unroll
        for (int sl = 0; sl < kSlabs; ++sl)
#pragma unroll
          for (int hr = 0; hr < 2; ++hr) {
            const float2 x = __fadd2_rn(make_float2(s[nt][sl][2 * hr], s[nt][sl][2 * hr + 1]), shift);
            const float2 p = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            sum = __fadd2_rn(sum, p);
            s[nt][sl][2 * hr] = p.x, s[nt][sl][2 * hr + 1] = p.y;
          }
        l[nt][0] = sum.x, l[nt][1] = sum.y;
      }
      // ---- 4 bits: the weights' factors
      if constexpr (BITS == 4) {
        if (moves) {
          float2 w[NT][kGroups];  // largest weights, times 2^-10 (p goes up to 2^8)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr) w[nt][gr] = make_float2(0.f, 0.f);
#pragma unroll
          for (int sl = 0; sl < kSlabs; ++sl)
#pragma unroll
            for (int hr = 0; hr < 2; ++hr) {
              uint32_t vp[kGroups];
              load_pairs(vp, st + Tl::kVP + (sl * 16 + g8 + 8 * hr) * Tl::kPairs);
#pragma unroll
              for (int gr = 0; gr < kGroups; ++gr) {
                float step = fabsf(__uint_as_float(vp[gr] << 16)) * 0x1p-10f;
                if (!(step < INFINITY)) step = 0.f;  // no number: does not count
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  w[nt][gr].x = fmaxf(w[nt][gr].x, s[nt][sl][2 * hr] * step);
                  w[nt][gr].y = fmaxf(w[nt][gr].y, s[nt][sl][2 * hr + 1] * step);
                }
              }
            }
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr) {
            float most = 0.f;  // of the columns that see something: the others' weights are zeros
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              // both columns' upper halves in one word
              uint32_t both = __byte_perm(__float_as_uint(w[nt][gr].x), __float_as_uint(w[nt][gr].y), 0x7632);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, d));
              // 2^(kWeightTop - exponent of the weight), from the exponent field of weight 2^-10; O's factor grows with the
              // maximum, up to kWeightFactorTop, and O stays
              auto next = [&](uint32_t field, float was, float alpha) {
                const float room = __uint_as_float(min(max(kWeightTop + 244 - static_cast<int>(field & 255u), 1), 227) << 23);
                return fminf(was * power_inverse(alpha), room);
              };
              const float2 a2 = make_float2(top[nt][0], top[nt][1]), was = f[nt][gr];
              const float2 now = make_float2(next(both >> 7, was.x, a2.x), next(both >> 23, was.y, a2.y));
              f[nt][gr] = now;
              most = fmaxf(most, fmaxf(m[nt][0] == -INFINITY ? 0.f : now.x, m[nt][1] == -INFINITY ? 0.f : now.y));
              const float2 r = __fmul2_rn(__fmul2_rn(now, a2), make_float2(power_inverse(was.x), power_inverse(was.y)));
#pragma unroll
              for (int i2 = 2 * gr; i2 < 2 * gr + 2; ++i2) {
                o[nt][i2][0] *= r.x, o[nt][i2][1] *= r.y;
                o[nt][i2][2] *= r.x, o[nt][i2][3] *= r.y;
              }
            }
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            limit[gr] = step_limit(most);
          }
        }
      }
      // ---- O^T += V^T P^T
      if constexpr (BITS == 16) {
        // an infinity or a NaN in the value of an entry that some row does not see would reach that row as 0 * inf
        bool odd = false;
        if (edge && n_new > 1) {
          for (int idx = lane; idx < kKeys * (D / 8); idx += 32) {
            const uint4 u = *reinterpret_cast<const uint4*>(st + Tl::kV + idx * 16);
            odd |= serving::any_nonfinite<T>(u.x) || serving::any_nonfinite<T>(u.y) ||
                   serving::any_nonfinite<T>(u.z) || serving::any_nonfinite<T>(u.w);
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        if (!odd) {
#pragma unroll
          for (int sl = 0; sl < kSlabs; ++sl) {
            uint32_t pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int hr = 0; hr < 2; ++hr)
                pb[nt][hr] = serving::movmatrix_trans(serving::pack2<T>(s[nt][sl][2 * hr], s[nt][sl][2 * hr + 1]));
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {
              // V^T: rows = dimensions mt * 16 .. + 15, columns = the slab's entries; transposed 8 x 8 blocks
              uint32_t va[4];
              const int r = sl * 16 + (lane & 7) + ((lane >> 4) << 3), ch = mt * 2 + ((lane >> 3) & 1);
              serving::ldsm_x4_trans(va, st + Tl::kV + r * Tl::kRow + ((ch ^ (r & 7)) * 16));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[nt][mt], va, pb[nt][0], pb[nt][1]);
            }
          }
        } else {  // rare: one entry after the other, hidden ones left out
#pragma unroll
          for (int sl = 0; sl < kSlabs; ++sl)
            for (int n = 0; n < 16; ++n) {
              const int r = sl * 16 + n;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  // entry n's row of the score block: half n / 8, lane group n % 8
                  const float p = __shfl_sync(0xffffffffu, n >> 3 ? s[nt][sl][2 + u] : s[nt][sl][u], (n & 7) * 4 + t4);
#pragma unroll
                  for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                      const int d = mt * 16 + hf * 8 + g8;
                      const float v = static_cast<float>(*(reinterpret_cast<const T*>(st + Tl::kV + r * Tl::kRow + (((d >> 3) ^ (r & 7)) * 16)) + (d & 7)));
                      if (key0 + r < sees[nt][u]) o[nt][mt][2 * hf + u] = fmaf(p, v, o[nt][mt][2 * hf + u]);
                    }
                }
            }
        }
      } else {
#pragma unroll
        for (int sl = 0; sl < kSlabs; ++sl) {
          // fp16 callers: what the rounding of the weights to fp16 left goes through the products as well
          constexpr bool kRest = std::is_same<T, __half>::value;
          uint32_t pb[NT][kGroups][2], pr[NT][kRest ? kGroups : 1][2];
#pragma unroll
          for (int hr = 0; hr < 2; ++hr) {
            uint32_t vp[kGroups];
            load_pairs(vp, st + Tl::kVP + (sl * 16 + g8 + 8 * hr) * Tl::kPairs);
            if (edge) {
              const int n = key0 + sl * 16 + g8 + 8 * hr;
#pragma unroll
              for (int gr = 0; gr < kGroups; ++gr) {
                // whatever stands in an entry that nobody sees counts nothing; a pair that is no number, of an entry
                // that some rows see: those get their NaN through the sum of p low (p = 0 would not keep it from the
                // others), and the codes count nothing
                const bool none = n >= sees_last || ((gone >> sl) & 1u);
                const bool fine = isfinite(__uint_as_float(vp[gr] << 16)) && isfinite(__uint_as_float(vp[gr] & 0xFFFF0000u));
                if (!none && !fine) {
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                      if (n < sees[nt][u]) om[nt][gr][u] = NAN;
                }
                if (none || !fine) vp[gr] = 0u;
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int gr = 0; gr < kGroups; ++gr) {
                const float step = __uint_as_float(vp[gr] << 16), low = __uint_as_float(vp[gr] & 0xFFFF0000u);
                const float2 p = make_float2(s[nt][sl][2 * hr], s[nt][sl][2 * hr + 1]);
                const float2 y = __fmul2_rn(p, __fmul2_rn(make_float2(step, step), f[nt][gr]));
                const float2 sum = __ffma2_rn(p, make_float2(low, low), make_float2(om[nt][gr][0], om[nt][gr][1]));
                om[nt][gr][0] = sum.x, om[nt][gr][1] = sum.y;
                const uint32_t yh = serving::pack2<__half>(y.x, y.y);
                pb[nt][gr][hr] = serving::movmatrix_trans(yh);
                if constexpr (kRest) {
                  const float2 f2 = serving::unpack2<__half>(yh), rest = __fadd2_rn(y, make_float2(-f2.x, -f2.y));
                  pr[nt][gr][hr] = serving::movmatrix_trans(serving::pack2<__half>(rest.x, rest.y));
                }
              }
          }
          // the half word g8 of each group's codes (dimensions 4 g8 .. + 3), of entries 2 t4 and 2 t4 + 1 (and + 8) in one
          // register: a transposed ldmatrix of half words
          uint32_t vw[kGroups][2];
#pragma unroll
          for (int gr = 0; gr < kGroups; gr += 2) {
            uint32_t w[4];
            serving::ldsm_x4_trans(w, st + Tl::kV + sl * 16 * Tl::kRow + code_at[gr / 2]);
            vw[gr][0] = w[0], vw[gr][1] = w[1], vw[gr + 1][0] = w[2], vw[gr + 1][1] = w[3];
          }
#pragma unroll
          for (int gr = 0; gr < kGroups; ++gr) {
            const uint32_t x0 = vw[gr][0], x1 = vw[gr][1];
            const uint32_t y0 = x0 >> 8, y1 = x1 >> 8;
            // rows g8 of the first product: dimension 4 g8, rows g8 + 8: 4 g8 + 1 (16 times); second: 4 g8 + 2, + 3
            const uint32_t a0[4] = {x0 & 0x000F000Fu, x0 & 0x00F000F0u, x1 & 0x000F000Fu, x1 & 0x00F000F0u};
            const uint32_t a1[4] = {y0 & 0x000F000Fu, y0 & 0x00F000F0u, y1 & 0x000F000Fu, y1 & 0x00F000F0u};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<__half>(o[nt][2 * gr], a0, pb[nt][gr][0], pb[nt][gr][1]);
              mma16816<__half>(o[nt][2 * gr + 1], a1, pb[nt][gr][0], pb[nt][gr][1]);
              if constexpr (kRest) {
                mma16816<__half>(o[nt][2 * gr], a0, pr[nt][gr][0], pr[nt][gr][1]);
                mma16816<__half>(o[nt][2 * gr + 1], a1, pr[nt][gr][0], pr[nt][gr][1]);
              }
            }
          }
        }
      }
      __syncwarp();
    }
    serving::copy_wait<0>();
    __syncthreads();  // every warp is done with its ring

    // ---- join the four warps
    float* js = reinterpret_cast<float*>(smem + warp * Sm::kPerWarp);  // [kRows][D + 1], then maxima, sums
    float* jm = js + kRows * (D + 1);
    float* jl = jm + kRows;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[nt][u] += __shfl_xor_sync(0xffffffffu, l[nt][u], d);
          if constexpr (BITS == 4) {
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr) om[nt][gr][u] += __shfl_xor_sync(0xffffffffu, om[nt][gr][u], d);
          }
        }
        const int r = nt * 8 + 2 * t4 + u;
        if (g8 == 0) {
          jm[r] = m[nt][u] == -INFINITY ? -INFINITY : ref[nt][u];
          jl[r] = l[nt][u];
        }
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          if constexpr (BITS == 16) {
            js[r * (D + 1) + mt * 16 + g8] = o[nt][mt][u];
            js[r * (D + 1) + mt * 16 + 8 + g8] = o[nt][mt][2 + u];
          } else {
            // 2^24 undoes the codes' subnormals, odd dimensions counted 16 times
            const int d = (mt >> 1) * 32 + 4 * g8 + 2 * (mt & 1);
            const float back = power_inverse(u ? f[nt][mt >> 1].y : f[nt][mt >> 1].x);
            js[r * (D + 1) + d] = fmaf(o[nt][mt][u] * 16777216.f, back, om[nt][mt >> 1][u]);
            js[r * (D + 1) + d + 1] = fmaf(o[nt][mt][2 + u] * 1048576.f, back, om[nt][mt >> 1][u]);
          }
        }
      }
    __syncthreads();
    const int slot_id = 2 * blockIdx.x + (cur > from ? 1 : 0);
    for (int idx = threadIdx.x; idx < kRows * (D / 2); idx += kWarps * 32) {
      const int r = idx / (D / 2), d = (idx % (D / 2)) * 2;
      if (r >= rows) break;
      float top = -INFINITY;
#pragma unroll
      for (int wv = 0; wv < kWarps; ++wv)
        top = fmaxf(top, reinterpret_cast<const float*>(smem + wv * Sm::kPerWarp)[kRows * (D + 1) + r]);
      float sum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
      for (int wv = 0; wv < kWarps; ++wv) {
        const float* p = reinterpret_cast<const float*>(smem + wv * Sm::kPerWarp);
        const float pm = p[kRows * (D + 1) + r];
        // a warp without entries (or with nothing visible) has sum 0; one whose scores are all NaN keeps its NaN
        const float f = pm == -INFINITY ? 1.f : ex2_approx(pm - top);
        sum = fmaf(f, p[kRows * (D + 1) + kRows + r], sum);
        o0 = fmaf(f, p[r * (D + 1) + d], o0);
        o1 = fmaf(f, p[r * (D + 1) + d + 1], o1);
      }
      if (whole) {
        const int row = row0 + r;
        const bool some = sum != 0.f;  // a NaN stays one
        const float inv = some ? __frcp_rn(sum) : 0.f;
        T* dst = static_cast<T*>(a.o) + static_cast<size_t>(sq.begin + row / a.g) * a.o_rs + (kh * a.g + row % a.g) * D + d;
        *reinterpret_cast<uint32_t*>(dst) = some ? serving::pack2<T>(o0 * inv, o1 * inv) : 0u;
      } else {
        float* p = a.part + static_cast<size_t>(slot_id) * kRows * (D + 2);
        *reinterpret_cast<float2*>(p + r * D + d) = make_float2(o0, o1);
        if (d == 0) *reinterpret_cast<float2*>(p + kRows * D + 2 * r) = make_float2(top, sum);
      }
    }
    cur = seg_end;
    __syncthreads();  // the join buffers are the next item's ring
  }
}

// Joins the partials of the items that the pieces' borders cut; CTA c takes the one that starts in piece c.  A warp takes
// a row and 8 parts at a time, all of whose loads are under way together (a lane D / 32 dimensions, every 8 lanes the
// parts' maxima and sums); what warps the rows leave over take further parts of the same rows, joined through shared
// memory.  Always in the line's order.  Short on purpose: it runs once per call, from a cold instruction cache.
constexpr int kPagedJoinWarps = 16;
constexpr int kPagedJoinParts = 8;

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kPagedJoinWarps * 32) paged_combine_kernel(const PagedAttnArgs a) {
  constexpr int kRows = 8 * NT, kSlot = kRows * (D + 2), kPer = D / 32, kParts = kPagedJoinParts;
  static_assert(kRows <= kPagedJoinWarps, "a warp per row");
  struct __align__(4 * kPer) Vec { float x[kPer]; };
  __shared__ Vec held[kPagedJoinWarps][32];
  __shared__ float2 held_ml[kPagedJoinWarps];
  pdl_wait();
  pdl_trigger();
  const int4 meta = a.meta[blockIdx.x], more = a.meta[gridDim.x + blockIdx.x];
  if (meta.x < 0) return;
  const int kh = meta.y, row0 = meta.z * kRows, parts = meta.w - static_cast<int>(blockIdx.x) + 1;
  const int first_slot = more.x, begin = more.y, n_new = more.z;
  const int rows = min(kRows, n_new * a.g - row0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int subs = kPagedJoinWarps / rows, used = min(subs, (parts + kParts - 1) / kParts);
  const int r = warp % rows, sub = warp / rows;

  Vec o;
#pragma unroll
  for (int i = 0; i < kPer; ++i) o.x[i] = 0.f;
  float top = -INFINITY, sum = 0.f;
  // factors of what is there and of a part with maximum m; nothing to see: sum 0, or NaN where all scores are NaN (kept)
  auto factor = [](float m, float t) { return m == -INFINITY ? 1.f : ex2_approx(m - t); };
  if (sub < used) {
    for (int c0 = sub * kParts; c0 < parts; c0 += used * kParts) {
      auto part = [&](int c) { return a.part + static_cast<size_t>(c == 0 ? first_slot : 2 * (static_cast<int>(blockIdx.x) + c)) * kSlot; };
      const int c = c0 + lane % kParts;
      const float2 ml = c < parts ? *reinterpret_cast<const float2*>(part(c) + kRows * D + 2 * r) : make_float2(-INFINITY, 0.f);
      Vec x[kParts];
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        if (c0 + i < parts) {
          x[i] = *reinterpret_cast<const Vec*>(part(c0 + i) + r * D + kPer * lane);
        } else {
#pragma unroll
          for (int j = 0; j < kPer; ++j) x[i].x[j] = 0.f;
        }
      }
      float t = fmaxf(top, ml.x);
#pragma unroll
      for (int d = 1; d < kParts; d <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
      const float old = factor(top, t), f = factor(ml.x, t);
      float l = f * ml.y;
#pragma unroll
      for (int d = 1; d < kParts; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      sum = fmaf(sum, old, l);
#pragma unroll
      for (int j = 0; j < kPer; ++j) o.x[j] *= old;
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const float fi = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
        for (int j = 0; j < kPer; ++j) o.x[j] = fmaf(fi, x[i].x[j], o.x[j]);
      }
      top = t;
    }
    held[warp][lane] = o;
    if (lane == 0) held_ml[warp] = make_float2(top, sum);
  }
  __syncthreads();
  if (sub > 0) return;
  for (int i = 1; i < used; ++i) {
    const float2 ml = held_ml[warp + i * rows];
    const Vec x = held[warp + i * rows][lane];
    const float t = fmaxf(top, ml.x), old = factor(top, t), f = factor(ml.x, t);
    sum = fmaf(sum, old, f * ml.y);
#pragma unroll
    for (int j = 0; j < kPer; ++j) o.x[j] = fmaf(f, x.x[j], o.x[j] * old);
    top = t;
  }
  const int row = row0 + r;
  const bool some = sum != 0.f;  // a NaN stays one
  const float inv = some ? __frcp_rn(sum) : 0.f;
  T* dst = static_cast<T*>(a.o) + static_cast<size_t>(begin + row / a.g) * a.o_rs + (kh * a.g + row % a.g) * D + kPer * lane;
#pragma unroll
  for (int j = 0; j < kPer; j += 2)
    *reinterpret_cast<uint32_t*>(dst + j) = some ? serving::pack2<T>(o.x[j] * inv, o.x[j + 1] * inv) : 0u;
}

}  // namespace svla
