// Attention over packed prompts: sequence b has queries cu_q[b] .. cu_q[b + 1] and keys cu_k[b] .. cu_k[b + 1] (n_q and
// n_k of them) of one packed tensor each; query i sees key j iff not causal, or j <= n_k - n_q + i (the queries are the
// last tokens);  o_i = sum_j softmax_j(scale q_i . k_j) v_j, zeros where no key weighs anything: where there is none to see,
// or every score is -infinity.
//
// One pass over the keys with the running maximum and sum of the softmax, fp32 scores and sums, probabilities rounded
// to the input type for the second product (as the framework's other attention kernels do).
//
// This form is for short prompts: 64 rows per CTA on mma.sync, whose start costs less than a tcgen05 tile's; bound by that
// start (place, first copies, cold code) and by instruction issue.  One prompt of 177 tokens at 15 / 5 heads of 64 takes
// 5.9 us: 7.8 with divisions from rows to tokens, scaled scores in the maximum and a walk to the tile's place, 7.1 with an
// eager running maximum, 6.4 with the numbering of many sequences.  64 prompts of 128 tokens 30 us, of 256 69 us.
//
// A query row is a (token, head) of one kv head, packed token-major (row r = token r / G, head r % G), so the G heads of
// a group share every key tile and the causal limit is nearly the same for all rows of a tile.  Whatever stands behind a
// sequence's last key -- the next sequence, padding, NaN -- is never multiplied in: those rows of V are zeros.  An
// infinity or a NaN in the value of a key that only later queries see is set to zero for the product and added to
// exactly the rows that see it afterwards.
#pragma once

#include "serving_common.cuh"

namespace svla {

struct PackedAttnArgs {
  const void *q, *k, *v;
  void* o;
  const int *cu_q, *cu_k;
  long long q_rs, k_rs, v_rs, o_rs;
  int batch, total_q, total_k, hq, hkv, g, qt;  // qt: tokens of a query tile
  unsigned g_magic;  // ceil(2^16 / g): row -> token, exact for the 64 rows of a tile and g <= 64
  int causal;
  float scale_log2;
};

namespace packed_detail {
constexpr int kWarps = 4;
constexpr int kRows = 16 * kWarps;  // query rows per CTA
constexpr int kKeys = 64;

// Tile number id of `qt` tokens of all sequences: its sequence and its place there; false: there is no such tile.  A warp
// calls it; ids go up to total / qt + batch.
//
// 2 to 128 sequences: longest first, by place from the largest down (a causal tile's keys grow with it), then by sequence.
// The place is found by bisection over the tiles that lie at a place or behind it, sum_b max(count_b - place, 0), with the
// counts in registers: half a microsecond of a CTA, for which a long sequence at the batch's end does not start last.
//
// One sequence, or more than registers hold: sequence b has the numbers from cu_q[b] / qt + b on (enough for its tiles, and
// a few that there are not), its longest tile first, so a search in cu_q finds them.  Measured, by place / by sequence: one
// prompt of 177 tokens 6.4 / 5.8 us, of 16384 654 / 641; 64 ragged prompts 57.2 / 57.9; 1024 prompts of 64 tokens, counts
// read again at every step, 527 / 217.
struct TileOrder {
  static constexpr int kHeld = 4;
  const int* cu_q;
  int batch, total, qt;

  __device__ __forceinline__ int count(int i) const {
    const serving::Span s = serving::span_of(cu_q, i, total);
    return (s.end - s.begin + qt - 1) / qt;
  }
  __device__ __forceinline__ bool find(int id, int lane, int& b, int& place) const {
    return batch > 1 && batch <= 32 * kHeld ? by_place(id, lane, b, place) : by_sequence(id, lane, b, place);
  }
  __device__ __forceinline__ bool by_place(int id, int lane, int& b, int& place) const {
    int held[kHeld], top = 0;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      held[u] = lane + 32 * u < batch ? count(lane + 32 * u) : 0;
      top = max(top, held[u]);
    }
    // from(place): tiles at `place` or behind it
    int behind = __reduce_max_sync(0xffffffffu, top), rank = id;  // from(behind) <= id < from(place), or place = 0 and
    place = 0;                                                    // there may be no such tile
#pragma unroll 1
    while (behind - place > 1) {
      const int mid = (place + behind) >> 1;
      int n = 0;
#pragma unroll
      for (int u = 0; u < kHeld; ++u) n += max(held[u] - mid, 0);
      n = __reduce_add_sync(0xffffffffu, n);
      if (n > id) {
        place = mid;
      } else {
        behind = mid;
        rank = id - n;
      }
    }
    b = -1;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {  // set bit number `rank` of the sequences that have this place
      const unsigned m = __ballot_sync(0xffffffffu, held[u] > place);
      if (rank >= 0 && rank < __popc(m)) {
        const bool me = ((m >> lane) & 1u) && __popc(m & ((1u << lane) - 1u)) == rank;
        b = 32 * u + __ffs(__ballot_sync(0xffffffffu, me)) - 1;
      }
      rank -= __popc(m);
    }
    return b >= 0;
  }
  __device__ __forceinline__ bool by_sequence(int id, int lane, int& b, int& place) const {
    auto start = [&](int i) { return min(max(__ldg(cu_q + i), 0), total) / qt + i; };
    int lo = 0, hi = batch;  // start(lo) <= id < start(hi)
#pragma unroll 1
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int at = lo + (lane + 1) * step;
      const bool below = at < hi && start(at) <= id;
      lo += __popc(__ballot_sync(0xffffffffu, below)) * step;
      hi = min(lo + step, hi);
    }
    b = lo;
    const int n = count(lo), j = id - start(lo);
    place = n - 1 - j;
    return j >= 0 && j < n;
  }
};
}  // namespace packed_detail

template <typename T, int D>
struct PackedSmem {
  static constexpr int kQ = 0, kTile = packed_detail::kKeys * D * 2, kK = packed_detail::kRows * D * 2,
                       kV = kK + 2 * kTile, kBytes = kV + 2 * kTile;
};

template <typename T, int D>
__global__ void __launch_bounds__(packed_detail::kWarps * 32) packed_attention_kernel(const PackedAttnArgs a) {
  using namespace packed_detail;
  using serving::copy16;
  using Sm = PackedSmem<T, D>;
  constexpr int kRow = D * 2, kChunks = D / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int place[2], odd_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  pdl_wait();
  pdl_trigger();
  const int kh = blockIdx.x % a.hkv;
  if (warp == 0) {
    int b = -1, j = 0;
    const TileOrder order{a.cu_q, a.batch, a.total_q, a.qt};
    const bool ok = order.find(static_cast<int>(blockIdx.x) / a.hkv, lane, b, j);
    if (lane == 0) {
      place[0] = ok ? b : -1;
      place[1] = j;
      odd_flag = 0;
    }
  }
  __syncthreads();
  const int b = place[0];
  if (b < 0) return;
  const serving::Span sq = serving::span_of(a.cu_q, b, a.total_q), sk = serving::span_of(a.cu_k, b, a.total_k);
  const int n_q = sq.end - sq.begin, n_k = sk.end - sk.begin;
  const int tok0 = place[1] * a.qt, toks = min(a.qt, n_q - tok0), rows = toks * a.g;
  const int past = n_k - n_q;
  auto seen = [&](int tok) { return a.causal ? min(max(past + tok + 1, 0), n_k) : n_k; };
  const int sees_last = seen(tok0 + toks - 1), sees_first = seen(tok0);
  const int n_tiles = (sees_last + kKeys - 1) / kKeys;

  auto token = [&](int r) { return static_cast<int>(static_cast<unsigned>(r) * a.g_magic >> 16); };
  {
    const T* qb = static_cast<const T*>(a.q) + static_cast<size_t>(sq.begin + tok0) * a.q_rs + kh * a.g * D;
#pragma unroll
    for (int u = 0; u < kRows * kChunks / (kWarps * 32); ++u) {
      const int idx = threadIdx.x + u * kWarps * 32, r = idx / kChunks, c = idx % kChunks, tk = token(r);
      const bool in = r < rows;
      const T* src = qb + (in ? static_cast<size_t>(tk) * a.q_rs + (r - tk * a.g) * D + c * 8 : 0);
      copy16(smem + Sm::kQ + r * kRow + ((c ^ (r & 7)) * 16), src, in ? 16 : 0);
    }
  }
  auto load = [&](int tile) {
    const T* kb = static_cast<const T*>(a.k) + static_cast<size_t>(sk.begin) * a.k_rs + kh * D;
    const T* vb = static_cast<const T*>(a.v) + static_cast<size_t>(sk.begin) * a.v_rs + kh * D;
    uint8_t* kd = smem + Sm::kK + (tile & 1) * Sm::kTile;
    uint8_t* vd = smem + Sm::kV + (tile & 1) * Sm::kTile;
#pragma unroll
    for (int u = 0; u < kKeys * kChunks / (kWarps * 32); ++u) {
      const int idx = threadIdx.x + u * kWarps * 32, r = idx / kChunks, c = idx % kChunks;
      const int key = tile * kKeys + r;
      const bool in = key < n_k;  // zeros behind the last key
      const int dst = r * kRow + ((c ^ (r & 7)) * 16);
      copy16(kd + dst, kb + (in ? static_cast<size_t>(key) * a.k_rs + c * 8 : 0), in ? 16 : 0);
      copy16(vd + dst, vb + (in ? static_cast<size_t>(key) * a.v_rs + c * 8 : 0), in ? 16 : 0);
    }
  };
  if (n_tiles > 0) load(0);
  serving::copy_commit();

  const int wr = warp * 16;
  int sees[2];  // keys that this thread's rows see
#pragma unroll
  for (int hr = 0; hr < 2; ++hr) sees[hr] = seen(tok0 + token(wr + g8 + 8 * hr));
  uint32_t qa[D / 16][4];
  float o[D / 8][4];
#pragma unroll
  for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, use[2] = {0.f, 0.f}, l[2] = {0.f, 0.f};

  for (int tile = 0; tile < n_tiles; ++tile) {
    if (tile + 1 < n_tiles) load(tile + 1);
    serving::copy_commit();
    serving::copy_wait<1>();
    __syncthreads();
    if (tile == 0) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int r = wr + (lane & 15), ch = kk * 2 + (lane >> 4);
        serving::ldsm_x4(qa[kk], smem + Sm::kQ + r * kRow + ((ch ^ (r & 7)) * 16));
      }
    }
    const uint8_t* kt = smem + Sm::kK + (tile & 1) * Sm::kTile;
    uint8_t* vt = smem + Sm::kV + (tile & 1) * Sm::kTile;
    const int key0 = tile * kKeys;
    const bool edge = key0 + kKeys > sees_first;
    if (edge && a.causal) {  // some row does not see some key of the tile: infinities and NaN leave V for now
      bool odd = false;
      for (int idx = threadIdx.x; idx < kKeys * kChunks; idx += kWarps * 32) {
        uint4 u = *reinterpret_cast<uint4*>(vt + idx * 16);
        if (serving::any_nonfinite<T>(u.x) || serving::any_nonfinite<T>(u.y) || serving::any_nonfinite<T>(u.z) ||
            serving::any_nonfinite<T>(u.w)) {
          odd = true;
          uint32_t uu[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (serving::any_nonfinite<T>(uu[i] & 0xFFFFu)) uu[i] &= 0xFFFF0000u;
            if (serving::any_nonfinite<T>(uu[i] & 0xFFFF0000u)) uu[i] &= 0xFFFFu;
          }
          *reinterpret_cast<uint4*>(vt + idx * 16) = make_uint4(uu[0], uu[1], uu[2], uu[3]);
        }
      }
      if (odd) odd_flag = 1;
      __syncthreads();
    }
    float s[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int np = 0; np < kKeys / 16; ++np) {
        uint32_t kb[4];
        const int r = np * 16 + (lane & 7) + ((lane >> 4) << 3), ch = kk * 2 + ((lane >> 3) & 1);
        serving::ldsm_x4(kb, kt + r * kRow + ((ch ^ (r & 7)) * 16));
        serving::mma16816<T>(s[2 * np], qa[kk], kb[0], kb[1]);
        serving::mma16816<T>(s[2 * np + 1], qa[kk], kb[2], kb[3]);
      }
    }
    if (edge) {
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key0 + n * 8 + 2 * t4 + (e & 1) >= sees[e >> 1]) s[n][e] = -INFINITY;
    }
    // The running maximum is lazy: it moves, and O is rescaled, only when a score of the warp passes its row's by more than
    // 8 in log2 units (weights up to 2^8 of the maximum's cancel in O / l)
    float top[2];
    bool pass = false;
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      top[hr] = fmaxf(s[0][2 * hr], s[0][2 * hr + 1]);
#pragma unroll
      for (int n = 1; n < kKeys / 8; ++n) top[hr] = fmaxf(top[hr], fmaxf(s[n][2 * hr], s[n][2 * hr + 1]));
      top[hr] *= a.scale_log2;
      pass |= top[hr] > m[hr] + 8.f;
    }
    if (__any_sync(0xffffffffu, pass)) {
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        float t = fmaxf(m[hr], top[hr]);
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
        const float alpha = m[hr] == -INFINITY ? 1.f : ex2_approx(m[hr] - t);
        m[hr] = t;
        use[hr] = t == -INFINITY ? 0.f : t - serving::kWeightLift<T>;
        l[hr] *= alpha;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][2 * hr] *= alpha;
          o[n][2 * hr + 1] *= alpha;
        }
      }
    }
    uint32_t pa[kKeys / 16][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = ex2_approx(fmaf(s[n][e], a.scale_log2, -use[e >> 1]));
        l[e >> 1] += p[e];
      }
      pa[n >> 1][(n & 1) * 2] = serving::pack2<T>(p[0], p[1]);
      pa[n >> 1][(n & 1) * 2 + 1] = serving::pack2<T>(p[2], p[3]);
    }
#pragma unroll
    for (int kk = 0; kk < kKeys / 16; ++kk) {
#pragma unroll
      for (int np = 0; np < D / 16; ++np) {
        uint32_t vb[4];
        const int r = kk * 16 + (lane & 15), ch = np * 2 + (lane >> 4);
        serving::ldsm_x4_trans(vb, vt + r * kRow + ((ch ^ (r & 7)) * 16));
        serving::mma16816<T>(o[2 * np], pa[kk], vb[0], vb[1]);
        serving::mma16816<T>(o[2 * np + 1], pa[kk], vb[2], vb[3]);
      }
    }
    __syncthreads();
  }
  serving::copy_wait<0>();
  __syncthreads();

#pragma unroll
  for (int hr = 0; hr < 2; ++hr) {
    l[hr] += __shfl_xor_sync(0xffffffffu, l[hr], 1);
    l[hr] += __shfl_xor_sync(0xffffffffu, l[hr], 2);
    const int r = wr + g8 + 8 * hr;
    if (r >= rows) continue;
    const int tk = token(r), tok = tok0 + tk, h = kh * a.g + r - tk * a.g;
    if (odd_flag) {  // rare: the infinities and NaN that left V, for the rows that see them
      for (int j = sees_first / kKeys * kKeys; j < sees[hr]; ++j) {
        const T* vr = static_cast<const T*>(a.v) + static_cast<size_t>(sk.begin + j) * a.v_rs + kh * D;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          const uint32_t u = *reinterpret_cast<const uint32_t*>(vr + n * 8 + 2 * t4);
          const float2 f = serving::unpack2<T>(u);
          if (!isfinite(f.x)) o[n][2 * hr] += f.x;
          if (!isfinite(f.y)) o[n][2 * hr + 1] += f.y;
        }
      }
    }
    const bool some = l[hr] != 0.f;  // 0: no key to see, or none whose score is above -infinity; a NaN stays one
    const float inv = some ? __frcp_rn(l[hr]) : 0.f;
    T* dst = static_cast<T*>(a.o) + static_cast<size_t>(sq.begin + tok) * a.o_rs + h * D + 2 * t4;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
      *reinterpret_cast<uint32_t*>(dst + n * 8) =
          some ? serving::pack2<T>(o[n][2 * hr] * inv, o[n][2 * hr + 1] * inv) : 0u;
  }
}

}  // namespace svla
