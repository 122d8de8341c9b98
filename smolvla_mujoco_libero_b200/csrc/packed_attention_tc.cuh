// Attention over packed prompts on the 5th-generation tensor cores (tcgen05): the operator of packed_attention.cuh, for
// prompts long enough to fill 128-row tiles.
//
// One CTA per SM takes two query tiles A and B of 128 packed rows (token-major, then the heads of the group; G * QT rows
// of each are real) of one sequence and kv head, one behind the other, and walks over their keys in tiles of 128 that
// both use.  384 threads:
//   warps 0-3, 4-7  softmax of A and of B: thread t owns TMEM lane t = one query row, so maximum and sum need no
//                   shuffles; the row's 128 scores are held in registers (setmaxnreg)
//   warp 8          TMA of Q, K and V; it also clears from the last V tiles what must not be multiplied (below)
//   warps 9, 10     MMA issuers of A and of B (9 owns the 512 columns of TMEM)
// While one tile's rows are in the softmax, the tensor pipe works for the other.
//
// TMEM.  D = 64: S_A, S_B (128 columns each), P_A, P_B (64), O_A, O_B (64): P has columns of its own, so the next scores
// are computed while the softmax still works on these.  D = 128: P_x over the first half of S_x, O_A, O_B (128): the next
// scores of a tile follow its P.V (the tensor pipe runs one thread's MMAs in order), and P.V starts with the first half of
// P (248 us for four prompts of 1024 to 4096 tokens, 257 with the whole).
//
// What the issuers wait for decides: a ready barrier asked by try_wait through one lane costs 200 cycles, by test_wait 41,
// and one issuer for both tiles needed 3100 cycles for an iteration's waits, MMAs and commits.  One 16384-token prompt at
// D = 64: 860 us; test_wait first: 734; an issuer per tile: 669; one pair of exponentials in eight as polynomials: 650
// (now 640, 800 TFLOP/s, in a graph; 695 where calls follow each other under the power cap).  64 ragged prompts of 1 to 1024
// tokens: 65 us with a CTA's tiles found by a walk through the sequences, 57 by bisection.
// Measured and left: two CTAs of one tile each per SM (715 us; 61 us for 64 ragged prompts where this took 65), the same
// as persistent CTAs that fetch ahead (785 and 63 us), scores read twice from TMEM instead of held (934 us).
//
// Exponentials are the bound at D = 64 (16 per clock and SM: 1024 cycles per 128 x 128 tile against 512 of MMA; the unit is
// 67% busy).  At D = 128 both pipes need 1024 cycles per tile and overlap little: 1800, and an item takes 6.5 us beside its
// tiles.  The running maximum is lazy (O is rescaled only when a row's maximum grows by more than 8 in log2 units, by the
// softmax threads themselves), exponent arguments and sums go through the packed fp32 pipe.
//
// What stands behind a sequence's last key belongs to its neighbour: scores there are masked, and the V rows of the tile
// are set to zero in shared memory before the product (0 * NaN would be NaN).  Under a causal mask the same holds inside
// the sequence for infinities and NaN in rows that some query of the CTA does not see; the epilogue then adds them to the
// rows that do.
#pragma once

#include <type_traits>

#include "packed_attention.cuh"

namespace svla {

struct PackedTcArgs {
  CUtensorMap tq;      // 3-D (dim, head, token): box 64 x G x QT, 128-byte swizzle
  CUtensorMap tk, tv;  // 3-D (dim, head, token): box 64 x 1 x 128
  const void* v;
  void* o;
  const int *cu_q, *cu_k;
  long long v_rs, o_rs;
  int batch, total_q, total_k, hq, hkv, g, qt;
  int causal;
  float scale_log2;
  int* err;
};

namespace ptc {
constexpr int kKeys = 128, kThreads = 384;
// registers: 384 threads x 168 at launch = 64512; the two softmax warpgroups take 208 each, the third keeps 88:
// 256 * 208 + 128 * 88 = 64512
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;

template <int D>
struct Cfg {
  static constexpr int kSub = D / 64;                 // 64-dimension blocks of a row (one 128-byte swizzle row each)
  static constexpr int kTile = 128 * D * 2;           // bytes of a Q, K or V tile
  static constexpr int kStages = D == 64 ? 4 : 2;     // K tiles and V tiles in their rings
  static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + kStages * kTile, kBar = kV + kStages * kTile;
  static constexpr int kSmem = kBar + 512 + 1024;     // + barriers + alignment slack
  static constexpr bool kOwnP = D == 64;              // P has its own columns
  static constexpr uint32_t kS = 0;                   // + 128 x
  static constexpr uint32_t kP = kOwnP ? 256 : 0;     // + 64 x, or over S_x
  static constexpr uint32_t kPStride = kOwnP ? 64 : 128;
  static constexpr uint32_t kO = kOwnP ? 384 : 256;   // + D x
};

using serving::elect_one;
using serving::wait_warp;

// instruction descriptor of kind::f16 for the type: fp32 accumulators, A and B of one type (fp16 0, bf16 1)
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int m, int n) {
  const uint32_t f = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^z for two z <= 15 or so on the fp32 pipe, by Cody and Waite's reduction (Software manual for the elementary functions,
// 1980): z = n + f with n = rint(z) (adding 1.5 * 2^23 leaves n in the low bits), 2^f by its minimax polynomial of degree 4
// on [-1/2, 1/2] (relative error 2.6e-6, found by exchanging extrema), times 2^n.  z is first raised to at least -127, whose
// power's exponent field is 0: a masked score's weight (z = -infinity), and every weight below 2^-126.5, is exactly 0, so
// no hidden value enters whatever its size.  A NaN stays one: the maximum keeps it, and so does the product (n added to the
// exponent's bits would not).
__device__ __forceinline__ float2 exp2_poly(float2 z) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(z.x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(z.y) : "f"(-127.f));
  auto both = [](float c) { return make_float2(c, c); };
  const float2 t = __fadd2_rn(z, both(12582912.f));
  const float2 f = __fadd2_rn(z, __ffma2_rn(t, both(-1.f), both(12582912.f)));
  float2 p = __ffma2_rn(f, both(0.0095701f), both(0.05591786f));
  p = __ffma2_rn(f, p, both(0.24024745f));
  p = __ffma2_rn(f, p, both(0.69312181f));
  p = __ffma2_rn(f, p, both(0.99999926f));
  auto power = [](float n) { return __uint_as_float((__float_as_uint(n) << 23) + 0x3F800000u); };  // of n's low bits
  return __fmul2_rn(p, make_float2(power(t.x), power(t.y)));
}
}  // namespace ptc

template <typename T, int D>
__global__ void __launch_bounds__(ptc::kThreads, 1) packed_attention_tc_kernel(const __grid_constant__ PackedTcArgs a) {
  using namespace ptc;
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::kBar);  // [2]
  uint64_t* k_full = q_full + 2;
  uint64_t* k_empty = k_full + C::kStages;
  uint64_t* v_full = k_empty + C::kStages;
  uint64_t* v_empty = v_full + C::kStages;
  uint64_t* v_clear = v_empty + C::kStages;  // an edge tile's V has been cleared
  uint64_t* s_full = v_clear + C::kStages;   // [2] scores are there
  uint64_t* s_free = s_full + 2;             // [2] (own P) scores are in registers
  uint64_t* p_half = s_free + 2;             // [2] the first 64 keys' probabilities are there
  uint64_t* p_full = p_half + 2;             // [2] all of them
  uint64_t* o_done = p_full + 2;             // [2] the tile's P.V so far is done
  uint64_t* all_done = o_done + 2;           // [2] everything the tile's issuer owes
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(all_done + 2);
  int* place = reinterpret_cast<int*>(tmem_slot + 1);  // [2] sequence, item
  int* odd_flag = place + 2;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == 8) {
    if (lane == 0) {
      for (int s = 0; s < C::kStages; ++s) {
        mbar_init(&k_full[s], 1);
        mbar_init(&k_empty[s], 2);  // both tiles' MMAs
        mbar_init(&v_full[s], 1);
        mbar_init(&v_empty[s], 2);
        mbar_init(&v_clear[s], 1);
      }
      for (int x = 0; x < 2; ++x) {
        mbar_init(&q_full[x], 1);
        mbar_init(&s_full[x], 1);
        mbar_init(&s_free[x], 4);
        mbar_init(&p_half[x], 4);
        mbar_init(&p_full[x], 4);
        mbar_init(&o_done[x], 1);
        mbar_init(&all_done[x], 1);
      }
      fence_mbar_init();
      *odd_flag = 0;
    }
  } else if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_wait();  // lengths, q, k, v are written by the previous kernel
  if (warp == 0) {
    int b = -1, j = 0;
    const packed_detail::TileOrder order{a.cu_q, a.batch, a.total_q, 2 * a.qt};
    const bool ok = order.find(static_cast<int>(blockIdx.x) / a.hkv, lane, b, j);
    if (lane == 0) {
      place[0] = ok ? b : -1;
      place[1] = j;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;
  const int b = place[0], kh = blockIdx.x % a.hkv;
  if (b >= 0) {
    const serving::Span sq = serving::span_of(a.cu_q, b, a.total_q), sk = serving::span_of(a.cu_k, b, a.total_k);
    const int n_q = sq.end - sq.begin, n_k = sk.end - sk.begin, past = n_k - n_q;
    auto seen = [&](int tok) { return a.causal ? min(max(past + tok + 1, 0), n_k) : n_k; };
    // tile x: tokens tok[x] .. of the sequence, toks[x] of them, n[x] key tiles
    int tok[2], toks[2], n[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      tok[x] = (2 * place[1] + x) * a.qt;
      toks[x] = min(max(n_q - tok[x], 0), a.qt);
      n[x] = toks[x] > 0 ? (seen(tok[x] + toks[x] - 1) + kKeys - 1) / kKeys : 0;
    }
    const int n_all = max(n[0], n[1]);
    // from this key tile on, V is cleared before it is multiplied: rows behind the sequence, rows that some query of the
    // CTA does not see
    const int first_clear = seen(tok[0]) / kKeys;

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 8) {
      // ---------------- producer
      if (lane == 0) {
        prefetch_tmap(&a.tq);
        prefetch_tmap(&a.tk);
        prefetch_tmap(&a.tv);
      }
      auto load_q = [&](int x) {
        mbar_arrive_expect_tx(&q_full[x], static_cast<uint32_t>(a.g * a.qt * D * 2));
#pragma unroll
        for (int c = 0; c < C::kSub; ++c)
          tma_load_3d(smem + C::kQ + x * C::kTile + c * 16384, &a.tq, &q_full[x], c * 64, kh * a.g, sq.begin + tok[x]);
      };
      auto load_kv = [&](const CUtensorMap* map, uint64_t* full, uint8_t* dst, int j) {
        mbar_arrive_expect_tx(full, C::kTile);
#pragma unroll
        for (int c = 0; c < C::kSub; ++c) tma_load_3d(dst + c * 16384, map, full, c * 64, kh, sk.begin + j * kKeys);
      };
      // sets what must not be multiplied in V tile j to zero, in shared memory
      auto clear = [&](int j) -> bool {
        const int s = j % C::kStages;
        if (!wait_warp(&v_full[s], (j / C::kStages) & 1, a.err)) return false;
        uint8_t* vt = smem + C::kV + s * C::kTile;
        const int behind = min(max(n_k - j * kKeys, 0), kKeys);                  // rows from here on are another's
        const int hidden = a.causal ? max(seen(tok[0]) - j * kKeys, 0) : kKeys;  // rows from here on some query does not see
#pragma unroll 1
        for (int c = 0; c < C::kSub; ++c) {
          for (int i = lane + behind * 8; i < 128 * 8; i += 32)
            *reinterpret_cast<uint4*>(vt + c * 16384 + i * 16) = make_uint4(0, 0, 0, 0);
          bool odd = false;
#pragma unroll 2
          for (int i = lane + hidden * 8; i < behind * 8; i += 32) {
            const uint4 u = *reinterpret_cast<const uint4*>(vt + c * 16384 + i * 16);
            odd |= serving::any_nonfinite<T>(u.x) || serving::any_nonfinite<T>(u.y) || serving::any_nonfinite<T>(u.z) ||
                   serving::any_nonfinite<T>(u.w);
          }
          if (odd) {
            *odd_flag = 1;
            for (int i = lane + hidden * 8; i < behind * 8; i += 32) {
              uint32_t* w = reinterpret_cast<uint32_t*>(vt + c * 16384 + i * 16);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (serving::any_nonfinite<T>(w[e] & 0xFFFFu)) w[e] &= 0xFFFF0000u;
                if (serving::any_nonfinite<T>(w[e] & 0xFFFF0000u)) w[e] &= 0xFFFFu;
              }
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_clear[s]);
        return true;
      };
      bool ok = true;
      int next_clear = first_clear, issued = 0;
      for (int j = 0; j < n_all && ok; ++j) {
        const int s = j % C::kStages;
        if (j >= C::kStages) {
          // the tile whose place this one takes has to be cleared before it can be multiplied
          while (ok && next_clear <= j - C::kStages) ok = clear(next_clear++);
          ok = ok && wait_warp(&k_empty[s], ((j / C::kStages) - 1) & 1, a.err);
        }
        if (ok && lane == 0) {
          if (j == 0 && n[0] > 0) load_q(0);
          load_kv(&a.tk, &k_full[s], smem + C::kK + s * C::kTile, j);
          if (j == 0 && n[1] > 0) load_q(1);
        }
        if (j >= C::kStages) ok = ok && wait_warp(&v_empty[s], ((j / C::kStages) - 1) & 1, a.err);
        if (ok && lane == 0) {
          load_kv(&a.tv, &v_full[s], smem + C::kV + s * C::kTile, j);
          issued = j + 1;
        }
      }
      while (ok && next_clear < n_all) ok = clear(next_clear++);
      if (!ok && lane == 0)  // a wait ran out: no copy may be in flight when the CTA ends
        for (int j = max(issued - C::kStages, 0); j < issued; ++j) {
          mbar_wait(&k_full[j % C::kStages], (j / C::kStages) & 1, a.err);
          mbar_wait(&v_full[j % C::kStages], (j / C::kStages) & 1, a.err);
        }
    } else if (warp < 11) {
      // ---------------- MMA issuer of tile x (warps 9, 10).  The whole warp walks through the loop and one elected lane
      // issues.  A warp of its own for each tile: waits, issue and commits of one iteration for both tiles took one warp
      // 3100 cycles, longer than the softmax that they serve.
      const int x = warp - 9, nx = x ? n[1] : n[0];
      const uint32_t id_qk = idesc<T>(128, kKeys);
      const uint32_t id_pv = idesc<T>(128, D) | (1u << 16);  // B (V) is MN-major
      const uint32_t k0 = smem_u32(smem + C::kK), v0 = smem_u32(smem + C::kV);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      // descriptors of a tile's first MMA; the others are constant distances (in 16-byte units) away
      const uint64_t qd = smem_desc_sw128(smem_u32(smem + C::kQ) + x * C::kTile);
      auto qk = [&](int j) {  // and the K tile is free again
        const uint64_t kd = smem_desc_sw128(k0 + (j % C::kStages) * C::kTile);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {  // 16 dimensions (32 bytes) per MMA
            const uint32_t off = ((kk / 4) * 16384 + (kk % 4) * 32) >> 4;
            mma_bf16(tm + C::kS + x * 128, qd + off, kd + off, id_qk, kk > 0 ? 1u : 0u);
          }
          mma_commit(&s_full[x]);
          mma_commit(&k_empty[j % C::kStages]);
        }
        __syncwarp();
      };
      // keys 16 first .. 16 last - 1 of the tile; after the last ones the V tile is free again
      auto pv = [&](int j, auto first, auto last) {
        const uint64_t vd = smem_desc_sw128_lbo(v0 + (j % C::kStages) * C::kTile, 16384);
        if (elect_one()) {
#pragma unroll
          for (int kk = first.value; kk < last.value; ++kk)  // 16 keys per MMA: 8 TMEM columns of P, 16 rows (2048 bytes) of V
            mma_bf16_tmem_a(tm + C::kO + x * D, tm + C::kP + x * C::kPStride + kk * 8, vd + kk * (2048 >> 4), id_pv,
                            (j > 0 || kk > 0) ? 1u : 0u);
          if (last.value == 8) {
            mma_commit(&o_done[x]);
            mma_commit(&v_empty[j % C::kStages]);
          }
        }
        __syncwarp();
      };
      using std::integral_constant;
      auto k_there = [&](int j) { return wait_warp(&k_full[j % C::kStages], (j / C::kStages) & 1, a.err); };
      auto v_there = [&](int j) {
        const int s = j % C::kStages;
        if (j >= first_clear) return wait_warp(&v_clear[s], ((j - first_clear) / C::kStages) & 1, a.err);
        return wait_warp(&v_full[s], (j / C::kStages) & 1, a.err);
      };
      bool ok = nx > 0 && wait_warp(&q_full[x], 0, a.err) && k_there(0);
      if (ok) qk(0);
      for (int j = 0; j < nx && ok; ++j) {
        if (C::kOwnP && j + 1 < nx) {  // the next scores as soon as these are in registers
          ok = k_there(j + 1) && wait_warp(&s_free[x], j & 1, a.err);
          tc_fence_after();
          if (ok) qk(j + 1);
        }
        ok = ok && v_there(j);
        if constexpr (C::kOwnP) {
          ok = ok && wait_warp(&p_full[x], j & 1, a.err);
          tc_fence_after();
          if (ok) pv(j, integral_constant<int, 0>{}, integral_constant<int, 8>{});
        } else {  // both pipes are the bound: start when half of P is there
          ok = ok && wait_warp(&p_half[x], j & 1, a.err);
          tc_fence_after();
          if (ok) pv(j, integral_constant<int, 0>{}, integral_constant<int, 4>{});
          ok = ok && wait_warp(&p_full[x], j & 1, a.err);
          tc_fence_after();
          if (ok) pv(j, integral_constant<int, 4>{}, integral_constant<int, 8>{});
        }
        if (!C::kOwnP && j + 1 < nx) {
          ok = ok && k_there(j + 1);
          if (ok) qk(j + 1);
        }
      }
      // Key tiles that only the other query tile uses: given back once they are there.  Not earlier: an arrival before
      // would count for the tile that had the place before, and the producer would arm a barrier whose copy is in flight.
      for (int j = nx; j < n_all && (ok || nx == 0); ++j) {
        if (!k_there(j)) break;
        if (lane == 0) mbar_arrive(&k_empty[j % C::kStages]);
        if (!wait_warp(&v_full[j % C::kStages], (j / C::kStages) & 1, a.err)) break;
        if (lane == 0) mbar_arrive(&v_empty[j % C::kStages]);
      }
      if (nx > 0) {  // every MMA and every arrival it owes is done before the TMEM and the CTA go
        if (elect_one()) mma_commit(&all_done[x]);
        __syncwarp();
        wait_warp(&all_done[x], 0, a.err);
      }
    }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
      // ---------------- softmax of tile x
      const int x = warp >> 2, wq = warp & 3;
      const int row = wq * 32 + lane, t = tok[x] + row / a.g, head = kh * a.g + row % a.g;
      const bool real = row < toks[x] * a.g;
      const int sees = real ? seen(t) : 0x7fffffff;  // rows that are not real are not stored, and need no mask
      const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
      const uint32_t tS = tmem + lanes + C::kS + x * 128, tP = tmem + lanes + C::kP + x * C::kPStride;
      const uint32_t tO = tmem + lanes + C::kO + x * D;
      const float c = a.scale_log2;
      float m = -INFINITY;
      float2 l = make_float2(0.f, 0.f);
      bool ok = true;
      for (int j = 0; j < n[x] && ok; ++j) {
        ok = wait_warp(&s_full[x], j & 1, a.err);
        if (!ok) break;
        tc_fence_after();
        const int left = sees - j * kKeys;  // keys of this tile that the row sees
        uint32_t r[kKeys];
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) tmem_ld32(tS + ch * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[ch * 32]));
        tmem_ld_wait();
        if constexpr (C::kOwnP) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[x]);
        }
        if (__any_sync(0xffffffffu, left < kKeys)) {
#pragma unroll
          for (int e = 0; e < kKeys; ++e)
            if (e >= left) r[e] = 0xFF800000u;  // -infinity
        }
        float mp[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) mp[u] = fmaxf(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1]));
#pragma unroll
        for (int e = 16; e < kKeys; e += 2)
          mp[(e >> 1) & 7] = max3(mp[(e >> 1) & 7], __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
        const float top = fmaxf(max3(mp[0], mp[1], mp[2]), max3(max3(mp[3], mp[4], mp[5]), mp[6], mp[7])) * c;
        // the tile's P.V before this one: it reads P (own columns) and adds to O, which may be rescaled below
        const bool grow = top > m + 8.f;
        if (j > 0 && (C::kOwnP || __any_sync(0xffffffffu, grow))) {
          ok = wait_warp(&o_done[x], (j - 1) & 1, a.err);
          if (!ok) break;
          tc_fence_after();
        }
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = !grow || m == -INFINITY ? 1.f : ex2_approx(m - top);
          if (grow) m = top;
          l = __fmul2_rn(l, make_float2(alpha, alpha));
          if (j > 0) {
#pragma unroll 1
            for (int ch = 0; ch < D / 16; ++ch) {
              uint32_t w[16];
              tmem_ld16(tO + ch * 16, w);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__fmul_rn(__uint_as_float(w[e]), alpha));
              tmem_st16(tO + ch * 16, w);
            }
          }
        }
        const float use = m == -INFINITY ? 0.f : m - serving::kWeightLift<T>;
        const float2 c2 = make_float2(c, c), nm2 = make_float2(-use, -use);
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const int k = ch * 32 + e;
            const float2 z = __ffma2_rn(make_float2(__uint_as_float(r[k]), __uint_as_float(r[k + 1])), c2, nm2);
            // one pair in eight leaves the exponential unit, where that is the bound (638 us; none 669, one in four 676)
            const float2 p = (D == 64 && (e / 2) % 8 == 0) ? exp2_poly(z) : make_float2(ex2_approx(z.x), ex2_approx(z.y));
            l = __fadd2_rn(l, p);
            pk[e / 2] = serving::pack2<T>(p.x, p.y);
          }
          tmem_st16(tP + ch * 16, pk);
          if (ch == 3 || (!C::kOwnP && ch == 1)) {
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ch == 1 ? &p_half[x] : &p_full[x]);
          }
        }
      }
      // ---------------- epilogue
      if (ok && n[x] > 0) {
        ok = wait_warp(&o_done[x], (n[x] - 1) & 1, a.err);
        tc_fence_after();
      }
      if (ok && toks[x] > 0) {
        const float sum = l.x + l.y;
        const bool some = sum != 0.f;  // 0: no key to see, or none whose score is above -infinity; a NaN stays one
        const float inv = some ? __frcp_rn(sum) : 0.f;
        T* dst = static_cast<T*>(a.o) + static_cast<size_t>(sq.begin + (real ? t : 0)) * a.o_rs + head * D;
        const bool odd = *reinterpret_cast<volatile int*>(odd_flag) != 0;
#pragma unroll
        for (int ch = 0; ch < D / 32; ++ch) {
          uint32_t r[32];
          __syncwarp();
          if (n[x] > 0) {
            tmem_ld32(tO + ch * 32, r);
            tmem_ld_wait();
          }
          if (!real) continue;
          if (odd) {  // rare: the infinities and NaN that left V, for the rows that see them
            for (int j = first_clear * kKeys; j < sees; ++j) {
              const T* vr = static_cast<const T*>(a.v) + static_cast<size_t>(sk.begin + j) * a.v_rs + kh * D + ch * 32;
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 f = serving::unpack2<T>(*reinterpret_cast<const uint32_t*>(vr + e));
                if (!isfinite(f.x)) r[e] = __float_as_uint(__uint_as_float(r[e]) + f.x);
                if (!isfinite(f.y)) r[e + 1] = __float_as_uint(__uint_as_float(r[e + 1]) + f.y);
              }
            }
          }
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)
            w[e] = some ? serving::pack2<T>(__uint_as_float(r[2 * e]) * inv, __uint_as_float(r[2 * e + 1]) * inv) : 0u;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *reinterpret_cast<uint4*>(dst + ch * 32 + u * 8) = make_uint4(w[4 * u], w[4 * u + 1], w[4 * u + 2], w[4 * u + 3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace svla
