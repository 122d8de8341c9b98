// The choice of a token from a row of logits l, given a uniform random number u:
//   w_i = round(2^44 exp((l_i - max l) / temperature)), whole numbers;
//   kept: the top_k largest logits with w_i >= min_p 2^44, of these the most likely up to the one with which their sum reaches
//   top_p of it; equal logits in the order of their indices (the lower one first);
//   the token is the first, by index, up to which the kept w add up to more than floor(u sum w).
// Whole numbers add up to the same in any order, so the answer depends neither on how a row is shared nor on timing.  2^44 leaves
// 2^18 tokens in 62 bits; a token below 2^-45 of the most likely one weighs nothing and is never drawn.
//
// A cluster of up to 8 CTAs holds a row in shared memory, read once from DRAM; every later pass is over shared memory, a
// thread's tokens next to each other (an odd number of them: no bank conflicts), so thread order is index order.  Without
// filters there is one pass of exponentials and a scan.  Filters need the place where a running count (top_k) or a running weight
// (top_p), in falling order of the logits, reaches a limit: a histogram over 2048 bins of (max - l) / temperature, whose bins
// the CTAs add up by shares through distributed shared memory, gives the bin; its few tokens are ranked by one CTA.  A bin
// of more than 512 tokens is divided again, by the bits of its logits; one of equal logits is cut by index.
//
// The exponential, P. T. P. Tang's table-driven method (Table-driven implementation of the exponential function in IEEE
// floating-point arithmetic, 1989) in 64 bits: (l - max) 32 log2(e) / temperature = n + f, 2^(n / 32) from a table of 32 and
// the exponent, 2^(f / 32) by Taylor's series up to f^5 (2.2e-15 relative, a 13th of the unit's half).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace svla {

struct SampleArgs {
  const void* logits;
  long long logits_rs;
  const float *u, *temperature, *top_p, *min_p;  // [batch]; temperature, top_p and min_p may be null: the values below
  const int* top_k;                              // likewise
  float temperature_value, top_p_value, min_p_value;
  int top_k_value;
  int* tokens;
  float* logprob;  // may be null
  int batch, vocab;
  int each;        // tokens of a thread, odd
};

namespace sample {
using u64 = unsigned long long;
constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 2048, kList = 512, kMaxCtas = 8;
constexpr double kUnit = 17592186044416.0;  // 2^44

__device__ const double kPowers[32] = {  // 2^(j / 32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};

struct alignas(16) Shared {
  unsigned hist[4][kBins];  // tokens, and the weights' bits 0-14, 15-29 and 30-44 (sums of 33024 of them stay in 32 bits)
  u64 list[kList], list_w[kList];
  double powers[32];
  u64 exch[2][2];           // what the CTAs tell one another, in turn
  u64 warp_sum[2][kWarps];
  u64 found[5];             // a crossing or a cut, written by the CTA that has it
  unsigned listed;
};

// order of logits as unsigned integers; larger is more likely
__device__ __forceinline__ unsigned key_of(float l) {
  const unsigned b = __float_as_uint(l);
  return b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
// falling logit, then rising index, as one number that falls
__device__ __forceinline__ u64 place_of(float l, unsigned index) { return (static_cast<u64>(key_of(l)) << 32) | (0xFFFFFFFFu - index); }

struct Weigh {
  double factor, top;  // 32 log2(e) / temperature, the largest logit
  const double* powers;
  __device__ __forceinline__ u64 operator()(float l) const {
    const double z = (static_cast<double>(l) - top) * factor;
    if (!(z > -1472.0)) return 0ull;                  // 46 octaves: rounds to 0
    constexpr double kMagic = 6755399441055744.0;     // 1.5 * 2^52: adding it rounds to an integer in the low bits
    const double t = z + kMagic;
    const int n = __double2loint(t);
    const double f = z - (t - kMagic);
    double p = fma(f, 3.973709984549416e-11, 9.172562701824643e-09);  // (ln 2 / 32)^k / k!
    p = fma(f, p, 1.693850972437182e-06);
    p = fma(f, p, 0.0002345961982022468);
    p = fma(f, p, 0.02166084939249829);
    p = fma(f, p, 1.0);
    p *= powers[n & 31];
    // times 2^(44 + n / 32), then rounded to an integer by adding 2^52
    p = __hiloint2double(__double2hiint(p) + ((44 + (n >> 5)) << 20), __double2loint(p));
    return static_cast<u64>(__double_as_longlong(p + 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
  }
};

__device__ __forceinline__ u64 remote_ld(const u64* p, unsigned rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned remote_ld(const unsigned* p, unsigned rank) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ void remote_st(u64* p, unsigned rank, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(p), rank)), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned remote_add(unsigned* p, unsigned rank, unsigned v) {
  unsigned old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(mapa_shared(smem_u32(p), rank)), "r"(v) : "memory");
  return old;
}

// every thread of the cluster; lanes may come from different branches
__device__ __forceinline__ void csync() {
  __syncwarp();
  cluster_sync();
}

struct Block {
  Shared& s;
  const unsigned rank, ctas;
  const int tid, lane, warp;
  unsigned turn, scan_turn;

  // all CTAs' (a, b), of which thread 0's count; lane r of every warp gets CTA r's, other lanes zeros
  __device__ __forceinline__ void exchange(u64& a, u64& b) {
    if (tid == 0) s.exch[turn][0] = a, s.exch[turn][1] = b;
    csync();
    a = b = 0ull;
    if (lane < static_cast<int>(ctas)) a = remote_ld(&s.exch[turn][0], lane), b = remote_ld(&s.exch[turn][1], lane);
    turn ^= 1u;  // the other place is free: every CTA has read it before it came to the barrier above
    __syncwarp();
  }
  // sum over the block before this thread; `total` is the block's
  __device__ __forceinline__ u64 scan(u64 v, u64& total) {
    u64 incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const u64 o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    if (lane == 31) s.warp_sum[scan_turn][warp] = incl;
    __syncthreads();
    u64 before = 0ull;
    total = 0ull;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const u64 o = s.warp_sum[scan_turn][w];
      if (w < warp) before += o;
      total += o;
    }
    scan_turn ^= 1u;
    return before + incl - v;
  }
  // sum of lanes 0 .. ctas - 1, and of those below this CTA's
  __device__ __forceinline__ u64 over_ctas(u64 v, u64& below) const {
    u64 total = 0ull;
    below = 0ull;
#pragma unroll
    for (int r = 0; r < kMaxCtas; ++r) {
      const u64 o = __shfl_sync(0xffffffffu, v, r);  // lanes from `ctas` on hold zeros
      total += o;
      if (r < static_cast<int>(rank)) below += o;
    }
    return total;
  }
};
}  // namespace sample

template <typename T>
__global__ void __launch_bounds__(sample::kThreads) sample_kernel(const SampleArgs a) {
  using namespace sample;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  float* logits = reinterpret_cast<float*>(smem_raw + sizeof(Shared));
  unsigned ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  Block k{s, cluster_ctarank(), ctas, static_cast<int>(threadIdx.x), static_cast<int>(threadIdx.x & 31), static_cast<int>(threadIdx.x >> 5), 0u, 0u};
  const int tid = k.tid, lane = k.lane;
  const long long row = blockIdx.x / ctas;
  if (tid < 32) s.powers[tid] = kPowers[tid];
  if (tid == 0) s.listed = 0u;
  pdl_wait();
  pdl_trigger();

  // ---------------- the row's share of this CTA, and the largest logit with its lowest index
  const int slice = a.each * kThreads, first = static_cast<int>(k.rank) * slice;
  const int count = max(0, min(slice, a.vocab - first));
  float best = -INFINITY;
  unsigned best_at = 0xFFFFFFFFu;
  bool nan = false;
  {
    const T* src = static_cast<const T*>(a.logits) + row * a.logits_rs + first;
    auto see = [&](float v, int i) {
      nan |= v != v;
      if (v > best) best = v, best_at = first + i;
      return v;
    };
    constexpr int kPer = 16 / sizeof(T);
    int done = 0;
    if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
      done = count / kPer * kPer;
#pragma unroll 4
      for (int i = tid * kPer; i < done; i += kThreads * kPer) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(src + i));
        const T* v = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int e = 0; e < kPer; e += 4) {
          // + 0: a negative zero equals a positive one
          const float4 f = make_float4(see(static_cast<float>(v[e]) + 0.f, i + e), see(static_cast<float>(v[e + 1]) + 0.f, i + e + 1),
                                       see(static_cast<float>(v[e + 2]) + 0.f, i + e + 2), see(static_cast<float>(v[e + 3]) + 0.f, i + e + 3));
          *reinterpret_cast<float4*>(logits + i + e) = f;
        }
      }
    }
    for (int i = done + tid; i < count; i += kThreads) logits[i] = see(static_cast<float>(src[i]) + 0.f, i);
  }
  u64 place = nan ? ~0ull : place_of(best, best_at);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) place = max(place, __shfl_xor_sync(0xffffffffu, place, d));
  if (lane == 0) s.warp_sum[0][k.warp] = place;
  __syncthreads();
  {
    u64 p = 0ull, other = 0ull;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) p = max(p, s.warp_sum[0][w]);
    k.scan_turn = 1u;
    k.exchange(p, other);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) p = max(p, __shfl_xor_sync(0xffffffffu, p, d));
    place = __shfl_sync(0xffffffffu, p, 0);
  }
  const unsigned top_key = static_cast<unsigned>(place >> 32);
  const float top = of_key(top_key);

  const float temperature = a.temperature ? __ldg(a.temperature + row) : a.temperature_value;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : a.top_p_value, min_p = a.min_p ? __ldg(a.min_p + row) : a.min_p_value;
  const int top_k = a.top_k ? __ldg(a.top_k + row) : a.top_k_value;
  const float u = __ldg(a.u + row);
  // a row without a finite largest logit or with a NaN, and settings that are none
  const bool bad = top_key >= 0xFF800000u || top_key <= 0x007FFFFFu || !(temperature >= 0.f) || temperature == INFINITY || !(top_p >= 0.f) ||
                   !(min_p >= 0.f) || !(u >= 0.f && u <= 1.f);
  const bool one = temperature == 0.f || top_k == 1 || top_p == 0.f || min_p > 1.f;  // the most likely one alone is kept
  if (bad || one) {
    if (k.rank == 0 && tid == 0) {
      a.tokens[row] = bad ? -1 : static_cast<int>(0xFFFFFFFFu - static_cast<unsigned>(place));
      if (a.logprob) a.logprob[row] = bad ? __int_as_float(0x7fc00000) : 0.f;
    }
    csync();  // no CTA leaves while another reads what it told
    return;
  }
  const Weigh weigh{46.16624130844683 / static_cast<double>(temperature), static_cast<double>(top), s.powers};
  const float* mine = logits + tid * a.each;
  const int mine_n = max(0, min(a.each, count - tid * a.each));
  const unsigned mine_first = first + tid * a.each;

  u64 cut = 0x0080000000000000ull;  // kept are places from here on (nothing at -infinity)
  if (min_p > 0.f) {
    // the smallest key whose weight reaches the bound, between one that does not and one that does: 33-fold search
    const double bound = static_cast<double>(min_p) * kUnit;
    unsigned lo = 0x007FFFFFu, hi = top_key;
    while (hi - lo > 1u) {
      const unsigned step = (hi - lo + 32u) / 33u, at = lo + step * (lane + 1u);
      const bool yes = at >= hi || at < lo || static_cast<double>(weigh(of_key(at))) >= bound;  // (at < lo: it wrapped)
      const int f = __ffs(__ballot_sync(0xffffffffu, yes));  // 1 + the first lane that does; 0: none
      if (f == 0) {
        lo += 32u * step;
      } else {
        hi = min(hi, lo + static_cast<unsigned>(f) * step);
        lo += static_cast<unsigned>(f - 1) * step;
      }
    }
    cut = static_cast<u64>(hi) << 32;
  }

  const bool by_count = top_k > 0 && top_k < a.vocab, by_weight = top_p < 1.f;
  if (by_count || by_weight) {
    const float to_bin = 64.f / temperature;
    auto linear_bin = [&](float l) {
      const float b = __fmul_rn(__fsub_rn(top, l), to_bin);  // not a number: 0 * infinity, the largest logit
      return b >= 2047.f ? kBins - 1 : __float2int_rz(b);
    };
    const int per = kBins / static_cast<int>(ctas), per_thread = per / kThreads;  // bins of a CTA, of a thread
    auto clear = [&]() {
      for (int i = tid; i < 4 * kBins; i += kThreads) (&s.hist[0][0])[i] = 0u;
      __syncthreads();
    };
    auto count_in = [&](int bin, float l) {
      atomicAdd(&s.hist[0][bin], 1u);
      if (by_weight) {
        const u64 w = weigh(l);
        atomicAdd(&s.hist[1][bin], static_cast<unsigned>(w) & 0x7FFFu);
        atomicAdd(&s.hist[2][bin], static_cast<unsigned>(w >> 15) & 0x7FFFu);
        atomicAdd(&s.hist[3][bin], static_cast<unsigned>(w >> 30));
      }
    };
    u64 c_before = 0ull, w_before = 0ull, c_total = 0ull, w_total = 0ull;  // before this thread's bins, over all bins
    // the CTAs' histograms added up: each CTA's share of the bins lies in its own hist[0] (tokens) and hist[1], hist[2] (weight)
    auto merge = [&]() {
      csync();
      u64 c = 0ull, w = 0ull;
      for (int j = 0; j < per_thread; ++j) {
        const int bin = static_cast<int>(k.rank) * per + tid * per_thread + j;
        unsigned n = 0u;
        u64 weight = 0ull;
        for (unsigned r = 0; r < ctas; ++r) {
          n += remote_ld(&s.hist[0][bin], r);
          if (by_weight)
            weight += remote_ld(&s.hist[1][bin], r) + (static_cast<u64>(remote_ld(&s.hist[2][bin], r)) << 15) +
                      (static_cast<u64>(remote_ld(&s.hist[3][bin], r)) << 30);
        }
        // (no other CTA reads this CTA's share)
        s.hist[0][bin] = n, s.hist[1][bin] = static_cast<unsigned>(weight), s.hist[2][bin] = static_cast<unsigned>(weight >> 32);
        c += n, w += weight;
      }
      u64 tc, tw;
      c_before = k.scan(c, tc);
      w_before = k.scan(w, tw);
      k.exchange(tc, tw);
      u64 below;
      c_total = k.over_ctas(tc, below);
      c_before += below;
      w_total = k.over_ctas(tw, below);
      w_before += below;
    };
    // the bin in which the running count (or weight) reaches `limit`, 1 <= limit <= its total
    unsigned bin, bin_n;
    u64 bin_c, bin_w;  // before the bin
    auto cross = [&](bool count, u64 limit) {
      u64 c = c_before, w = w_before;
      for (int j = 0; j < per_thread; ++j) {
        const int b = static_cast<int>(k.rank) * per + tid * per_thread + j;
        const u64 n = s.hist[0][b], weight = (static_cast<u64>(s.hist[2][b]) << 32) | s.hist[1][b];
        const u64 at = count ? c : w, size = count ? n : weight;
        if (at < limit && limit <= at + size)
          for (unsigned r = 0; r < ctas; ++r) {
            remote_st(&s.found[0], r, b);
            remote_st(&s.found[1], r, n);
            remote_st(&s.found[2], r, c);
            remote_st(&s.found[3], r, w);
          }
        c += n, w += weight;
      }
      csync();
      bin = static_cast<unsigned>(s.found[0]), bin_n = static_cast<unsigned>(s.found[1]), bin_c = s.found[2], bin_w = s.found[3];
    };
    bool divided = false;  // the histogram is one of a bin's
    // the cut inside a bin: after `need` tokens of it, or after the token with which their weight reaches `need`.
    // -> the weight of what is kept of it
    auto resolve = [&](bool count, u64 need) {
      bool ranged = false;  // members: of the linear bin, or with keys from lo to hi
      unsigned lo = 0u, hi = 0u, n = bin_n;
      const int in_bin = static_cast<int>(bin);
      const unsigned floor_key = static_cast<unsigned>(cut >> 32);
      auto member = [&](float l) {
        const unsigned key = key_of(l);
        return key >= floor_key && (ranged ? key >= lo && key <= hi : linear_bin(l) == in_bin);
      };
      u64 kept_w = 0ull;
      // (a division takes 11 of the keys' 32 bits, so the fourth round at the latest has few or equal ones)
      for (int round = 0; round < 4; ++round) {
        if (n <= kList) {
          for (int j = 0; j < mine_n; ++j) {
            const float l = mine[j];
            if (!member(l)) continue;
            const unsigned at = remote_add(&s.listed, 0, 1u);
            if (at < kList) remote_st(&s.list[at], 0, place_of(l, mine_first + j));
          }
          csync();
          if (k.rank == 0) {
            const int m = static_cast<int>(min(s.listed, static_cast<unsigned>(kList)));
            if (by_weight) {
              for (int i = tid; i < m; i += kThreads) s.list_w[i] = weigh(of_key(static_cast<unsigned>(s.list[i] >> 32)));
            }
            __syncthreads();
            u64 last = ~0ull, sum = 0ull;  // of the kept: the least likely place, the weight
            for (int i = tid; i < m; i += kThreads) {
              const u64 own = s.list[i];
              u64 before = 0ull;
              for (int j = 0; j < m; ++j)
                if (s.list[j] > own) before += count ? 1ull : s.list_w[j];
              if (before < need) {
                last = min(last, own);
                if (by_weight) sum += s.list_w[i];
              }
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) last = min(last, __shfl_xor_sync(0xffffffffu, last, d));
            u64 total;
            k.scan(sum, total);
            __syncthreads();
            if (lane == 0) s.list[k.warp] = last;
            __syncthreads();
            if (tid == 0) {
              for (int w = 0; w < kWarps; ++w) last = min(last, s.list[w]);
              s.listed = 0u;
              for (unsigned r = 0; r < ctas; ++r) remote_st(&s.found[0], r, last), remote_st(&s.found[1], r, total);
            }
            __syncwarp();
          }
          csync();
          cut = s.found[0];
          return kept_w + s.found[1];
        }
        // too many: the range of their keys
        unsigned least = 0xFFFFFFFFu, most = 0u;
        for (int j = 0; j < mine_n; ++j)
          if (member(mine[j])) least = min(least, key_of(mine[j])), most = max(most, key_of(mine[j]));
        least = __reduce_min_sync(0xffffffffu, least), most = __reduce_max_sync(0xffffffffu, most);
        __syncthreads();
        if (lane == 0) s.warp_sum[0][k.warp] = (static_cast<u64>(least) << 32) | most;
        __syncthreads();
        u64 l64 = 0xFFFFFFFFull, m64 = 0ull;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) l64 = min(l64, s.warp_sum[0][w] >> 32), m64 = max(m64, s.warp_sum[0][w] & 0xFFFFFFFFull);
        k.scan_turn = 1u;
        k.exchange(l64, m64);
        if (lane >= static_cast<int>(ctas)) l64 = 0xFFFFFFFFull;
        least = __reduce_min_sync(0xffffffffu, static_cast<unsigned>(l64)), most = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(m64));
        if (least == most) {  // equal logits: the first ones by index
          const u64 w = weigh(of_key(most)), r = count ? need : (need + w - 1ull) / w;
          u64 here = 0ull, total, below, none = 0ull;
          for (int j = 0; j < mine_n; ++j) here += key_of(mine[j]) == most;
          u64 before = k.scan(here, total);
          k.exchange(total, none);
          k.over_ctas(total, below);
          before += below;
          if (before < r && r <= before + here) {
            u64 at = before;
            int j = 0;
            for (; j < mine_n; ++j)
              if (key_of(mine[j]) == most && ++at == r) break;
            for (unsigned q = 0; q < ctas; ++q) remote_st(&s.found[0], q, place_of(of_key(most), mine_first + j));
          }
          csync();
          cut = s.found[0];
          return kept_w + r * w;
        }
        const int bits = 32 - __clz(most - least), shift = bits > 11 ? bits - 11 : 0;
        clear();
        for (int j = 0; j < mine_n; ++j)
          if (member(mine[j])) count_in(static_cast<int>((most - key_of(mine[j])) >> shift), mine[j]);
        __syncwarp();
        merge();
        cross(count, need);
        need -= count ? bin_c : bin_w;
        kept_w += bin_w;
        hi = most - (bin << shift);
        lo = max(least, hi - ((1u << shift) - 1u));
        ranged = divided = true;
        n = bin_n;
      }
      return kept_w;
    };

    auto count_all = [&]() {
      clear();
      const unsigned floor_key = static_cast<unsigned>(cut >> 32);
      for (int j = 0; j < mine_n; ++j) {
        const float l = mine[j];
        const int b = linear_bin(l);
        if (b < kBins - 1 && key_of(l) >= floor_key) count_in(b, l);  // (what falls into the last bin weighs nothing)
      }
      merge();
    };
    count_all();
    u64 kept_w = w_total;
    if (by_count && static_cast<u64>(top_k) < c_total) {
      cross(true, static_cast<u64>(top_k));
      const u64 w_at = bin_w;
      kept_w = w_at + resolve(true, static_cast<u64>(top_k) - bin_c);
      if (by_weight && divided) count_all();
    }
    if (by_weight) {
      const u64 limit = max(1ull, static_cast<u64>(ceil(static_cast<double>(top_p) * static_cast<double>(kept_w))));
      cross(false, limit);
      resolve(false, limit - bin_w);
    }
  }

  // ---------------- the token
  u64 sum = 0ull, total, none = 0ull, below;
  for (int j = 0; j < mine_n; ++j)
    if (place_of(mine[j], mine_first + j) >= cut) sum += weigh(mine[j]);
  u64 before = k.scan(sum, total);
  k.exchange(total, none);
  const u64 all = k.over_ctas(total, below);
  before += below;
  const u64 target = min(static_cast<u64>(static_cast<double>(u) * static_cast<double>(all)), all - 1ull);
  if (before <= target && target < before + sum) {
    for (int j = 0; j < mine_n; ++j) {
      const u64 w = place_of(mine[j], mine_first + j) >= cut ? weigh(mine[j]) : 0ull;
      before += w;
      if (before > target) {
        a.tokens[row] = static_cast<int>(mine_first + j);
        if (a.logprob) a.logprob[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(all)));
        break;
      }
    }
  }
  csync();  // no CTA leaves while another reads what it told
}

}  // namespace svla
