// The choice of a token from a row of logits l, given a uniform random number u:
//   w_i = round(2^44 exp((l_i - max l) / temperature)), whole numbers;
//   kept: the top_k largest logits with w_i >= min_p 2^44, of these the most likely up to the one with which their sum reaches
//   top_p of it; equal logits in the order of their indices (the lower one first);
//   the token is the first, by index, up to which the kept w add up to more than floor(u sum w).
// Whole numbers add up to the same in any order, so the answer depends neither on how a row is shared nor on timing.  2^44 leaves
// 2^18 tokens in 62 bits; a token below 2^-45 of the most likely one weighs nothing and is never drawn.
//
// A cluster of up to 8 CTAs holds a row in shared memory, read once from DRAM; every later pass is over shared memory, a
// thread's tokens next to each other (an odd number of words: no bank conflicts), so thread order is index order.  Without
// filters there is one pass of exponentials and a scan.  Filters need the place where a running count (top_k) or a running weight
// (top_p), in falling order of the logits, reaches a limit: a histogram over 2048 bins of (max - l) / temperature, whose bins
// the CTAs add up by shares through distributed shared memory, gives the bin.  Up to 512 tokens are then ranked by one CTA: all
// that top_k leaves, and the token is found among them at once, or those of the bin.  A bin of more is divided again, by the bits
// of its logits; one of equal logits is cut by index.
//
// The exponential, P. T. P. Tang's table-driven method (Table-driven implementation of the exponential function in IEEE
// floating-point arithmetic, 1989) in 64 bits: (l - max) 64 log2(e) / temperature = n + f, 2^(n / 64) from a table of 64 and the
// exponent, 2^(f / 64) by the polynomial of degree 4 through Chebyshev's points (4.9e-15 relative, a twelfth of a unit at the
// most likely token): 10 operations in 64 bits, of which an SM does 64 a cycle.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"
#include "serving_common.cuh"

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
  int words;       // 32-bit words of logits per thread, odd
};

namespace sample {
using u64 = unsigned long long;
constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 2048, kList = 512, kMaxCtas = 8;
constexpr double kUnit = 17592186044416.0;  // 2^44

__device__ const double kPowers[64] = {  // 2^(j / 64)
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951};

struct alignas(16) Shared {
  unsigned hist[4][kBins];  // tokens, and the weights' bits 0-14, 15-29 and 30-44 (sums of 2^16 of them stay in 32 bits)
  u64 list[kList], list_w[kList];
  u64 own[kList];           // of this CTA, on their way to the list of CTA 0
  double powers[64];
  u64 exch[2][2];           // what the CTAs tell one another, in turn
  u64 warp_sum[2][kWarps];
  u64 found[4];             // a crossing or a cut, written by the CTA that has it
  unsigned listed[2], own_n, own_at;
};

// order of logits as unsigned integers; larger is more likely, both zeros are one
__device__ __forceinline__ unsigned key_of(float l) {
  const unsigned b = __float_as_uint(l + 0.f);
  return b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
// falling logit, then rising index, as one number that falls
__device__ __forceinline__ u64 place_of(float l, int index) { return (static_cast<u64>(key_of(l)) << 32) | ~static_cast<unsigned>(index); }

struct Weigh {
  double factor, top;  // 64 log2(e) / temperature, the largest logit
  const double* powers;
  // the weight of a logit less than 33 temperatures below the largest
  __device__ __forceinline__ u64 operator()(float l) const {
    const double d = static_cast<double>(l) - top;
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer in the low bits
    const double t = fma(d, factor, kMagic);
    const int n = __double2loint(t);
    const double f = fma(d, factor, kMagic - t);
    double p = fma(f, 5.732857292414682e-10, 2.1173168200092995e-07);
    p = fma(f, p, 5.864904955054418e-05);
    p = fma(f, p, 0.010830424696239445);
    p = fma(f, p, 1.0);
    p *= powers[n & 63];
    // times 2^(44 + n / 64), then rounded to an integer by adding 2^52
    p = __hiloint2double(__double2hiint(p) + ((44 + (n >> 6)) << 20), __double2loint(p)) + 4503599627370496.0;
    return static_cast<u64>(__double_as_longlong(p)) & 0xFFFFFFFFFFFFFull;
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

// the two halves of a csync
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
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
  // a value of every warp to all threads, joined by f
  template <typename F>
  __device__ __forceinline__ u64 over_warps(u64 v, F f) {
    if (lane == 0) s.warp_sum[scan_turn][warp] = v;
    __syncthreads();
    v = s.warp_sum[scan_turn][0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v = f(v, s.warp_sum[scan_turn][w]);
    scan_turn ^= 1u;
    return v;
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

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// the logits of a word, one or two of them
template <typename T>
__device__ __forceinline__ float2 logits_of(unsigned w) {
  if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w), -INFINITY);
  else return serving::unpack2<T>(w);
}
}  // namespace sample

template <typename T>
__global__ void __launch_bounds__(sample::kThreads) sample_kernel(const SampleArgs a) {
  using namespace sample;
  constexpr int kIn = 4 / sizeof(T);  // logits of a word
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& s = *reinterpret_cast<Shared*>(smem_raw);
  unsigned* row_words = reinterpret_cast<unsigned*>(smem_raw + sizeof(Shared));
  unsigned ctas;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  Block k{s, cluster_ctarank(), ctas, static_cast<int>(threadIdx.x), static_cast<int>(threadIdx.x & 31), static_cast<int>(threadIdx.x >> 5), 0u, 0u};
  const int tid = k.tid, lane = k.lane;
  const long long row = blockIdx.x / ctas;
  if (tid < 64) s.powers[tid] = kPowers[tid];
  if (tid < 2) s.listed[tid] = 0u;
  pdl_wait();
  pdl_trigger();

  // ---------------- this CTA's share of the row, -infinity behind its end, and the largest logit
  const int slice = a.words * kThreads * kIn, first = static_cast<int>(k.rank) * slice;
  const int count = max(0, min(slice, a.vocab - first));
  float top = -INFINITY;
  {
    const T* src = static_cast<const T*>(a.logits) + row * a.logits_rs + first;
    constexpr int kPer = 16 / sizeof(T);
    int done = 0;
    if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
      done = count / kPer * kPer;
#pragma unroll 4
      for (int i = tid; i < done / kPer; i += kThreads) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(src) + i);
        reinterpret_cast<uint4*>(row_words)[i] = w;
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 l = logits_of<T>(u[e]);
          top = max_nan(top, l.x);
          if constexpr (kIn == 2) top = max_nan(top, l.y);
        }
      }
    }
    T* dst = reinterpret_cast<T*>(row_words);
    for (int i = done + tid; i < slice; i += kThreads) {
      const T v = i < count ? src[i] : static_cast<T>(-INFINITY);
      dst[i] = v;
      top = max_nan(top, static_cast<float>(v));
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
  auto larger = [](u64 x, u64 y) { return x > y ? x : y; };
  auto smaller = [](u64 x, u64 y) { return x < y ? x : y; };
  {
    u64 p = k.over_warps(top != top ? ~0ull : key_of(top), larger), none = 0ull;
    k.exchange(p, none);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) p = larger(p, __shfl_xor_sync(0xffffffffu, p, d));
    p = __shfl_sync(0xffffffffu, p, 0);
    top = p == ~0ull ? INFINITY : of_key(static_cast<unsigned>(p));
  }

  const float temperature = a.temperature ? __ldg(a.temperature + row) : a.temperature_value;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : a.top_p_value, min_p = a.min_p ? __ldg(a.min_p + row) : a.min_p_value;
  const int top_k = a.top_k ? __ldg(a.top_k + row) : a.top_k_value;
  const float u = __ldg(a.u + row);
  const unsigned* mine = row_words + tid * a.words;
  const int mine_first = first + tid * a.words * kIn;
  auto for_mine = [&](auto f) {  // f(logit, index) of this thread's tokens
#pragma unroll 4
    for (int j = 0; j < a.words; ++j) {
      const float2 l = logits_of<T>(mine[j]);
      f(l.x, mine_first + j * kIn);
      if constexpr (kIn == 2) f(l.y, mine_first + j * kIn + 1);
    }
  };
  // a row without a finite largest logit or with a NaN, and settings that are none
  const bool bad = !(fabsf(top) < INFINITY) || !(temperature >= 0.f && temperature < INFINITY) || !(top_p >= 0.f) || !(min_p >= 0.f) || !(u >= 0.f && u <= 1.f);
  if (bad) {
    if (k.rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.logprob) a.logprob[row] = __int_as_float(0x7fc00000);
    }
    csync();  // no CTA leaves while another reads what it told
    return;
  }
  if (temperature == 0.f || top_k == 1 || top_p == 0.f || min_p > 1.f) {  // the most likely token alone is kept
    unsigned at = 0xFFFFFFFFu;
    for_mine([&](float l, int i) {
      if (l == top) at = min(at, static_cast<unsigned>(i));
    });
    at = __reduce_min_sync(0xffffffffu, at);
    u64 p = k.over_warps(at, smaller), none = 0ull;
    k.exchange(p, none);
    if (lane >= static_cast<int>(ctas)) p = ~0ull;
    at = __reduce_min_sync(0xffffffffu, static_cast<unsigned>(p));
    if (k.rank == 0 && tid == 0) {
      a.tokens[row] = static_cast<int>(at);
      if (a.logprob) a.logprob[row] = 0.f;
    }
    csync();
    return;
  }
  const Weigh weigh{92.33248261689366 / static_cast<double>(temperature), static_cast<double>(top), s.powers};
  // Kept are logits above cut_l, and of those that equal it the ones up to index cut_i.  At first what weighs something: less
  // than 45 octaves, 31.2 temperatures below the largest (rounded so that nothing is lost)
  float cut_l = __fsub_rd(top, __fmul_ru(33.f, temperature));
  int cut_i = -1;
  bool filtered = false;
  auto keeps = [&](float l, int i) { return l > cut_l || (l == cut_l && i <= cut_i); };

  if (min_p > 0.f) {
    // the smallest key whose weight reaches the bound, between one that does not and one that does: 33-fold search
    const double bound = static_cast<double>(min_p) * kUnit;
    unsigned lo = max(key_of(cut_l), 0x007FFFFFu), hi = key_of(top);
    while (hi - lo > 1u) {
      const unsigned step = (hi - lo + 32u) / 33u, at = lo + step * (lane + 1u);
      const bool yes = at >= hi || static_cast<double>(weigh(of_key(at))) >= bound;
      const int f = __ffs(__ballot_sync(0xffffffffu, yes));  // 1 + the first lane that does; 0: none
      if (f == 0) {
        lo += 32u * step;
      } else {
        hi = min(hi, lo + static_cast<unsigned>(f) * step);
        lo += static_cast<unsigned>(f - 1) * step;
      }
    }
    cut_l = of_key(hi), cut_i = 0x7FFFFFFF, filtered = true;
  }

  const bool by_count = top_k > 0 && top_k < a.vocab;
  const bool by_weight = top_p < 1.f;
  if (by_count || by_weight) {
    filtered = true;
    const float to_bin = 64.f / temperature;
    auto linear_bin = [&](float l) {  // (0 * infinity, the largest logit's, is bin 0 too)
      return min(__float2int_rz(__fmul_rn(__fsub_rn(top, l), to_bin)), kBins - 1);
    };
    const int per = kBins / static_cast<int>(ctas), per_thread = per > kThreads ? per / kThreads : 1;  // bins of a CTA, of a thread
    const int my_bin = static_cast<int>(k.rank) * per + tid * per_thread, my_bins = tid * per_thread < per ? per_thread : 0;
    bool counting = false, weighing = false;  // what the histogram holds
    auto clear = [&]() {
      for (int i = tid; i < kBins; i += kThreads) reinterpret_cast<uint4*>(&s.hist[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
    };
    auto count_in = [&](int bin, float l) {
      if (counting) atomicAdd(&s.hist[0][bin], 1u);
      if (weighing) {
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
      for (int j = 0; j < my_bins; ++j) {
        const int bin = my_bin + j;
        unsigned n = 0u;
        u64 weight = 0ull;
#pragma unroll
        for (unsigned r = 0; r < kMaxCtas; ++r) {
          if (r >= ctas) break;
          if (counting) n += remote_ld(&s.hist[0][bin], r);
          if (weighing)
            weight += remote_ld(&s.hist[1][bin], r) + (static_cast<u64>(remote_ld(&s.hist[2][bin], r)) << 15) +
                      (static_cast<u64>(remote_ld(&s.hist[3][bin], r)) << 30);
        }
        // (no other CTA reads this CTA's share)
        s.hist[0][bin] = n, s.hist[1][bin] = static_cast<unsigned>(weight), s.hist[2][bin] = static_cast<unsigned>(weight >> 32);
        c += n, w += weight;
      }
      u64 tc = 0ull, tw = 0ull, below;
      if (counting) c_before = k.scan(c, tc);
      if (weighing) w_before = k.scan(w, tw);
      k.exchange(tc, tw);
      c_total = k.over_ctas(tc, below), c_before += below;
      w_total = k.over_ctas(tw, below), w_before += below;
    };
    // the bin in which the running count (or weight) reaches `limit`, 1 <= limit <= its total
    int bin = 0;
    u64 bin_n = 0ull, bin_c = 0ull, bin_w = 0ull;  // its tokens; before the bin: tokens, weight
    auto cross = [&](bool count, u64 limit) {
      u64 c = c_before, w = w_before;
      for (int b = my_bin; b < my_bin + my_bins; ++b) {
        const u64 n = s.hist[0][b], weight = (static_cast<u64>(s.hist[2][b]) << 32) | s.hist[1][b];
        const u64 at = count ? c : w, size = count ? n : weight;
        if (at < limit && limit <= at + size)
          for (unsigned r = 0; r < ctas; ++r) {
            remote_st(&s.found[0], r, static_cast<u64>(b));
            remote_st(&s.found[1], r, n);
            remote_st(&s.found[2], r, c);
            remote_st(&s.found[3], r, w);
          }
        c += n, w += weight;
      }
      csync();
      bin = static_cast<int>(s.found[0]), bin_n = s.found[1], bin_c = s.found[2], bin_w = s.found[3];
    };
    // the tokens that `member` says, to the list of CTA 0 as far as it takes them; -> how many there are
    unsigned gather_turn = 0u;
    auto gather = [&](auto member) -> unsigned {
      if (tid == 0) s.own_n = 0u;
      __syncthreads();
      for_mine([&](float l, int i) {
        if (!member(l, i)) return;
        const unsigned at = atomicAdd(&s.own_n, 1u);
        if (at < kList) s.own[at] = place_of(l, i);
      });
      __syncthreads();
      const unsigned n = s.own_n;
      if (tid == 0 && n) s.own_at = remote_add(&s.listed[gather_turn], 0, n);
      __syncthreads();
      if (n) {
        const unsigned at = s.own_at;
        for (unsigned i = tid; i < n && at + i < kList; i += kThreads) remote_st(&s.list[at + i], 0, s.own[i]);
      }
      csync();
      const unsigned all = remote_ld(&s.listed[gather_turn], 0);
      gather_turn ^= 1u;
      if (k.rank == 0 && tid == 0) s.listed[gather_turn] = 0u;  // (every CTA has read it before it came to the barrier above)
      return all;
    };
    // CTA 0: for token i of the list, how many of the m come before it and what they weigh
    auto rank_of = [&](int i, int m, unsigned& rank, u64& weight) {
      const u64 own = s.list[i];
      rank = 0u, weight = 0ull;
#pragma unroll 4
      for (int j = 0; j < m; ++j) {
        const bool before = s.list[j] > own;
        rank += before;
        if (before) weight += s.list_w[j];
      }
    };
    auto weigh_list = [&](int m) {
      for (int i = tid; i < m; i += kThreads) s.list_w[i] = weigh(of_key(static_cast<unsigned>(s.list[i] >> 32)));
      __syncthreads();
    };
    bool divided = false;  // the histogram is one of a bin's
    // the cut inside a bin: after `need` tokens of it, or after the token with which their weight reaches `need`.
    // -> the weight of what is kept of it
    auto resolve = [&](bool count, u64 need) -> u64 {
      bool ranged = false;  // members: of the linear bin, or with keys from lo to hi
      unsigned lo = 0u, hi = 0u;
      const int in_bin = bin;
      auto member = [&](float l, int i) {
        if (!keeps(l, i)) return false;
        const unsigned key = key_of(l);
        return ranged ? key >= lo && key <= hi : linear_bin(l) == in_bin;
      };
      u64 kept_w = 0ull;
      // (a division takes 11 of the keys' 32 bits, so the fourth round at the latest has few or equal ones)
      for (int round = 0; round < 4; ++round) {
        if (!count || bin_n <= kList) {
          const int m = static_cast<int>(gather(member));
          if (m <= kList) {
            if (k.rank == 0) {
              weigh_list(m);
              u64 last = ~0ull, sum = 0ull;  // of the kept: the least likely place, the weight
              for (int i = tid; i < m; i += kThreads) {
                unsigned rank;
                u64 before;
                rank_of(i, m, rank, before);
                if ((count ? rank : before) < need) last = smaller(last, s.list[i]), sum += s.list_w[i];
              }
#pragma unroll
              for (int d = 16; d > 0; d >>= 1) last = smaller(last, __shfl_xor_sync(0xffffffffu, last, d));
              last = k.over_warps(last, smaller);
              u64 total;
              k.scan(sum, total);
              if (tid < static_cast<int>(ctas)) remote_st(&s.found[0], tid, last), remote_st(&s.found[1], tid, total);
            }
            csync();
            cut_l = of_key(static_cast<unsigned>(s.found[0] >> 32)), cut_i = static_cast<int>(~static_cast<unsigned>(s.found[0]));
            return kept_w + s.found[1];
          }
        }
        // too many: the range of their keys
        unsigned least = 0xFFFFFFFFu, most = 0u;
        for_mine([&](float l, int i) {
          if (member(l, i)) least = min(least, key_of(l)), most = max(most, key_of(l));
        });
        least = __reduce_min_sync(0xffffffffu, least), most = __reduce_max_sync(0xffffffffu, most);
        u64 range = (static_cast<u64>(~least) << 32) | most, none = 0ull;  // (both as maxima)
        auto both = [](u64 x, u64 y) {
          const unsigned h = max(static_cast<unsigned>(x >> 32), static_cast<unsigned>(y >> 32)), l = max(static_cast<unsigned>(x), static_cast<unsigned>(y));
          return (static_cast<u64>(h) << 32) | l;
        };
        range = k.over_warps(range, both);
        k.exchange(range, none);
        least = ~__reduce_max_sync(0xffffffffu, static_cast<unsigned>(range >> 32)), most = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(range));
        if (least == most) {  // equal logits: the first ones by index
          const float l0 = of_key(most);
          const u64 w = weigh(l0), r = count ? need : (need + w - 1ull) / w;
          u64 here = 0ull, total, below;
          for_mine([&](float l, int i) { here += l == l0; });
          u64 before = k.scan(here, total);
          k.exchange(total, none);
          k.over_ctas(total, below);
          before += below;
          if (before < r && r <= before + here) {
            u64 at = before;
            for_mine([&](float l, int i) {
              if (l == l0 && ++at == r)
                for (unsigned q = 0; q < ctas; ++q) remote_st(&s.found[0], q, static_cast<u64>(i));
            });
          }
          csync();
          cut_l = l0, cut_i = static_cast<int>(s.found[0]);
          return kept_w + r * w;
        }
        const int bits = 32 - __clz(most - least), shift = bits > 11 ? bits - 11 : 0;
        clear();
        for_mine([&](float l, int i) {
          if (member(l, i)) count_in(static_cast<int>((most - key_of(l)) >> shift), l);
        });
        merge();
        cross(count, need);
        need -= count ? bin_c : bin_w;
        kept_w += bin_w;
        hi = most - (static_cast<unsigned>(bin) << shift);
        lo = max(least, hi - ((1u << shift) - 1u));
        ranged = divided = true;
      }
      return kept_w;
    };
    auto count_all = [&]() {
      clear();
      for_mine([&](float l, int i) {
        if (keeps(l, i)) count_in(linear_bin(l), l);
      });
      merge();
    };

    u64 kept_w = 0ull;
    if (by_count) {
      counting = true;
      count_all();
      const bool all = c_total <= static_cast<u64>(top_k);  // (what weighs nothing is not counted)
      u64 most = c_total;
      if (!all) {
        cross(true, static_cast<u64>(top_k));
        most = bin_c + bin_n;
      }
      if (most <= kList) {
        // all that can be kept is few: CTA 0 ranks it and finds the token
        const int last_bin = bin;
        const int m = static_cast<int>(gather([&](float l, int i) { return keeps(l, i) && (all || linear_bin(l) <= last_bin); }));
        if (k.rank == 0) {
          constexpr int kEach = kList / kThreads;
          weigh_list(m);
          unsigned rank[kEach];
          u64 weight[kEach], w[kEach], sum = 0ull, total;
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            const int i = tid + e * kThreads;
            w[e] = 0ull, rank[e] = 0u, weight[e] = 0ull;
            if (i >= m) continue;
            rank_of(i, m, rank[e], weight[e]);
            if (rank[e] < static_cast<unsigned>(top_k)) w[e] = s.list_w[i];
            sum += w[e];
          }
          k.scan(sum, total);
          if (by_weight) {
            const u64 limit = larger(1ull, static_cast<u64>(ceil(static_cast<double>(top_p) * static_cast<double>(total))));
            sum = 0ull;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
              if (weight[e] >= limit) w[e] = 0ull;
              sum += w[e];
            }
            k.scan(sum, total);
          }
          __syncthreads();
#pragma unroll
          for (int e = 0; e < kEach; ++e)
            if (tid + e * kThreads < m) s.list_w[tid + e * kThreads] = w[e];
          __syncthreads();
          const u64 target = smaller(static_cast<u64>(static_cast<double>(u) * static_cast<double>(total)), total - 1ull);
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            if (w[e] == 0ull) continue;
            const unsigned own = static_cast<unsigned>(s.list[tid + e * kThreads]);
            u64 before = 0ull;
#pragma unroll 4
            for (int j = 0; j < m; ++j)
              if (static_cast<unsigned>(s.list[j]) > own) before += s.list_w[j];  // (of a lower index)
            if (before <= target && target < before + w[e]) {
              a.tokens[row] = static_cast<int>(~own);
              if (a.logprob) a.logprob[row] = static_cast<float>(log(static_cast<double>(w[e]) / static_cast<double>(total)));
            }
          }
        }
        csync();
        return;
      }
      if (!all) resolve(true, static_cast<u64>(top_k) - bin_c);
    }
    if (by_weight) {
      counting = false, weighing = true;
      count_all();
      kept_w = w_total;
      const u64 limit = larger(1ull, static_cast<u64>(ceil(static_cast<double>(top_p) * static_cast<double>(kept_w))));
      cross(false, limit);
      resolve(false, limit - bin_w);
    }
  }

  // ---------------- the token
  u64 sum = 0ull, total, none = 0ull, below;
  if (filtered) {
    for_mine([&](float l, int i) {  // few of them: a warp without one skips the exponential
      if (keeps(l, i)) sum += weigh(l);
    });
  } else {
    for_mine([&](float l, int) {
      const u64 w = weigh(l);
      sum += l > cut_l ? w : 0ull;
    });
  }
  u64 before = k.scan(sum, total);
  k.exchange(total, none);
  cluster_arrive();  // this CTA has read what the others told
  const u64 all = k.over_ctas(total, below);
  before += below;
  const u64 target = smaller(static_cast<u64>(static_cast<double>(u) * static_cast<double>(all)), all - 1ull);
  const unsigned hit = __ballot_sync(0xffffffffu, before <= target && target < before + sum);
  if (hit) {
    // the warp looks through the tokens of the thread that has it, a token per lane
    const int lucky = __ffs(hit) - 1;
    before = __shfl_sync(0xffffffffu, before, lucky);
    const int n = a.words * kIn, from = (k.warp * 32 + lucky) * n;
    for (int j = 0; j < n; j += 32) {
      const int at = from + j + lane;
      const float l = j + lane < n ? static_cast<float>(reinterpret_cast<const T*>(row_words)[at]) : -INFINITY;
      const u64 w = keeps(l, first + at) ? weigh(l) : 0ull;
      u64 upto = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const u64 o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
      }
      if (before + upto - w <= target && target < before + upto) {
        a.tokens[row] = first + at;
        if (a.logprob) a.logprob[row] = static_cast<float>(log(static_cast<double>(w) / static_cast<double>(all)));
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  cluster_wait();  // no CTA leaves while another reads what it told
}

}  // namespace svla
