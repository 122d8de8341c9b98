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
// (top_p), in falling order of the logits, reaches a limit.  Tokens are counted in 4096 bins of (max - l) / temperature, whose bins
// the CTAs add up by shares through distributed shared memory.  That gives the bin where top_k cuts; where all that is left is
// up to 256 tokens, one CTA ranks them and finds the token at once.  Otherwise counts times weights at the bins' middles say
// between which logits top_p cuts, one pass of exponentials gives the exact sums around them, and what lies between is noted:
// up to 256 of them one CTA ranks, more are divided by the bits of their logits, equal ones are cut by index.
//
// The exponential, P. T. P. Tang's table-driven method (Table-driven implementation of the exponential function in IEEE
// floating-point arithmetic, 1989) in 64 bits: (l - max) 64 log2(e) / temperature = n + f, 2^(n / 64) from a table of 64 and the
// exponent, 2^(f / 64) by the polynomial of degree 4 through Chebyshev's points (4.9e-15 relative, a twelfth of a unit at the
// most likely token): 10 operations in 64 bits, of which an SM does 64 a cycle.
//
// Measured: one row of 49280, top_k and top_p, 12.8 us; 256 rows with settings of their own 45; 512 rows (bf16) without filters
// 44; 64 rows of 131072 (bf16), top_p keeping thousands, 60.  A CTA's life is a chain of load, joins between CTAs and scans
// with 2 to 4 CTAs per SM to fill it: issue slots are 40 to 50% busy, the 64-bit pipe 33% without filters.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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
constexpr int kThreads = 256, kWarps = kThreads / 32, kBinBits = 9, kBins = 1 << kBinBits, kFine = 8 * kBins, kList = 256, kMaxCtas = 8;
constexpr int kNear = 4 * kBins * 2;
constexpr double kUnit = 17592186044416.0;  // 2^44

__device__ const double kPowers[64] = {  // 2^(j / 64); shared memory holds them times 2^44
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
  union {
    unsigned fine[kFine];        // at first: tokens per bin
    struct {
      unsigned hist[4][kBins];   // then: tokens, and the weights' bits 0-14, 15-29 and 30-44 (sums of 2^16 of them stay in 32 bits)
      unsigned short near[kNear];  // this CTA's tokens about the cut, by their places in its share
    };
  };
  u64 list[kList];
  u64 list_w[kList];        // CTA 0's; before that, in every CTA, the tokens that go to CTA 0's list
  double powers[64];
  u64 exch[2][3];           // what the CTAs tell one another, in turn
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
  __device__ __forceinline__ u64 operator()(float l) const { return bits(l) & 0xFFFFFFFFFFFFFull; }
  // the same in the low bits of 2^52 + weight
  __device__ __forceinline__ u64 bits(float l) const {
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
    // times 2^(n / 64), whole octaves in the exponent, then rounded to an integer by adding 2^52
    p = __hiloint2double(__double2hiint(p) + ((n << 14) & 0xFFF00000), __double2loint(p)) + 4503599627370496.0;
    return static_cast<u64>(__double_as_longlong(p));
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
__device__ __forceinline__ uint4 remote_ld4(const unsigned* p, unsigned rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(mapa_shared(smem_u32(p), rank))
               : "memory");
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

  // all CTAs' (a, b, c), of which thread 0's count; lane r of every warp gets CTA r's, other lanes zeros
  __device__ __forceinline__ void exchange(u64& a, u64& b, u64& c) {
    if (tid == 0) s.exch[turn][0] = a, s.exch[turn][1] = b, s.exch[turn][2] = c;
    csync();
    a = b = c = 0ull;
    if (lane < static_cast<int>(ctas)) {
      a = remote_ld(&s.exch[turn][0], lane);
      b = remote_ld(&s.exch[turn][1], lane);
      c = remote_ld(&s.exch[turn][2], lane);
    }
    turn ^= 1u;  // the other place is free: every CTA has read it before it came to the barrier above
    __syncwarp();
  }
  __device__ __forceinline__ void exchange(u64& a) {
    if (tid == 0) s.exch[turn][0] = a;
    csync();
    a = lane < static_cast<int>(ctas) ? remote_ld(&s.exch[turn][0], lane) : 0ull;
    turn ^= 1u;
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
// the larger ones of two pairs of 16-bit logits, NaN where one is
template <typename T>
__device__ __forceinline__ unsigned max2(unsigned a, unsigned b) {
  unsigned r;
  if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// the low bits that are 0 in every logit of the type, as fp32
template <typename T>
constexpr int kZeroBits = 0;
template <>
constexpr int kZeroBits<__nv_bfloat16> = 16;
template <>
constexpr int kZeroBits<__half> = 13;

// the logits of a word, one or two of them
template <typename T>
__device__ __forceinline__ float2 logits_of(unsigned w) {
  if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w), -INFINITY);
  else return serving::unpack2<T>(w);
}
}  // namespace sample

template <typename T>
__global__ void __launch_bounds__(sample::kThreads, 4) sample_kernel(const SampleArgs a) {
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
  if (tid < 64) s.powers[tid] = kPowers[tid] * kUnit;
  if (tid < 2) s.listed[tid] = 0u;
  pdl_wait();
  pdl_trigger();

  const float temperature = a.temperature ? __ldg(a.temperature + row) : a.temperature_value;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : a.top_p_value, min_p = a.min_p ? __ldg(a.min_p + row) : a.min_p_value;
  const int top_k = a.top_k ? __ldg(a.top_k + row) : a.top_k_value;
  const float u = __ldg(a.u + row);

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
        if constexpr (kIn == 1) {
          top = max_nan(max_nan(top, max_nan(__uint_as_float(w.x), __uint_as_float(w.y))), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
        } else {
          const float2 l = logits_of<T>(max2<T>(max2<T>(w.x, w.y), max2<T>(w.z, w.w)));
          top = max_nan(top, max_nan(l.x, l.y));
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
    u64 p = k.over_warps(top != top ? ~0ull : key_of(top), larger);
    k.exchange(p);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) p = larger(p, __shfl_xor_sync(0xffffffffu, p, d));
    p = __shfl_sync(0xffffffffu, p, 0);
    top = p == ~0ull ? INFINITY : of_key(static_cast<unsigned>(p));
  }

  const unsigned* mine = row_words + tid * a.words;
  const int mine_first = first + tid * a.words * kIn;
  // f(four logits, index of the first) over this thread's tokens; -infinity behind the last
  auto for_mine = [&](auto f) {
    constexpr int kGroup = 4 / kIn;
    int j = 0;
    for (; j + kGroup <= a.words; j += kGroup) {
      float l[4];
#pragma unroll
      for (int e = 0; e < kGroup; ++e) {
        const float2 v = logits_of<T>(mine[j + e]);
        l[e * kIn] = v.x;
        if constexpr (kIn == 2) l[e * kIn + 1] = v.y;
      }
      f(l, mine_first + j * kIn);
    }
    float l[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // (an odd number of words: there is a rest)
#pragma unroll
    for (int e = 0; e < kGroup - 1; ++e) {
      if (j + e >= a.words) break;
      const float2 v = logits_of<T>(mine[j + e]);
      l[e * kIn] = v.x;
      if constexpr (kIn == 2) l[e * kIn + 1] = v.y;
    }
    f(l, mine_first + j * kIn);
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
    for_mine([&](const float (&l)[4], int i) {
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (l[e] == top) at = min(at, static_cast<unsigned>(i + e));
    });
    at = __reduce_min_sync(0xffffffffu, at);
    u64 p = k.over_warps(at, smaller);
    k.exchange(p);
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
  float cut_l = fmaxf(__fsub_rd(top, __fmul_ru(33.f, temperature)), -3.4028234663852886e38f);
  if (static_cast<double>(top) - static_cast<double>(cut_l) > 34.0 * static_cast<double>(temperature))
    cut_l = of_key(key_of(cut_l) + 1u);  // one step of the logits is more than that
  int cut_i = 0x7FFFFFFF;
  auto keeps = [&](float l, int i) { return l >= cut_l && !(l == cut_l && i > cut_i); };
  // the smallest key from lo to hi for which `yes`, which holds for hi and all above the smallest: 33-fold search
  auto smallest = [&](unsigned lo, unsigned hi, auto yes) {
    while (lo < hi) {
      const unsigned step = (hi - lo + 32u) / 33u, at = lo + step * lane + (step - 1u);  // (the last of each piece)
      const int f = __ffs(__ballot_sync(0xffffffffu, at >= hi || yes(of_key(at))));       // 1 + the first that does; 0: none
      if (f == 0) {
        lo += 32u * step;
      } else {
        const unsigned before = lo + static_cast<unsigned>(f - 1) * step;
        hi = min(hi, before + step - 1u);
        lo = before;
      }
    }
    return hi;
  };

  // the sum of all weights, 2^52 in front of each taken off at the end; what is raised to cut_l weighs nothing
  auto weight_of_all = [&](auto more) {
    u64 all = 0ull;
    for_mine([&](const float (&l)[4], int i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u64 w = weigh.bits(fmaxf(l[e], cut_l));
        all += w;
        more(l, e, i, w & 0xFFFFFFFFFFFFFull);
      }
    });
    return all - static_cast<u64>((a.words * kIn + 3) / 4 * 4) * 0x4330000000000000ull;
  };

  if (min_p > 0.f) {
    const double bound = static_cast<double>(min_p) * kUnit;
    auto reaches = [&](float l) { return static_cast<double>(weigh(l)) >= bound; };
    const unsigned lo = key_of(cut_l), hi = key_of(top);
    // the border is at top + temperature ln(min_p): nearly always within 16 steps of that in fp32
    const unsigned guess = key_of(fminf(fmaxf(top + temperature * __logf(min_p), cut_l), top)), from = guess - min(guess - lo, 16u);
    const unsigned yes = __ballot_sync(0xffffffffu, from + lane >= hi || reaches(of_key(from + lane)));
    cut_l = of_key((yes & 1u) || yes == 0u ? smallest(lo, hi, reaches) : from + __ffs(yes) - 1u);
  }

  const bool by_count = top_k > 0 && top_k < a.vocab, by_weight = top_p < 1.f;
  // (cut_l weighs something where -3.4e38 does)
  const bool dense = !by_count && min_p == 0.f && weigh(cut_l) == 0ull;
  u64 sum = 0ull;  // of this thread's kept tokens
  if (by_count || by_weight) {
    // At first bins of 1 / 120 of the temperature: what is kept lies less than 33 (or one step of the logits) below the largest.
    // Differences are taken in halves, so that those above 3.4e38 stay finite, where the temperature is above 1, and times 2^64
    // where it is so small that 120 / temperature leaves fp32 (with larger logits than that allows, one step is more than 33
    // temperatures and only equal logits are left: any bins do).
    const float unit = temperature >= 1.f ? 0.5f : temperature < 5.421010862427522e-20f && fabsf(top) < 4.611686018427388e18f ? 18446744073709551616.f : 1.f;
    const float to_bin = fminf(120.f / __fmul_rn(temperature, unit), 3.4028234663852886e38f), top_units = __fmul_rn(top, unit);
    auto fine_bin = [&](float l) {
      return __float2int_rn(fminf(__fmul_rn(__fmaf_rn(l, -unit, top_units), to_bin), static_cast<float>(kFine - 1)));
    };
    unsigned* fine = s.fine;
    int my_bin = 0, my_bins = 0;  // this thread's of this CTA's share of the bins
    auto share = [&](int bins) {
      const int per = bins / static_cast<int>(ctas), per_thread = max(4, per / kThreads);
      my_bin = static_cast<int>(k.rank) * per + tid * per_thread, my_bins = tid * per_thread < per ? per_thread : 0;
    };
    auto clear = [&]() {
      for (int i = tid; i < kBins; i += kThreads) reinterpret_cast<uint4*>(&s.hist[0][0])[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
    };
    // f(logit, index) of this CTA's kept tokens from one logit to another: from the list of those about the cut, once it is
    // there and holds them, or from all
    int near_n = -1;
    auto for_members = [&](float from, float to, auto f) {
      if (near_n >= 0 && near_n <= kNear) {
        for (int j = tid; j < near_n; j += kThreads) {
          const int at = s.near[j];
          const float l = static_cast<float>(reinterpret_cast<const T*>(row_words)[at]);
          if (l >= from && l <= to && keeps(l, first + at)) f(l, first + at);
        }
      } else {
        for_mine([&](const float (&l)[4], int i) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (l[e] >= from && l[e] <= to && keeps(l[e], i + e)) f(l[e], i + e);
        });
      }
    };
    // the CTAs' histograms added up: each CTA's share of the bins lies in its own hist[0] (tokens) and hist[1], hist[2] (weight)
    u64 c_before = 0ull, w_before = 0ull, c_total = 0ull;  // tokens and weight before this thread's bins, tokens of all bins
    auto merge = [&](bool weights) {
      csync();
      u64 c = 0ull, w = 0ull;
      for (int bin = my_bin; bin < my_bin + my_bins; bin += 4) {  // four bins of every CTA at once
        uint4 n = make_uint4(0u, 0u, 0u, 0u);
        u64 weight[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (unsigned r = 0; r < kMaxCtas; ++r) {
          if (r >= ctas) break;
          const uint4 v = remote_ld4(&fine[bin], r);
          n.x += v.x, n.y += v.y, n.z += v.z, n.w += v.w;
          if (weights) {
            const uint4 w0 = remote_ld4(&s.hist[1][bin], r), w1 = remote_ld4(&s.hist[2][bin], r), w2 = remote_ld4(&s.hist[3][bin], r);
            weight[0] += w0.x + (static_cast<u64>(w1.x) << 15) + (static_cast<u64>(w2.x) << 30);
            weight[1] += w0.y + (static_cast<u64>(w1.y) << 15) + (static_cast<u64>(w2.y) << 30);
            weight[2] += w0.z + (static_cast<u64>(w1.z) << 15) + (static_cast<u64>(w2.z) << 30);
            weight[3] += w0.w + (static_cast<u64>(w1.w) << 15) + (static_cast<u64>(w2.w) << 30);
          }
        }
        *reinterpret_cast<uint4*>(&fine[bin]) = n;  // (no other CTA reads this CTA's share)
        c += static_cast<u64>(n.x) + n.y + n.z + n.w;
        if (weights)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s.hist[1][bin + e] = static_cast<unsigned>(weight[e]), s.hist[2][bin + e] = static_cast<unsigned>(weight[e] >> 32);
            w += weight[e];
          }
      }
      u64 tc = 0ull, tw = 0ull, none = 0ull, below;
      c_before = k.scan(c, tc);
      if (weights) w_before = k.scan(w, tw);
      k.exchange(tc, tw, none);
      c_total = k.over_ctas(tc, below), c_before += below;
      if (weights) k.over_ctas(tw, below), w_before += below;
    };
    auto count_of = [&](int b) { return static_cast<u64>(fine[b]); };
    auto weight_of = [&](int b) { return (static_cast<u64>(s.hist[2][b]) << 32) | s.hist[1][b]; };
    auto tell = [&](int slot, u64 v) {
      for (unsigned r = 0; r < ctas; ++r) remote_st(&s.found[slot], r, v);
    };
    // the bin in which a running size, `before` in front of this thread's bins, reaches `limit` (from 1 to the sum of sizes)
    int bin = 0;
    u64 bin_n = 0ull, bin_before = 0ull;  // its tokens, the size before it
    auto cross = [&](u64 limit, u64 before, auto size_of) {
      for (int b = my_bin; b < my_bin + my_bins; ++b) {
        const u64 size = size_of(b);
        if (before < limit && limit <= before + size) tell(0, b), tell(1, fine[b]), tell(2, before);
        before += size;
      }
      csync();
      bin = static_cast<int>(s.found[0]), bin_n = s.found[1], bin_before = s.found[2];
    };
    // the tokens from one logit to another, as far as they are kept, to the list of CTA 0; -> how many there are, at most kList
    unsigned gather_turn = 0u;
    auto gather = [&](float from, float to) -> int {
      if (tid == 0) s.own_n = 0u;
      __syncthreads();
      for_members(from, to, [&](float l, int i) {
        const unsigned at = atomicAdd(&s.own_n, 1u);
        if (at < kList) s.list_w[at] = place_of(l, i);
      });
      __syncthreads();
      const unsigned n = min(s.own_n, static_cast<unsigned>(kList));
      if (tid == 0 && n) s.own_at = remote_add(&s.listed[gather_turn], 0, n);
      __syncthreads();
      if (n) {
        const unsigned at = s.own_at;
        for (unsigned i = tid; i < n && at + i < kList; i += kThreads) remote_st(&s.list[at + i], 0, s.list_w[i]);
      }
      csync();
      const unsigned all = min(remote_ld(&s.listed[gather_turn], 0), static_cast<unsigned>(kList));
      gather_turn ^= 1u;
      if (k.rank == 0 && tid == 0) s.listed[gather_turn] = 0u;  // (every CTA has read it before it came to the barrier above)
      return static_cast<int>(all);
    };
    // CTA 0: for token i of the list, how many of the m come before it and what they weigh
    auto rank_of = [&](int i, int m, unsigned& rank, u64& weight) {
      const u64 own = s.list[i];
      rank = 0u, weight = 0ull;
#pragma unroll 4
      for (int j = 0; j < m; ++j) {
        const bool before = s.list[j] > own;
        rank += before;
        weight += before ? s.list_w[j] : 0ull;
      }
    };
    auto weigh_list = [&](int m) {
      for (int i = tid; i < m; i += kThreads) s.list_w[i] = weigh(of_key(static_cast<unsigned>(s.list[i] >> 32)));
      __syncthreads();
    };
    // the cut inside a range of logits with at most n kept tokens: after `need` of them, or after the one with which their
    // weight reaches `need`
    auto resolve = [&](bool count, u64 need, float from, float to, u64 n) {
      constexpr unsigned kZeros = (1u << kZeroBits<T>) - 1u;
      // (a division takes kBinBits of the keys' 32 bits, so the last round has few or equal ones)
      for (int round = 0; round <= (31 + kBinBits) / kBinBits; ++round) {
        if (n <= kList) {
          const int m = gather(from, to);
          if (k.rank == 0) {
            weigh_list(m);
            u64 last = ~0ull;  // of the kept: the least likely place
            for (int i = tid; i < m; i += kThreads) {
              unsigned rank;
              u64 before;
              rank_of(i, m, rank, before);
              if ((count ? rank : before) < need) last = smaller(last, s.list[i]);
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) last = smaller(last, __shfl_xor_sync(0xffffffffu, last, d));
            last = k.over_warps(last, smaller);
            if (tid < static_cast<int>(ctas)) remote_st(&s.found[0], tid, last);
          }
          csync();
          cut_l = of_key(static_cast<unsigned>(s.found[0] >> 32)), cut_i = static_cast<int>(~static_cast<unsigned>(s.found[0]));
          return;
        }
        // (the keys of both signs end in the type's zero bits, negative ones inverted: all ones)
        unsigned lo = key_of(fmaxf(from, cut_l)), hi = key_of(to);
        lo = (lo & 0x80000000u) ? (lo + kZeros) & ~kZeros : lo | kZeros;
        hi = (hi & 0x80000000u) ? hi & ~kZeros : (hi & kZeros) == kZeros ? hi : (hi | kZeros) - (kZeros + 1u);
        if (lo >= hi) {  // equal logits: the first ones by index
          const float l0 = of_key(hi);
          const u64 r = count ? need : (need + weigh(l0) - 1ull) / weigh(l0);
          u64 here = 0ull, total, below;
          for_mine([&](const float (&l)[4], int i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) here += l[e] == l0;
          });
          u64 before = k.scan(here, total);
          k.exchange(total);
          k.over_ctas(total, below);
          before += below;
          if (before < r && r <= before + here) {
            u64 at = before;
            const T* tokens = reinterpret_cast<const T*>(mine);
            for (int j = 0; j < a.words * kIn; ++j)
              if (static_cast<float>(tokens[j]) == l0 && ++at == r)
                tell(0, mine_first + j);
          }
          csync();
          cut_l = l0, cut_i = static_cast<int>(s.found[0]);
          return;
        }
        const int bits = 32 - __clz(hi - lo), shift = bits > kBinBits ? bits - kBinBits : 0;
        clear();
        share(kBins);
        for_members(from, to, [&](float l, int) {
          const int b = static_cast<int>((hi - key_of(l)) >> shift);
          atomicAdd(&s.hist[0][b], 1u);
          if (count) return;
          const u64 w = weigh(l);
          atomicAdd(&s.hist[1][b], static_cast<unsigned>(w) & 0x7FFFu);
          atomicAdd(&s.hist[2][b], static_cast<unsigned>(w >> 15) & 0x7FFFu);
          atomicAdd(&s.hist[3][b], static_cast<unsigned>(w >> 30));
        });
        __syncwarp();
        merge(!count);
        if (count) cross(need, c_before, count_of);
        else cross(need, w_before, weight_of);
        need -= bin_before, n = bin_n;
        hi -= static_cast<unsigned>(bin) << shift;
        lo = max(lo, hi - ((1u << shift) - 1u));
        from = of_key(lo), to = of_key(hi);
      }
    };
    // the logits whose bins are at most b, and at least b
    auto lowest_of = [&](int b) { return b >= kFine - 1 ? cut_l : of_key(smallest(key_of(cut_l), key_of(top), [&](float l) { return fine_bin(l) <= b; })); };
    auto highest_of = [&](int b) { return b <= 0 ? top : of_key(smallest(key_of(cut_l), key_of(top), [&](float l) { return fine_bin(l) < b; }) - 1u); };

    // tokens per bin
    for (int i = tid; i < kFine / 4; i += kThreads) reinterpret_cast<uint4*>(fine)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    share(kFine);
    for_mine([&](const float (&l)[4], int) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (l[e] >= cut_l) atomicAdd(&fine[fine_bin(l[e])], 1u);
    });
    merge(false);
    const bool cuts = by_count && static_cast<u64>(top_k) < c_total;  // (what weighs nothing is not counted)
    u64 candidates = c_total;
    int last_bin = kFine - 1;
    if (cuts) {
      cross(static_cast<u64>(top_k), c_before, count_of);
      candidates = bin_before + bin_n, last_bin = bin;
    }
    const float last_l = lowest_of(last_bin);
    if (candidates <= kList) {
      // all that can be kept is few: CTA 0 ranks it and finds the token
      const int m = gather(last_l, top);
      if (k.rank == 0) {
        constexpr int kEach = (kList + kThreads - 1) / kThreads;
        const unsigned most = by_count ? static_cast<unsigned>(top_k) : kList;
        weigh_list(m);
        unsigned rank[kEach];
        u64 weight[kEach], w[kEach], total;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int i = tid + e * kThreads;
          w[e] = 0ull, rank[e] = 0u, weight[e] = 0ull;
          if (i >= m) continue;
          rank_of(i, m, rank[e], weight[e]);
          if (rank[e] < most) w[e] = s.list_w[i];
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
          for (int j = 0; j < m; ++j) before += static_cast<unsigned>(s.list[j]) > own ? s.list_w[j] : 0ull;  // (of a lower index)
          if (before <= target && target < before + w[e]) {
            a.tokens[row] = static_cast<int>(~own);
            if (a.logprob) a.logprob[row] = static_cast<float>(log(static_cast<double>(w[e]) / static_cast<double>(total)));
          }
        }
      }
      csync();
      return;
    }
    float from = cut_l, to = top;  // between which top_p cuts
    u64 window = 0ull;             // tokens there
    if (by_weight) {
      // A bin's tokens times the weight at its middle is right to 1 / 240 in the exponent, sums of it and the limit that they
      // are compared with too: the cut lies between the bins where 0.991 and 1.009 of the limit are reached
      auto about = [&](int b) {
        u64 n = fine[b];
        if (cuts && b >= last_bin) n = b == last_bin ? static_cast<u64>(top_k) - bin_before : 0ull;
        return n * static_cast<u64>(ex2_approx(static_cast<float>(b) * (-1.4426950408889634f / 120.f)) * 1099511627776.f);
      };
      u64 size = 0ull, total, below, c = c_before;
      for (int b = my_bin; b < my_bin + my_bins; ++b) size += about(b);
      u64 before = k.scan(size, total);
      k.exchange(total);
      const u64 all = k.over_ctas(total, below);
      before += below;
      const double limit = static_cast<double>(top_p) * static_cast<double>(all);
      const u64 least = larger(1ull, static_cast<u64>(0.991 * limit)), most = smaller(all, static_cast<u64>(1.009 * limit) + 1ull);
      for (int b = my_bin; b < my_bin + my_bins; ++b) {
        const u64 after = before + about(b);
        if (before < least && least <= after) tell(0, b), tell(1, c);
        c += fine[b];
        if (before < most && most <= after) tell(2, b), tell(3, c);
        before = after;
      }
      csync();
      const int b0 = static_cast<int>(s.found[0]), b1 = static_cast<int>(s.found[2]);
      from = most == all ? cut_l : lowest_of(b1), to = highest_of(b0);  // (tokens of weight 0 here stand behind the last bin)
      window = (most == all ? c_total : s.found[3]) - s.found[1];
      csync();  // every CTA has read what it was told
    }
    if (cuts) resolve(true, static_cast<u64>(top_k) - bin_before, last_l, highest_of(last_bin), bin_n);
    if (by_weight) {
      // exact sums: of all that is kept, and of what lies above the window; the window's tokens are noted
      if (tid == 0) s.own_n = 0u;
      __syncthreads();
      auto note = [&](const float (&l)[4], int e, int i, u64 w) {
        if (l[e] > to) sum += w;
        else if (l[e] >= from) {
          const unsigned at = atomicAdd(&s.own_n, 1u);
          if (at < kNear) s.near[at] = static_cast<unsigned short>(i + e - first);
        }
      };
      u64 all = 0ull, t_all, t_above, below, none = 0ull;
      if (dense) {
        all = weight_of_all(note);
      } else {
        for_mine([&](const float (&l)[4], int i) {
          if (!__any_sync(0xffffffffu, fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= cut_l)) return;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const u64 w = weigh(l[e]);
            if (!keeps(l[e], i + e)) continue;
            all += w;
            note(l, e, i, w);
          }
        });
      }
      __syncwarp();
      k.scan(all, t_all), k.scan(sum, t_above);
      near_n = static_cast<int>(s.own_n);
      k.exchange(t_all, t_above, none);
      all = k.over_ctas(t_all, below);
      const u64 limit = larger(1ull, static_cast<u64>(ceil(static_cast<double>(top_p) * static_cast<double>(all))));
      resolve(false, limit - k.over_ctas(t_above, below), from, to, window);
      // what is kept of the window, added to the threads whose tokens it is: bits 0-21 and 22-44 of the weights
      unsigned* extra = &s.hist[0][0];
      for (int i = tid; i < 2 * kThreads; i += kThreads) extra[i] = 0u;
      __syncthreads();
      for_members(from, to, [&](float l, int i) {
        const u64 w = weigh(l);
        const int owner = (i - first) / (a.words * kIn);
        atomicAdd(&extra[owner], static_cast<unsigned>(w) & 0x3FFFFFu);
        atomicAdd(&extra[kThreads + owner], static_cast<unsigned>(w >> 22));
      });
      __syncthreads();
      sum += extra[tid] + (static_cast<u64>(extra[kThreads + tid]) << 22);
    }
  }
  if (!by_weight) {
    if (dense) {
      sum = weight_of_all([](const float (&)[4], int, int, u64) {});
    } else {
      for_mine([&](const float (&l)[4], int i) {
        // (a warp without any skips the exponentials)
        if (!__any_sync(0xffffffffu, fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= cut_l)) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u64 w = weigh(l[e]);
          sum += keeps(l[e], i + e) ? w : 0ull;
        }
      });
    }
  }

  // ---------------- the token
  u64 total, below;
  u64 before = k.scan(sum, total);
  k.exchange(total);
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
