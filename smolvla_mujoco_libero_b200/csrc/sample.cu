// C-ABI entry point of the choice of tokens (include/svla.h).
#include <cmath>
#include <cstring>

#include "answer_host.cuh"
#include "sample.cuh"

namespace svla {
namespace {

constexpr int kSampleVocab = 1 << 18;

template <typename T>
int32_t launch_sample(SampleArgs& a, cudaStream_t st) {
  static bool configured[64] = {false};
  auto kern = sample_kernel<T>;
  constexpr int kIn = 4 / static_cast<int>(sizeof(T)), kRound = sample::kThreads * kIn;  // tokens of a word, of a word per thread
  auto words = [](int vocab, int ctas) { return ((vocab + ctas * kRound - 1) / (ctas * kRound)) | 1; };
  auto bytes = [](int words) { return static_cast<int>(sizeof(sample::Shared)) + words * sample::kThreads * 4; };
  if (int32_t rc = allow_smem(kern, bytes(words(kSampleVocab, sample::kMaxCtas)), configured)) return rc;
  // CTAs of about a thousand tokens or more each, up to 8, which is the fastest for what fits the GPU at once (one row of 49280
  // tokens with top_k and top_p: 12.8 us, 14.7 with 4, 18.9 with 2; 64 bf16 rows of 131072 with top_p: 60.4, 66.3 with 4); many rows
  // have less to begin, to tell one another and to join with as few as leave three CTAs to an SM (256 mixed rows in fp32: 45 us
  // with 4, 62 with 2, 54 with 8; 512 rows without filters in bf16: 44 with 2, 49 with 4, 69 with 8)
  int ctas = 1;
  while (ctas < sample::kMaxCtas && a.vocab > 1024 * ctas) ctas *= 2;
  if (2ll * a.batch > sm_count())
    while (ctas > 2 && bytes(words(a.vocab, ctas / 2)) <= 75 * 1024) ctas /= 2;
  a.words = words(a.vocab, ctas);
  return launch_cluster(kern, dim3(static_cast<unsigned>(a.batch) * ctas), dim3(sample::kThreads), bytes(a.words), st, "sample_kernel",
                        static_cast<unsigned>(ctas), a);
}

}  // namespace
}  // namespace svla

using namespace svla;

extern "C" {

int32_t svla_sample_tokens(const svla_sample_desc* d, svla_stream_t stream) {
  const char* who = "svla_sample_tokens";
  if (!d) return fail(SVLA_ERR_ARG, "%s: null descriptor", who);
  if (d->dtype != SVLA_DT_BF16 && d->dtype != SVLA_DT_HALF && d->dtype != SVLA_DT_FLOAT)
    return fail(SVLA_ERR_ARG, "%s: dtype must be BF16, HALF or FLOAT (got %d)", who, d->dtype);
  if (d->vocab < 1 || d->vocab > kSampleVocab) return fail(SVLA_ERR_ARG, "%s: vocab must be 1 to %d (got %d)", who, kSampleVocab, d->vocab);
  if (d->batch < 0 || d->batch > (1 << 27)) return fail(SVLA_ERR_ARG, "%s: batch must be 0 to 2^27 (got %d)", who, d->batch);
  if (!d->temperature && !(d->temperature_value >= 0.f && !std::isinf(d->temperature_value)))
    return fail(SVLA_ERR_ARG, "%s: temperature must be finite and not negative (got %g)", who, d->temperature_value);
  if (!d->top_p && !(d->top_p_value >= 0.f)) return fail(SVLA_ERR_ARG, "%s: top_p must not be negative (got %g)", who, d->top_p_value);
  if (!d->min_p && !(d->min_p_value >= 0.f)) return fail(SVLA_ERR_ARG, "%s: min_p must not be negative (got %g)", who, d->min_p_value);
  if (d->batch == 0) return SVLA_OK;
  if (int32_t rc = check_rows(who, "logits", d->logits, d->logits_rs, d->vocab, d->dtype == SVLA_DT_FLOAT ? 4 : 2)) return rc;
  if (!d->u || !d->tokens) return fail(SVLA_ERR_ARG, "%s: u or tokens is null", who);
  const void* words[] = {d->u, d->temperature, d->top_k, d->top_p, d->min_p, d->tokens, d->logprob};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(SVLA_ERR_ARG, "%s: an argument is not aligned to its elements", who);
  SampleArgs a;
  std::memset(&a, 0, sizeof(a));
  a.logits = d->logits, a.logits_rs = d->logits_rs, a.u = d->u;
  a.temperature = d->temperature, a.top_k = d->top_k, a.top_p = d->top_p, a.min_p = d->min_p;
  a.temperature_value = d->temperature_value, a.top_k_value = d->top_k_value, a.top_p_value = d->top_p_value, a.min_p_value = d->min_p_value;
  a.tokens = d->tokens, a.logprob = d->logprob, a.batch = d->batch, a.vocab = d->vocab;
  if (d->dtype == SVLA_DT_FLOAT) return launch_sample<float>(a, cs(stream));
  if (d->dtype == SVLA_DT_HALF) return launch_sample<__half>(a, cs(stream));
  return launch_sample<__nv_bfloat16>(a, cs(stream));
}

}  // extern "C"
