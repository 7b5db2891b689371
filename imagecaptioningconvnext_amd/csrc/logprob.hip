// Log-probabilities of given tokens, entropy and top alternatives of logit rows, and their backward.
//   m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m)
//   logp = (x_target - m) - ln s      H = ln s - t / s      p_j = e^(x_j - m - ln s)
//   d x_j = g (1[j = target] - p_j) - h p_j (ln p_j + H)      for upstream g of logp, h of H
// The forward leaves (m, ln s) rather than their sum: x - m is exact near the maximum, so the
// backward's p keeps full fp32 accuracy however large the logits are.
// Logits of -inf (banned words) have weight zero and add nothing; a row of them alone gives
// logp -inf, H 0 and no gradient.  NaN and +inf reach every output of their row.
#include "common.h"

namespace imgcap {

// order of the alternatives: larger value first, NaN behind every number, ties to the lower index
DEV uint32_t order_key(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 -> +0
  return x != x ? 0u : (u >> 31) ? ~u : (u | 0x80000000u);
}
DEV uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t u = ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), o, 64) << 32) | (uint32_t)__shfl_xor((int)v, o, 64);
    v = u > v ? u : v;
  }
  return v;
}

constexpr int LP_MAX_TOP = 64;

template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_kernel(int V, int top, const T* __restrict__ logits, long ld,
                                                             const int64_t* __restrict__ tgt, float* __restrict__ logp,
                                                             float* __restrict__ entropy, float* __restrict__ stats,
                                                             float* __restrict__ top_logp, int64_t* __restrict__ top_ids) {
  __shared__ float red[4];
  __shared__ uint64_t redk[4];
  const long row = blockIdx.x;
  const T* x = logits + row * ld;
  const int w = threadIdx.x >> 6;
  float m = -INFINITY;
  for (int c = threadIdx.x; c < V; c += 256) m = fmaxf(m, to_f(x[c]));
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ms = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
  for (int c = threadIdx.x; c < V; c += 256) {
    const float y = to_f(x[c]) - ms, e = __expf(y);
    s += e;
    t += e == 0.f ? 0.f : e * y;
  }
  s = block_sum(s, red);
  t = block_sum(t, red);
  const float ls = logf(s);
  const bool none = s == 0.f;  // every logit -inf
  if (threadIdx.x == 0) {
    stats[2 * row] = m;
    stats[2 * row + 1] = none ? 0.f : ls;
    entropy[row] = none ? 0.f : ls - t / s;
    if (tgt) {
      const long k = tgt[row];
      logp[row] = k < 0 || k >= V ? 0.f : none ? -INFINITY : (to_f(x[k]) - m) - ls;
    }
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (int c = threadIdx.x; c < V; c += 256) {
      const uint64_t key = ((uint64_t)order_key(to_f(x[c])) << 32) | (0xffffffffu - (uint32_t)c);
      if (key < last && key > best) best = key;
    }
    best = wave_max_u64(best);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) redk[w] = best;
    __syncthreads();
    for (int i = 0; i < 4; ++i) best = redk[i] > best ? redk[i] : best;
    last = best;
    if (threadIdx.x == 0) {
      const uint32_t id = 0xffffffffu - (uint32_t)best;
      top_ids[row * top + k] = id;
      top_logp[row * top + k] = none ? -INFINITY : (to_f(x[id]) - m) - ls;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(int V, const T* logits, long ld,
                                                                 const int64_t* __restrict__ tgt,
                                                                 const float* __restrict__ stats,
                                                                 const float* __restrict__ entropy,
                                                                 const float* __restrict__ dlogp,
                                                                 const float* __restrict__ dentropy, T* dx, long ldd) {
  const long row = blockIdx.x;
  const T* x = logits + row * ld;
  T* o = dx + row * ldd;
  const long k = tgt ? tgt[row] : -1;
  const float m = stats[2 * row], ls = stats[2 * row + 1];
  const float g = dlogp && k >= 0 && k < V ? dlogp[row] : 0.f, h = dentropy ? dentropy[row] : 0.f;
  const float a = -g - h * entropy[row];
  const bool none = m == -INFINITY && ls == 0.f;  // every logit -inf: no gradient
  for (int c = threadIdx.x; c < V; c += 256) {
    const float y = none ? -INFINITY : (to_f(x[c]) - m) - ls;
    const float p = __expf(y);
    const float d = p == 0.f ? 0.f : p * (a - h * y);
    o[c] = from_f<T>(c == k ? d + g : d);
  }
}

}  // namespace imgcap

using namespace imgcap;

extern "C" int imgcap_token_logprobs(int dtype, int n, int V, int top, const void* logits, int64_t ld,
                                     const int64_t* targets, float* logp, float* entropy, float* stats,
                                     float* top_logp, int64_t* top_ids, void* stream) {
  IMGCAP_REQUIRE(dtype == IMGCAP_F32 || dtype == IMGCAP_BF16, "imgcap_token_logprobs: dtype must be fp32 or bf16");
  IMGCAP_REQUIRE(n >= 0 && V > 0 && ld >= V, "imgcap_token_logprobs: bad n / V / ld");
  IMGCAP_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= V, "imgcap_token_logprobs: top must be 0 .. min(64, V)");
  if (n == 0) return 0;
  IMGCAP_REQUIRE(logits && entropy && stats && (!targets || logp) && (top == 0 || (top_logp && top_ids)),
                 "imgcap_token_logprobs: NULL operand");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == IMGCAP_BF16)
    hipLaunchKernelGGL(token_logprobs_kernel<bf16>, dim3(n), dim3(256), 0, st, V, top, (const bf16*)logits, (long)ld,
                       targets, logp, entropy, stats, top_logp, top_ids);
  else
    hipLaunchKernelGGL(token_logprobs_kernel<float>, dim3(n), dim3(256), 0, st, V, top, (const float*)logits, (long)ld,
                       targets, logp, entropy, stats, top_logp, top_ids);
  IMGCAP_CHECK_LAUNCH("imgcap_token_logprobs");
  return 0;
}

extern "C" int imgcap_token_logprobs_bwd(int dtype, int n, int V, const void* logits, int64_t ld,
                                         const int64_t* targets, const float* stats, const float* entropy,
                                         const float* dlogp, const float* dentropy, void* dlogits, int64_t ldd,
                                         void* stream) {
  IMGCAP_REQUIRE(dtype == IMGCAP_F32 || dtype == IMGCAP_BF16, "imgcap_token_logprobs_bwd: dtype must be fp32 or bf16");
  IMGCAP_REQUIRE(n >= 0 && V > 0 && ld >= V && ldd >= V, "imgcap_token_logprobs_bwd: bad n / V / ld / ldd");
  if (n == 0) return 0;
  IMGCAP_REQUIRE(logits && stats && entropy && dlogits && (!dlogp || targets),
                 "imgcap_token_logprobs_bwd: NULL operand");
  IMGCAP_REQUIRE(logits != dlogits || ld == ldd, "imgcap_token_logprobs_bwd: in place needs equal pitches");
  hipStream_t st = (hipStream_t)stream;
  if (dtype == IMGCAP_BF16)
    hipLaunchKernelGGL(token_logprobs_bwd_kernel<bf16>, dim3(n), dim3(256), 0, st, V, (const bf16*)logits, (long)ld,
                       targets, stats, entropy, dlogp, dentropy, (bf16*)dlogits, (long)ldd);
  else
    hipLaunchKernelGGL(token_logprobs_bwd_kernel<float>, dim3(n), dim3(256), 0, st, V, (const float*)logits, (long)ld,
                       targets, stats, entropy, dlogp, dentropy, (float*)dlogits, (long)ldd);
  IMGCAP_CHECK_LAUNCH("imgcap_token_logprobs_bwd");
  return 0;
}
