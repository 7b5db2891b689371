// Log-probabilities of given tokens, entropy and top alternatives of logit rows, and their backward.
//   m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m)
//   logp = (x_target - m) - ln s      H = ln s - t / s      p_j = e^(x_j - m - ln s)
//   d x_j = g (1[j = target] - p_j) - h p_j (ln p_j + H)      for upstream g of logp, h of H
// The forward leaves (m, log2 s) rather than their sum: x - m is exact near the maximum, so the
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

constexpr int LP_MAX_TOP = 64, LP_CAND = 512;
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.69314718055994531f;

// One row of V elements of any alignment as 16-byte vectors from the aligned address below its
// first element: element e of vector q is e + q * VEC - skew.  A vector is read only if an element
// of the row is in it.
template <typename T> struct Row {
  static constexpr int VEC = 16 / sizeof(T);
  const uint4* base;
  int skew, nvec, V;
  DEV Row(const T* x, int V_) : V(V_) {
    skew = (int)(((uintptr_t)x & 15) / sizeof(T));
    base = (const uint4*)((const char*)x - skew * sizeof(T));
    nvec = (V + skew + VEC - 1) / VEC;
  }
  // -inf in the places of vector q outside the row (the first and the last vector can have such);
  // on words, so that a row in registers stays one
  DEV void trim(uint4& u, int q) const {
    const int c0 = q * VEC - skew;
    uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 4) {
        if (c0 + i < 0 || c0 + i >= V) w[i] = 0xff800000u;
      } else {
        if (c0 + 2 * i < 0 || c0 + 2 * i >= V) w[i] = (w[i] & 0xffff0000u) | 0xff80u;
        if (c0 + 2 * i + 1 < 0 || c0 + 2 * i + 1 >= V) w[i] = (w[i] & 0xffffu) | 0xff800000u;
      }
    }
    u = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T> DEV void unpack(const uint4& u, float (&v)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __builtin_bit_cast(float, u.x); v[1] = __builtin_bit_cast(float, u.y);
    v[2] = __builtin_bit_cast(float, u.z); v[3] = __builtin_bit_cast(float, u.w);
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __builtin_bit_cast(float, w[i] << 16);
      v[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
    }
  }
}

// The packed words stay what is kept between two passes over a row: without this the compiler keeps
// the first pass's unpacked floats instead, twice the registers, and spills.
template <int NV> DEV void keep_packed(uint4 (&u)[NV]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) asm volatile("" : "+v"(u[j].x), "+v"(u[j].y), "+v"(u[j].z), "+v"(u[j].w));
}

// (maximum, sum, weighted sum) of two parts of a row; e^(m - M) of a part without weight is not
// taken, and a difference that passes the float range weighs nothing
DEV void lp_join(float& m, float& s, float& t, float m2, float s2, float t2) {
  const float M = fmaxf(m, m2), ms = M == -INFINITY ? 0.f : M;
  const float d = fmaxf((m - ms) * LOG2E, -200.f), d2 = fmaxf((m2 - ms) * LOG2E, -200.f);
  const float f = __builtin_amdgcn_exp2f(d), f2 = __builtin_amdgcn_exp2f(d2);
  t = f * fmaf(d, s, t) + f2 * fmaf(d2, s2, t2);
  s = f * s + f2 * s2;
  m = M;
}

// A row per workgroup.  The row is read once into registers, NV vectors a thread (a LONG row in
// segments of that).  Every thread sums relative to its own running maximum, so the row needs one
// exchange between waves.  Alternatives: the top-th largest of 64 partial maxima (one per lane,
// over the waves) is a value that at least `top` elements reach; the few elements that reach it are
// gathered in LDS and ranked there.  Where more than LP_CAND do (long ties), or too few (NaN), the
// alternatives are found one by one, in passes over the row.
template <typename T, int TPB, int NV, bool LONG>
__global__ __launch_bounds__(TPB) __attribute__((amdgpu_waves_per_eu(4))) void token_logprobs_kernel(
    int V, int top, const T* __restrict__ logits, long ld, const int64_t* __restrict__ tgt, float* __restrict__ logp,
    float* __restrict__ entropy, float* __restrict__ stats, float* __restrict__ top_logp,
    int64_t* __restrict__ top_ids) {
  constexpr int VEC = 16 / sizeof(T), NW = TPB / 64, SEG = TPB * NV;
  __shared__ float part[NW][3];
  __shared__ float lane_max[NW][64];
  __shared__ uint64_t cand[LP_CAND];
  __shared__ int ncand;
  const long row = blockIdx.x;
  const T* x = logits + row * ld;
  const Row<T> r(x, V);
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const long k = tgt ? tgt[row] : -1;
  const bool hit = k >= 0 && k < V;
  float xt = 0.f;
  if (tid == 0) ncand = 0;
  constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
  uint4 u[NV];
  float m = -INFINITY, s = 0.f, t = 0.f;
  for (int q0 = 0; q0 < (LONG ? r.nvec : 1); q0 += SEG) {
    const int last = r.nvec - 1 - q0;
#pragma unroll
    for (int j = 0; j < NV; ++j)  // all in flight before the first is used: under no branch, the end again where past it
      u[j] = r.base[q0 + min(j * TPB + tid, last)];
    if (q0 == 0 && tid == 0) r.trim(u[0], 0);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (last >= j * TPB && last < (j + 1) * TPB) {
        if (j * TPB + tid > last) u[j] = make_uint4(NONE, NONE, NONE, NONE);
        if (j * TPB + tid == last) r.trim(u[j], q0 + last);
      }
    float mx = m;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (last >= j * TPB) {
        float v[VEC];
        unpack<T>(u[j], v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) mx = fmaxf(mx, v[e]);
      }
      __builtin_amdgcn_sched_barrier(0);  // one vector's floats at a time: more of them at once only spill
    }
    if constexpr (sizeof(T) == 2) keep_packed(u);
    if (q0 == 0 && hit) xt = to_f(x[k]);
    const float ms = mx == -INFINITY ? 0.f : mx;
    if (LONG && q0 > 0) lp_join(m, s, t, mx, 0.f, 0.f);
    m = mx;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (last >= j * TPB) {
        float v[VEC];
        unpack<T>(u[j], v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float z = (v[e] - ms) * LOG2E, p = __builtin_amdgcn_exp2f(z);
          s += p;
          t = fmaf(p, fmaxf(z, -200.f), t);  // p is 0 long before -200: a finite factor beside it
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  lane_max[w][lane] = m;
  float ms = m, ss = s, ts = t;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    lp_join(ms, ss, ts, __shfl_xor(ms, o, 64), __shfl_xor(ss, o, 64), __shfl_xor(ts, o, 64));
  if (lane == 0) {
    part[w][0] = ms;
    part[w][1] = ss;
    part[w][2] = ts;
  }
  __syncthreads();
  float M = part[lane % NW][0], S = part[lane % NW][1], Z = part[lane % NW][2];
#pragma unroll
  for (int o = 1; o < NW; o <<= 1) lp_join(M, S, Z, __shfl_xor(M, o, 64), __shfl_xor(S, o, 64), __shfl_xor(Z, o, 64));
  // the lanes join in different orders and may differ in the last bit: lane 0's holds for all, or an
  // alternative's value would go by the place that it got in the list
  M = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, M)));
  S = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, S)));
  Z = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, Z)));
  const bool none = S == 0.f;  // every logit -inf
  const float l2 = none ? 0.f : log2f(S), ls = l2 * LN2;
  if (tid == 0) {
    stats[2 * row] = M;
    stats[2 * row + 1] = l2;
    entropy[row] = none ? 0.f : (l2 - Z / S) * LN2;
    if (tgt) logp[row] = !hit ? 0.f : none ? -INFINITY : (xt - M) - ls;
  }
  if (top == 0) return;
  // the largest 16-bit key that at least `top` of the 64 partial maxima reach
  float lm = lane_max[0][lane];
  for (int i = 1; i < NW; ++i) lm = fmaxf(lm, lane_max[i][lane]);
  const uint32_t key = order_key(lm) >> 16;
  uint32_t bar = 0;
#pragma unroll
  for (int b = 15; b >= 0; --b)
    if (__popcll(__ballot(key >= (bar | 1u << b))) >= top) bar |= 1u << b;
  const float least = bar <= 0x007fu ? -INFINITY
                                     : __builtin_bit_cast(float, bar & 0x8000u ? (bar << 16) & 0x7fffffffu : ~(bar << 16));
  // a thread with such an element goes over its part of the row again: few do, and it is in the cache
  if (m >= least)
    for (int q = tid; q < r.nvec; q += TPB) {
      float v[VEC];
      unpack<T>(r.base[q], v);
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (v[e] >= least) {
          const int c = q * VEC + e - r.skew;
          if (c >= 0 && c < V) {
            const int at = atomicAdd(&ncand, 1);
            if (at < LP_CAND) cand[at] = ((uint64_t)order_key(v[e]) << 32) | (0xffffffffu - (uint32_t)c);
          }
        }
    }
  __syncthreads();
  const int nc = ncand;
  if (nc >= top && nc <= LP_CAND) {
    for (int i = tid; i < nc; i += TPB) {
      const uint64_t mine = cand[i];
      int rank = 0;
      for (int o = 0; o < nc; ++o) rank += cand[o] > mine;
      if (rank < top) {
        const uint32_t id = 0xffffffffu - (uint32_t)mine;
        top_ids[row * top + rank] = id;
        top_logp[row * top + rank] = none ? -INFINITY : (to_f(x[id]) - M) - ls;
      }
    }
    return;
  }
  uint64_t last = ~0ull;
  for (int a = 0; a < top; ++a) {
    uint64_t best = 0;
    for (int c = tid; c < V; c += TPB) {
      const uint64_t c64 = ((uint64_t)order_key(to_f(x[c])) << 32) | (0xffffffffu - (uint32_t)c);
      if (c64 < last && c64 > best) best = c64;
    }
    best = wave_max_u64(best);
    __syncthreads();
    if (lane == 0) cand[w] = best;
    __syncthreads();
    for (int i = 0; i < NW; ++i) best = cand[i] > best ? cand[i] : best;
    last = best;
    if (tid == 0) {
      const uint32_t id = 0xffffffffu - (uint32_t)best;
      top_ids[row * top + a] = id;
      top_logp[row * top + a] = none ? -INFINITY : (to_f(x[id]) - M) - ls;
    }
  }
}

// 16 bytes in, 16 bytes out per thread and step; a row's constants are the same for its workgroup
template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(int V, int blocks, const T* logits, long ld,
                                                                 const int64_t* __restrict__ tgt,
                                                                 const float* __restrict__ stats,
                                                                 const float* __restrict__ entropy,
                                                                 const float* __restrict__ dlogp,
                                                                 const float* __restrict__ dentropy, T* dx, long ldd) {
  constexpr int VEC = 16 / sizeof(T), STEPS = 4;
  const long row = blockIdx.x / blocks;
  const T* x = logits + row * ld;
  T* o = dx + row * ldd;
  const Row<T> r(x, V);
  const bool whole = (((uintptr_t)o ^ (uintptr_t)x) & 15) == 0;  // both rows lie alike: vector stores
  const long k = tgt ? tgt[row] : -1;
  float m = stats[2 * row];
  const float l2 = stats[2 * row + 1];
  if (m == -INFINITY && l2 == 0.f) m = 0.f;  // every logit -inf: p = 0 throughout
  const float g = dlogp && k >= 0 && k < V ? dlogp[row] : 0.f, h = dentropy ? dentropy[row] : 0.f;
  const float a = -g - h * entropy[row], b = -h * LN2;
  const int q0 = (blockIdx.x % blocks) * (256 * STEPS) + threadIdx.x;
  uint4 u[STEPS];
#pragma unroll
  for (int j = 0; j < STEPS; ++j)
    if (q0 + 256 * j < r.nvec) u[j] = r.base[q0 + 256 * j];
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    const int q = q0 + 256 * j, c0 = q * VEC - r.skew;
    if (q >= r.nvec) break;
    float v[VEC];
    unpack<T>(u[j], v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float z = fmaf(v[e] - m, LOG2E, -l2);  // log2 p
      v[e] = __builtin_amdgcn_exp2f(z) * fmaf(b, fmaxf(z, -200.f), a);
    }
    if (k >= c0 && k < c0 + VEC) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c0 + e == k) v[e] += g;
    }
    if (whole && c0 >= 0 && c0 + VEC <= V) {
      st_g<T, VEC>(o + c0, v);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c0 + e >= 0 && c0 + e < V) o[c0 + e] = from_f<T>(v[e]);
    }
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
#define LP_(T, TPB, NV, LONG)                                                                             \
  hipLaunchKernelGGL((token_logprobs_kernel<T, TPB, NV, LONG>), dim3(n), dim3(TPB), 0, st, V, top,        \
                     (const T*)logits, (long)ld, targets, logp, entropy, stats, top_logp, top_ids)
#define LP_T(T)                                               \
  do {                                                        \
    const int vec = 16 / (int)sizeof(T), nvec = (V + 2 * vec - 2) / vec; \
    if (nvec <= 256 * 8 && n > 512) LP_(T, 256, 8, false);    \
    else if (nvec <= 1024 * 8) LP_(T, 1024, 8, false);        \
    else if (nvec <= 1024 * 16) LP_(T, 1024, 16, false);      \
    else LP_(T, 1024, 8, true);                               \
  } while (0)
  if (dtype == IMGCAP_BF16) LP_T(bf16);
  else LP_T(float);
#undef LP_T
#undef LP_
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
  IMGCAP_REQUIRE(logits != dlogits || ld == ldd || n == 1, "imgcap_token_logprobs_bwd: in place needs equal pitches");
  hipStream_t st = (hipStream_t)stream;
#define LPB_(T)                                                                                                     \
  do {                                                                                                              \
    const int vec = 16 / (int)sizeof(T), blocks = ((V + 2 * vec - 2) / vec + 1023) / 1024;                          \
    IMGCAP_REQUIRE((int64_t)n * blocks < (1ll << 31), "imgcap_token_logprobs_bwd: too many rows");                  \
    hipLaunchKernelGGL(token_logprobs_bwd_kernel<T>, dim3((unsigned)n * blocks), dim3(256), 0, st, V, blocks,       \
                       (const T*)logits, (long)ld, targets, stats, entropy, dlogp, dentropy, (T*)dlogits, (long)ldd); \
  } while (0)
  if (dtype == IMGCAP_BF16) LPB_(bf16);
  else LPB_(float);
#undef LPB_
  IMGCAP_CHECK_LAUNCH("imgcap_token_logprobs_bwd");
  return 0;
}
