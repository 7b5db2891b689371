// Log-probabilities of given tokens, entropy and top alternatives of logit rows, and their backward.
//   m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m)
//   logp = (x_target - m) - ln s      H = ln s - t / s      p_j = e^(x_j - m - ln s)
//   d x_j = g (1[j = target] - p_j) - h p_j (ln p_j + H)      for upstream g of logp, h of H
// The forward leaves (m, log2 s) rather than their sum: x - m is exact near the maximum, so the
// backward's p keeps full fp32 accuracy however large the logits are.
// Logits of -inf (banned words) have weight zero, add nothing and get no gradient, but for a target
// among them, which keeps its g (1 - p = g); a row of them alone gives logp -inf and H 0.  NaN and +inf
// reach every output of their row.
#include "common.h"

namespace imgcap {

// order of the alternatives: larger value first, NaN behind every number, ties to the lower index
DEV uint32_t order_key(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 -> +0
  return x != x ? 0u : (u >> 31) ? ~u : (u | 0x80000000u);
}
// the number that an order_key of a number stands for
DEV float key_value(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
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
  const char* base;
  int skew, nvec, V;
  DEV uint4 at(int q) const { return *(const uint4*)(base + (uint32_t)q * 16u); }  // rows end below 2^32 bytes
  DEV Row(const T* x, int V_) : V(V_) {
    skew = (int)(((uintptr_t)x & 15) / sizeof(T));
    base = (const char*)x - skew * sizeof(T);
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

// Wave-wide maximum / sum, one instruction a step: row_shr 1, 2, 4, 8 within 16 lanes, then row_bcast
// 15 and 31; a lane without a source keeps its value, lane 63 has the result, and all get it.  (Waits:
// two states between writing a register and a permuted read of it.)
#define LP_FOLD(op)                                                   \
  asm("s_nop 1\n\t" op " %0, %0, %0 row_shr:1\n\t"                    \
      "s_nop 1\n\t" op " %0, %0, %0 row_shr:2\n\t"                    \
      "s_nop 1\n\t" op " %0, %0, %0 row_shr:4\n\t"                    \
      "s_nop 1\n\t" op " %0, %0, %0 row_shr:8\n\t"                    \
      "s_nop 1\n\t" op " %0, %0, %0 row_bcast:15 row_mask:0xa\n\t"    \
      "s_nop 1\n\t" op " %0, %0, %0 row_bcast:31 row_mask:0xc\n\t"    \
      "s_nop 1"                                                       \
      : "+v"(v));                                                     \
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63))
DEV float wave_all_max(float v) { LP_FOLD("v_max_f32_dpp"); }
DEV float wave_all_sum(float v) { LP_FOLD("v_add_f32_dpp"); }
#undef LP_FOLD
// the lanes' parts (reference c, -inf: nothing yet; sum s, weighted sum t) as one, in every lane; a
// difference that passes the float range weighs nothing
DEV void lp_join_lanes(float& c, float& s, float& t) {
  const float C = wave_all_max(c), cs = C == -INFINITY ? 0.f : C;
  const float d = fmaxf((c - cs) * LOG2E, -1000.f), f = __builtin_amdgcn_exp2f(d);
  t = wave_all_sum(f * fmaf(d, s, t));
  s = wave_all_sum(f * s);
  c = C;
}

// A row per workgroup, read once: NV vectors a thread in flight, taken as they come.  A thread keeps
// its maximum m and sums relative to a reference c, a logit that follows m when m has passed it by 5
// or more (rare after the first vector, so no second look at the data and no rescaling as a rule):
// with z = (x - c) log2 e, s = sum 2^z and t = sum 2^z z.  c is a logit itself, so the row of a single
// word has s = 1 exactly.  DPP joins the lanes, LDS the waves.
// Alternatives: the top-th largest of 64 partial maxima (one per lane, over the waves) is a value
// that at least `top` elements reach; the few elements that reach it are gathered in LDS and ranked
// there.  Where more than LP_CAND do (long ties), or too few (NaN), the alternatives are found one by
// one, in passes over the row.
// Bound by vector issue beside HBM: 8.4 instructions a logit (the exponential at a quarter of the rate)
// and some 300 a wave.  MI355X, calls one after another: 3264 x 9490 bf16 with 5 alternatives 17.0 us
// (62 MB; 12.7 at the rate of a large copy), 1000 x 131072 bf16 with 20 58.4 us (4.5 TB/s), 777 x 50257
// fp32 with 10 32.3 us (4.8 TB/s), 5 x 9490 fp32 5.5 us.
template <typename T, int TPB, bool LONG>
__global__ __launch_bounds__(TPB) void token_logprobs_kernel(int V, int top, const T* __restrict__ logits, long ld,
                                                             const int64_t* __restrict__ tgt, float* __restrict__ logp,
                                                             float* __restrict__ entropy, float* __restrict__ stats,
                                                             float* __restrict__ top_logp, int64_t* __restrict__ top_ids) {
  constexpr int VEC = 16 / sizeof(T), NW = TPB / 64, NV = 8, SEG = TPB * NV;
  __shared__ float part[NW][3];
  __shared__ float lane_max[NW][64];
  __shared__ uint64_t cand[LP_CAND];
  __shared__ int ncand, nbusy;
  __shared__ uint16_t busy[TPB];
  const long row = blockIdx.x;
  const T* x = logits + row * ld;
  const Row<T> r(x, V);
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const long k = tgt ? tgt[row] : -1;
  const bool hit = k >= 0 && k < V;
  if (tid == 0) ncand = nbusy = 0;
  constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
  float m = -INFINITY, c = -INFINITY, s = 0.f, t = 0.f;
  uint4 u[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j)  // all in flight before the first is used: under no branch, the end again where past it
    u[j] = r.at(min(j * TPB + tid, r.nvec - 1));
  if (tid == 0) r.trim(u[0], 0);
  for (int q0 = 0; q0 < (LONG ? r.nvec : 1); q0 += SEG) {
    const int last = r.nvec - 1 - q0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (last >= j * TPB) {
        if (last < (j + 1) * TPB) {
          if (j * TPB + tid > last) u[j] = make_uint4(NONE, NONE, NONE, NONE);
          if (j * TPB + tid == last) r.trim(u[j], q0 + last);
        }
        float v[VEC];
        unpack<T>(u[j], v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = fmaxf(m, v[e]);
        if (m - c > 5.f) {
          const float d = fmaxf((c - m) * LOG2E, -1000.f), f = __builtin_amdgcn_exp2f(d);
          t = f * fmaf(d, s, t);
          s *= f;
          c = m;
        }
        const float cs = c == -INFINITY ? 0.f : c;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float z = (v[e] - cs) * LOG2E, p = __builtin_amdgcn_exp2f(z);
          s += p;
          t = fmaf(p, fmaxf(z, -200.f), t);  // p is 0 long before -200: a finite factor beside it
        }
      }
      if (LONG) u[j] = r.at(min(q0 + SEG + j * TPB + tid, r.nvec - 1));  // its place in the next segment
      __builtin_amdgcn_sched_barrier(0);  // one vector's floats at a time: more of them at once only spill
    }
  }
  const float xt = hit && w == 0 ? to_f(x[k]) : 0.f;
  lane_max[w][lane] = m;
  lp_join_lanes(c, s, t);
  if (lane == 0) {
    part[w][0] = c;
    part[w][1] = s;
    part[w][2] = t;
  }
  __syncthreads();
  float lm = lane_max[0][lane];
#pragma unroll
  for (int i = 1; i < NW; ++i) lm = fmaxf(lm, lane_max[i][lane]);
  // the first wave joins the parts and puts out what is one to a row
  float M = 0.f, ls = 0.f;
  bool none = false;
  if (w == 0) {
    float C = lane < NW ? part[lane][0] : -INFINITY, S = lane < NW ? part[lane][1] : 0.f, Z = lane < NW ? part[lane][2] : 0.f;
    M = wave_all_max(lm);
    lp_join_lanes(C, S, Z);
    none = S == 0.f;  // every logit -inf
    const float ls2 = log2f(S), l2 = none ? 0.f : fmaf(C - M, LOG2E, ls2);
    ls = l2 * LN2;
    if (lane == 0) {
      stats[2 * row] = M;
      stats[2 * row + 1] = l2;
      entropy[row] = none ? 0.f : (ls2 - Z / S) * LN2;
      if (tgt) logp[row] = !hit ? 0.f : none ? -INFINITY : (xt - M) - ls;
    }
  }
  if (top == 0) return;
  // the largest 16-bit key that at least `top` of the 64 partial maxima reach
  const uint32_t key = order_key(lm) >> 16;
  uint32_t bar = 0;
#pragma unroll
  for (int b = 15; b >= 0; --b)
    if (__popcll(__ballot(key >= (bar | 1u << b))) >= top) bar |= 1u << b;
  const float least = bar <= 0x007fu ? -INFINITY
                                     : __builtin_bit_cast(float, bar & 0x8000u ? (bar << 16) & 0x7fffffffu : ~(bar << 16));
  // the threads with such an element are few: their parts of the row are gone over again, a vector a
  // thread of the whole group, out of the cache
  if (m >= least) busy[atomicAdd(&nbusy, 1)] = (uint16_t)tid;
  __syncthreads();
  const int per = (r.nvec + TPB - 1) / TPB;
  for (int i0 = tid; i0 < nbusy * per; i0 += TPB) {
    const int q = busy[i0 / per] + i0 % per * TPB;
    if (q < r.nvec) {
      float v[VEC], mx = -INFINITY;
      unpack<T>(r.at(q), v);
#pragma unroll
      for (int e = 0; e < VEC; ++e) mx = fmaxf(mx, v[e]);
      if (mx < least) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (v[e] >= least) {
          const int i = q * VEC + e - r.skew;
          if (i >= 0 && i < V) {
            const int at = atomicAdd(&ncand, 1);
            if (at < LP_CAND) cand[at] = ((uint64_t)order_key(v[e]) << 32) | (0xffffffffu - (uint32_t)i);
          }
        }
    }
  }
  __syncthreads();
  const int nc = ncand;
  if (nc >= top && nc <= LP_CAND) {
    if (w > 0) return;
    for (int i = lane; i < nc; i += 64) {
      const uint64_t mine = cand[i];
      int rank = 0;
      for (int o = 0; o < nc; ++o) rank += cand[o] > mine;
      if (rank < top) {
        const uint32_t id = 0xffffffffu - (uint32_t)mine;
        top_ids[row * top + rank] = id;
        top_logp[row * top + rank] = none ? -INFINITY : (key_value((uint32_t)(mine >> 32)) - M) - ls;
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

// 16 bytes in, 16 bytes out per thread and step; a row's constants are the same for its workgroup.
// Bound by HBM.  Rows go from the last back, so the logits that the forward read last come from the
// memory-side cache; where logits and gradient together pass its 256 MB the stores are streaming, or
// they push out what is still to be read (777 x 50257 fp32 forward and gradient 103 -> 86 us; 3264 x
// 9490 bf16, 124 MB in all, 45.6 -> 44.7 by the order alone, and its stores stay cached for the
// product that reads them next).  A row is cut into even shares of up to 1024 vectors: at 9490 words
// two of 594, not 1024 and 163, 25.9 -> 20.5 us (6 TB/s of reads and writes, the reads cached).
template <typename T>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(int V, int blocks, const T* logits, long ld,
                                                                 const int64_t* __restrict__ tgt,
                                                                 const float* __restrict__ stats,
                                                                 const float* __restrict__ entropy,
                                                                 const float* __restrict__ dlogp,
                                                                 const float* __restrict__ dentropy, T* dx, long ldd,
                                                                 int stream_out) {
  constexpr int VEC = 16 / sizeof(T), STEPS = 4;
  const long row = (gridDim.x - 1 - blockIdx.x) / blocks;  // from the last row back: the forward's latest are still cached
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
  const int per = (r.nvec + blocks - 1) / blocks, begin = (blockIdx.x % blocks) * per;  // even shares of the row
  const int end = min(begin + per, r.nvec), q0 = begin + threadIdx.x;
  uint4 u[STEPS];
#pragma unroll
  for (int j = 0; j < STEPS; ++j)
    if (q0 + 256 * j < end) u[j] = r.at(q0 + 256 * j);
#pragma unroll
  for (int j = 0; j < STEPS; ++j) {
    const int q = q0 + 256 * j, c0 = q * VEC - r.skew;
    if (q >= end) break;
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
      if (stream_out) {
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        u32x4 words;
        T* es = (T*)&words;
#pragma unroll
        for (int e = 0; e < VEC; ++e) es[e] = from_f<T>(v[e]);
        __builtin_nontemporal_store(words, (u32x4*)(o + c0));
      } else {
        st_g<T, VEC>(o + c0, v);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c0 + e >= 0 && c0 + e < V) o[c0 + e] = from_f<T>(v[e]);
    }
  }
}

}  // namespace imgcap

using namespace imgcap;

static int lp_check(const imgcap_logprob_desc* d, const char* name) {
  const std::string at = std::string(name) + ": ";
  IMGCAP_REQUIRE(d != nullptr, at + "desc NULL");
  IMGCAP_REQUIRE(d->dtype == IMGCAP_F32 || d->dtype == IMGCAP_BF16, at + "dtype must be fp32 or bf16");
  IMGCAP_REQUIRE(d->n >= 0 && d->V > 0 && d->V <= (1 << 28) && (d->n <= 1 || d->ld >= d->V), at + "bad n / V / ld");
  return 0;
}

extern "C" int imgcap_token_logprobs(const imgcap_logprob_desc* d, void* stream) {
  if (int rc = lp_check(d, "imgcap_token_logprobs")) return rc;
  const int n = d->n, V = d->V, top = d->top;
  IMGCAP_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= V, "imgcap_token_logprobs: top must be 0 .. min(64, V)");
  if (n == 0) return 0;
  IMGCAP_REQUIRE(d->logits && d->entropy && d->stats && (!d->targets || d->logp) &&
                     (top == 0 || (d->top_logp && d->top_ids)),
                 "imgcap_token_logprobs: NULL operand");
  hipStream_t st = (hipStream_t)stream;
  // Few rows: 1024 threads each, for latency (5 x 9490 5.5 us).  More than 512: 256 threads for rows that
  // these hold in registers or nearly (3264 x 9490 bf16 17.0 us, 24.0 with 512; 2000 x 9490 fp32 16.9,
  // 18.0), 512 beyond (1280 x 50257 fp32 46.1 us, 50.1 with 256; 1000 x 131072 bf16 58.4, 60.8).
  const int vec = d->dtype == IMGCAP_BF16 ? 8 : 4, nvec = (V + 2 * vec - 2) / vec;
  const int tpb = n <= 512 ? 1024 : nvec <= 512 * 8 ? 256 : 512;
  IMGCAP_REQUIRE((int64_t)n * tpb < (1ll << 32), "imgcap_token_logprobs: too many rows for a launch (2^32 threads)");
#define LP_(T, TPB, LONG)                                                                                 \
  hipLaunchKernelGGL((token_logprobs_kernel<T, TPB, LONG>), dim3(n), dim3(TPB), 0, st, V, top,            \
                     (const T*)d->logits, (long)d->ld, d->targets, d->logp, d->entropy, d->stats, d->top_logp, d->top_ids)
#define LP_T(T)                                                                                           \
  do {                                                                                                    \
    if (tpb == 256) {                                                                                     \
      if (nvec <= 256 * 8) LP_(T, 256, false);                                                            \
      else LP_(T, 256, true);                                                                             \
    } else if (tpb == 512) {                                                                              \
      LP_(T, 512, true);                                                                                  \
    } else {                                                                                              \
      if (nvec <= 1024 * 8) LP_(T, 1024, false);                                                          \
      else LP_(T, 1024, true);                                                                            \
    }                                                                                                     \
  } while (0)
  if (d->dtype == IMGCAP_BF16) LP_T(bf16);
  else LP_T(float);
#undef LP_T
#undef LP_
  IMGCAP_CHECK_LAUNCH("imgcap_token_logprobs");
  return 0;
}

extern "C" int imgcap_token_logprobs_bwd(const imgcap_logprob_desc* d, void* stream) {
  if (int rc = lp_check(d, "imgcap_token_logprobs_bwd")) return rc;
  const int n = d->n, V = d->V;
  IMGCAP_REQUIRE(n <= 1 || d->ldd >= V, "imgcap_token_logprobs_bwd: bad ldd");
  if (n == 0) return 0;
  IMGCAP_REQUIRE(d->logits && d->stats && d->entropy && d->dlogits && (!d->dlogp || d->targets),
                 "imgcap_token_logprobs_bwd: NULL operand");
  IMGCAP_REQUIRE(d->logits != d->dlogits || d->ld == d->ldd || n == 1,
                 "imgcap_token_logprobs_bwd: in place needs equal pitches");
  hipStream_t st = (hipStream_t)stream;
#define LPB_(T)                                                                                                     \
  do {                                                                                                              \
    const int vec = 16 / (int)sizeof(T), blocks = ((V + 2 * vec - 2) / vec + 1023) / 1024;                          \
    IMGCAP_REQUIRE((int64_t)n * blocks < (1ll << 24),                                                               \
                   "imgcap_token_logprobs_bwd: too many rows for a launch (2^32 threads)");                         \
    hipLaunchKernelGGL(token_logprobs_bwd_kernel<T>, dim3((unsigned)n * blocks), dim3(256), 0, st, V, blocks,       \
                       (const T*)d->logits, (long)d->ld, d->targets, d->stats, d->entropy, d->dlogp,                \
                       d->dentropy, (T*)d->dlogits, (long)d->ldd,                                                   \
                       (int64_t)n * V * (int64_t)sizeof(T) > (128ll << 20) ? 1 : 0);                                \
  } while (0)
  if (d->dtype == IMGCAP_BF16) LPB_(bf16);
  else LPB_(float);
#undef LPB_
  IMGCAP_CHECK_LAUNCH("imgcap_token_logprobs_bwd");
  return 0;
}
