// Fused ConvNeXt block MLP (torchvision CNBlock, reached via encoder.py:18-24):
//   x[m, :] += gamma * sd[m / rows_per_sample] * (GELU(z[m, :] W1^T + b1) W2^T + b2)
// with z = LN(y), y = dwconv7(x) (the LayerNorm runs in this kernel's prologue when ln_w is
// given, else z is taken as already normalised), W1 [4C, C], W2 [C, 4C] (nn.Linear), bf16.
// The 4C-wide hidden activation never leaves the chip: the block walks the hidden dimension
// in chunks of HC, computing H = GELU(Z W1c^T + b1c) and immediately accumulating
// O += H W2c^T; HBM traffic per row is z + x read and x written (6C bytes) instead of the
// unfused 6C + 16C (hidden written by Linear1 and read back by Linear2).
//
// Block = 4 waves, BM rows; wave w owns rows [w*BM/4, +BM/4) of BOTH GEMMs, so its hidden
// chunk goes accumulator -> LDS (per-wave region, layout change C-fragment -> A-fragment) ->
// MFMA without a block barrier.  The Z rows of a wave stay in registers as A fragments for
// the whole chunk loop; the W1/W2 chunks are shared by the 4 waves through a double-buffered
// LDS stage (global loads of chunk i+1 in flight under chunk i's MFMAs).  Epilogue: fp32
// tile through LDS, 8 columns per thread (16-byte residual loads and stores).
#include "mfma.h"

#include <algorithm>

namespace imgcap {

#ifndef MLP_GELU
#define MLP_GELU 2  // polynomial erf on two values at once (|err| <= 1.5e-7, common.h gelu_fast2); 0 = libm erff
#endif
#ifndef MLP_TAG
#define MLP_TAG "erf"
#endif
#ifndef MLP_EPI_BATCH
#define MLP_EPI_BATCH 0
#endif
#ifndef MLP96_BM
#define MLP96_BM 128
#endif
#ifndef MLP96_WPE
#define MLP96_WPE 2
#endif
#ifndef MLP96_HC
#define MLP96_HC 64
#endif
#ifndef MLP192_HC
#define MLP192_HC 32
#endif
#ifndef MLP192_BM
#define MLP192_BM 64
#endif
#ifndef MLP192_WPE
#define MLP192_WPE 2
#endif
#ifdef MLP_STAMPS  // kernel-bench diagnostics only (tools/kbench): s_memtime at phase edges
__device__ long long* g_mlp_stamps;
#define MLP_STAMP(k)                                                                       \
  do {                                                                                     \
    if (g_mlp_stamps && threadIdx.x == 0 && blockIdx.x < 64) {                             \
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");                          \
      g_mlp_stamps[blockIdx.x * 64 + (k)] = (long long)__builtin_amdgcn_s_memtime();       \
    }                                                                                      \
  } while (0)
#else
#define MLP_STAMP(k) do { } while (0)
#endif

// GELU of the hidden activation.  MLP_GELU (kernel-variant experiments, tools/kbench): 0 =
// erf form (torch nn.GELU default), 1 = identity (timing only), 2 = fast erf.
DEV float mlp_gelu(float v) {
#if MLP_GELU == 1
  return v;
#elif MLP_GELU == 2
  return gelu_fast(v);
#else
  return gelu_erf(v);
#endif
}

template <int C, int BM, int HC, bool ZL>
struct MlpCfg {
  static constexpr int WR = BM / 4;           // rows per wave
  static constexpr int TM = WR / 16;
  static constexpr int TN1 = HC / 16;         // hidden-chunk fragments per wave
  static constexpr int TN2 = C / 16;          // output fragments per wave
  static constexpr int KS1 = C / 32;          // k-steps of GEMM1
  static constexpr int KS2 = HC / 32;         // k-steps of GEMM2
  static constexpr int LD1 = C + 8;           // W1c image [HC][C] row stride (bf16)
  static constexpr int LD2 = HC + 8;          // W2c image [C][HC]
  static constexpr int LDH = HC + 8;          // per-wave hidden image [WR][HC]
  static constexpr int BUFE = HC * LD1 + C * LD2;
  static constexpr int HE = WR * LDH;
  static constexpr int V1 = HC * C / 8 / 256;  // 16-byte vectors per thread per W1 chunk
  static constexpr int V2 = C * HC / 8 / 256;
  static constexpr int LDO = C + 4;            // fp32 epilogue image row stride
  static constexpr int LDZ = C + 8;           // Z image [BM][C] (ZL: A fragments read from LDS)
  static constexpr int ZE = ZL ? BM * LDZ : 0;
  static constexpr int STAGE_BYTES = (BUFE + 4 * HE + ZE) * 2;
  static constexpr int EPI_BYTES = BM * LDO * 4;
  static constexpr int SMEM = STAGE_BYTES > EPI_BYTES ? STAGE_BYTES : EPI_BYTES;
  static_assert(WR % 16 == 0 && C % 32 == 0 && HC % 32 == 0, "tile shape");
  static_assert(V1 * 8 * 256 == HC * C && V2 * 8 * 256 == C * HC, "chunk must split evenly over 256 threads");
  static_assert(SMEM <= 160 * 1024, "LDS budget");
};

// weight chunk staging: W1 rows [h0, h0+HC) -> image [HC][C]; W2 columns [h0, h0+HC) ->
// image [C][HC]; one chunk in flight in registers while the previous one is consumed
template <int C, int HC, int V1, int V2>
DEV void mlp_load(uint4 (&r1)[V1], uint4 (&r2)[V2], const bf16* __restrict__ w1, const bf16* __restrict__ w2,
                  int h0) {
#pragma unroll
  for (int i = 0; i < V1; ++i) {
    const int v = threadIdx.x + i * 256, r = v / (C / 8), c = (v % (C / 8)) * 8;
    r1[i] = *(const uint4*)(w1 + (long)(h0 + r) * C + c);
  }
#pragma unroll
  for (int i = 0; i < V2; ++i) {
    const int v = threadIdx.x + i * 256, n = v / (HC / 8), c = (v % (HC / 8)) * 8;
    r2[i] = *(const uint4*)(w2 + (long)n * (4 * C) + h0 + c);
  }
}
template <int C, int HC, int LD1, int LD2, int V1, int V2>
DEV void mlp_store(bf16* buf, const uint4 (&r1)[V1], const uint4 (&r2)[V2]) {
#pragma unroll
  for (int i = 0; i < V1; ++i) {
    const int v = threadIdx.x + i * 256, r = v / (C / 8), c = (v % (C / 8)) * 8;
    *(uint4*)(buf + r * LD1 + c) = r1[i];
  }
#pragma unroll
  for (int i = 0; i < V2; ++i) {
    const int v = threadIdx.x + i * 256, n = v / (HC / 8), c = (v % (HC / 8)) * 8;
    *(uint4*)(buf + HC * LD1 + n * LD2 + c) = r2[i];
  }
}

// WPE: waves per SIMD the register budget must allow (1 = up to 512 registers per lane, 2 = 256:
// two resident blocks per CU, one block's prologue/epilogue latency under the other's MFMAs)
template <int C, int BM, int HC, bool ZL, int WPE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) void cnblock_mlp_kernel(int M, const bf16* __restrict__ z,
                                                          const bf16* __restrict__ w1, const float* __restrict__ b1,
                                                          const bf16* __restrict__ w2, const float* __restrict__ b2,
                                                          const float* __restrict__ gamma,
                                                          const float* __restrict__ sd, int rows_per_sample,
                                                          const float* __restrict__ lnw,
                                                          const float* __restrict__ lnb, bf16* __restrict__ x) {
  using G = MlpCfg<C, BM, HC, ZL>;
  __shared__ __attribute__((aligned(16))) char smem[G::SMEM];
  bf16* wbuf = (bf16*)smem;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  bf16* hbuf = wbuf + G::BUFE + w * G::HE;
  bf16* zimg = wbuf + G::BUFE + 4 * G::HE;  // ZL only
  const int m0 = blockIdx.x * BM;
  const int wr0 = m0 + w * G::WR;
  MLP_STAMP(0);

  // this wave's Z rows as A fragments (row fr of each 16-row slab, k = 8*fq..): kept in
  // registers for the whole chunk loop, or (ZL, wide C) staged once into an LDS image
  constexpr int ZR = ZL ? 1 : G::TM, ZK = ZL ? 1 : G::KS1;
  bf16x8 zf[ZR][ZK];
  if constexpr (ZL) {
    for (int v = threadIdx.x; v < BM * (C / 8); v += 256) {
      const int r = v / (C / 8), c = (v % (C / 8)) * 8;
      const int row = m0 + r;
      const uint4 u = *(const uint4*)(z + (long)(row < M ? row : 0) * C + c);
      *(uint4*)(zimg + r * G::LDZ + c) = row < M ? u : make_uint4(0u, 0u, 0u, 0u);
    }
  } else {
#pragma unroll
    for (int tm = 0; tm < G::TM; ++tm) {
      const int row = wr0 + tm * 16 + fr;
      const bool ok = row < M;
      const bf16* zp = z + (long)(ok ? row : 0) * C + 8 * fq;
#pragma unroll
      for (int ks = 0; ks < G::KS1; ++ks) {
        const uint4 u = *(const uint4*)(zp + ks * 32);
        zf[tm][ks] = __builtin_bit_cast(bf16x8, ok ? u : make_uint4(0u, 0u, 0u, 0u));
      }
    }
    if (lnw) {
      // z = LayerNorm(y) (torchvision LayerNorm2d, eps 1e-6), two-pass in fp32: row fr's C values
      // sit in lanes fr, fr+16, fr+32, fr+48; the result is rounded to bf16 like a stored z
#pragma unroll
      for (int tm = 0; tm < G::TM; ++tm) {
        float s = 0.f;
#pragma unroll
        for (int ks = 0; ks < G::KS1; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) s += (float)zf[tm][ks][j];
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        const float mean = s * (1.f / C);
        float q = 0.f;
#pragma unroll
        for (int ks = 0; ks < G::KS1; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) { const float dd = (float)zf[tm][ks][j] - mean; q += dd * dd; }
        q += __shfl_xor(q, 16, 64);
        q += __shfl_xor(q, 32, 64);
        const float rstd = rsqrtf(q * (1.f / C) + 1e-6f);
#pragma unroll
        for (int ks = 0; ks < G::KS1; ++ks) {
          const int k = ks * 32 + 8 * fq;
          const f32x4 g0 = *(const f32x4*)(lnw + k), g1 = *(const f32x4*)(lnw + k + 4);
          const f32x4 c0 = *(const f32x4*)(lnb + k), c1 = *(const f32x4*)(lnb + k + 4);
          const float gg[8] = {g0[0], g0[1], g0[2], g0[3], g1[0], g1[1], g1[2], g1[3]};
          const float cc[8] = {c0[0], c0[1], c0[2], c0[3], c1[0], c1[1], c1[2], c1[3]};
#pragma unroll
          for (int j = 0; j < 8; ++j) zf[tm][ks][j] = (bf16)(((float)zf[tm][ks][j] - mean) * rstd * gg[j] + cc[j]);
        }
      }
    }
  }
  f32x4 acc2[G::TM][G::TN2];
#pragma unroll
  for (int tm = 0; tm < G::TM; ++tm)
#pragma unroll
    for (int tn = 0; tn < G::TN2; ++tn) acc2[tm][tn] = f32x4{0.f, 0.f, 0.f, 0.f};
  MLP_STAMP(1);

  uint4 r1[G::V1], r2[G::V2];
  mlp_load<C, HC>(r1, r2, w1, w2, 0);
  mlp_store<C, HC, G::LD1, G::LD2>(wbuf, r1, r2);
  __syncthreads();  // (also publishes the Z image)
  MLP_STAMP(2);

  constexpr int NCH = 4 * C / HC;
  for (int ch = 0; ch < NCH; ++ch) {
    const bf16* cur = wbuf;
    // unconditional (the last iteration re-loads chunk 0, never stored to a live buffer):
    // a conditional load would make the compiler keep r1/r2 in scratch across the branch
    mlp_load<C, HC>(r1, r2, w1, w2, ((ch + 1) % NCH) * HC);
    // GEMM1: H[WR, HC] = Z W1c^T
    f32x4 acc1[G::TM][G::TN1];
#pragma unroll
    for (int tm = 0; tm < G::TM; ++tm)
#pragma unroll
      for (int tn = 0; tn < G::TN1; ++tn) acc1[tm][tn] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < G::KS1; ++ks) {
#pragma unroll
      for (int tn = 0; tn < G::TN1; ++tn) {
        const bf16x8 bfr = *(const bf16x8*)(cur + (tn * 16 + fr) * G::LD1 + ks * 32 + 8 * fq);
#pragma unroll
        for (int tm = 0; tm < G::TM; ++tm) {
          bf16x8 za;
          if constexpr (ZL)
            za = *(const bf16x8*)(zimg + (w * G::WR + tm * 16 + fr) * G::LDZ + ks * 32 + 8 * fq);
          else
            za = zf[tm < ZR ? tm : 0][ks < ZK ? ks : 0];
          // operands swapped: the tile is H^T (rows = hidden units, columns = rows of Z), so each
          // lane ends with 4 CONSECUTIVE hidden units of one row -- one 8-byte LDS write below
          acc1[tm][tn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bfr, za, acc1[tm][tn], 0, 0, 0);
        }
      }
    }
    if (ch < 8) MLP_STAMP(3 + 4 * ch);
    // bias + GELU -> bf16 hidden chunk in this wave's LDS image: lane (row fr, units 4fq..4fq+3)
    const int h0 = ch * HC;
#pragma unroll
    for (int tn = 0; tn < G::TN1; ++tn) {
      const f32x4 bb = *(const f32x4*)(b1 + h0 + tn * 16 + 4 * fq);
#pragma unroll
      for (int tm = 0; tm < G::TM; ++tm) {
        bf16x4 hv;
#if MLP_GELU == 2
        // (gelu_sig here measured slower: C = 192 59 -> 71 us, tools/kbench)
        const f32x2 g01 = gelu_fast2(f32x2{acc1[tm][tn][0] + bb[0], acc1[tm][tn][1] + bb[1]});
        const f32x2 g23 = gelu_fast2(f32x2{acc1[tm][tn][2] + bb[2], acc1[tm][tn][3] + bb[3]});
        hv[0] = (bf16)g01[0]; hv[1] = (bf16)g01[1]; hv[2] = (bf16)g23[0]; hv[3] = (bf16)g23[1];
#else
#pragma unroll
        for (int r = 0; r < 4; ++r) hv[r] = (bf16)mlp_gelu(acc1[tm][tn][r] + bb[r]);
#endif
        *(bf16x4*)(hbuf + (tm * 16 + fr) * G::LDH + tn * 16 + 4 * fq) = hv;
      }
    }
    if (ch < 8) MLP_STAMP(4 + 4 * ch);
    // GEMM2: O[WR, C] += H W2c^T   (the hidden image is written and read by this wave only)
    const bf16* w2c = cur + HC * G::LD1;
#pragma unroll
    for (int ks = 0; ks < G::KS2; ++ks) {
      bf16x8 hf[G::TM];
#pragma unroll
      for (int tm = 0; tm < G::TM; ++tm) hf[tm] = *(const bf16x8*)(hbuf + (tm * 16 + fr) * G::LDH + ks * 32 + 8 * fq);
#pragma unroll
      for (int tn = 0; tn < G::TN2; ++tn) {
        const bf16x8 bfr = *(const bf16x8*)(w2c + (tn * 16 + fr) * G::LD2 + ks * 32 + 8 * fq);
#pragma unroll
        for (int tm = 0; tm < G::TM; ++tm)
          acc2[tm][tn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hf[tm], bfr, acc2[tm][tn], 0, 0, 0);
      }
    }
    if (ch < 8) MLP_STAMP(5 + 4 * ch);
    __syncthreads();  // every wave is done with the staged chunk
    mlp_store<C, HC, G::LD1, G::LD2>(wbuf, r1, r2);
    __syncthreads();
    if (ch < 8) MLP_STAMP(6 + 4 * ch);
  }

  // epilogue: fp32 tile through LDS, then x += gamma * sd * (o + b2) on 8-column vectors
  constexpr int NV = C / 8;
  constexpr int NIT = BM * NV / 256;
  static_assert(NIT * 256 == BM * NV, "epilogue split");
  float* tile = (float*)smem;
#pragma unroll
  for (int tm = 0; tm < G::TM; ++tm)
#pragma unroll
    for (int tn = 0; tn < G::TN2; ++tn)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        tile[(w * G::WR + tm * 16 + 4 * fq + r) * G::LDO + tn * 16 + fr] = acc2[tm][tn][r];
  __syncthreads();
  MLP_STAMP(40);
#if MLP_EPI_BATCH
  // residual rows of all NIT iterations loaded at once (one memory round trip)
  bf16x8 xres[NIT];
#pragma unroll
  for (int u = 0; u < NIT; ++u) {
    const int e = threadIdx.x + u * 256, r = e / NV, c = (e % NV) * 8;
    xres[u] = *(const bf16x8*)(x + (long)min(m0 + r, M - 1) * C + c);
  }
#endif
#pragma unroll
  for (int u = 0; u < NIT; ++u) {
    const int e = threadIdx.x + u * 256, r = e / NV, c = (e % NV) * 8;
    const int m = m0 + r;
    if (m >= M) continue;
#if MLP_EPI_BATCH
    const bf16x8 xv = xres[u];
#else
    const bf16x8 xv = *(const bf16x8*)(x + (long)m * C + c);
#endif
    const float s = sd ? sd[m / rows_per_sample] : 1.f;
    const f32x4 t0 = *(const f32x4*)(tile + r * G::LDO + c), t1 = *(const f32x4*)(tile + r * G::LDO + c + 4);
    const f32x4 g0 = *(const f32x4*)(gamma + c), g1 = *(const f32x4*)(gamma + c + 4);
    const f32x4 c0 = *(const f32x4*)(b2 + c), c1 = *(const f32x4*)(b2 + c + 4);
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[j] = (bf16)((float)xv[j] + (t0[j] + c0[j]) * g0[j] * s);
      o[j + 4] = (bf16)((float)xv[j + 4] + (t1[j] + c1[j]) * g1[j] * s);
    }
    *(bf16x8*)(x + (long)m * C + c) = o;
  }
  MLP_STAMP(41);
}

// z = LayerNorm(y) (torchvision LayerNorm2d, eps 1e-6) on GEMM-operand fragments, two-pass in
// fp32: row fr of slab tm sits in lanes fr, fr+16, fr+32, fr+48 (k = 32 ks + 8 fq ..); the result
// is rounded to bf16 like a stored z
template <int C, int TM, int KS>
DEV void mlp_ln_frags(bf16x8 (&zf)[TM][KS], const float* __restrict__ lnw, const float* __restrict__ lnb, int fq) {
#pragma unroll
  for (int tm = 0; tm < TM; ++tm) {
    float s = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += (float)zf[tm][ks][j];
    s += __shfl_xor(s, 16, 64);
    s += __shfl_xor(s, 32, 64);
    const float mean = s * (1.f / C);
    float q = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) { const float dd = (float)zf[tm][ks][j] - mean; q += dd * dd; }
    q += __shfl_xor(q, 16, 64);
    q += __shfl_xor(q, 32, 64);
    const float rstd = rsqrtf(q * (1.f / C) + 1e-6f);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int k = ks * 32 + 8 * fq;
      const f32x4 g0 = *(const f32x4*)(lnw + k), g1 = *(const f32x4*)(lnw + k + 4);
      const f32x4 c0 = *(const f32x4*)(lnb + k), c1 = *(const f32x4*)(lnb + k + 4);
      const float gg[8] = {g0[0], g0[1], g0[2], g0[3], g1[0], g1[1], g1[2], g1[3]};
      const float cc[8] = {c0[0], c0[1], c0[2], c0[3], c1[0], c1[1], c1[2], c1[3]};
#pragma unroll
      for (int j = 0; j < 8; ++j) zf[tm][ks][j] = (bf16)(((float)zf[tm][ks][j] - mean) * rstd * gg[j] + cc[j]);
    }
  }
}

// W2 k order inside a 32-wide hidden step, as GEMM1's swapped output leaves the hidden values in a
// lane: 4-element piece p = 4s + q (hidden 16s + 4q .. +3) sits at position 8q + 4s.  Stores the
// 16-byte source vector holding hidden [c, c + 8) of one W2 row (c % 8 == 0) into `row`.
// swz: XOR applied to the 16-byte granule index (4j + q) of the destination (0: none).
DEV void w2_store_permuted(bf16* row, int c, const uint4& u, int swz = 0) {
  const int j = c / 32, p = (c % 32) / 4;  // p even
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int pp = p + e, s = pp / 4, q = pp % 4;
    *(uint2*)(row + 8 * ((4 * j + q) ^ swz) + 4 * s) = e ? make_uint2(u.z, u.w) : make_uint2(u.x, u.y);
  }
}

// ---- narrow stages (C = 96): both weight matrices resident in LDS ---------------------------
// The chunked kernel above re-streams W1 and W2 (2 * 4C * C bf16 = 144 KB at C = 96) from L2
// into LDS for every 128-row block: 115 MB of L2 -> LDS traffic per launch at the Tiny stage-1
// shape, at the per-CU LDS-fill rate that is most of its time.  Here one 512-thread workgroup per
// CU fills LDS with W1, W2 (and b1) ONCE and then its waves walk 32-row units.  The hidden activation never touches LDS either: GEMM1 runs with the
// operands swapped (H^T = W1 Z^T), so a lane ends with hidden units {32j + 4q .. +3} and
// {32j + 16 + 4q .. +3} of row fr -- after bias + GELU these 8 values ARE the lane's B fragment of
// GEMM2's k-step j, provided W2's k order inside each 32-wide step is permuted the same way (done
// once while filling LDS).  GEMM2 is swapped as well (O^T = W2 H^T): each lane ends with 4
// consecutive output channels of one row, so the residual update is 8-byte loads and stores
// straight from the accumulators.  Per row: z read once, x read and written once (6C bytes).
#ifndef MLP_RES_TM
#define MLP_RES_TM 2
#endif
#ifndef MLP_RES_PIPE
#define MLP_RES_PIPE 0  // 1: GEMM1 of step j+1 issued before step j's GELU (measured 34.4 vs 32.7 us at C = 96)
#endif
namespace {
template <int C>
struct ResCfg {
  static constexpr int HID = 4 * C;
  // ds_read_b128 serves a wave in 4 fixed groups of 16 lanes (MI355X_MICROARCH.md §LDS): the 16
  // lanes of a fragment group (rows fr, granules fq) must cover the 64 banks once.  W1 rows padded
  // by 32 B (C + 8 was 2-way: SQ_LDS_BANK_CONFLICT 3.3 per LDS instruction); W2 rows unpadded with
  // the 16-byte granule index XOR'ed by (row & 15) (tools: the bank model in DESIGN.md §3d)
  static constexpr int LD1 = C + 16;   // W1 image [HID][C]
  static constexpr int LD2 = HID;      // W2 image [C][HID]: k permuted per 32-step, granules swizzled
  static constexpr int W1E = HID * LD1;
  static constexpr int W2E = C * LD2;
  static constexpr int SMEM = (W1E + W2E) * 2 + HID * 4;
  static constexpr int KS1 = C / 32;   // GEMM1 k-steps
  static constexpr int NJ = HID / 32;  // GEMM2 k-steps (hidden chunks of 32)
  static constexpr int TN2 = C / 16;   // output-channel fragments
  static constexpr int TM = MLP_RES_TM;  // 16-row slabs per unit
  static constexpr int UR = 16 * TM;   // rows per unit
  static constexpr int WAVES = 8;
  static_assert(SMEM <= 160 * 1024, "LDS budget");
  static_assert(C % 32 == 0 && NJ % 2 == 0, "C");
};
}  // namespace


template <int C>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void cnblock_mlp_res_kernel(
    int M, const bf16* __restrict__ z, const bf16* __restrict__ w1, const float* __restrict__ b1,
    const bf16* __restrict__ w2, const float* __restrict__ b2, const float* __restrict__ gamma,
    const float* __restrict__ sd, int rows_per_sample, const float* __restrict__ lnw,
    const float* __restrict__ lnb, bf16* __restrict__ x) {
  using G = ResCfg<C>;
  extern __shared__ __attribute__((aligned(16))) char smem_dyn[];
  bf16* w1s = (bf16*)smem_dyn;
  bf16* w2s = w1s + G::W1E;
  float* b1s = (float*)(w2s + G::W2E);
  const int lane = threadIdx.x & 63;
  const int fr = lane & 15, fq = lane >> 4;
  const int nunits = (M + G::UR - 1) / G::UR;

  // 32-row units dealt round robin over the waves of the grid.  (A launch-wide counter that
  // waves pull units from measured 92 us against 40 us for this static deal at the Tiny stage-1
  // shape: same-address returning atomics from 2048 waves serialise.)
  const int nw = gridDim.x * G::WAVES;
  int unit = blockIdx.x * G::WAVES + (threadIdx.x >> 6);

  auto load_z = [&](int u, bf16x8 (&zf)[G::TM][G::KS1]) {
#pragma unroll
    for (int tm = 0; tm < G::TM; ++tm) {
      const int row = u * G::UR + tm * 16 + fr;
      const bool ok = row < M;
      const bf16* zp = z + (long)(ok ? row : 0) * C + 8 * fq;
#pragma unroll
      for (int ks = 0; ks < G::KS1; ++ks) {
        const uint4 q = *(const uint4*)(zp + ks * 32);
        zf[tm][ks] = __builtin_bit_cast(bf16x8, ok ? q : make_uint4(0u, 0u, 0u, 0u));
      }
    }
  };
  // the first unit's Z rows requested ahead of the fill, so they land under it
  bf16x8 zf[G::TM][G::KS1];
  if (unit < nunits) load_z(unit, zf);

  // every load of the fill issued before the first LDS store (one memory round trip)
  constexpr int NV = G::HID * C / 8 / 512;
  static_assert(NV * 512 * 8 == G::HID * C, "fill split");
  uint4 f1[NV], f2[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * 512;
    f1[i] = *(const uint4*)(w1 + (long)v * 8);
    f2[i] = *(const uint4*)(w2 + (long)v * 8);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * 512;
    {
      const int r = v / (C / 8), c = (v % (C / 8)) * 8;
      *(uint4*)(w1s + r * G::LD1 + c) = f1[i];
    }
    const int n = v / (G::HID / 8), c = (v % (G::HID / 8)) * 8;
    w2_store_permuted(w2s + n * G::LD2, c, f2[i], n & 15);
  }
  for (int v = threadIdx.x; v < G::HID; v += 512) b1s[v] = b1[v];
  MLP_STAMP(1);
  __syncthreads();
  MLP_STAMP(2);
  int nu = 0;

  // Z fragments of a unit (B operand of GEMM1: column fr = row, k = 32 ks + 8 fq), LayerNorm'd
  while (unit < nunits) {
    // next unit's index and Z rows, and this unit's residual rows, in flight under the MFMAs
    const int next = unit + nw;
    const int r0 = unit * G::UR;
    uint2 xres[G::TM][G::TN2];
#pragma unroll
    for (int tm = 0; tm < G::TM; ++tm) {
      const int row = min(r0 + tm * 16 + fr, M - 1);
#pragma unroll
      for (int tn = 0; tn < G::TN2; ++tn) xres[tm][tn] = *(const uint2*)(x + (long)row * C + tn * 16 + 4 * fq);
    }
    if (lnw) mlp_ln_frags<C, G::TM, G::KS1>(zf, lnw, lnb, fq);
    bf16x8 zc[G::TM][G::KS1];
#pragma unroll
    for (int tm = 0; tm < G::TM; ++tm)
#pragma unroll
      for (int ks = 0; ks < G::KS1; ++ks) zc[tm][ks] = zf[tm][ks];
    if (next < nunits) load_z(next, zf);

    f32x4 acc2[G::TM][G::TN2];
#pragma unroll
    for (int tm = 0; tm < G::TM; ++tm)
#pragma unroll
      for (int tn = 0; tn < G::TN2; ++tn) acc2[tm][tn] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (nu < 4) MLP_STAMP(3 + 3 * nu);

    // GEMM1 (swapped): a1[t][tm] = b1 + W1[32j + 16t + .., :] Z^T -> hidden 32j+16t+4fq+r of row fr
    auto gemm1 = [&](int j, f32x4 (&a1)[2][G::TM]) {
      const f32x4 bb0 = *(const f32x4*)(b1s + 32 * j + 4 * fq);
      const f32x4 bb1 = *(const f32x4*)(b1s + 32 * j + 16 + 4 * fq);
#pragma unroll
      for (int tm = 0; tm < G::TM; ++tm) {
        a1[0][tm] = bb0;
        a1[1][tm] = bb1;
      }
      bf16x8 a[G::KS1][2];  // every fragment requested before the first MFMA (the compiler
                            // otherwise pairs each LDS read with its MFMA and waits it out)
#pragma unroll
      for (int ks = 0; ks < G::KS1; ++ks)
#pragma unroll
        for (int t = 0; t < 2; ++t) a[ks][t] = *(const bf16x8*)(w1s + (32 * j + 16 * t + fr) * G::LD1 + ks * 32 + 8 * fq);
      asm volatile("" ::: "memory");
#pragma unroll
      for (int ks = 0; ks < G::KS1; ++ks)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int tm = 0; tm < G::TM; ++tm)
            a1[t][tm] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[ks][t], zc[tm][ks], a1[t][tm], 0, 0, 0);
    };
    // GELU -> the lane's GEMM2 B fragment (hidden 32j+4fq+{0..3}, 32j+16+4fq+{0..3}), then
    // GEMM2 (swapped): acc2[tm][tn] += W2[16tn + .., step j] H^T -> channels 16tn+4fq+r of row fr
    auto gemm2 = [&](int j, const f32x4 (&a1)[2][G::TM]) {
      bf16x8 hf[G::TM];
#pragma unroll
      for (int tm = 0; tm < G::TM; ++tm)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) hf[tm][4 * t + r] = (bf16)gelu_sig(a1[t][tm][r]);
      bf16x8 a[G::TN2];
#pragma unroll
      for (int tn = 0; tn < G::TN2; ++tn) a[tn] = *(const bf16x8*)(w2s + (tn * 16 + fr) * G::LD2 + 8 * ((4 * j + fq) ^ fr));
      asm volatile("" ::: "memory");
#pragma unroll
      for (int tn = 0; tn < G::TN2; ++tn)
#pragma unroll
        for (int tm = 0; tm < G::TM; ++tm)
          acc2[tm][tn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[tn], hf[tm], acc2[tm][tn], 0, 0, 0);
    };
    // software-pipelined by one step: step j+1's GEMM1 MFMAs are issued before step j's GELU, so
    // the matrix core works under the VALU (a wave's GELU otherwise waits on its own GEMM1)
    f32x4 a1a[2][G::TM], a1b[2][G::TM];
#if MLP_RES_PIPE
    gemm1(0, a1a);
    for (int j = 0; j < G::NJ; j += 2) {
      gemm1(j + 1, a1b);
      gemm2(j, a1a);
      if (j + 2 < G::NJ) gemm1(j + 2, a1a);
      gemm2(j + 1, a1b);
    }
#else
    for (int j = 0; j < G::NJ; ++j) {
      gemm1(j, a1a);
      gemm2(j, a1a);
    }
#endif

    if (nu < 4) MLP_STAMP(4 + 3 * nu);
    // x += gamma * sd * (o + b2): 4 consecutive channels of row fr per fragment
#pragma unroll
    for (int tm = 0; tm < G::TM; ++tm) {
      const int row = r0 + tm * 16 + fr;
      if (row < M) {
        const float s = sd ? sd[row / rows_per_sample] : 1.f;
#pragma unroll
        for (int tn = 0; tn < G::TN2; ++tn) {
          const int c = tn * 16 + 4 * fq;
          const f32x4 g = *(const f32x4*)(gamma + c), bb = *(const f32x4*)(b2 + c);
          const bf16x4 xv = __builtin_bit_cast(bf16x4, xres[tm][tn]);
          bf16x4 o;
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = (bf16)((float)xv[r] + (acc2[tm][tn][r] + bb[r]) * g[r] * s);
          *(bf16x4*)(x + (long)row * C + c) = o;
        }
      }
    }
    if (nu < 4) MLP_STAMP(5 + 3 * nu);
    ++nu;
    unit = next;
  }
  MLP_STAMP(20);
}

// ---- wider stages (C = 128, 192): weights streamed through LDS, hidden chained in registers ----
// W1/W2 (2 * 4C * C bf16: 256 / 576 KB) do not fit in LDS.  One 512-thread workgroup per 128 rows
// (8 waves x one 16-row slab); the hidden dimension is walked in 32-unit steps whose W1 rows and
// (k-permuted) W2 columns pass through a 3-deep LDS ring, loaded two steps ahead into alternating
// register sets, so one barrier per step and a step's load has two steps of compute to land.
// GEMM1 -> GELU -> GEMM2 run on the registers exactly as in the resident kernel above.
namespace {
template <int C>
struct StrCfg {
  static constexpr int HID = 4 * C;
  static constexpr int LD1 = C + 16;  // W1 chunk image [32][C]: rows padded by 32 B (see ResCfg: +16 B was 2-way)
  static constexpr int LD2 = 48;      // W2 chunk image [C][32] (+16): 96-B rows
  static constexpr int STE = 32 * LD1 + C * LD2;  // one ring stage (bf16 elements)
  static constexpr int NS = 3;
  static constexpr int SMEM = NS * STE * 2 + HID * 4;  // + b1 (a global bias load in the loop
                                                        // would wait out every weight load before it)
  static constexpr int KS1 = C / 32;
  static constexpr int NJ = HID / 32;
  static constexpr int TN2 = C / 16;
  static constexpr int WAVES = 8;
  static constexpr int BM = 16 * WAVES;
  static constexpr int NW1 = 32 * C / 8;        // 16-byte W1 vectors per step (as many of W2)
  static constexpr int NV = 2 * NW1 / 512;      // per thread (index v < NW1: W1, else W2)
  static_assert(NV * 512 == 2 * NW1 && NW1 % 512 % 64 == 0, "step split (wave-uniform matrix choice)");
  static_assert(SMEM <= 160 * 1024 && NJ % 2 == 0, "ring");
};
// Branch-free (addresses selected, not code paths): a conditional load or store here makes the
// compiler's vmcnt bookkeeping conservative, and the store of step j + 2 would wait out the loads
// of step j + 3 as well.
template <int C>
DEV void str_load(uint4 (&r)[StrCfg<C>::NV], const bf16* __restrict__ w1, const bf16* __restrict__ w2, int j) {
  using G = StrCfg<C>;
#pragma unroll
  for (int i = 0; i < G::NV; ++i) {
    const int v = threadIdx.x + i * 512, u = v - G::NW1;
    const bf16* p1 = w1 + (long)(32 * j + v / (C / 8)) * C + (v % (C / 8)) * 8;
    const bf16* p2 = w2 + (long)(u / 4) * G::HID + 32 * j + (u % 4) * 8;
    r[i] = *(const uint4*)(v < G::NW1 ? p1 : p2);
  }
}
template <int C>
DEV void str_store(bf16* st, const uint4 (&r)[StrCfg<C>::NV]) {
  using G = StrCfg<C>;
#pragma unroll
  for (int i = 0; i < G::NV; ++i) {
    const int v = threadIdx.x + i * 512, u = v - G::NW1;
    // W1: 8 elements at [h][c]; W2: hidden pieces 2a, 2a+1 of row n to their permuted slots
    const int o1 = (v / (C / 8)) * G::LD1 + (v % (C / 8)) * 8;
    const int p = (u % 4) * 2;  // first 4-element piece of the 8 (within the 32-wide step)
    const int o2 = 32 * G::LD1 + (u / 4) * G::LD2;
    const bool a = v < G::NW1;
    const int lo = a ? o1 : o2 + 8 * (p % 4) + 4 * (p / 4);
    const int hi = a ? o1 + 4 : o2 + 8 * ((p + 1) % 4) + 4 * ((p + 1) / 4);
    *(uint2*)(st + lo) = make_uint2(r[i].x, r[i].y);
    *(uint2*)(st + hi) = make_uint2(r[i].z, r[i].w);
  }
}
}  // namespace

template <int C>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void cnblock_mlp_str_kernel(
    int M, const bf16* __restrict__ z, const bf16* __restrict__ w1, const float* __restrict__ b1,
    const bf16* __restrict__ w2, const float* __restrict__ b2, const float* __restrict__ gamma,
    const float* __restrict__ sd, int rows_per_sample, const float* __restrict__ lnw,
    const float* __restrict__ lnb, bf16* __restrict__ x) {
  using G = StrCfg<C>;
  extern __shared__ __attribute__((aligned(16))) char smem_dyn[];
  bf16* ring = (bf16*)smem_dyn;
  float* b1s = (float*)(ring + G::NS * G::STE);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const int row = blockIdx.x * G::BM + w * 16 + fr;
  for (int v = threadIdx.x; v < G::HID; v += 512) b1s[v] = b1[v];
  const bool ok = row < M;

  uint4 ra[G::NV], rb[G::NV];
  str_load<C>(ra, w1, w2, 0);
  str_load<C>(rb, w1, w2, 1);
  // this wave's slab: Z as GEMM1 B fragments, the residual as 4-channel pieces
  bf16x8 zf[1][G::KS1];
  {
    const bf16* zp = z + (long)(ok ? row : 0) * C + 8 * fq;
#pragma unroll
    for (int ks = 0; ks < G::KS1; ++ks) {
      const uint4 q = *(const uint4*)(zp + ks * 32);
      zf[0][ks] = __builtin_bit_cast(bf16x8, ok ? q : make_uint4(0u, 0u, 0u, 0u));
    }
  }
  uint2 xres[G::TN2];
#pragma unroll
  for (int tn = 0; tn < G::TN2; ++tn) xres[tn] = *(const uint2*)(x + (long)(ok ? row : M - 1) * C + tn * 16 + 4 * fq);
  str_store<C>(ring, ra);
  str_store<C>(ring + G::STE, rb);
  str_load<C>(ra, w1, w2, 2);
  str_load<C>(rb, w1, w2, 3);
  if (lnw) mlp_ln_frags<C, 1, G::KS1>(zf, lnw, lnb, fq);
  __syncthreads();

  f32x4 acc2[G::TN2];
#pragma unroll
  for (int tn = 0; tn < G::TN2; ++tn) acc2[tn] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto gemm1 = [&](int j, f32x4 (&a1)[2]) {
    const bf16* st = ring + (j % G::NS) * G::STE;
    a1[0] = *(const f32x4*)(b1s + 32 * j + 4 * fq);
    a1[1] = *(const f32x4*)(b1s + 32 * j + 16 + 4 * fq);
    bf16x8 a[G::KS1][2];  // every fragment requested before the first MFMA (see the resident kernel)
#pragma unroll
    for (int ks = 0; ks < G::KS1; ++ks)
#pragma unroll
      for (int t = 0; t < 2; ++t) a[ks][t] = *(const bf16x8*)(st + (16 * t + fr) * G::LD1 + ks * 32 + 8 * fq);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int ks = 0; ks < G::KS1; ++ks)
#pragma unroll
      for (int t = 0; t < 2; ++t) a1[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[ks][t], zf[0][ks], a1[t], 0, 0, 0);
  };
  auto gemm2 = [&](int j, const f32x4 (&a1)[2]) {
    bf16x8 hf;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) hf[4 * t + r] = (bf16)gelu_sig(a1[t][r]);
    const bf16* w2c = ring + (j % G::NS) * G::STE + 32 * G::LD1;
    bf16x8 a[G::TN2];
#pragma unroll
    for (int tn = 0; tn < G::TN2; ++tn) a[tn] = *(const bf16x8*)(w2c + (tn * 16 + fr) * G::LD2 + 8 * fq);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int tn = 0; tn < G::TN2; ++tn) acc2[tn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[tn], hf, acc2[tn], 0, 0, 0);
  };
  // Software-pipelined as in the resident kernel: step j+1's GEMM1 (its stage landed before the
  // barrier that closed step j-1) is issued before step j's GELU.  After step j: step j+2 goes
  // into the stage step j-1 used (every wave passed the barrier after it), then step j+4 is
  // requested into the same registers.  The loop body is unconditional (the tail is peeled) so
  // the vmcnt waits count the register sets exactly.
  f32x4 a1a[2], a1b[2];
  gemm1(0, a1a);
  for (int j = 0; j < G::NJ - 4; j += 2) {
    gemm1(j + 1, a1b);
    gemm2(j, a1a);
    str_store<C>(ring + ((j + 2) % G::NS) * G::STE, ra);
    str_load<C>(ra, w1, w2, j + 4);
    __syncthreads();
    gemm1(j + 2, a1a);
    gemm2(j + 1, a1b);
    str_store<C>(ring + ((j + 3) % G::NS) * G::STE, rb);
    str_load<C>(rb, w1, w2, j + 5);
    __syncthreads();
  }
  gemm1(G::NJ - 3, a1b);
  gemm2(G::NJ - 4, a1a);
  str_store<C>(ring + ((G::NJ - 2) % G::NS) * G::STE, ra);
  __syncthreads();
  gemm1(G::NJ - 2, a1a);
  gemm2(G::NJ - 3, a1b);
  str_store<C>(ring + ((G::NJ - 1) % G::NS) * G::STE, rb);
  __syncthreads();
  gemm1(G::NJ - 1, a1b);
  gemm2(G::NJ - 2, a1a);
  gemm2(G::NJ - 1, a1b);

  if (ok) {
    const float s = sd ? sd[row / rows_per_sample] : 1.f;
#pragma unroll
    for (int tn = 0; tn < G::TN2; ++tn) {
      const int c = tn * 16 + 4 * fq;
      const f32x4 g = *(const f32x4*)(gamma + c), bb = *(const f32x4*)(b2 + c);
      const bf16x4 xv = __builtin_bit_cast(bf16x4, xres[tn]);
      bf16x4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (bf16)((float)xv[r] + (acc2[tn][r] + bb[r]) * g[r] * s);
      *(bf16x4*)(x + (long)row * C + c) = o;
    }
  }
}

}  // namespace imgcap

using namespace imgcap;

namespace {
bool mlp_res_enabled() {
  static int v = -1;
  if (v < 0) {
    const char* e = getenv("IMGCAP_MLP_RES");  // A/B switch for kernel benchmarks (default on)
    v = (e && e[0] == '0') ? 0 : 1;
  }
  return v == 1;
}
}  // namespace

extern "C" int imgcap_cnblock_mlp(int M, int C, const void* z, const float* ln_w, const float* ln_b, const void* w1,
                                  const float* b1, const void* w2, const float* b2, const float* gamma, const float* sd,
                                  int rows_per_sample, void* x, void* stream) {
  if (M == 0) return 0;
  IMGCAP_REQUIRE(aligned16(z) && aligned16(w1) && aligned16(w2) && aligned16(x) && aligned16(b1) &&
                     aligned16(b2) && aligned16(gamma),
                 "imgcap_cnblock_mlp: operands must be 16-byte aligned");
  IMGCAP_REQUIRE(sd == nullptr || rows_per_sample > 0, "imgcap_cnblock_mlp: rows_per_sample");
  IMGCAP_REQUIRE((ln_w == nullptr) == (ln_b == nullptr) && (ln_w == nullptr || (aligned16(ln_w) && aligned16(ln_b))),
                 "imgcap_cnblock_mlp: ln_w / ln_b");
  hipStream_t st = (hipStream_t)stream;
  if (C == 96 && mlp_res_enabled()) {
    using G = ResCfg<96>;
    (void)hipFuncSetAttribute((const void*)cnblock_mlp_res_kernel<96>, hipFuncAttributeMaxDynamicSharedMemorySize,
                              G::SMEM);  // per device, so on every call
    int dev = 0;
    IMGCAP_REQUIRE(hipGetDevice(&dev) == hipSuccess && dev >= 0 && dev < 64, "imgcap_cnblock_mlp: device");
    static int ncu_of[64];
    if (!ncu_of[dev]) {
      ncu_of[dev] = 256;
      (void)hipDeviceGetAttribute(&ncu_of[dev], hipDeviceAttributeMultiprocessorCount, dev);
    }
    const int ncu = ncu_of[dev];
    const int units = (M + G::UR - 1) / G::UR;
    const int grid = std::max(1, std::min(ncu, (units + G::WAVES - 1) / G::WAVES));
    hipLaunchKernelGGL(cnblock_mlp_res_kernel<96>, dim3(grid), dim3(512), G::SMEM, st, M, (const bf16*)z,
                       (const bf16*)w1, b1, (const bf16*)w2, b2, gamma, sd, rows_per_sample, ln_w, ln_b, (bf16*)x);
    IMGCAP_CHECK_LAUNCH("imgcap_cnblock_mlp");
    return 0;
  }
  if ((C == 128 || C == 192) && mlp_res_enabled()) {
    auto launch = [&](auto kern, int smem) {
      (void)hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
      hipLaunchKernelGGL(kern, dim3((M + 127) / 128), dim3(512), smem, st, M, (const bf16*)z, (const bf16*)w1, b1,
                         (const bf16*)w2, b2, gamma, sd, rows_per_sample, ln_w, ln_b, (bf16*)x);
    };
    if (C == 128) launch(cnblock_mlp_str_kernel<128>, StrCfg<128>::SMEM);
    else launch(cnblock_mlp_str_kernel<192>, StrCfg<192>::SMEM);
    IMGCAP_CHECK_LAUNCH("imgcap_cnblock_mlp");
    return 0;
  }
#define MLP_(CC, BM, HC, ZL, WPE)                                                                            \
  hipLaunchKernelGGL((cnblock_mlp_kernel<CC, BM, HC, ZL, WPE>), dim3((M + BM - 1) / BM), dim3(256), 0, st, M,         \
                     (const bf16*)z, (const bf16*)w1, b1, (const bf16*)w2, b2, gamma, sd, rows_per_sample, ln_w, \
                     ln_b, (bf16*)x)
  switch (C) {
    case 96: MLP_(96, MLP96_BM, MLP96_HC, false, MLP96_WPE); break;
    case 128: MLP_(128, 128, 64, false, 1); break;
    case 192: MLP_(192, MLP192_BM, MLP192_HC, false, MLP192_WPE); break;
    default: return fail(IMGCAP_EUNSUPPORTED, "imgcap_cnblock_mlp: C must be 96, 128 or 192");
  }
#undef MLP_
  IMGCAP_CHECK_LAUNCH("imgcap_cnblock_mlp");
  return 0;
}
