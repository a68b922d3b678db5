// Residual addition + RMSNorm + 8-bit quantization of whole rows, in one pass:
//   h  <- bf16(x + y)                 (stored; without y, h = x)
//   v  <- h * w / sqrt(mean(h^2) + eps)
//   INT8: s = max(max|v| / 127, 1e-10), q = clamp(rint(v / s), -127, 127)
//   E4M3: s = max(max|v| / 448, 1e-12), q = e4m3_rn(v / s), saturating
// and optionally v rounded to bf16.  The one rounding to fewer bits before the
// codes is that of h, which is the residual stream's own type: the row that is
// normalized is the row that is stored.  v itself stays in fp32.
//
// Mathematics: with r = 1 / sqrt(mean(h^2) + eps), v = (h w) r and
// max|v| = r max|h w|, so sum(h^2) and max|h w| come out of ONE reduction over
// the row.  Where s is not its floor, r cancels from v / s: the quotient is
// (h w) k with k = 127 / max|h w| (448 for E4M3); h w and the maximum are exact
// in fp32 (16 bits).  k is held as k_hi + k_lo, and the code is that of
// fma(h w, k_hi, (h w) k_lo), the quotient rounded once: codes fall as those of
// exact arithmetic do, ties included (the product (h w) (r / s) tipped one in
// 10^5, for one packed operation per two elements less, 1 % of the time of 16384 x 8192).
//
// Bound: HBM, 2 D in (+ 2 D of y), D codes out (+ 2 D of h) per row; 16384 x 8192
// with residual 145 us in bursts, 159 in loops of a thousand calls and more.
// A row lives in the registers of T threads (16-byte chunks, C per thread)
// between the reduction and the codes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "dit_fused.cuh"
#include "launch_count.cuh"
#include "quantize_act.cuh"
#include "quantize_nvfp4.cuh"

namespace qib {

constexpr int kRmsMaxDim = 16384;

struct RmsQuantParams {
  const __nv_bfloat16* x;  // [M, ldx]
  long long ldx;
  const __nv_bfloat16* y;  // [M, ldy] or nullptr
  long long ldy;
  __nv_bfloat16* h;        // [M, ldh] where x + y goes (may be x), used with y
  long long ldh;
  const __nv_bfloat16* w;  // [D]
  uint8_t* q;              // [M, D] codes, or nullptr
  float* s;                // [M] (with q)
  __nv_bfloat16* xn;       // [M, D] or nullptr
  int M, D;
  float eps;
};

// Four codes of t = v / s (INT8: |t| <= 127 up to rounding).
template <bool FP8>
__device__ __forceinline__ uint32_t rms_codes4(float a, float b, float c, float d) {
  if constexpr (FP8) {
    return e4m3x2_rn_sat(a, b) | (e4m3x2_rn_sat(c, d) << 16);
  } else {
    auto code = [](float t) {
      return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(t)))) & 0xFFu;
    };
    return code(a) | (code(b) << 8) | (code(c) << 16) | (code(d) << 24);
  }
}

// The larger one; NaN where either is one (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// T threads per row (whole warps, at most 512), blockDim.x / T rows per CTA,
// C chunks of 8 elements per thread.  FMT: 0 bf16 only, 1 INT8, 2 E4M3.
template <int C, int FMT>
__global__ void __launch_bounds__(512) k_rms_quant(const RmsQuantParams p, int T) {
  __shared__ float2 red[16];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = threadIdx.x % T;
  const int row = blockIdx.x * (blockDim.x / T) + threadIdx.x / T;
  const bool live = row < p.M;
  const int nvec = p.D >> 3;
  const uint4* xr = reinterpret_cast<const uint4*>(p.x + (live ? row : 0) * p.ldx);
  const uint4* yr = p.y == nullptr ? nullptr : reinterpret_cast<const uint4*>(p.y + (live ? row : 0) * p.ldy);
  const uint4* wr = reinterpret_cast<const uint4*>(p.w);

  uint4 hv[C], yv[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int j = c * T + t;
    hv[c] = yv[c] = make_uint4(0u, 0u, 0u, 0u);
    if (live && j < nvec) {
      hv[c] = xr[j];
      if (yr != nullptr) yv[c] = yr[j];
    }
  }
  float ss = 0.f, mx = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int j = c * T + t;
    if (!live || j >= nvec) continue;
    float2 f[4];
    unpack8x2(hv[c], f);
    if (yr != nullptr) {
      float2 g[4];
      unpack8x2(yv[c], g);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = round2(__fadd2_rn(f[e], g[e]));
      hv[c] = pack8x2_exact(f);
      reinterpret_cast<uint4*>(p.h + row * p.ldh)[j] = hv[c];
    }
    float2 w[4];
    unpack8x2(wr[j], w);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ss = fmaf(f[e].x, f[e].x, ss);
      ss = fmaf(f[e].y, f[e].y, ss);
      mx = max_nan(mx, max_nan(fabsf(f[e].x * w[e].x), fabsf(f[e].y * w[e].y)));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (T > 32) {
    if (lane == 0) red[warp] = make_float2(ss, mx);
    __syncthreads();
    const int w0 = threadIdx.x / T * (T >> 5);
    ss = 0.f;
    for (int w = 0; w < (T >> 5); ++w) {
      const float2 v = red[w0 + w];
      ss += v.x;
      mx = max_nan(mx, v.y);
    }
  }
  const float r = rsqrtf(ss / static_cast<float>(p.D) + p.eps);
  // a row with an infinity or NaN, its own or the weight's, has no scale: NaN (h w is one
  // of the two wherever h or w is), and so has one whose sum of squares or product is
  // beyond fp32
  constexpr float kInf = __builtin_huge_valf();
  const float amax = ss < kInf && mx < kInf ? mx * r : __int_as_float(0x7fffffff);
  float s = 1.f;
  if (FMT == 1) s = amax == amax ? fmaxf(__fdiv_rn(amax, 127.0f), 1e-10f) : amax;
  if (FMT == 2) s = amax == amax ? fmaxf(__fdiv_rn(amax, 448.0f), 1e-12f) : amax;
  // v / s = (h w) (k_hi + k_lo).  k_hi lies below k by 2^-22 to 2^-20 of it, more
  // than the reciprocal's error, so k_lo is positive and a zero keeps its sign; the
  // residual is exact (20 bits), and the sum is right to 2^-40 of k
  constexpr float kTop = FMT == 1 ? 127.f : 448.f, kFloor = FMT == 1 ? 1e-10f : 1e-12f;
  const float inv = rcp_approx(mx);
  float k_hi = inv * (kTop - kTop * 0x1p-21f);
  float k_lo = fmaf(-k_hi, mx, kTop) * inv;
  if (!(amax >= kFloor * kTop && mx > 0x1p-80f && mx < 0x1p80f)) {  // s is its floor, or the row has none
    k_hi = __fdiv_rn(r, s);
    k_lo = 0.f;
  }
  if (FMT != 0 && live && t == 0) p.s[row] = s;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int j = c * T + t;
    if (!live || j >= nvec) continue;
    float2 f[4], w[4];
    unpack8x2(hv[c], f);
    unpack8x2(wr[j], w);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __fmul2_rn(f[e], w[e]);
    if (FMT != 0) {
      float2 v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = __ffma2_rn(f[e], make_float2(k_hi, k_hi), __fmul2_rn(f[e], make_float2(k_lo, k_lo)));
      reinterpret_cast<uint2*>(p.q + static_cast<long long>(row) * p.D)[j] =
          make_uint2(rms_codes4<FMT == 2>(v[0].x, v[0].y, v[1].x, v[1].y),
                     rms_codes4<FMT == 2>(v[2].x, v[2].y, v[3].x, v[3].y));
    }
    if (p.xn != nullptr) {
      const float2 r2 = make_float2(r, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = __fmul2_rn(f[e], r2);
      reinterpret_cast<uint4*>(p.xn + static_cast<long long>(row) * p.D)[j] = pack8x2(f);
    }
  }
}

}  // namespace qib
