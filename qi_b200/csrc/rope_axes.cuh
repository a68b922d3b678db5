// Rotary positions with several axes (one for text; frame, height and width
// for video), applied to the q and k columns of a fused projection, and
// optionally the write of the rotated k and of v into a paged cache.
//
// Pair i of a head turns by the angle pos[axis(i)] * freq(i):
//   (x, y) -> (x cos - y sin, x sin + y cos)
// with (x, y) the elements (2i, 2i+1) of the head (INTERLEAVED) or (i, i+P);
// elements from 2P on pass unchanged.
//
// Angles: the turn pos * freq / (2 pi) is formed and reduced to [-1/2, 1/2]
// in 64 bits (an fp32 product is off by up to 2^-24 of the whole angle: 0.06
// rad at position 10^6), and sin / cos of the reduced turn are taken in fp32,
// with a first-order step for what the fp32 turn leaves out.
// They depend on the token and the pair only, so a CTA computes them once for
// its tokens and every head reads them from shared memory; no table per token
// exists in memory.
//
// Bound: HBM, every q / k / v element read once and written once.  A thread
// handles 8 pairs (two 16-byte chunks) at a time; the loads of its first
// units are issued before the angles are computed, which hides their latency.
// Measured: 16384 rows of 32 / 8 heads of 128 into an E4M3 cache 70 us (5.3
// TB/s; 102 us with integer divisions for the places of a unit and unpacked
// arithmetic), 3120 rows of 24 / 24 heads 16.3 us (4.7 TB/s), 64 rows 2.9 us.
// Even / odd pairs take 70 to 77 registers, so three CTAs an SM: the 1,560 CTAs of
// those 3120 rows are 3.5 waves; (i, i + P) pairs take 64, four CTAs.
// A warp per token: 3120 rows 14 us, but the prompt 74 at best; 128, 192, 384 or
// 512 threads or 8 tokens a CTA: the prompt no faster.
// The units whose loads a thread keeps in flight: 2 or 3 the same, 6 slower
// (registers).
//
// Cache rows: token m goes to slot s = slots[m], page s / page_size, place
// s % page_size.  A negative slot writes nothing (a padding row); one behind
// the last page writes nothing and sets the device status word.  E4M3 caches
// hold e4m3_rn(value / scale) with a scale per tensor or per key head.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "dit_fused.cuh"
#include "launch_count.cuh"
#include "quantize_act.cuh"
#include "sm100_ptx.cuh"

namespace qib {

constexpr unsigned int kTagRope = 0x700u;
constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 256;
constexpr int kRopeMaxTokens = 4;  // tokens per CTA
// 32-bit offsets inside a CTA, and exact products with the reciprocals: 4 units^2 < 2^32
constexpr long long kRopeMaxStride = 1ll << 28;
constexpr long long kRopeMaxUnits = 1ll << 15;
constexpr int kRopeAhead = 4;      // units whose loads a thread keeps in flight

struct RopeAxesParams {
  const __nv_bfloat16* in[3];  // q, k, v rows
  long long ld_in[3];
  __nv_bfloat16* out[2];       // q, k (with a cache k's may be nullptr)
  long long ld_out[2];
  int heads, kv_heads, head_dim, pairs, axes;
  const void* pos;             // [axes, M] int32 or int64
  int pos64;
  const double* freq;          // [pairs] radians per position
  const int* axis;             // [pairs]
  int M, tokens;               // tokens per CTA
  unsigned inv_token, inv_units;  // ceil(2^32 / units per token), ceil(2^32 / units per head)
  // cache (element strides; unit stride inside a head)
  void* cache[2];
  long long page_stride[2], slot_stride[2], head_stride[2];
  long long slots_total;       // pages * page_size
  int page_size;
  const void* slots;           // [M] int32 or int64
  int slots64;
  const float* scale[2];       // E4M3: [1] or [kv_heads]
  int scale_per_head[2];
};

__device__ __forceinline__ long long load_index(const void* p, long long i, int is64) {
  return is64 ? static_cast<const long long*>(p)[i] : static_cast<long long>(static_cast<const int*>(p)[i]);
}

// Two E4M3 codes of f / s, the reciprocal of s as a sum hi + lo: the quotient is
// rounded once, so that a value on a code's border falls as the quotient does.
// hi is rounded towards zero and lo positive: a zero keeps its sign, and an
// infinity does not meet a zero.  Not for scales whose reciprocal or its
// residual leaves fp32's normal range.  (Two codes from a bracketed reciprocal
// took 74 us for the prompt above.)
__device__ __forceinline__ uint32_t rope_codes2(float2 f, float hi, float lo) {
  const float2 v = __ffma2_rn(f, make_float2(hi, hi), __fmul2_rn(f, make_float2(lo, lo)));
  return e4m3x2_rn_sat(v.x, v.y);
}

// The codes of a unit whose scale is beyond rope_codes2: one branch a unit (a
// branch at each pair took 4 us more, a call 18).
__device__ __forceinline__ uint4 rope_divided_codes(const float2 (&fa)[4], const float2 (&fb)[4], float s) {
  uint32_t o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 u = e < 2 ? fa[2 * e] : fb[2 * e - 4], v = e < 2 ? fa[2 * e + 1] : fb[2 * e - 3];
    o[e] = e4m3x2_rn_sat(__fdiv_rn(u.x, s), __fdiv_rn(u.y, s)) |
           (e4m3x2_rn_sat(__fdiv_rn(v.x, s), __fdiv_rn(v.y, s)) << 16);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// CACHE: 0 none, 1 bf16, 2 E4M3.
template <bool INTERLEAVED, int CACHE>
__global__ void __launch_bounds__(kRopeThreads) k_rope_axes(const RopeAxesParams p) {
  __shared__ __align__(16) float cs[2][kRopeMaxTokens * kRopeMaxPairs];  // cos, sin
  __shared__ long long row_of[2][kRopeMaxTokens];  // element offset of each token's cache row (K, V), -1: none
  griddep_wait();
  griddep_launch_dependents();
  const int m0 = blockIdx.x * p.tokens;
  const int nt = min(p.tokens, p.M - m0);
  const int U = p.head_dim >> 4;                // units of 16 elements per head
  const int rot = p.pairs >> 3;                 // of them rotated
  const int per_tok = (p.heads + (CACHE ? 2 : 1) * p.kv_heads) * U;
  const int total = nt * per_tok;
  // this CTA's rows; offsets from them fit 32 bits
  const __nv_bfloat16* in_q = p.in[0] + m0 * p.ld_in[0];
  const __nv_bfloat16* in_k = p.in[1] + m0 * p.ld_in[1];
  const __nv_bfloat16* in_v = CACHE ? p.in[2] + m0 * p.ld_in[2] : nullptr;
  const int ld_q = static_cast<int>(p.ld_in[0]), ld_k = static_cast<int>(p.ld_in[1]);
  const int ld_v = CACHE ? static_cast<int>(p.ld_in[2]) : 0;

  struct Where {
    int tok, part, head, a, b, u;  // a, b: element offsets of the unit's two chunks inside the head
  };
  // units run over tokens, then q, k, v heads, then a head's columns; both
  // divisions are products with a rounded-up reciprocal, exact below 2^32 / divisor
  auto where = [&](int i) {
    Where w;
    w.tok = per_tok == 1 ? i : __umulhi(i, p.inv_token);
    const int r = i - w.tok * per_tok;
    int h = U == 1 ? r : __umulhi(r, p.inv_units);
    w.u = r - h * U;
    w.part = 0;
    if (h >= p.heads) {
      h -= p.heads;
      w.part = 1;
      if (CACHE && h >= p.kv_heads) {
        h -= p.kv_heads;
        w.part = 2;
      }
    }
    w.head = h;
    if (!INTERLEAVED && w.part < 2 && w.u < rot) {
      w.a = w.u * 8;
      w.b = p.pairs + w.u * 8;
    } else {
      w.a = w.u * 16;
      w.b = w.a + 8;
    }
    return w;
  };
  auto load = [&](int i, uint4& a, uint4& b) {
    const Where w = where(i);
    const __nv_bfloat16* src = w.part == 0 ? in_q + w.tok * ld_q : (w.part == 1 ? in_k + w.tok * ld_k : in_v + w.tok * ld_v);
    src += w.head * p.head_dim;
    a = *reinterpret_cast<const uint4*>(src + w.a);
    b = *reinterpret_cast<const uint4*>(src + w.b);
  };
  uint4 va[kRopeAhead], vb[kRopeAhead];
#pragma unroll
  for (int n = 0; n < kRopeAhead; ++n) {
    const int i = threadIdx.x + n * kRopeThreads;
    if (i < total) load(i, va[n], vb[n]);
  }

  for (int i = threadIdx.x; i < nt * p.pairs; i += kRopeThreads) {
    const int tok = i / p.pairs, pair = i - tok * p.pairs;  // one or two per thread
    const int ax = p.axis[pair];
    double turn = 0.0;
    if (ax >= 0 && ax < p.axes)
      turn = static_cast<double>(load_index(p.pos, static_cast<long long>(ax) * p.M + m0 + tok, p.pos64)) *
             (p.freq[pair] * 0.15915494309189533577);  // 1 / (2 pi)
    else
      record_error(kDevBadIndex, kTagRope, 1);
    turn -= rint(turn);
    // the half turns as a sum of two floats; sin and cos of the first, turned on by the second
    const double half = 2.0 * turn;
    const float hi = static_cast<float>(half);
    const float lo = static_cast<float>(half - static_cast<double>(hi)) * 3.14159265f;
    float sn, c;
    sincospif(hi, &sn, &c);
    cs[0][i] = fmaf(-sn, lo, c);
    cs[1][i] = fmaf(c, lo, sn);
  }
  if (CACHE && threadIdx.x < nt) {
    long long s = load_index(p.slots, m0 + threadIdx.x, p.slots64);
    if (s >= p.slots_total) {
      record_error(kDevBadIndex, kTagRope, 2);
      s = -1;
    }
    const long long page = s / p.page_size, place = s - page * p.page_size;
#pragma unroll
    for (int c = 0; c < 2; ++c)
      row_of[c][threadIdx.x] = s < 0 ? -1 : page * p.page_stride[c] + place * p.slot_stride[c];
  }
  __syncthreads();

  auto finish = [&](int i, const uint4& a, const uint4& b) {
    const Where w = where(i);
    // x and y of the 8 pairs, two pairs to a register pair
    float2 x[4], y[4];
    if (INTERLEAVED) {
      const uint32_t wa[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = make_float2(__uint_as_float(wa[2 * e] << 16), __uint_as_float(wa[2 * e + 1] << 16));
        y[e] = make_float2(__uint_as_float(wa[2 * e] & 0xffff0000u), __uint_as_float(wa[2 * e + 1] & 0xffff0000u));
      }
    } else {
      unpack8x2(a, x);
      unpack8x2(b, y);
    }
    if (w.part < 2 && w.u < rot) {
      const int at = w.tok * p.pairs + w.u * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 c4 = *reinterpret_cast<const float4*>(cs[0] + at + 4 * h);
        const float4 s4 = *reinterpret_cast<const float4*>(cs[1] + at + 4 * h);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 c = e ? make_float2(c4.z, c4.w) : make_float2(c4.x, c4.y);
          const float2 s = e ? make_float2(s4.z, s4.w) : make_float2(s4.x, s4.y);
          const float2 u = x[2 * h + e], v = y[2 * h + e];
          x[2 * h + e] = __ffma2_rn(u, c, __fmul2_rn(v, make_float2(-s.x, -s.y)));
          y[2 * h + e] = __ffma2_rn(u, s, __fmul2_rn(v, c));
        }
      }
    }
    // back to the two chunks as they lie in memory
    float2 fa[4], fb[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (INTERLEAVED) {
        (e < 2 ? fa : fb)[2 * (e & 1)] = make_float2(x[e].x, y[e].x);
        (e < 2 ? fa : fb)[2 * (e & 1) + 1] = make_float2(x[e].y, y[e].y);
      } else {
        fa[e] = x[e];
        fb[e] = y[e];
      }
    }
    if (w.part == 0 || (w.part == 1 && p.out[1] != nullptr)) {
      __nv_bfloat16* dst = w.part == 0 ? p.out[0] + (m0 + w.tok) * p.ld_out[0] : p.out[1] + (m0 + w.tok) * p.ld_out[1];
      dst += w.head * p.head_dim;
      *reinterpret_cast<uint4*>(dst + w.a) = pack8x2(fa);
      *reinterpret_cast<uint4*>(dst + w.b) = pack8x2(fb);
    }
    if (w.part == 0 || CACHE == 0) return;
    const int c = w.part - 1;
    const long long row = row_of[c][w.tok];
    if (row < 0) return;
    const long long at = row + w.head * (c ? p.head_stride[1] : p.head_stride[0]);
    void* cache = c ? p.cache[1] : p.cache[0];
    if (CACHE == 1) {
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(cache) + at;
      *reinterpret_cast<uint4*>(dst + w.a) = pack8x2(fa);
      *reinterpret_cast<uint4*>(dst + w.b) = pack8x2(fb);
    } else {
      const float s = c ? p.scale[1][p.scale_per_head[1] ? w.head : 0] : p.scale[0][p.scale_per_head[0] ? w.head : 0];
      uint4 o;
      if (__builtin_expect(s > 0x1p-80f && s < 0x1p80f, 1)) {
        const float hi = __frcp_rz(s), lo = fmaxf(fmaf(-hi, s, 1.f), 0x1p-60f) * hi;
        o.x = rope_codes2(fa[0], hi, lo) | (rope_codes2(fa[1], hi, lo) << 16);
        o.y = rope_codes2(fa[2], hi, lo) | (rope_codes2(fa[3], hi, lo) << 16);
        o.z = rope_codes2(fb[0], hi, lo) | (rope_codes2(fb[1], hi, lo) << 16);
        o.w = rope_codes2(fb[2], hi, lo) | (rope_codes2(fb[3], hi, lo) << 16);
      } else {
        o = rope_divided_codes(fa, fb, s);
      }
      uint8_t* dst = static_cast<uint8_t*>(cache) + at;
      *reinterpret_cast<uint2*>(dst + w.a) = make_uint2(o.x, o.y);
      *reinterpret_cast<uint2*>(dst + w.b) = make_uint2(o.z, o.w);
    }
  };
#pragma unroll
  for (int n = 0; n < kRopeAhead; ++n) {
    const int i = threadIdx.x + n * kRopeThreads;
    if (i < total) finish(i, va[n], vb[n]);
  }
  for (int i = threadIdx.x + kRopeAhead * kRopeThreads; i < total; i += kRopeThreads) {
    uint4 a, b;
    load(i, a, b);
    finish(i, a, b);
  }
}

}  // namespace qib
