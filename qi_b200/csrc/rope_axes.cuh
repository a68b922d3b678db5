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
// rad at position 10^6), and sin / cos of the reduced turn are taken in fp32.
// They depend on the token and the pair only, so a CTA computes them once for
// its tokens and every head reads them from shared memory; no table per token
// exists in memory.
//
// Bound: HBM, every q / k / v element read once and written once.  A thread
// handles 8 pairs (two 16-byte chunks) at a time; the loads of its first
// units are issued before the angles are computed, which hides their latency.
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

// CACHE: 0 none, 1 bf16, 2 E4M3.
template <bool INTERLEAVED, int CACHE>
__global__ void __launch_bounds__(kRopeThreads) k_rope_axes(const RopeAxesParams p) {
  __shared__ float2 cs[kRopeMaxTokens * kRopeMaxPairs];
  __shared__ long long row_of[kRopeMaxTokens];  // cache slot of each token, -1 to write nothing
  griddep_wait();
  griddep_launch_dependents();
  const int m0 = blockIdx.x * p.tokens;
  const int nt = min(p.tokens, p.M - m0);
  const int U = p.head_dim >> 4;                // units of 16 elements per head
  const int rot = p.pairs >> 3;                 // of them rotated
  const int per_tok = (p.heads + (CACHE ? 2 : 1) * p.kv_heads) * U;
  const int total = nt * per_tok;

  struct Where {
    int tok, part, head, a, b, u;  // a, b: element offsets of the unit's two chunks inside the head
  };
  auto where = [&](int i) {
    Where w;
    w.tok = i / per_tok;
    const int r = i - w.tok * per_tok;
    int h = r / U;
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
    const __nv_bfloat16* src =
        p.in[w.part] + static_cast<long long>(m0 + w.tok) * p.ld_in[w.part] + w.head * p.head_dim;
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
    const int tok = i / p.pairs, pair = i - tok * p.pairs;
    const int ax = p.axis[pair];
    double turn = 0.0;
    if (ax >= 0 && ax < p.axes)
      turn = static_cast<double>(load_index(p.pos, static_cast<long long>(ax) * p.M + m0 + tok, p.pos64)) *
             (p.freq[pair] * 0.15915494309189533577);  // 1 / (2 pi)
    else
      record_error(kDevBadIndex, kTagRope, 1);
    turn -= rint(turn);
    float sn, c;
    sincospif(2.0f * static_cast<float>(turn), &sn, &c);
    cs[i] = make_float2(c, sn);
  }
  if (CACHE && threadIdx.x < nt) {
    long long s = load_index(p.slots, m0 + threadIdx.x, p.slots64);
    if (s >= p.slots_total) {
      record_error(kDevBadIndex, kTagRope, 2);
      s = -1;
    }
    row_of[threadIdx.x] = s;
  }
  __syncthreads();

  auto finish = [&](int i, const uint4& a, const uint4& b) {
    const Where w = where(i);
    float fa[8], fb[8];
    unpack8(a, fa);
    unpack8(b, fb);
    if (w.part < 2 && w.u < rot) {
      const float2* t = cs + w.tok * p.pairs + w.u * 8;
      if (INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float* f = e < 4 ? fa : fb;
          const int k = 2 * (e & 3);
          const float2 v = t[e];
          const float x = f[k], y = f[k + 1];
          f[k] = fmaf(x, v.x, -(y * v.y));
          f[k + 1] = fmaf(x, v.y, y * v.x);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 v = t[e];
          const float x = fa[e], y = fb[e];
          fa[e] = fmaf(x, v.x, -(y * v.y));
          fb[e] = fmaf(x, v.y, y * v.x);
        }
      }
    }
    if (w.part == 0 || (w.part == 1 && p.out[1] != nullptr)) {
      __nv_bfloat16* dst =
          p.out[w.part] + static_cast<long long>(m0 + w.tok) * p.ld_out[w.part] + w.head * p.head_dim;
      *reinterpret_cast<uint4*>(dst + w.a) = pack8(fa);
      *reinterpret_cast<uint4*>(dst + w.b) = pack8(fb);
    }
    if (w.part == 0 || CACHE == 0) return;
    const long long slot = row_of[w.tok];
    if (slot < 0) return;
    const int c = w.part - 1;
    const long long page = slot / p.page_size;
    const long long at = page * p.page_stride[c] + (slot - page * p.page_size) * p.slot_stride[c] +
                         w.head * p.head_stride[c];
    if (CACHE == 1) {
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.cache[c]) + at;
      *reinterpret_cast<uint4*>(dst + w.a) = pack8(fa);
      *reinterpret_cast<uint4*>(dst + w.b) = pack8(fb);
    } else {
      const float s = p.scale[c][p.scale_per_head[c] ? w.head : 0];
      const float r = QuantFp8::aux(s);
      auto codes = [&](const float (&f)[8]) {
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = QuantFp8::q2(make_float2(f[2 * e], f[2 * e + 1]), s, r);
        return make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
      };
      uint8_t* dst = static_cast<uint8_t*>(p.cache[c]) + at;
      *reinterpret_cast<uint2*>(dst + w.a) = codes(fa);
      *reinterpret_cast<uint2*>(dst + w.b) = codes(fb);
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
