// Attention of one new token per sequence over a paged key-value cache:
//   o_b = softmax(scale q_b K_b^T) V_b   per head, grouped heads,
// K_b, V_b being the first lengths[b] rows that the page table of sequence b
// names.  Bound: HBM, every cached row is read once and serves all query
// heads of its key head.
//
// Split: the work of all (sequence, key head, chunk of 16 query heads) items,
// counted in units of kPagedUnit tokens, is laid end to end and cut into
// gridDim.x equal ranges, one per CTA, so every SM streams the same number of
// bytes whatever the lengths are.  An item inside one range is finished there;
// an item cut by range borders leaves partial results (row maximum, sum,
// unnormalized output, all fp32) in the workspace, which k_attn_paged_join
// adds up in range order: the result does not depend on timing.
//
// Inside a CTA the warps take blocks of the range in turn.  Each warp runs
// its own ring of cp.async stages (no barrier between warps while it streams)
// and its own running softmax: S = Q K^T and O += P V with mma.sync m16n8k16,
// the query heads of the item as the 16 rows.  The tensor work is a few
// per cent of what the SM can do, so the legacy instruction is enough; what
// counts are the bytes in flight (8 warps x 2 stages x 8 KB per SM).
//
// E4M3 caches: codes are widened exactly to fp16 and multiplied in fp16 with
// fp32 sums; q is scaled by a power of two per row so that it fits fp16, the
// key scale goes into the softmax scale and the value scale into the output.
//
// A page index outside the cache, or a length behind the page table, reads
// nothing: those keys take no part, and the device status word is set.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "attn_short.cuh"
#include "launch_count.cuh"
#include "sm100_ptx.cuh"

namespace qib {

constexpr unsigned int kTagPaged = 0x800u;
constexpr int kPagedUnit = 64;      // tokens per unit of work
constexpr int kPagedWarps = 8;
constexpr int kPagedRows = 16;      // query heads per item
constexpr int kPagedStageBytes = 8192;

struct PagedParams {
  const __nv_bfloat16* q;
  long long ldq;
  const uint8_t* cache[2];                 // K, V
  long long page_stride[2], slot_stride[2], head_stride[2];  // bytes
  const int* pages;                        // [B, ld_pages]
  long long ld_pages;
  const int* lengths;                      // [B]
  __nv_bfloat16* out;
  long long ldo;
  float* lse;                              // [B, heads] or nullptr
  float* ws;
  const float* scale[2];                   // E4M3: k_scale, v_scale, [1] or [kv_heads]
  int scale_per_head[2];
  int B, heads, kv_heads, group, chunks;   // chunks of kPagedRows query heads per key head
  int page_size, max_pages, num_pages;
  float scale_log2e;
};

// Floats of one partial result: maxima, sums, output rows.
template <int D>
__host__ __device__ constexpr int paged_part_floats() { return kPagedRows * (D + 2); }

__device__ __forceinline__ int paged_length(const PagedParams& p, int b) {
  const int n = p.lengths[b];
  const long long most = static_cast<long long>(p.max_pages) * p.page_size;
  if (n > most) {
    record_error(kDevBadIndex, kTagPaged, 1);
    return static_cast<int>(most);
  }
  return n < 0 ? 0 : n;
}
__device__ __forceinline__ int paged_units(int len) { return (len + kPagedUnit - 1) / kPagedUnit; }

// Ranges that T units are cut into: none of them is empty, so the partial
// results of an item are those of consecutive CTAs.
__device__ __forceinline__ long long paged_ranges(long long T, int ctas) { return T < ctas ? T : ctas; }

// CTA whose range [c T / G, (c + 1) T / G) holds unit u.
__device__ __forceinline__ int paged_owner(long long u, long long T, long long G) {
  return static_cast<int>(((u + 1) * G - 1) / T);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two E4M3 codes (low 16 bits) -> two fp16, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(v)));
  return r;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <int D, bool FP8>
struct PagedCfg {
  static constexpr int ELT = FP8 ? 1 : 2;
  static constexpr int ROW = D * ELT;                       // bytes of one cached head row
  static constexpr int BT = kPagedStageBytes / (2 * ROW);   // tokens per block: 16 ... 64
  static constexpr int CH = ROW / 16;                       // 16-byte chunks per row: 4, 8 or 16
  static constexpr int STAGES = 3;
  static constexpr int THREADS = kPagedWarps * 32;
  static constexpr int RING = kPagedWarps * STAGES * kPagedStageBytes;
  static constexpr int MERGE = kPagedWarps * kPagedRows * (D + 2) * 4;
  static constexpr int SMEM = (RING > MERGE ? RING : MERGE) + 256;
  // byte offset of chunk c of row r: 128-byte lines whose 16-byte chunks are
  // permuted so that the 8 rows ldmatrix reads at once hit 8 different chunks
  __device__ static __forceinline__ uint32_t at(int r, int c) {
    if constexpr (CH >= 8) return r * ROW + ((c ^ (r & 7)) << 4);
    else return r * ROW + ((c ^ ((r >> 1) & 3)) << 4);
  }
};

// ROWS8: at most 8 query heads per item (rows 8-15 of the MMA are zero).
template <int D, bool FP8, bool ROWS8>
__global__ void __launch_bounds__(kPagedWarps * 32, 1) k_attn_paged(const PagedParams p) {
  using C = PagedCfg<D, FP8>;
  constexpr int BT = C::BT, ST = C::STAGES;
  constexpr int NT = D / 8;        // output column tiles
  constexpr int NR = ROWS8 ? 1 : 2;
  extern __shared__ __align__(128) uint8_t paged_sm[];
  __shared__ long long scan[kPagedWarps];
  __shared__ int start_b;
  __shared__ long long start_u;
  __shared__ uint32_t masks[kPagedWarps][ST][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_wait();
  griddep_launch_dependents();

  // the range of this CTA and the sequence it starts in
  const long long per_unit = static_cast<long long>(p.kv_heads) * p.chunks;
  const int per_thread = (p.B + C::THREADS - 1) / C::THREADS;
  const int b_lo = min(p.B, tid * per_thread), b_hi = min(p.B, b_lo + per_thread);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += paged_units(paged_length(p, b)) * per_unit;
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  long long T = 0, before = 0;
#pragma unroll
  for (int w = 0; w < kPagedWarps; ++w) {
    if (w < warp) before += scan[w];
    T += scan[w];
  }
  if (T == 0) return;
  const long long G = paged_ranges(T, gridDim.x);
  long long u = T * blockIdx.x / G;
  const long long u_end = blockIdx.x < G ? T * (blockIdx.x + 1) / G : u;
  before += incl - mine;
  if (u < u_end && before <= u && u < before + mine) {
    long long at = before;
    for (int b = b_lo; b < b_hi; ++b) {
      const long long n = paged_units(paged_length(p, b)) * per_unit;
      if (u < at + n) {
        start_b = b;
        start_u = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  if (u >= u_end) return;
  int b = start_b;
  long long b_first = start_u;  // first unit of sequence b
  uint8_t* ring = paged_sm + warp * ST * kPagedStageBytes;
  const uint32_t ring_u = smem_u32(ring);
  const int g = lane >> 2, t4 = lane & 3;

  while (u < u_end) {
    int len = paged_length(p, b);
    int n_units = paged_units(len);
    while (u >= b_first + n_units * per_unit) {  // next sequence with keys
      b_first += n_units * per_unit;
      ++b;
      len = paged_length(p, b);
      n_units = paged_units(len);
    }
    const long long rel = u - b_first;
    const int item = static_cast<int>(rel / n_units);           // key head and chunk
    const int unit0 = static_cast<int>(rel - static_cast<long long>(item) * n_units);
    const int unit1 = static_cast<int>(min(static_cast<long long>(n_units), unit0 + (u_end - u)));
    const int kvh = item / p.chunks, chunk = item - kvh * p.chunks;
    const int head0 = kvh * p.group + chunk * kPagedRows;
    const int rows = min(kPagedRows, p.group - chunk * kPagedRows);
    const int tok0 = unit0 * kPagedUnit, tok1 = min(len, unit1 * kPagedUnit);
    u += unit1 - unit0;

    // Q as the A operand, rows g and g + 8
    uint32_t qa[D / 16][4];
    float row_scale[2] = {1.f, 1.f};
    {
      float qmax[2] = {0.f, 0.f};
      uint32_t raw[D / 16][4];
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v = 0;
            if (r < NR && g + 8 * r < rows) {
              // fp16 path: the thread's 4 columns of a 16-column step are consecutive (as its 4 codes of K are)
              const int col = ks * 16 + (FP8 ? 4 * t4 + 2 * h : 2 * t4 + 8 * h);
              v = *reinterpret_cast<const uint32_t*>(p.q + static_cast<long long>(b) * p.ldq +
                                                     static_cast<long long>(head0 + g + 8 * r) * D + col);
            }
            raw[ks][r + 2 * h] = v;
            if (FP8) {
              const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
              qmax[r] = fmaxf(qmax[r], fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          }
      if (FP8) {
        float down[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          qmax[r] = fmaxf(qmax[r], __shfl_xor_sync(0xffffffffu, qmax[r], 1));
          qmax[r] = fmaxf(qmax[r], __shfl_xor_sync(0xffffffffu, qmax[r], 2));
          // 2^e with e the exponent of the row's largest element, kept so that 2^-e is a normal number
          int e = static_cast<int>(__float_as_uint(qmax[r]) >> 23) - 127;
          e = max(-100, min(100, e));
          row_scale[r] = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
          down[r] = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        }
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks][i]));
            qa[ks][i] = pack_pair<true>(f.x * down[i & 1], f.y * down[i & 1]);
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int i = 0; i < 4; ++i) qa[ks][i] = raw[ks][i];
      }
    }
    float sl2[2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      sl2[r] = p.scale_log2e * (FP8 ? row_scale[r] * p.scale[0][p.scale_per_head[0] ? kvh : 0] : 1.f);

    // this warp's blocks: tok0 + (warp + i * kPagedWarps) * BT
    const int n_blocks = (tok1 - tok0 + BT - 1) / BT;
    const int my_blocks = n_blocks > warp ? (n_blocks - warp - 1) / kPagedWarps + 1 : 0;
    const int* pg = p.pages + static_cast<long long>(b) * p.ld_pages;
    auto issue = [&](int i) {
      const int st = i % ST;
      const int t0 = tok0 + (warp + i * kPagedWarps) * BT;
#pragma unroll
      for (int half = 0; half < (BT + 31) / 32; ++half) {
        constexpr int R = BT < 32 ? BT : 32;  // rows whose addresses the lanes look up at once
        const int tok = t0 + half * 32 + (lane % R);
        long long off[2] = {0, 0};
        bool ok = tok < tok1;
        if (ok) {
          const int pi = tok / p.page_size, place = tok - pi * p.page_size;
          const int page = pg[pi];
          if (page < 0 || page >= p.num_pages) {
            record_error(kDevBadIndex, kTagPaged, 2);
            ok = false;
          } else {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              off[c] = page * p.page_stride[c] + place * p.slot_stride[c] + kvh * p.head_stride[c];
          }
        }
        const uint32_t m = __ballot_sync(0xffffffffu, ok);
        if (lane == 0) masks[warp][st][half] = BT < 32 ? (m & ((1u << (BT & 31)) - 1u)) : m;
        constexpr int RPI = 32 / C::CH;       // rows copied per instruction
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i2 = 0; i2 < R / RPI; ++i2) {
            const int r = i2 * RPI + lane / C::CH, ch = lane % C::CH;
            const long long o = __shfl_sync(0xffffffffu, off[c], r);
            cp_async16(ring_u + st * kPagedStageBytes + c * (kPagedStageBytes / 2) + C::at(half * 32 + r, ch),
                       p.cache[c] + o + ch * 16, (m >> r) & 1u);
          }
      }
    };

    float o[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      if (i < my_blocks) issue(i);
      cp_async_commit();
    }
#pragma unroll 1
    for (int i = 0; i < my_blocks; ++i) {
      __syncwarp();  // every lane has read stage (i - 1) % ST, which is filled next
      if (i + ST - 1 < my_blocks) issue(i + ST - 1);
      cp_async_commit();
      cp_async_wait<ST - 1>();
      __syncwarp();
      const uint32_t sk = ring_u + (i % ST) * kPagedStageBytes, sv = sk + kPagedStageBytes / 2;

      // S = Q K^T, 8 tokens per tile
      float s[BT / 8][4];
#pragma unroll
      for (int n = 0; n < BT / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = 0.f;
      if constexpr (!FP8) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int n = 0; n < BT / 16; ++n) {
            uint32_t k[4];  // (tokens 0-7, 8-15) x (dims 0-7, 8-15)
            ldsm_x4(k, sk + C::at(n * 16 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
            mma_16816<false>(s[2 * n], qa[ks], k[0], k[1]);
            mma_16816<false>(s[2 * n + 1], qa[ks], k[2], k[3]);
          }
      } else {
#pragma unroll
        for (int kg = 0; kg < D / 32; ++kg)
#pragma unroll
          for (int n = 0; n < BT / 16; ++n) {
            uint32_t k[4];  // (tokens 0-7, 8-15) x (dims 0-15, 16-31), 4 codes per register
            ldsm_x4(k, sk + C::at(n * 16 + (lane & 7) + ((lane >> 4) << 3), kg * 2 + ((lane >> 3) & 1)));
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mma_16816<true>(s[2 * n + (j >> 1)], qa[kg * 2 + (j & 1)], e4m3x2_to_half2(k[j]),
                              e4m3x2_to_half2(k[j] >> 16));
          }
      }

      // running softmax, in powers of two
      float nm[2] = {mx[0], mx[1]};
      uint32_t mk[2] = {masks[warp][i % ST][0], BT > 32 ? masks[warp][i % ST][1] : 0u};
#pragma unroll
      for (int n = 0; n < BT / 8; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int tok = n * 8 + 2 * t4 + j;
          const bool ok = (mk[tok >> 5] >> (tok & 31)) & 1u;
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const float v = ok ? s[n][2 * r + j] * sl2[r] : -INFINITY;
            s[n][2 * r + j] = v;
            nm[r] = fmaxf(nm[r], v);
          }
        }
      bool grew = false;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        nm[r] = fmaxf(nm[r], __shfl_xor_sync(0xffffffffu, nm[r], 1));
        nm[r] = fmaxf(nm[r], __shfl_xor_sync(0xffffffffu, nm[r], 2));
        grew |= nm[r] > mx[r];
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float f = nm[r] > mx[r] ? ex2_approx(mx[r] - nm[r]) : 1.f;  // 2^-inf = 0: nothing summed yet
          mx[r] = nm[r];
          sum[r] *= f;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            o[n][2 * r] *= f;
            o[n][2 * r + 1] *= f;
          }
        }
      }
      uint32_t pa[BT / 16][4];
#pragma unroll
      for (int n = 0; n < BT / 8; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint32_t v = 0;
          if (r < NR) {
            const float base = mx[r] == -INFINITY ? 0.f : mx[r];
            const float e0 = ex2_approx(s[n][2 * r] - base), e1 = ex2_approx(s[n][2 * r + 1] - base);
            sum[r] += e0 + e1;
            v = pack_pair<FP8>(e0, e1);
          }
          pa[n >> 1][(n & 1) * 2 + r] = v;
        }

      // O += P V
      if constexpr (!FP8) {
#pragma unroll
        for (int ks = 0; ks < BT / 16; ++ks)
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            uint32_t v[4];  // (tokens 0-7, 8-15) x (dims 0-7, 8-15), transposed
            ldsm_x4_t(v, sv + C::at(ks * 16 + (lane & 15), n * 2 + (lane >> 4)));
            mma_16816<false>(o[2 * n], pa[ks], v[0], v[1]);
            mma_16816<false>(o[2 * n + 1], pa[ks], v[2], v[3]);
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < BT / 16; ++ks)
#pragma unroll
          for (int n = 0; n < D / 32; ++n) {
            uint32_t v[4];  // (tokens 0-7, 8-15) x (dims 0-15, 16-31); a register: 2 tokens x 2 dims
            ldsm_x4_t(v, sv + C::at(ks * 16 + (lane & 15), n * 2 + (lane >> 4)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // even dims (bytes 0, 2) and odd dims (bytes 1, 3) of the 16 make one column tile each
              mma_16816<true>(o[4 * n + 2 * h], pa[ks], e4m3x2_to_half2(__byte_perm(v[2 * h], 0, 0x4420)),
                              e4m3x2_to_half2(__byte_perm(v[2 * h + 1], 0, 0x4420)));
              mma_16816<true>(o[4 * n + 2 * h + 1], pa[ks], e4m3x2_to_half2(__byte_perm(v[2 * h], 0, 0x4431)),
                              e4m3x2_to_half2(__byte_perm(v[2 * h + 1], 0, 0x4431)));
            }
          }
      }
    }
    cp_async_wait<0>();
    __syncthreads();  // the rings are free: they take the warps' results

    // the warps' results -> shared memory: maxima, sums, rows
    float* mg = reinterpret_cast<float*>(paged_sm);
    float* mg_m = mg + kPagedWarps * kPagedRows * D;
    float* mg_l = mg_m + kPagedWarps * kPagedRows;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      const int row = g + 8 * r;
      if (t4 == 0) {
        mg_m[warp * kPagedRows + row] = mx[r];
        mg_l[warp * kPagedRows + row] = sum[r];
      }
      float* dst = mg + (warp * kPagedRows + row) * D;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if constexpr (!FP8) {
          *reinterpret_cast<float2*>(dst + n * 8 + 2 * t4) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
        } else {
          const int d0 = (n >> 1) * 16 + 4 * t4 + (n & 1);  // column tiles hold the even or the odd dims of 16
          dst[d0] = o[n][2 * r];
          dst[d0 + 2] = o[n][2 * r + 1];
        }
      }
    }
    __syncthreads();
    const bool whole = unit0 == 0 && unit1 == n_units;
    float* part = p.ws + (2ll * blockIdx.x + (unit0 == 0 ? 1 : 0)) * paged_part_floats<D>();
    const float v_scale = FP8 ? p.scale[1][p.scale_per_head[1] ? kvh : 0] : 1.f;
    for (int i = tid; i < rows * (D / 2); i += C::THREADS) {
      const int row = i / (D / 2), d = (i - row * (D / 2)) * 2;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) m = fmaxf(m, mg_m[w * kPagedRows + row]);
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      float2 acc = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) {
        const float f = ex2_approx(mg_m[w * kPagedRows + row] - base);
        l = fmaf(mg_l[w * kPagedRows + row], f, l);
        const float2 v = *reinterpret_cast<const float2*>(mg + (w * kPagedRows + row) * D + d);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
      }
      if (whole) {
        const float inv = l > 0.f ? v_scale / l : 0.f;
        *reinterpret_cast<__nv_bfloat162*>(p.out + static_cast<long long>(b) * p.ldo +
                                           static_cast<long long>(head0 + row) * D + d) =
            __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
        if (p.lse != nullptr && d == 0)
          p.lse[static_cast<long long>(b) * p.heads + head0 + row] = (m + log2f(l)) * 0.69314718055994531f;
      } else {
        if (d == 0) {
          part[row] = m;
          part[kPagedRows + row] = l;
        }
        *reinterpret_cast<float2*>(part + 2 * kPagedRows + row * D + d) = make_float2(acc.x * v_scale, acc.y * v_scale);
      }
    }
    __syncthreads();  // the rings are filled again for the next item
  }
}

// Adds up the partial results of the items that were cut, and writes the rows
// of sequences without keys (zeros).  One CTA per (sequence, query head), one
// thread per two columns; ctas is the first kernel's grid.
template <int D>
__global__ void __launch_bounds__(D / 2 < 32 ? 32 : D / 2) k_attn_paged_join(const PagedParams p, int ctas) {
  __shared__ long long red[2][4];
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.y, head = blockIdx.x;
  const int kvh = head / p.group, in_group = head - kvh * p.group;
  const int chunk = in_group / kPagedRows, row = in_group - chunk * kPagedRows;
  const long long per_unit = static_cast<long long>(p.kv_heads) * p.chunks;
  long long before = 0, T = 0;
  for (int i = threadIdx.x; i < p.B; i += blockDim.x) {
    const long long n = paged_units(paged_length(p, i)) * per_unit;
    T += n;
    if (i < b) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    T += __shfl_xor_sync(0xffffffffu, T, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  if ((threadIdx.x & 31) == 0) {
    red[0][threadIdx.x >> 5] = T;
    red[1][threadIdx.x >> 5] = before;
  }
  __syncthreads();
  T = before = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    T += red[0][w];
    before += red[1][w];
  }
  const int n_units = paged_units(paged_length(p, b));
  const int d = threadIdx.x * 2;
  __nv_bfloat16* dst = p.out + static_cast<long long>(b) * p.ldo + static_cast<long long>(head) * D + d;
  float* lse = p.lse == nullptr ? nullptr : p.lse + static_cast<long long>(b) * p.heads + head;
  if (n_units == 0) {
    *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(0.f, 0.f);
    if (lse != nullptr && d == 0) *lse = -INFINITY;
    return;
  }
  const long long G = paged_ranges(T, ctas);
  const long long u0 = before + (static_cast<long long>(kvh) * p.chunks + chunk) * n_units;
  const int c0 = paged_owner(u0, T, G), c1 = paged_owner(u0 + n_units - 1, T, G);
  if (c0 == c1) return;  // finished by its CTA
  auto part = [&](int c) { return p.ws + (2ll * c + (c == c0 ? 1 : 0)) * paged_part_floats<D>(); };
  float m = -INFINITY;
  for (int c = c0; c <= c1; ++c) m = fmaxf(m, part(c)[row]);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float2 acc = make_float2(0.f, 0.f);
  for (int c = c0; c <= c1; ++c) {
    const float* w = part(c);
    const float f = ex2_approx(w[row] - base);
    l = fmaf(w[kPagedRows + row], f, l);
    const float2 v = *reinterpret_cast<const float2*>(w + 2 * kPagedRows + row * D + d);
    acc.x = fmaf(v.x, f, acc.x);
    acc.y = fmaf(v.y, f, acc.y);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  *reinterpret_cast<__nv_bfloat162*>(dst) = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
  if (lse != nullptr && d == 0) *lse = (m + log2f(l)) * 0.69314718055994531f;
}

}  // namespace qib
