// Attention of one new token per sequence over a paged key-value cache:
//   o_b = softmax(scale q_b K_b^T) V_b   per head, grouped heads,
// K_b, V_b being the first lengths[b] rows that the page table of sequence b
// names.  Bound: HBM, every cached row is read once for every 16 query heads of
// its key head (8 sequences of 32768 tokens, one key head of 128, bf16: 37 us with
// 16 query heads, 46 with 24, 48 with 32).
//
// An item is a sequence, a group of 1 to 8 key heads and a chunk of 16 query
// heads of each.  Where the heads of a cached token lie next to each other, the
// warps of a CTA form one team per key head and read the same tokens together:
// a head row of 64 to 256 bytes by itself leaves DRAM pages open for too little
// (64 sequences of up to 8192 tokens, 8 key heads: bf16 rows of 256 bytes
// 176 us with one head at a time, 168 / 162 / 161 with 2 / 4 / 8; E4M3 rows of
// 128 bytes 151, 126, 121, 115).
//
// Split: the work of all items, counted in units of 16 tokens or more, is laid
// end to end and cut into gridDim.x equal ranges, one per CTA, so every SM
// streams the same number of bytes whatever the lengths are.  An item inside
// one range is finished there; an item cut by range borders leaves partial
// results (row maximum, sum, unnormalized output, all fp32) in the workspace,
// which k_attn_paged_join adds up in range order: the result does not depend on
// timing.
//
// Inside a CTA the warps take blocks of the range in turn.  Each warp runs
// its own ring of cp.async stages (no barrier between warps while it streams)
// and its own running softmax, transposed so that the query heads of a key head
// are the 8 columns of mma.sync m16n8k16: S^T = K Q^T (16 tokens x 8 heads) and
// O^T += V^T P^T (16 columns x 8 heads); 9 to 16 heads take two column tiles
// over the same K and V fragments.  P^T goes from S^T's accumulator layout to
// the operand layout with one 8 x 8 transpose per 8 tokens.  Powers P = 2^(s - base)
// are taken above a base that follows the maximum; bf16 caches let it lag by
// up to 2^8, so most blocks need one vote and no reduction.  The tensor work is a
// few per cent of what the SM can do, so the legacy instruction is enough; what counts are the bytes in flight
// (128 KB per SM) and the instructions per byte.
//
// E4M3 caches: codes are widened exactly to fp16 and multiplied in fp16 with
// fp32 sums; q is scaled by a power of two per head so that it fits fp16, the
// key scale goes into the softmax scale and the value scale into the quotient
// of output and sum (the sums before it may pass fp32 with it).
// P is rounded to fp16, whose range ends at 2^-24: what lies far below a row's
// maximum would be lost, although it makes up the output where the maximum's own
// value is near zero.  So the base is 2^15 below the maximum and does not lag:
// P reaches up to 2^15 and keeps its 11 bits down to 2^-29 of the maximum (20
// nats), and no probability is off by more than 2^-40.
//
// A page index outside the cache, or a length behind the page table, reads
// nothing: those keys take no part, and the device status word is set.  So it is
// for a negative length, which counts as 0.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "attn_short.cuh"
#include "attn_split.h"
#include "launch_count.cuh"
#include "sm100_ptx.cuh"

namespace qib {

constexpr unsigned int kTagPaged = 0x800u;
constexpr int kPagedUnitShift = 6;  // log2 of tokens per unit of work times key heads per item (a block at least)
constexpr int kPagedRows = 16;      // query heads per item
constexpr int kPagedWarps = 8;

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
  const float* scale[2];                   // E4M3: k_scale, v_scale, [1] or [kv_heads]; else nullptr
  int scale_per_head[2];
  int B, heads, kv_heads, group, chunks;   // chunks of kPagedRows query heads per key head
  int team_shift, groups;                  // log2 of the key heads per item; kv_heads in such groups
  int unit_shift;                          // log2 of the tokens per unit of work
  int page_size, max_pages, num_pages;
  int page_shift;                          // log2 of page_size, or -1
  float scale_log2e;
};

// Floats of one partial result of one key head: maxima, sums, output rows.
template <int D>
__host__ __device__ constexpr int paged_part_floats() { return kPagedRows * (D + 2); }

__device__ __forceinline__ int paged_length(const PagedParams& p, int b) {
  const int n = p.lengths[b];
  const long long most = static_cast<long long>(p.max_pages) * p.page_size;
  if (n > most) {
    record_error(kDevBadIndex, kTagPaged, 1);
    return static_cast<int>(most);
  }
  if (n < 0) record_error(kDevBadIndex, kTagPaged, 3);
  return max(n, 0);
}
// Tokens per unit: 2^unit_shift.
__device__ __forceinline__ int paged_units(const PagedParams& p, int len) {
  return paged_unit_count(len, p.unit_shift);
}
// The item that a CTA begins and later ones go on with, up to CTA `last`.
struct PagedRecord {
  int used, b, kv_group, chunk, last;
};
template <int D>
__device__ __forceinline__ PagedRecord* paged_records(const PagedParams& p, int ctas) {
  return reinterpret_cast<PagedRecord*>(p.ws + ((2ll * ctas) << p.team_shift) * paged_part_floats<D>());
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
// Transpose of an 8 x 8 matrix of 16-bit elements, a row of it in every 4 lanes.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
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
  static constexpr int WARPS = kPagedWarps;
  static constexpr int STAGE = ROW == 64 ? 4096 : 8192;
  static constexpr int BT = STAGE / (2 * ROW);              // tokens per block: 16 or 32
  static_assert(BT == (ROW == 256 ? 16 : 32), "the entry point sizes the units of work by it");
  static constexpr int CH = ROW / 16;                       // 16-byte chunks per row: 4, 8 or 16
  static constexpr int STAGES = 24576 / STAGE;              // 192 KB in all
  static constexpr int THREADS = WARPS * 32;
  // the base lies BELOW binary places below the maximum and moves when a score is TOP places above it
  static constexpr float BELOW = FP8 ? 15.f : 0.f, TOP = FP8 ? 15.f : 8.f;
  static constexpr int RING = WARPS * STAGES * STAGE;
  // byte offset of chunk c of row r: 128-byte lines whose 16-byte chunks are
  // permuted so that the 8 rows ldmatrix reads at once hit 8 different chunks
  __device__ static __forceinline__ uint32_t at(int r, int c) {
    if constexpr (CH >= 8) return r * ROW + ((c ^ (r & 7)) << 4);
    else return r * ROW + ((c ^ ((r >> 1) & 3)) << 4);
  }
};
template <int D, bool FP8, int HT>
__host__ __device__ constexpr int paged_smem() {
  const int merge = PagedCfg<D, FP8>::WARPS * 8 * HT * (D + 2) * 4;
  return (PagedCfg<D, FP8>::RING > merge ? PagedCfg<D, FP8>::RING : merge) + 256;
}

// HT column tiles of 8 query heads per item: 1 or 2.
template <int D, bool FP8, int HT>
__global__ void __launch_bounds__(PagedCfg<D, FP8>::THREADS, 1) k_attn_paged(const PagedParams p) {
  using C = PagedCfg<D, FP8>;
  constexpr int BT = C::BT, ST = C::STAGES, W = C::WARPS;
  constexpr int KS = D / 16;       // 16-column steps of a head
  constexpr int R = 8 * HT;        // heads of an item
  extern __shared__ __align__(128) uint8_t paged_sm[];
  __shared__ long long scan[W];
  __shared__ int start_b;
  __shared__ long long start_u;
  __shared__ uint32_t masks[W][ST];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_wait();
  griddep_launch_dependents();

  PagedRecord* rec = paged_records<D>(p, gridDim.x) + blockIdx.x;
  if (tid == 0) rec->used = 0;
  // zeros for sequences without keys
  for (int b = blockIdx.x; b < p.B; b += gridDim.x)
    if (paged_length(p, b) == 0) {
      for (int i = tid; i < p.heads * D; i += C::THREADS)
        p.out[static_cast<long long>(b) * p.ldo + i] = __float2bfloat16_rn(0.f);
      if (p.lse != nullptr)
        for (int i = tid; i < p.heads; i += C::THREADS) p.lse[static_cast<long long>(b) * p.heads + i] = -INFINITY;
    }

  // the range of this CTA and the sequence it starts in
  const long long per_unit = static_cast<long long>(p.groups) * p.chunks;
  const int per_thread = (p.B + C::THREADS - 1) / C::THREADS;
  const int b_lo = min(p.B, tid * per_thread), b_hi = min(p.B, b_lo + per_thread);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += paged_units(p, paged_length(p, b)) * per_unit;
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
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += scan[w];
    T += scan[w];
  }
  if (T == 0) return;
  const long long G = paged_ranges(T, gridDim.x);
  long long u = paged_range_begin(blockIdx.x, T, G);
  const long long u_end = blockIdx.x < G ? paged_range_begin(blockIdx.x + 1, T, G) : u;
  before += incl - mine;
  if (u < u_end && before <= u && u < before + mine) {
    long long at = before;
    for (int b = b_lo; b < b_hi; ++b) {
      const long long n = paged_units(p, paged_length(p, b)) * per_unit;
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
  const uint32_t ring_u = smem_u32(paged_sm + warp * ST * C::STAGE);
  const int g = lane >> 2, t4 = lane & 3;
  // a block lies in one page: units, where ranges begin, are multiples of BT
  const bool whole_pages = p.page_shift >= 0 && (1 << p.page_shift) >= BT && (1 << p.unit_shift) >= BT;

  while (u < u_end) {
    int len = paged_length(p, b);
    int n_units = paged_units(p, len);
    while (u >= b_first + n_units * per_unit) {  // next sequence with keys
      b_first += n_units * per_unit;
      ++b;
      len = paged_length(p, b);
      n_units = paged_units(p, len);
    }
    const long long rel = u - b_first;
    const int item = static_cast<int>(rel / n_units);           // group of key heads, and chunk
    const int unit0 = static_cast<int>(rel - static_cast<long long>(item) * n_units);
    const int unit1 = static_cast<int>(min(static_cast<long long>(n_units), unit0 + (u_end - u)));
    const int kv_group = item / p.chunks, chunk = item - kv_group * p.chunks;
    const int rows = min(kPagedRows, p.group - chunk * kPagedRows);
    const int tok0 = unit0 << p.unit_shift;
    const int tok1 = static_cast<int>(min(static_cast<long long>(len), static_cast<long long>(unit1) << p.unit_shift));
    u += unit1 - unit0;
    // this warp's key head, and the blocks of its team: tok0 + (mate + i * mates) * BT
    const int team = warp & ((1 << p.team_shift) - 1), mate = warp >> p.team_shift, mates = W >> p.team_shift;
    const int kvh = (kv_group << p.team_shift) + team;
    const int head0 = kvh * p.group + chunk * kPagedRows;

    const int n_blocks = (tok1 - tok0 + BT - 1) / BT;
    const int my_blocks = n_blocks > mate ? (n_blocks - mate - 1) / mates + 1 : 0;
    const int* pg = p.pages + static_cast<long long>(b) * p.ld_pages;
    constexpr int RPI = 32 / C::CH;       // rows copied per instruction
    const int row0 = lane / C::CH, ch = lane % C::CH;
    const uint8_t* lane_src[2];           // this lane's chunk of the first rows of page 0
#pragma unroll
    for (int c = 0; c < 2; ++c)
      lane_src[c] = p.cache[c] + kvh * p.head_stride[c] + row0 * p.slot_stride[c] + ch * 16;
    auto issue = [&](int i) {
      const int st = i % ST;
      const int t0 = tok0 + (mate + i * mates) * BT;
      if (whole_pages) {
        // the block lies in one page: one look-up, rows at fixed distances
        const int pi = t0 >> p.page_shift, place = t0 - (pi << p.page_shift);
        const int page = pg[pi];
        const bool good = page >= 0 && page < p.num_pages;
        if (!good) record_error(kDevBadIndex, kTagPaged, 2);
        const int n = good ? min(BT, tok1 - t0) : 0;
        if (lane == 0) masks[warp][st] = n >= 32 ? 0xffffffffu : (1u << n) - 1u;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint8_t* src = lane_src[c];
          if (good) src += page * p.page_stride[c] + place * p.slot_stride[c];
          const long long step = RPI * p.slot_stride[c];
#pragma unroll
          for (int i2 = 0; i2 < BT / RPI; ++i2) {
            const int r = i2 * RPI + row0;
            cp_async16(ring_u + st * C::STAGE + c * (C::STAGE / 2) + C::at(r, ch), src + i2 * step, r < n);
          }
        }
        return;
      }
      // any page size: every lane looks up a token, the copies take the addresses from there
      const int tok = t0 + (lane % BT);
      long long off[2] = {0, 0};
      bool ok = tok < tok1;
      if (ok) {
        const int pi = p.page_shift >= 0 ? tok >> p.page_shift : tok / p.page_size;
        const int place = tok - pi * p.page_size;
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
      if (lane == 0) masks[warp][st] = m;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i2 = 0; i2 < BT / RPI; ++i2) {
          const int r = i2 * RPI + row0;
          const long long o = __shfl_sync(0xffffffffu, off[c], r);
          cp_async16(ring_u + st * C::STAGE + c * (C::STAGE / 2) + C::at(r, ch), p.cache[c] + o + ch * 16,
                     (m >> r) & 1u);
        }
    };
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      if (i < my_blocks) issue(i);
      cp_async_commit();
    }

    // Q^T as the B operand: head 8 h + g, columns of a 16-column step by the lane
    uint32_t qb[HT][KS][2];
    float sl2[HT][2];  // scale of heads 8 h + 2 t4, 8 h + 2 t4 + 1, in powers of two
#pragma unroll
    for (int h = 0; h < HT; ++h) {
      float qmax = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // fp16 path: the lane's 4 columns are consecutive, as its 4 codes of K are
          const int col = ks * 16 + (FP8 ? 4 * t4 + 2 * j : 2 * t4 + 8 * j);
          uint32_t v = 0;
          if (8 * h + g < rows)
            v = *reinterpret_cast<const uint32_t*>(p.q + static_cast<long long>(b) * p.ldq +
                                                   static_cast<long long>(head0 + 8 * h + g) * D + col);
          qb[h][ks][j] = v;
          if (FP8) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
            qmax = fmaxf(qmax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
      float up = 1.f;
      if (FP8) {
        qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, 1));
        qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, 2));
        // the row's largest element goes to fp16's last binade (at most 255 2^8 there), so that
        // small ones beside it keep their bits down to 2^-29 of it; both powers stay normal
        const int e = max(-126, static_cast<int>(__float_as_uint(qmax) >> 23) - 127 - 15);
        up = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qb[h][ks][j]));
            qb[h][ks][j] = pack_pair<true>(f.x * down, f.y * down);
          }
      }
      const float base = p.scale_log2e * (FP8 ? p.scale[0][p.scale_per_head[0] ? kvh : 0] : 1.f);
#pragma unroll
      for (int j = 0; j < 2; ++j) sl2[h][j] = base * (FP8 ? __shfl_sync(0xffffffffu, up, 4 * (2 * t4 + j)) : 1.f);
    }

    float o[HT][KS][4];
#pragma unroll
    for (int h = 0; h < HT; ++h)
#pragma unroll
      for (int n = 0; n < KS; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[h][n][i] = 0.f;
    float base2[HT][2], sum[HT][2];
#pragma unroll
    for (int h = 0; h < HT; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        base2[h][j] = -INFINITY;
        sum[h][j] = 0.f;
      }
#pragma unroll 1
    for (int i = 0; i < my_blocks; ++i) {
      __syncwarp();  // every lane has read stage (i - 1) % ST, which is filled next
      if (i + ST - 1 < my_blocks) issue(i + ST - 1);
      cp_async_commit();
      cp_async_wait<ST - 1>();
      __syncwarp();
      const uint32_t sk = ring_u + (i % ST) * C::STAGE, sv = sk + C::STAGE / 2;
      const uint32_t mask = masks[warp][i % ST];
#pragma unroll
      for (int tb = 0; tb < BT / 16; ++tb) {
        // S^T = K Q^T of 16 tokens
        float s[HT][4];
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[h][j] = 0.f;
        if constexpr (!FP8) {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t k[4];  // (tokens 0-7, 8-15) of columns 0-7, then of 8-15
            ldsm_x4(k, sk + C::at(tb * 16 + (lane & 15), ks * 2 + (lane >> 4)));
#pragma unroll
            for (int h = 0; h < HT; ++h) mma_16816<false>(s[h], k, qb[h][ks][0], qb[h][ks][1]);
          }
        } else {
#pragma unroll
          for (int kg = 0; kg < KS / 2; ++kg) {
            uint32_t k[4];  // (tokens 0-7, 8-15) of columns 0-15, then of 16-31; 4 codes per register
            ldsm_x4(k, sk + C::at(tb * 16 + (lane & 15), kg * 2 + (lane >> 4)));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t a[4] = {e4m3x2_to_half2(k[2 * j]), e4m3x2_to_half2(k[2 * j + 1]),
                                     e4m3x2_to_half2(k[2 * j] >> 16), e4m3x2_to_half2(k[2 * j + 1] >> 16)};
#pragma unroll
              for (int h = 0; h < HT; ++h) mma_16816<true>(s[h], a, qb[h][2 * kg + j][0], qb[h][2 * kg + j][1]);
            }
          }
        }
        // running softmax: elements (token g, g + 8) x (head 2 t4, 2 t4 + 1)
        const bool ok0 = (mask >> (tb * 16 + g)) & 1u, ok1 = (mask >> (tb * 16 + 8 + g)) & 1u;
        bool grew = false;
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[h][j] = ok0 ? s[h][j] * sl2[h][j] : -INFINITY;
            s[h][2 + j] = ok1 ? s[h][2 + j] * sl2[h][j] : -INFINITY;
            grew |= fmaxf(s[h][j], s[h][2 + j]) - base2[h][j] > C::TOP;
          }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float top = fmaxf(s[h][j], s[h][2 + j]);
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
              float nb = top - C::BELOW;
              if (top - nb > C::TOP) nb = top;  // scores so large that the difference is rounded
              nb = fmaxf(nb, base2[h][j]);
              const float f = nb > base2[h][j] ? ex2_approx(base2[h][j] - nb) : 1.f;  // 2^-inf = 0: nothing summed yet
              base2[h][j] = nb;
              sum[h][j] *= f;
#pragma unroll
              for (int n = 0; n < KS; ++n) {
                o[h][n][j] *= f;
                o[h][n][2 + j] *= f;
              }
            }
        }
        uint32_t pb[HT][2];
#pragma unroll
        for (int h = 0; h < HT; ++h) {
          const float m0 = base2[h][0] == -INFINITY ? 0.f : base2[h][0];
          const float m1 = base2[h][1] == -INFINITY ? 0.f : base2[h][1];
          const float e00 = ex2_approx(s[h][0] - m0), e01 = ex2_approx(s[h][1] - m1);
          const float e10 = ex2_approx(s[h][2] - m0), e11 = ex2_approx(s[h][3] - m1);
          sum[h][0] += e00 + e10;
          sum[h][1] += e01 + e11;
          pb[h][0] = transpose8x8(pack_pair<FP8>(e00, e01));
          pb[h][1] = transpose8x8(pack_pair<FP8>(e10, e11));
        }
        // O^T += V^T P^T
        if constexpr (!FP8) {
#pragma unroll
          for (int n = 0; n < KS; ++n) {
            uint32_t v[4];  // columns (0-7, 8-15) of tokens 0-7, then of 8-15, transposed
            ldsm_x4_t(v, sv + C::at(tb * 16 + (lane & 7) + ((lane >> 4) << 3), n * 2 + ((lane >> 3) & 1)));
#pragma unroll
            for (int h = 0; h < HT; ++h) mma_16816<false>(o[h][n], v, pb[h][0], pb[h][1]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < KS / 2; ++n) {
            uint32_t v[4];  // tokens (0-7, 8-15) of columns 0-15, then of 16-31; a register: 2 tokens x 2 columns
            ldsm_x4_t(v, sv + C::at(tb * 16 + (lane & 15), n * 2 + (lane >> 4)));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // rows 0-7 of the tile are the even columns of the 16 (bytes 0, 2), rows 8-15 the odd ones (1, 3)
              const uint32_t a[4] = {e4m3x2_to_half2(__byte_perm(v[2 * j], 0, 0x4420)),
                                     e4m3x2_to_half2(__byte_perm(v[2 * j], 0, 0x4431)),
                                     e4m3x2_to_half2(__byte_perm(v[2 * j + 1], 0, 0x4420)),
                                     e4m3x2_to_half2(__byte_perm(v[2 * j + 1], 0, 0x4431))};
#pragma unroll
              for (int h = 0; h < HT; ++h) mma_16816<true>(o[h][2 * n + j], a, pb[h][0], pb[h][1]);
            }
          }
        }
      }
    }
    cp_async_wait<0>();
    __syncthreads();  // the rings are free: they take the warps' results

    // the warps' results -> shared memory: rows, bases (as maxima below), sums
    float* mg = reinterpret_cast<float*>(paged_sm);
    float* mg_m = mg + W * R * D;
    float* mg_l = mg_m + W * R;
#pragma unroll
    for (int h = 0; h < HT; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = sum[h][j];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int row = 8 * h + 2 * t4 + j;
        if (g == 0) {
          mg_m[warp * R + row] = base2[h][j];
          mg_l[warp * R + row] = l;
        }
        float* dst = mg + (warp * R + row) * D;
#pragma unroll
        for (int n = 0; n < KS; ++n) {
          dst[n * 16 + (FP8 ? 2 * g : g)] = o[h][n][j];
          dst[n * 16 + (FP8 ? 2 * g + 1 : g + 8)] = o[h][n][2 + j];
        }
      }
    __syncthreads();
    const bool whole = unit0 == 0 && unit1 == n_units;
    if (tid == 0 && unit0 == 0 && !whole)
      *rec = {1, b, kv_group, chunk, paged_owner(b_first + static_cast<long long>(item + 1) * n_units - 1, T, G)};
    float* parts = p.ws + ((2ll * blockIdx.x + (unit0 == 0 ? 1 : 0)) << p.team_shift) * paged_part_floats<D>();
    for (int i = tid; i < (rows * (D / 2)) << p.team_shift; i += C::THREADS) {
      const int r = i / (D / 2), d = (i - r * (D / 2)) * 2;
      const int of = r / rows, row = r - of * rows;  // key head of the group, query head of its chunk
      const int kv = (kv_group << p.team_shift) + of, head = kv * p.group + chunk * kPagedRows + row;
      float m = -INFINITY;
      for (int w = of; w < W; w += 1 << p.team_shift) m = fmaxf(m, mg_m[w * R + row]);
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      float2 acc = make_float2(0.f, 0.f);
      for (int w = of; w < W; w += 1 << p.team_shift) {
        const float f = ex2_approx(mg_m[w * R + row] - base);
        l = fmaf(mg_l[w * R + row], f, l);
        const float2 v = *reinterpret_cast<const float2*>(mg + (w * R + row) * D + d);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
      }
      if (whole) {
        const float inv = l != 0.f ? 1.f / l : 0.f;  // a sum of NaN stays one
        const float v_scale = FP8 ? p.scale[1][p.scale_per_head[1] ? kv : 0] : 1.f;
        *reinterpret_cast<__nv_bfloat162*>(p.out + static_cast<long long>(b) * p.ldo + static_cast<long long>(head) * D +
                                           d) = __floats2bfloat162_rn(acc.x * inv * v_scale, acc.y * inv * v_scale);
        if (p.lse != nullptr && d == 0)
          p.lse[static_cast<long long>(b) * p.heads + head] = (m + log2f(l)) * 0.69314718055994531f;
      } else {
        float* part = parts + of * paged_part_floats<D>();
        if (d == 0) {
          part[row] = m;
          part[kPagedRows + row] = l;
        }
        *reinterpret_cast<float2*>(part + 2 * kPagedRows + row * D + d) = acc;
      }
    }
    __syncthreads();  // the rings are filled again for the next item
  }
}

// Adds up the partial results of the items that were cut: CTA (c, y) query
// head y of the item that CTA c of the first kernel began and did not finish.
// Its warps take the parts in turn, four loads ahead, and add their sums up in
// warp order; a lane holds D / 32 columns.
constexpr int kPagedJoinWarps = 4;
template <int D>
__global__ void __launch_bounds__(kPagedJoinWarps * 32) k_attn_paged_join(const PagedParams p, int ctas) {
  constexpr int N = D / 32;
  __shared__ float sm_m[kPagedJoinWarps], sm_l[kPagedJoinWarps], sm_o[kPagedJoinWarps][D];
  griddep_wait();
  griddep_launch_dependents();
  const int c0 = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PagedRecord r = paged_records<D>(p, ctas)[c0];
  if (!r.used) return;
  const int rows = min(kPagedRows, p.group - r.chunk * kPagedRows);
  const int of = blockIdx.y / rows, row = blockIdx.y - of * rows;  // key head of the group, query head of its chunk
  if (of >> p.team_shift) return;
  float m = -INFINITY, l = 0.f, acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
#pragma unroll 4
  for (int c = c0 + warp; c <= r.last; c += kPagedJoinWarps) {
    const float* w = p.ws + (((2ll * c + (c == c0 ? 1 : 0)) << p.team_shift) + of) * paged_part_floats<D>();
    float v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = w[2 * kPagedRows + row * D + 32 * k + lane];
    const float pm = w[row], pl = w[kPagedRows + row];
    const float nm = fmaxf(m, pm), base = nm == -INFINITY ? 0.f : nm;
    const float f0 = ex2_approx(m - base), f1 = ex2_approx(pm - base);
    m = nm;
    l = l * f0 + pl * f1;
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = acc[k] * f0 + v[k] * f1;
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) sm_o[warp][32 * k + lane] = acc[k];
  __syncthreads();
  const int kv = (r.kv_group << p.team_shift) + of, head = kv * p.group + r.chunk * kPagedRows + row;
  const float v_scale = p.scale[1] != nullptr ? p.scale[1][p.scale_per_head[1] ? kv : 0] : 1.f;
  for (int d = threadIdx.x; d < D; d += kPagedJoinWarps * 32) {
    float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kPagedJoinWarps; ++w) top = fmaxf(top, sm_m[w]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kPagedJoinWarps; ++w) {
      const float f = ex2_approx(sm_m[w] - base);
      sum = fmaf(sm_l[w], f, sum);
      o = fmaf(sm_o[w][d], f, o);
    }
    p.out[static_cast<long long>(r.b) * p.ldo + static_cast<long long>(head) * D + d] =
        __float2bfloat16_rn(sum != 0.f ? o / sum * v_scale : 0.f);
    if (p.lse != nullptr && d == 0)
      p.lse[static_cast<long long>(r.b) * p.heads + head] = (top + log2f(sum)) * 0.69314718055994531f;
  }
}

}  // namespace qib
