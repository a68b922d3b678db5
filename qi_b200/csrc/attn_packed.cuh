// Attention over whole prompts: packed sequences, grouped heads, causal or not.
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j
// over the keys j of query i's own sequence, and with `causal` only those with
// j <= i + (lk - lq) (the last query sees every key).  Sequence b has query
// rows cu_q[b] .. cu_q[b+1] and key rows cu_k[b] .. cu_k[b+1]; a query that
// sees no key gives zeros.
//
// One work item = two 128-row query tiles that share their key head: 256
// consecutive tokens of one head, or, when the group size is even, the same
// 128 tokens of two heads (short sequences then fill both tiles, and both have
// the same causal extent).  Per 128-key step and tile:
//   S = Q K^T      tcgen05.mma (shared x shared) -> TMEM, fp32
//   P = 2^(S - m)  one thread per row: running maximum and sum in registers,
//                  P rounded to bf16 and stored over S in TMEM
//   O += P V       tcgen05.mma (TMEM x shared; V as it lies, MN-major) -> TMEM
// The two tiles alternate, so one tile's softmax runs beside the other's
// products.  O is rescaled only when a row's maximum has grown by more than
// 2^8 since the value in use (the sums use the same value, so the result is
// the same up to rounding); keys run from the last step to the first, so the
// maximum rarely grows.
//
// Roles: warps 0-3 and 4-7 softmax and epilogue of tile 0 and 1, warp 8 TMA,
// warp 9 MMA, warp 10 the list of items, warp 11 zeros for the rows outside every
// sequence where they are asked for.  A softmax thread holds a whole row of S, so
// the softmax warpgroups take 208 registers a thread and the third leaves them all but 88 (of 168 at launch: 256 x 208 +
// 128 x 88 = 64,512, all of them).  CTAs are persistent; each takes every
// gridDim.x-th item, longest items first, the direction alternating from round
// to round.  The order is a function of cu_q alone: level L (the L-th query
// block of every sequence that has one) from the last to the first; warp 10
// walks it and hands the items over in shared memory, four in flight.
//
// What bounds it: the chain of one tile, softmax (about 2,200 clocks, 1,024 of
// them exponentials) then P V and S (1,300 clocks, 1,024 of them products),
// 3,600 clocks per 128-key step where the products of both tiles take 2,048.
// At D = 64 the products take half of that and the exponentials as much as before.
// (TMEM is full at D = 128; at D = 64 columns 384 to 511 are free, and a third S
// buffer there has not been tried.)
// Measured on the way (16384 tokens, 24 / 8 heads of 128, causal, us in a short
// burst; 1,266 is 1,303 TFLOP/s; calls back to back for a second take 1,450 to
// 1,500 under the 1000 W cap): products issued by lane 0 with 64-bit descriptors
// formed on the spot 1,842, by an elected thread 1,645, item list in a warp of its own and
// descriptors as constants to a base 1,371, all MMA operands warp-uniform 1,330,
// S loaded in one go 1,297, the masked keys in one branch 1,266.  Two threads
// per row (16 softmax warps) 1,433; half of P handed over early 1,359; 64-key
// steps with S double-buffered 1,457 (the products read shared memory at its
// full rate then, and every barrier waits behind them); a quarter of the
// exponentials as polynomials on the FP32 pipe 1,365; masks by 32-key chunk
// 1,351 (branches between the loads and the maximum).
// A short item costs about 4 us beside its further steps: both tiles' softmax
// fall together, then the output.
//
// Rows behind a sequence's end belong to its neighbour: scores of such keys
// are replaced (not added to), the V rows of the last 16-key step behind the
// end are zeroed in shared memory, further steps are not multiplied, and
// output rows are stored one by one.  So nothing, NaN included, passes from
// one sequence to another.  Later keys of a query's own sequence take part in
// its last step with probability zero, which times an infinity or a NaN is a
// NaN: a row whose sum is finite and whose output is not is looked at again
// (packed_mend), and one that saw no key at all is overwritten with zeros, so
// that what a row does not see does not reach it either (the look at the outputs
// takes 0.2 us of a short item's 4).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <type_traits>

#include "attn_short.cuh"
#include "attn_split.h"
#include "launch_count.cuh"
#include "sm100_ptx.cuh"

namespace qib {

constexpr unsigned int kTagPacked = 0x900u;

struct PackedParams : PackedShape {
  const int* cu_q;   // [n_seq + 1]
  const int* cu_k;
  int n_seq, total_q, total_k;
  int kv_heads, group;
  int zero_rest;     // 1: rows of out outside every sequence become zeros
  float scale_log2e;
  __nv_bfloat16* out;
  long long ldo;
  float* lse;        // [total_q, heads] or nullptr
  float* ws;         // partial results and records, or nullptr: items are never cut
  const __nv_bfloat16 *q, *k, *v;  // as in the tensor maps, for packed_mend
  long long ldq, ldk, ldv;
};

// Shared-memory descriptors as two words.  The high word is a constant (8-row
// groups 1024 B apart, version 1, 128-byte swizzle); the low word holds the
// address / 16 and the leading offset / 16: unused (1) for K-major operands;
// for V, whose rows are the K extent (MN-major), the distance of its blocks of
// 64 columns.  Products of a tile differ in the low word by constants.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr, uint32_t lead) {
  return ((smem_addr & 0x3FFFFu) >> 4) | ((lead >> 4) << 16);
}
__device__ __forceinline__ void tc_commit_if(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_bf16_lo(uint32_t leader, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi), "r"(leader));
}
__device__ __forceinline__ void mma_bf16_ts_lo(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo,
                                               uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 b, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHi), "r"(leader));
}

// What the roles of a CTA tell each other: one gave up; warps that look at rows
// once more (packed_mend).
struct PackedFlags {
  int abort, mending;
};

// The softmax warps' wait: mbar_wait_hot, but the limit does not run while a warp
// is in packed_mend, which ends by itself and takes time by the length of the
// sequence (32 rows over 300,000 keys take longer than the limit).
__device__ __forceinline__ bool packed_wait(uint64_t* bar, uint32_t parity, volatile PackedFlags* flags,
                                            unsigned int tag, unsigned int site) {
#pragma unroll 1
  for (int i = 0; i < 512; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = globaltimer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (flags->abort) return false;
    if (flags->mending) {
      t0 = globaltimer_ns();
    } else if (globaltimer_ns() - t0 > QI_WAIT_TIMEOUT_NS) {
      record_error(kDevWaitTimeout, tag, site);
      flags->abort = 1;
      return false;
    }
  }
}
// The other roles only have to outlast it: where the pipeline stalls the softmax
// warps wait too, and give up for the CTA after the usual limit.  (With the
// check in their waits as well, chunks after prefixes at D = 64 took 2 % longer.)
constexpr unsigned long long kPackedRoleLimit = 600000000000ull;  // 600 s: a mend over 80 million keys

template <int D>
struct PackedCfg {
  static constexpr int TILE = 128 * D * 2;       // bytes of a 128-row operand tile (D / 64 swizzled blocks)
  static constexpr int BLOCK = 128 * 128;        // bytes of one 64-column block
  static constexpr int STAGES = 4;               // K and V of two steps
  static constexpr int THREADS = 384;
  static constexpr int STAGING = 8 * 4096;       // 32 rows x 128 B of output per softmax warp
  static constexpr int SMEM = (2 + STAGES) * TILE + STAGING + 1024 + 512;
  static constexpr int TMEM_COLS = 512;
  __host__ __device__ static constexpr uint32_t S_COL(int t) { return t * 128; }
  __host__ __device__ static constexpr uint32_t O_COL(int t) { return 256 + t * D; }
  static constexpr uint32_t IDESC_S = make_idesc(kDF32, kFmtBF16, kFmtBF16, 128, 128);
  static constexpr uint32_t IDESC_O = make_idesc(kDF32, kFmtBF16, kFmtBF16, 128, D) | (1u << 16);  // B is MN-major
};

constexpr int kPackedItems = 4;  // items in flight

// Rows of sequence b, clamped to the tensor (bad prefix sums read and write inside it).
__device__ __forceinline__ void packed_span(const int* cu, int b, int total, int& first, int& len) {
  first = min(max(cu[b], 0), total);
  len = min(max(cu[b + 1], first), total) - first;
}

__device__ __forceinline__ PackedSpan packed_load(const PackedParams& p, int b) {
  PackedSpan s = {0, 0, 0, 0};
  if (b < p.n_seq) {
    packed_span(p.cu_q, b, p.total_q, s.q0, s.lq);
    packed_span(p.cu_k, b, p.total_k, s.k0, s.lk);
  }
  return s;
}
__device__ __forceinline__ PackedSpan packed_from_lane(const PackedSpan& s, int lane) {
  return {__shfl_sync(0xffffffffu, s.q0, lane), __shfl_sync(0xffffffffu, s.lq, lane),
          __shfl_sync(0xffffffffu, s.k0, lane), __shfl_sync(0xffffffffu, s.lk, lane)};
}
// One partial result in the workspace: per tile 128 maxima, 128 sums and D
// columns of 128 fp32 output elements.
template <int D>
__host__ __device__ constexpr int packed_part_floats() { return 2 * 128 * (D + 2); }
// The rows of a warp (a lane each) once more whose sum is finite and whose
// output holds a NaN (`bad`), where a key behind the row's last visible one
// (`limit`) and inside the steps that were multiplied (`end`) has a value that
// is not finite: 8 lanes to a key, 4 keys at a time, from global memory.  k and
// v point at the sequence's first key, q_row and out_row at the lane's row, m
// and inv are its maximum and 1 / sum.  `only` >= 0: just that eighth of the
// columns is written.
template <int D>
__device__ __noinline__ void packed_mend(bool bad, int limit, int end, const __nv_bfloat16* q_row,
                                         const __nv_bfloat16* k, long long ldk, const __nv_bfloat16* v, long long ldv,
                                         __nv_bfloat16* out_row, float scale_log2e, float m, float inv, int only) {
  constexpr int E = D / 8;
  const int lane = threadIdx.x & 31, part = lane & 7, group = lane >> 3;
  __syncwarp();  // the rows' first results are stored
  int worst = -1;
  for (int j = __reduce_min_sync(0xffffffffu, bad ? limit + 1 : end) + lane; j < end; j += 32) {
    const uint4* at = reinterpret_cast<const uint4*>(v + j * ldv);
    uint32_t most = 0;  // largest exponent field
#pragma unroll
    for (int c = 0; c < D / 8; ++c) {
      const uint4 w = at[c];
      most = __vmaxu2(most, __vmaxu2(__vmaxu2(w.x & 0x7f807f80u, w.y & 0x7f807f80u),
                                     __vmaxu2(w.z & 0x7f807f80u, w.w & 0x7f807f80u)));
    }
    if ((most & 0xffffu) == 0x7f80u || (most >> 16) == 0x7f80u) worst = j;
  }
  worst = __reduce_max_sync(0xffffffffu, worst);
  unsigned todo = __ballot_sync(0xffffffffu, bad && limit < worst);
  auto row_of = [](unsigned long long ptr, int src) { return __shfl_sync(0xffffffffu, ptr, src); };
  auto widen = [](const __nv_bfloat16* src, float (&f)[E]) {
#pragma unroll
    for (int c = 0; c < E / 8; ++c) {
      const uint4 w4 = reinterpret_cast<const uint4*>(src)[c];
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[8 * c + 2 * i] = __uint_as_float(w[i] << 16);
        f[8 * c + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  };
  while (todo) {
    const int src = __ffs(todo) - 1;
    todo &= todo - 1;
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(row_of(reinterpret_cast<uintptr_t>(q_row), src));
    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(row_of(reinterpret_cast<uintptr_t>(out_row), src));
    const int n = __shfl_sync(0xffffffffu, limit, src) + 1;
    const float row_m = __shfl_sync(0xffffffffu, m, src), row_inv = __shfl_sync(0xffffffffu, inv, src);
    float qf[E], acc[E];
    widen(q + part * E, qf);
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = 0.f;
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += 4) {
      const int j = min(j0 + group, n - 1);
      float kf[E], vf[E];
      widen(k + j * ldk + part * E, kf);
      widen(v + j * ldv + part * E, vf);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) dot = fmaf(qf[i], kf[i], dot);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      const float w = __bfloat162float(__float2bfloat16(ex2_approx(fmaf(dot, scale_log2e, -row_m))));
      if (j0 + group < n) {
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = fmaf(w, vf[i], acc[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 8);
      acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 16);
      acc[i] *= row_inv;
    }
    if (group == 0 && (only < 0 || only == part)) {
#pragma unroll
      for (int c = 0; c < E / 8; ++c) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = acc[8 * c + i];
        reinterpret_cast<uint4*>(out + part * E)[c] = pack8(f);
      }
    }
  }
  __syncwarp();
}

// The items of this CTA one after another to `put` (the whole warp calls it).
// A lane holds the span of a sequence, 32 sequences at a time.
template <int D, class Put>
__device__ __forceinline__ void packed_schedule(const PackedParams& p, Put put) {
  const int lane = threadIdx.x & 31;
  const int heads_items = packed_head_items(p);
  const int G = gridDim.x, me = blockIdx.x;
  PackedSpan span = packed_load(p, lane);
  auto blocks = [&](const PackedSpan& s) { return packed_blocks(p, s); };
  auto end_of_items = [&]() {
    PackedItem end = {};
    end.last = 1;
    put(end);
  };
  int most = 0, longest = 0, count = 0;
  int chunk_most = 0;  // most blocks of a sequence in the lane's chunk of 32 (of the first 32 chunks)
  long long total = 0;
  for (int chunk = 0; chunk < p.n_seq; chunk += 32) {
    const PackedSpan s = chunk ? packed_load(p, chunk + lane) : span;
    const int chunk_max = __reduce_max_sync(0xffffffffu, blocks(s));
    most = max(most, chunk_max);
    if (lane == chunk >> 5) chunk_most = chunk_max;
    if (p.ws != nullptr) {
      total += packed_seq_cost(p, s, longest);
      count += blocks(s);
    }
  }
  if (p.ws != nullptr) {
    PackedRecord* rec = reinterpret_cast<PackedRecord*>(p.ws + 2ll * G * packed_part_floats<D>()) + 2 * me;
    if (lane < 2) rec[lane].used = 0;
    __syncwarp();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
      count += __shfl_xor_sync(0xffffffffu, count, o);
    }
    total *= heads_items;
    if (packed_even_split(total, static_cast<long long>(count) * heads_items, longest, G, p.causal)) {
      const long long cuts = packed_cuts(total, G);
      const long long lo = packed_cut_begin(total, cuts, me), hi = packed_cut_begin(total, cuts, me + 1);
      auto scan = [&](long long v) {  // inclusive, over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long u = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += u;
        }
        return v;
      };
      auto cost_of = [&](int steps) { return packed_cost(steps) * static_cast<long long>(heads_items); };
      long long before = 0;  // cost of the sequences in front of the chunk
      int idle = 0;          // blocks without steps so far (zeros to write: the CTAs take turns at them)
      for (int chunk = 0; chunk < p.n_seq; chunk += 32) {
        if (chunk) span = packed_load(p, chunk + lane);
        const long long mine = packed_seq_cost(p, span, longest) * heads_items;
        const long long end = before + scan(mine);
        unsigned todo = __ballot_sync(0xffffffffu, end > lo && end - mine < hi && mine > 0);
        while (todo) {
          const int i = __ffs(todo) - 1;
          todo &= todo - 1;
          const PackedSpan s = packed_from_lane(span, i);
          const int nb = blocks(s);
          long long at = __shfl_sync(0xffffffffu, end - mine, i);
          for (int l0 = 0; l0 < nb && at < hi; l0 += 32) {
            const int s_lane = l0 + lane < nb ? packed_steps(p, s, l0 + lane) : 0;
            const long long l_end = at + scan(cost_of(s_lane));
            unsigned levels = __ballot_sync(0xffffffffu, s_lane > 0 && l_end > lo && l_end - cost_of(s_lane) < hi);
            while (levels) {
              const int j = __ffs(levels) - 1;
              levels &= levels - 1;
              const int n = __shfl_sync(0xffffffffu, s_lane, j), per = packed_cost(n);
              const long long first = __shfl_sync(0xffffffffu, l_end, j) - cost_of(n);
              int h = first < lo ? static_cast<int>((lo - first) / per) : 0;
              for (long long u = first + static_cast<long long>(h) * per; h < heads_items && u < hi; ++h, u += per) {
                const PackedCut c = packed_cut_item(u, n, lo, hi);
                if (c.from >= c.to) continue;
                const PackedItem it = packed_item(p, s, l0 + j, h, n - c.to, n - c.from, c.part);
                if (c.part >= 0 && lane == 0) rec[c.part] = packed_record(p, s, l0 + j, n, c.to, it);
                if (!put(it)) return;
              }
            }
            at = __shfl_sync(0xffffffffu, l_end, 31);
          }
        }
        before = __shfl_sync(0xffffffffu, end, 31);
        int none = 0;
        for (int level = 0; level < blocks(span); ++level) none += packed_steps(p, span, level) == 0;
        unsigned with = __ballot_sync(0xffffffffu, none > 0);
        while (with) {
          const int i = __ffs(with) - 1;
          with &= with - 1;
          const PackedSpan s = packed_from_lane(span, i);
          const int nb = blocks(s);
          for (int level = 0; level < nb; ++level) {
            if (packed_steps(p, s, level) > 0) continue;
            for (int h = (me + idle) % G; h < heads_items; h += G)
              if (!put(packed_item(p, s, level, h, 0, 0, -1))) return;
            ++idle;
          }
        }
      }
      end_of_items();
      return;
    }
  }
  // longest first: level by level from the last
  int base = 0, round = 0;  // items before this (level, chunk); rounds of G items begun
  for (int level = most - 1; level >= 0; --level) {
    const unsigned with = __ballot_sync(0xffffffffu, chunk_most > level);
    for (int chunk = 0; chunk < p.n_seq; chunk += 32) {
      if (chunk < 1024 && !((with >> (chunk >> 5)) & 1u)) continue;
      if (p.n_seq > 32) span = packed_load(p, chunk + lane);
      const unsigned active = __ballot_sync(0xffffffffu, blocks(span) > level);
      const int n = __popc(active) * heads_items;
      while (true) {
        const int idx = round * G + ((round & 1) ? G - 1 - me : me) - base;
        if (idx >= n) break;
        ++round;
        const int nth = idx / heads_items, hi = idx - nth * heads_items;
        unsigned mm = active;
        for (int i = 0; i < nth; ++i) mm &= mm - 1;
        const PackedSpan s = packed_from_lane(span, __ffs(mm) - 1);
        if (!put(packed_item(p, s, level, hi, 0, packed_steps(p, s, level), -1))) return;
      }
      base += n;
    }
  }
  end_of_items();
}

template <int D>
__global__ void __launch_bounds__(384, 1)
k_attn_packed(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
              const __grid_constant__ CUtensorMap tmV, const PackedParams p) {
  using C = PackedCfg<D>;
  constexpr int NB = D / 64;  // 64-column blocks of a tile
  extern __shared__ uint8_t packed_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(packed_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * C::TILE;
  uint8_t* staging = ring + C::STAGES * C::TILE;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(staging + C::STAGING);        // [2]
  uint64_t* q_empty = q_full + 2;                                              // [2]
  uint64_t* s_full = q_full + 4;                                               // [2]
  uint64_t* p_full = q_full + 6;                                               // [2]
  uint64_t* o_done = q_full + 8;                                               // [2]
  uint64_t* drain = q_full + 10;
  uint64_t* kv_full = q_full + 11;                                             // [STAGES]
  uint64_t* kv_empty = kv_full + C::STAGES;                                    // [STAGES]
  uint64_t* it_full = kv_empty + C::STAGES;                                    // [kPackedItems]
  uint64_t* it_empty = it_full + kPackedItems;                                 // [kPackedItems]
  PackedItem* items = reinterpret_cast<PackedItem*>(it_empty + kPackedItems);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + kPackedItems);
  volatile PackedFlags* flags = reinterpret_cast<volatile PackedFlags*>(tmem_slot + 1);
  volatile int* abort_flag = &flags->abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
    }
    mbar_init(drain, 1);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int i = 0; i < kPackedItems; ++i) {
      mbar_init(&it_full[i], 1);
      mbar_init(&it_empty[i], 10);  // the softmax warps, TMA and MMA
    }
    flags->abort = flags->mending = 0;
    fence_mbar_init();
    tma_prefetch_map(&tmQ);
    tma_prefetch_map(&tmK);
    tma_prefetch_map(&tmV);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  griddep_wait();
  griddep_launch_dependents();

  // the next item (nullptr: none, or the CTA gives up), and its release
  uint32_t n_it = 0;
  auto next_item = [&]() -> const PackedItem* {
    if (!packed_wait(&it_full[n_it % kPackedItems], (n_it / kPackedItems) & 1u, flags, kTagPacked, 11))
      return nullptr;
    const PackedItem* it = &items[n_it % kPackedItems];
    return it->last ? nullptr : it;
  };
  auto release_item = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&it_empty[n_it % kPackedItems]);
    ++n_it;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 10) {
      // ---- items ----
      packed_schedule<D>(p, [&](const PackedItem& it) {
        const int i = n_it % kPackedItems;
        if (!mbar_wait_hot<kPackedRoleLimit>(&it_empty[i], ((n_it / kPackedItems) & 1u) ^ 1u, abort_flag, kTagPacked, 12))
          return false;
        if (lane == 0) {
          items[i] = it;
          mbar_arrive(&it_full[i]);
        }
        __syncwarp();
        ++n_it;
        return true;
      });
    } else if (warp == 11) {
      // ---- rows in front of the first sequence and behind the last ----
      if (p.zero_rest) {
        const int front = min(max(p.cu_q[0], 0), p.total_q), back = min(max(p.cu_q[p.n_seq], front), p.total_q);
        const int width = p.heads * (D / 8);
        for (int r = blockIdx.x; r < front + p.total_q - back; r += gridDim.x) {
          uint4* to = reinterpret_cast<uint4*>(p.out + static_cast<long long>(r < front ? r : back + r - front) * p.ldo);
          for (int i = lane; i < width; i += 32) to[i] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
    } else if (warp == 8) {
      // ---- TMA ----
      int stage = 0, issued = 0;
      uint32_t use = 0;  // times the ring has been gone round
      bool ok = true;
      int q_pend[2] = {0, 0};  // Q loads issued
      auto load = [&](const CUtensorMap* map, int col, int row) {
        ok = ok && mbar_wait_hot<kPackedRoleLimit>(&kv_empty[stage], (use & 1u) ^ 1u, abort_flag, kTagPacked, 21);
        if (!ok) return;
        if (lane == 0) {
          mbar_expect_tx(&kv_full[stage], C::TILE);
#pragma unroll
          for (int b = 0; b < NB; ++b)
            tma_load_2d(ring + stage * C::TILE + b * C::BLOCK, map, &kv_full[stage], col + b * 64, row);
        }
        ++issued;
        if (++stage == C::STAGES) {
          stage = 0;
          ++use;
        }
      };
      while (const PackedItem* it = next_item()) {
        const int steps = max(it->n[0], it->n[1]);
        const int q0 = it->q0, k0 = it->k0, col = it->head[0] / p.group * D;
        // the first K goes ahead of Q, whose places are free later
        if (steps > 0) load(&tmK, col, k0 + (steps - 1) * 128);
        if (steps > 0) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (it->n[t] == 0 || !ok) continue;
            ok = mbar_wait_hot<kPackedRoleLimit>(&q_empty[t], (q_pend[t] & 1) ^ 1, abort_flag, kTagPacked, 22);
            if (ok && lane == 0) {
              mbar_expect_tx(&q_full[t], C::TILE);
#pragma unroll
              for (int b = 0; b < NB; ++b)
                tma_load_2d(smem + t * C::TILE + b * C::BLOCK, &tmQ, &q_full[t], it->head[t] * D + b * 64,
                            q0 + it->m[t]);
            }
            if (ok) ++q_pend[t];
          }
        }
        release_item();
        for (int j = steps - 1; j >= 0 && ok; --j) {
          if (j < steps - 1) load(&tmK, col, k0 + j * 128);
          load(&tmV, col, k0 + j * 128);
        }
        if (!ok) break;
      }
      if (*abort_flag) {
        // let the copies in flight land before the CTA exits
        for (int i = max(0, issued - C::STAGES); i < issued; ++i)
          mbar_wait_drain(&kv_full[i % C::STAGES], static_cast<uint32_t>(i / C::STAGES) & 1u);
        for (int t = 0; t < 2; ++t)
          if (q_pend[t] > 0) mbar_wait_drain(&q_full[t], static_cast<uint32_t>(q_pend[t] - 1) & 1u);
      }
    } else if (warp == 9) {
      // ---- MMA ----
      // The whole warp runs this with warp-uniform values (counts are broadcast,
      // waits end in a vote), one elected thread issues: operands then stay in
      // uniform registers.  Step by step, tile by tile: P V of the step before (the
      // last step of the item before, at an item's first step), then S of this step.
      const uint32_t q_lo = desc_lo(smem_u32(smem), 16), k_lo = desc_lo(smem_u32(ring), 16);
      const uint32_t v_lo = desc_lo(smem_u32(ring) + C::TILE, C::BLOCK);
      const uint32_t leader = elect_one();
      int n_k = 0;             // steps begun: K is ring load 2 n_k, V is 2 n_k + 1
      uint32_t q_use0 = 0, q_use1 = 0, p_use0 = 0, p_use1 = 0;
      bool pv0 = false, pv1 = false;      // P V of the step before to do, per tile
      uint32_t more0 = 0, more1 = 0;      // it adds to O
      bool last = false;                  // it is its item's last
      int valid = 0;                      // keys of the step before that lie inside the sequence
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
        return __all_sync(0xffffffffu, mbar_wait_hot<kPackedRoleLimit>(bar, parity, abort_flag, kTagPacked, site)) != 0;
      };
      auto full = [&](int i, int site) {
        return wait(&kv_full[i % C::STAGES], static_cast<uint32_t>(i / C::STAGES) & 1u, site);
      };
      // V of the step before has arrived; zero its rows behind the end up to a multiple of 16
      auto v_ready = [&]() {
        const int vt = 2 * n_k - 1;
        if (!full(vt, 32)) return false;
        if (valid & 15) {
          uint8_t* v = ring + (vt % C::STAGES) * C::TILE;
          const int n16 = (16 - (valid & 15)) * (D / 8);
          for (int i = lane; i < n16; i += 32) {
            const int r = valid + i / (D / 8), c = i % (D / 8);
            *reinterpret_cast<uint4*>(v + (c >> 3) * C::BLOCK + r * 128 + ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_shared();
          __syncwarp();
        }
        return true;
      };
      // V of step n_k - 1
      auto issue_pv = [&](auto tile, uint32_t& use, uint32_t more) {
        constexpr int t = decltype(tile)::value;
        if (!wait(&p_full[t], use & 1u, 33)) return false;
        ++use;
        tc_fence_after();
        const uint32_t vd = v_lo + ((n_k - 1) & 1) * (2 * C::TILE / 16);
        if (valid > 112) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // 16 keys: 2048 bytes further
            mma_bf16_ts_lo(leader, tmem + C::O_COL(t), tmem + C::S_COL(t) + kk * 8, vd + kk * 128, C::IDESC_O,
                           kk > 0 ? 1u : more);
        } else {
          for (int kk = 0; kk * 16 < valid; ++kk)
            mma_bf16_ts_lo(leader, tmem + C::O_COL(t), tmem + C::S_COL(t) + kk * 8, vd + kk * 128, C::IDESC_O,
                           kk > 0 ? 1u : more);
        }
        if (last) tc_commit_if(leader, &o_done[t]);
        return true;
      };
      auto issue_s = [&](auto tile, uint32_t& use, bool first, bool end) {
        constexpr int t = decltype(tile)::value;
        if (first) {
          if (!wait(&q_full[t], use & 1u, 35)) return false;
          ++use;
        }
        tc_fence_after();
        const uint32_t qd = q_lo + t * (C::TILE / 16), kd = k_lo + (n_k & 1) * (2 * C::TILE / 16);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 16 columns: 32 bytes further
            mma_bf16_lo(leader, tmem + C::S_COL(t), qd + b * (C::BLOCK / 16) + kk * 2,
                        kd + b * (C::BLOCK / 16) + kk * 2, C::IDESC_S, (b | kk) != 0 ? 1u : 0u);
        tc_commit_if(leader, &s_full[t]);
        if (end) tc_commit_if(leader, &q_empty[t]);
        return true;
      };
      using Zero = std::integral_constant<int, 0>;
      using One = std::integral_constant<int, 1>;
      auto finish = [&]() {  // P V of the last step, where no S follows
        if (!pv0 && !pv1) return true;
        if (!v_ready()) return false;
        if (pv0 && !issue_pv(Zero(), p_use0, more0)) return false;
        if (pv1 && !issue_pv(One(), p_use1, more1)) return false;
        tc_commit_if(leader, &kv_empty[(2 * n_k - 1) % C::STAGES]);
        pv0 = pv1 = false;
        return true;
      };
      while (const PackedItem* it = next_item()) {
        const int n0 = __shfl_sync(0xffffffffu, it->n[0], 0), n1 = __shfl_sync(0xffffffffu, it->n[1], 0);
        const int lk = __shfl_sync(0xffffffffu, it->lk, 0), steps = max(n0, n1);
        release_item();
        // an item without keys brings no step, and many of them may follow: the
        // softmax warps have to get through the item before without one
        if (steps == 0) ok = finish();
        for (int j = steps - 1; j >= 0; --j) {
          const bool any = pv0 || pv1, s0 = j < n0, s1 = j < n1;
          if (!(ok = !any || v_ready())) break;
          if (!(ok = full(2 * n_k, 31))) break;
          if (pv0 && !(ok = issue_pv(Zero(), p_use0, more0))) break;
          if (s0 && !(ok = issue_s(Zero(), q_use0, j == n0 - 1, j == 0))) break;
          if (pv1 && !(ok = issue_pv(One(), p_use1, more1))) break;
          if (s1 && !(ok = issue_s(One(), q_use1, j == n1 - 1, j == 0))) break;
          tc_commit_if(leader, &kv_empty[(2 * n_k) % C::STAGES]);
          if (any) tc_commit_if(leader, &kv_empty[(2 * n_k - 1) % C::STAGES]);
          pv0 = s0, pv1 = s1;
          more0 = j + 1 < n0, more1 = j + 1 < n1;
          last = j == 0;
          valid = min(128, lk - j * 128);
          ++n_k;
        }
        if (!ok) break;
      }
      if (ok) ok = finish();
      // every product and every arrival of its commits has happened before the CTA exits
      tc_commit_if(leader, drain);
      mbar_wait_drain(drain, 0);
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax and epilogue: tile t, one row per thread ----
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + C::S_COL(t), t_o = t_lane + C::O_COL(t);
    uint32_t n_s = 0, n_items = 0;  // steps and items done so far (phases of s_full and o_done)
    bool ok = true;
    while (const PackedItem* it = next_item()) {
      const int steps = it->n[t];
      // last visible key of this row, and of the warp's first
      const int reach = it->m[t] + (warp & 3) * 32 + it->diag, last_key = it->lk - 1;
      const int limit = min(last_key, reach + lane), first_limit = min(last_key, reach);
      float m_use = -INFINITY;
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      for (int j = steps - 1; j >= 0; --j) {
        ok = packed_wait(&s_full[t], n_s & 1u, flags, kTagPacked, 41);
        if (!ok) break;
        tc_fence_after();
        uint32_t r[4][32];
        tmem_ld_32x32b_x32(t_s, r[0]);
        tmem_ld_32x32b_x32(t_s + 32, r[1]);
        tmem_ld_32x32b_x32(t_s + 64, r[2]);
        tmem_ld_32x32b_x32(t_s + 96, r[3]);
        tmem_ld_wait();
        if (j * 128 + 127 > first_limit) {
          const int lim = limit - j * 128;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i > lim) r[c][i] = 0xff800000u;  // -inf
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // independent chains
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            mx4[(i >> 1) & 3] = fmaxf(mx4[(i >> 1) & 3], fmaxf(__uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1])));
        }
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        // powers of two of scaled scores; the maximum in use follows when some row of the warp outgrew it
        mx = fmaxf(mx * p.scale_log2e, m_use);
        if (__any_sync(0xffffffffu, mx > m_use + 8.f)) {
          const float f = mx == -INFINITY ? 1.f : ex2_approx(m_use - mx);
          m_use = mx;
          sum2[0] = __fmul2_rn(sum2[0], make_float2(f, f));
          sum2[1] = __fmul2_rn(sum2[1], make_float2(f, f));
          if (j != steps - 1) {  // S of this step was multiplied after P V of the step before: O is at rest
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(t_o + 16 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st_32x32b_x16(t_o + 16 * c, o);
            }
          }
        }
        const float off = m_use == -INFINITY ? 0.f : -m_use;
        const float2 off2 = make_float2(off, off), scale2 = make_float2(p.scale_log2e, p.scale_log2e);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int k = (c & 1) * 16 + 2 * i;
            const float2 x = __ffma2_rn(
                make_float2(__uint_as_float(r[c >> 1][k]), __uint_as_float(r[c >> 1][k + 1])), scale2, off2);
            const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
            sum2[i & 1] = __fadd2_rn(sum2[i & 1], e);
            const __nv_bfloat162 b = __floats2bfloat162_rn(e.x, e.y);
            pk[i] = *reinterpret_cast<const uint32_t*>(&b);
          }
          tmem_st_32x32b_x8(t_s + 8 * c, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        ++n_s;
      }
      if (!ok) break;
      const int head = it->head[t], rows = min(128, it->lq - it->m[t]) - (warp & 3) * 32;  // rows of this warp's 32
      const long long first = it->q0 + it->m[t] + (warp & 3) * 32;
      __nv_bfloat16* dst = p.out + first * p.ldo + head * D;
      float* lse = p.lse != nullptr && lane < rows ? p.lse + (first + lane) * p.heads + head : nullptr;
      if (it->part >= 0) {
        // a part: maxima, sums and unnormalized output to the workspace, row fastest
        float* part = p.ws + (2ll * blockIdx.x + it->part) * packed_part_floats<D>() + t * (128 * (D + 2)) + row;
        part[0] = m_use;
        part[128] = (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
        if (steps > 0) {
          ok = packed_wait(&o_done[t], n_items++ & 1u, flags, kTagPacked, 44);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(t_o + 32 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) part[(2 + 32 * c + i) * 128] = __uint_as_float(o[i]);
          }
          tc_fence_before();
        }
        release_item();
        continue;
      }
      float inv = 0.f;  // a row that saw no key gives zeros
      bool finite = false;
      if (steps > 0) {
        ok = packed_wait(&o_done[t], n_items++ & 1u, flags, kTagPacked, 43);
        if (!ok) break;
        tc_fence_after();
        const float sum = (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
        // a sum of NaN (with a maximum that is still -inf where every score is one) stays one
        if (sum != 0.f) inv = 1.f / sum;
        finite = sum > 0.f && sum < INFINITY;
        if (lse != nullptr) *lse = sum != 0.f ? (m_use + log2f(sum)) * 0.69314718055994531f : -INFINITY;
      } else if (lse != nullptr) {
        *lse = -INFINITY;
      }
      // 64 columns at a time through shared memory (chunks permuted by the row, so
      // that neither side has bank conflicts), so that a store covers whole lines;
      // a row per thread would touch 32 lines with each
      uint8_t* box = staging + warp * 4096;
      // a lane stores chunk lane % 8 of rows lane / 8, lane / 8 + 4, ... (their places alternate between two)
      const uint8_t* box_even = box + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
      const uint8_t* box_odd = box + (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3) + 4)) << 4);
      __nv_bfloat16* lane_dst = dst + (lane >> 3) * p.ldo + (lane & 7) * 8;
      uint32_t o[D / 32][32];
      if (steps > 0) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) tmem_ld_32x32b_x32(t_o + 32 * c, o[c]);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) o[c][i] = 0u;
      }
      float2 nan2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};  // stays 0 but for infinities and NaN
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              f[e] = __fmul2_rn(make_float2(__uint_as_float(o[2 * c + h][8 * i + 2 * e]),
                                            __uint_as_float(o[2 * c + h][8 * i + 2 * e + 1])),
                                make_float2(inv, inv));
            *reinterpret_cast<uint4*>(box + lane * 128 + (((4 * h + i) ^ (lane & 7)) << 4)) = pack8x2(f);
#pragma unroll
            for (int e = 0; e < 4; ++e) nan2[e & 1] = __ffma2_rn(f[e], make_float2(0.f, 0.f), nan2[e & 1]);
          }
        __syncwarp();
        __nv_bfloat16* to = lane_dst + 64 * c;
        if (rows >= 32) {
#pragma unroll
          for (int i = 0; i < 8; ++i, to += 4 * p.ldo)
            *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(i & 1 ? box_odd + i * 512 : box_even + i * 512);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i, to += 4 * p.ldo)
            if (4 * i + (lane >> 3) < rows)
              *reinterpret_cast<uint4*>(to) =
                  *reinterpret_cast<const uint4*>(i & 1 ? box_odd + i * 512 : box_even + i * 512);
        }
        __syncwarp();
      }
      tc_fence_before();
      const int end = min(it->lk, 128 * steps);
      const bool odd = lane < rows && !((nan2[0].x + nan2[0].y) + (nan2[1].x + nan2[1].y) == 0.f);
      const bool bad = odd && finite && limit + 1 < end;
      // a row that saw no key, in a tile whose step multiplied an infinity or a NaN
      // (0 times which is a NaN): zeros
      const bool blank = odd && inv == 0.f;
      if (__any_sync(0xffffffffu, blank)) {
        __syncwarp();  // the rows' first results are stored
        if (blank)
          for (int c = 0; c < D / 8; ++c) reinterpret_cast<uint4*>(dst + lane * p.ldo)[c] = make_uint4(0u, 0u, 0u, 0u);
      }
      if (__any_sync(0xffffffffu, bad)) {
        const int col = head / p.group * D;
        int* mending = const_cast<int*>(&flags->mending);
        if (lane == 0) atomicAdd(mending, 1);
        packed_mend<D>(bad, limit, end, p.q + (first + lane) * p.ldq + head * D, p.k + it->k0 * p.ldk + col, p.ldk,
                       p.v + it->k0 * p.ldv + col, p.ldv, dst + lane * p.ldo, p.scale_log2e, m_use, inv, -1);
        if (lane == 0) atomicSub(mending, 1);
      }
      release_item();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) {
    __syncwarp();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Joins the partial results of the items that k_attn_packed cut.  CTA (c, y)
// looks at the item that CTA c of that kernel began and did not finish, tile
// y / 4, 32 rows: the parts are its place 1, then place 0 of the CTAs behind it
// up to the one that ends the item, added up in that order.  A warp per D / 8
// columns, a lane per row.
template <int D>
__global__ void __launch_bounds__(256) k_attn_packed_join(const PackedParams p, int ctas) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int N = D / 8;
  const PackedRecord* rec = reinterpret_cast<const PackedRecord*>(p.ws + 2ll * ctas * packed_part_floats<D>());
  const int c0 = blockIdx.x, t = blockIdx.y >> 2;
  const PackedRecord r = rec[2 * c0 + 1];
  if (!r.used) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = (blockIdx.y & 3) * 32 + lane;
  const bool live = row < (t ? r.rows[1] : r.rows[0]);
  if (!__any_sync(0xffffffffu, live)) return;
  auto part = [&](int c) {
    return p.ws + (2ll * c + (c == c0 ? 1 : 0)) * packed_part_floats<D>() + t * (128 * (D + 2)) + row;
  };
  int c1 = c0 + 1;
  while (c1 < ctas - 1 && !rec[2 * c1].ends) ++c1;
  float m = -INFINITY;
  for (int c = c0; c <= c1; ++c) m = fmaxf(m, part(c)[0]);
  float sum = 0.f, acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  for (int c = c0; c <= c1; ++c) {
    const float* w = part(c);
    if (w[128] == 0.f) continue;  // saw no key: nothing was written behind the sum
    const float f = ex2_approx(w[0] - m);
    sum = fmaf(w[128], f, sum);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = fmaf(w[(2 + warp * N + i) * 128], f, acc[i]);
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  const long long grow = (t ? r.row[1] : r.row[0]) + row;
  const int head = t ? r.head[1] : r.head[0];
  __nv_bfloat16* dst = p.out + grow * p.ldo + head * D;
  float nan = 0.f;  // stays 0 but for infinities and NaN
#pragma unroll
  for (int i = 0; i < N; ++i) nan = fmaf(acc[i], 0.f, nan);
  if (live) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = acc[8 * i + e] * inv;
      reinterpret_cast<uint4*>(dst + warp * N)[i] = pack8(f);
    }
    if (p.lse != nullptr && warp == 0)
      p.lse[grow * p.heads + head] = sum != 0.f ? (m + log2f(sum)) * 0.69314718055994531f : -INFINITY;
  }
  const int end = t ? r.end[1] : r.end[0], limit = min(end - 1, (t ? r.limit[1] : r.limit[0]) + row);
  const bool bad = live && sum > 0.f && sum < INFINITY && limit + 1 < end && !(nan == 0.f);
  if (__any_sync(0xffffffffu, bad)) {
    const int col = head / p.group * D;
    packed_mend<D>(bad, limit, end, p.q + grow * p.ldq + head * D, p.k + r.k0 * p.ldk + col, p.ldk,
                   p.v + r.k0 * p.ldv + col, p.ldv, dst, p.scale_log2e, m, inv, warp);
  }
}

}  // namespace qib
