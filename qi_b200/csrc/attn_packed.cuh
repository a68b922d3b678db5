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
// warp 9 MMA (10 and 11 fill up their warpgroup).  A softmax thread holds a
// whole row of S, so the softmax warpgroups take 216 registers a thread and
// the third leaves them all but 72 (of 168 at launch: 256 x 216 + 128 x 72 =
// 64,512, all of them).  CTAs are persistent; each takes every gridDim.x-th item, longest
// items first, the direction alternating from round to round.  The order is a
// function of cu_q alone: level L (the L-th query block of every sequence that
// has one) from the last to the first, so no list of items is stored.
//
// Rows behind a sequence's end belong to its neighbour: scores of such keys
// are replaced (not added to), the V rows of the last 16-key step behind the
// end are zeroed in shared memory, further steps are not multiplied, and
// output rows are stored one by one.  So nothing, NaN included, passes from
// one sequence to another.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "attn_short.cuh"
#include "launch_count.cuh"
#include "sm100_ptx.cuh"

namespace qib {

constexpr unsigned int kTagPacked = 0x900u;

struct PackedParams {
  const int* cu_q;   // [n_seq + 1]
  const int* cu_k;
  int n_seq, total_q, total_k;
  int heads, kv_heads, group;
  int pair_heads;    // 1: an item is two heads x 128 tokens, 0: one head x 256 tokens
  int causal;
  float scale_log2e;
  __nv_bfloat16* out;
  long long ldo;
  float* lse;        // [total_q, heads] or nullptr
};

// Descriptor of an operand whose rows are the K extent (MN-major): rows of 64
// elements (128 B, 128-byte swizzle), 8-row groups 1024 B apart, blocks of 64
// MN elements `lead` bytes apart.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_addr, uint32_t lead) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(lead >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
      "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

template <int D>
struct PackedCfg {
  static constexpr int TILE = 128 * D * 2;       // bytes of a 128-row operand tile (D / 64 swizzled blocks)
  static constexpr int BLOCK = 128 * 128;        // bytes of one 64-column block
  static constexpr int STAGES = D == 128 ? 4 : 8;
  static constexpr int THREADS = 384;
  static constexpr int SMEM = (2 + STAGES) * TILE + 1024 + 256;
  static constexpr int TMEM_COLS = 512;
  __host__ __device__ static constexpr uint32_t S_COL(int t) { return t * 128; }
  __host__ __device__ static constexpr uint32_t O_COL(int t) { return 256 + t * D; }
  static constexpr uint32_t IDESC_S = make_idesc(kDF32, kFmtBF16, kFmtBF16, 128, 128);
  static constexpr uint32_t IDESC_O = make_idesc(kDF32, kFmtBF16, kFmtBF16, 128, D) | (1u << 16);  // B is MN-major
};

// One work item.
struct PackedItem {
  int q0, lq, k0, lk;  // first rows and lengths of the sequence
  int m[2], head[2];   // first token (inside the sequence) and head of the two tiles
  int n[2];            // 128-key steps of the two tiles (0: nothing visible, or no rows)
};

// The items of one CTA in order; every warp walks the same sequence.
struct PackedSched {
  const PackedParams& p;
  int lane, rows_per_item, heads_items;
  int level, chunk;
  int base;            // items before the current (level, chunk)
  int round;
  unsigned mask;       // active sequences of the chunk
  int blocks0;         // query blocks of sequence `lane` (chunk 0)

  __device__ __forceinline__ int seq_blocks(int b) const {
    if (b >= p.n_seq) return 0;
    int q0, lq;
    span(p.cu_q, b, p.total_q, q0, lq);
    return (lq + rows_per_item - 1) / rows_per_item;
  }
  // rows of sequence b, clamped to the tensor (bad prefix sums read and write inside it)
  __device__ __forceinline__ static void span(const int* cu, int b, int total, int& first, int& len) {
    first = min(max(cu[b], 0), total);
    len = min(max(cu[b + 1], first), total) - first;
  }
  __device__ __forceinline__ PackedSched(const PackedParams& pp) : p(pp) {
    lane = threadIdx.x & 31;
    rows_per_item = p.pair_heads ? 128 : 256;
    heads_items = p.pair_heads ? p.heads / 2 : p.heads;
    int most = 0;
    for (int b = lane; b < p.n_seq; b += 32) most = max(most, seq_blocks(b));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    blocks0 = seq_blocks(lane);
    level = most - 1;
    chunk = 0;
    base = 0;
    round = 0;
    mask = __ballot_sync(0xffffffffu, blocks0 > level);
  }
  __device__ __forceinline__ bool next(PackedItem& it) {
    const int G = gridDim.x;
    const int target = round * G + ((round & 1) ? G - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x));
    if (level < 0) return false;
    while (target >= base + __popc(mask) * heads_items) {
      base += __popc(mask) * heads_items;
      chunk += 32;
      if (chunk >= p.n_seq) {
        chunk = 0;
        if (--level < 0) return false;
      }
      mask = __ballot_sync(0xffffffffu, (chunk == 0 ? blocks0 : seq_blocks(chunk + lane)) > level);
    }
    ++round;
    const int idx = target - base;
    const int nth = idx / heads_items, hi = idx - nth * heads_items;
    unsigned mm = mask;
    for (int i = 0; i < nth; ++i) mm &= mm - 1;
    const int b = chunk + __ffs(mm) - 1;
    span(p.cu_q, b, p.total_q, it.q0, it.lq);
    span(p.cu_k, b, p.total_k, it.k0, it.lk);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      it.head[t] = p.pair_heads ? 2 * hi + t : hi;
      it.m[t] = level * rows_per_item + (p.pair_heads ? 0 : 128 * t);
      const int rows = min(128, it.lq - it.m[t]);
      const int visible = p.causal ? min(it.lk, it.m[t] + rows + it.lk - it.lq) : it.lk;
      it.n[t] = rows > 0 && visible > 0 ? (visible + 127) / 128 : 0;
    }
    return true;
  }
};

template <int D>
__global__ void __launch_bounds__(384, 1)
k_attn_packed(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
              const __grid_constant__ CUtensorMap tmV, const PackedParams p) {
  using C = PackedCfg<D>;
  constexpr int NB = D / 64;  // 64-column blocks of a tile
  extern __shared__ uint8_t packed_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(packed_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * C::TILE;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(ring + C::STAGES * C::TILE);  // [2]
  uint64_t* q_empty = q_full + 2;                                              // [2]
  uint64_t* s_full = q_full + 4;                                               // [2]
  uint64_t* p_half = q_full + 6;                                               // [2]
  uint64_t* p_full = q_full + 8;                                               // [2]
  uint64_t* o_done = q_full + 10;                                              // [2]
  uint64_t* drain = q_full + 12;
  uint64_t* kv_full = q_full + 13;                                             // [STAGES]
  uint64_t* kv_empty = kv_full + C::STAGES;                                    // [STAGES]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kv_empty + C::STAGES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_half[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_done[t], 1);
    }
    mbar_init(drain, 1);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    *abort_flag = 0;
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
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    PackedSched sched(p);
    PackedItem it;
    if (warp == 8) {
      // ---- TMA ----
      int stage = 0, issued = 0;
      uint32_t use = 0;  // times the ring has been gone round
      bool ok = true;
      int q_pend[2] = {0, 0};  // Q loads issued
      auto load = [&](const CUtensorMap* map, int col, int row) {
        ok = ok && mbar_wait_hot(&kv_empty[stage], (use & 1u) ^ 1u, abort_flag, kTagPacked, 21);
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
      while (ok && sched.next(it)) {
        const int steps = max(it.n[0], it.n[1]);
        if (steps == 0) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (it.n[t] == 0 || !ok) continue;
          ok = mbar_wait_hot(&q_empty[t], (q_pend[t] & 1) ^ 1, abort_flag, kTagPacked, 22);
          if (ok && lane == 0) {
            mbar_expect_tx(&q_full[t], C::TILE);
#pragma unroll
            for (int b = 0; b < NB; ++b)
              tma_load_2d(smem + t * C::TILE + b * C::BLOCK, &tmQ, &q_full[t], it.head[t] * D + b * 64, it.q0 + it.m[t]);
          }
          if (ok) ++q_pend[t];
        }
        const int col = it.head[0] / p.group * D;
        for (int j = steps - 1; j >= 0 && ok; --j) {
          load(&tmK, col, it.k0 + j * 128);
          load(&tmV, col, it.k0 + j * 128);
        }
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
      // Step by step, tile by tile: P V of the step before (the last step of the
      // item before, at an item's first step), then S of this step.
      const uint32_t smem_q = smem_u32(smem), ring_u = smem_u32(ring);
      int n_k = 0;             // steps begun: K is ring load 2 n_k, V is 2 n_k + 1
      int q_use[2] = {0, 0}, p_use[2] = {0, 0};
      bool ok = true;
      bool pv[2] = {false, false}, more[2] = {false, false};  // P V to do; it adds to O
      int valid = 0;           // keys of the step before that lie inside the sequence
      auto full = [&](int i, int site) {
        return mbar_wait_hot(&kv_full[i % C::STAGES], static_cast<uint32_t>(i / C::STAGES) & 1u, abort_flag, kTagPacked,
                         site);
      };
      // V of the step before has arrived; zero its rows behind the end up to a multiple of 16
      auto v_ready = [&](int vt) {
        if (!full(vt, 32)) return false;
        if (valid & 15) {
          const int n16 = (16 - (valid & 15)) * (D / 8);
          for (int i = lane; i < n16; i += 32) {
            const int r = valid + i / (D / 8), c = i % (D / 8);
            *reinterpret_cast<uint4*>(ring + (vt % C::STAGES) * C::TILE + (c >> 3) * C::BLOCK + r * 128 +
                                      (((c & 7) ^ (r & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_async_shared();
          __syncwarp();
        }
        return true;
      };
      auto issue_pv = [&](int t, int vt) {
        if (!mbar_wait_hot(&p_full[t], static_cast<uint32_t>(p_use[t]++) & 1u, abort_flag, kTagPacked, 33)) return false;
        tc_fence_after();
        const int k16 = (valid + 15) / 16;
        if (elect_one()) {
          const uint64_t vd = sw128_mnmajor_desc(ring_u + (vt % C::STAGES) * C::TILE, C::BLOCK);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)  // 16 keys: 2048 bytes further
            if (kk < k16)
              mma_bf16_ts(tmem + C::O_COL(t), tmem + C::S_COL(t) + kk * 8, vd + kk * 128, C::IDESC_O,
                          kk > 0 || more[t] ? 1u : 0u);
          tc_commit(&o_done[t]);
        }
        __syncwarp();
        return true;
      };
      while (ok && sched.next(it)) {
        const int steps = max(it.n[0], it.n[1]);
        for (int j = steps - 1; j >= 0 && ok; --j) {
          const int kt = 2 * n_k, vt = kt - 1;
          const bool any = pv[0] || pv[1];
          if (any) ok = v_ready(vt);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && pv[t]) ok = issue_pv(t, vt);
            if (t == 0 && ok) ok = full(kt, 31);
            const bool s = j < it.n[t];
            if (ok && s) {
              if (j == it.n[t] - 1)
                ok = mbar_wait_hot(&q_full[t], static_cast<uint32_t>(q_use[t]++) & 1u, abort_flag, kTagPacked, 35);
              tc_fence_after();
              if (ok && elect_one()) {
                const uint64_t qd = sw128_kmajor_desc(smem_q + t * C::TILE);
                const uint64_t kd = sw128_kmajor_desc(ring_u + (kt % C::STAGES) * C::TILE);
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                  for (int kk = 0; kk < 4; ++kk)  // 16 columns: 32 bytes further
                    mma_bf16(tmem + C::S_COL(t), qd + b * (C::BLOCK / 16) + kk * 2, kd + b * (C::BLOCK / 16) + kk * 2,
                             C::IDESC_S, (b | kk) != 0 ? 1u : 0u);
                tc_commit(&s_full[t]);
                if (j == 0) tc_commit(&q_empty[t]);
              }
              __syncwarp();
            }
            pv[t] = s;
            more[t] = j + 1 < it.n[t];
          }
          if (!ok) break;
          if (elect_one()) {
            tc_commit(&kv_empty[kt % C::STAGES]);
            if (any) tc_commit(&kv_empty[vt % C::STAGES]);
          }
          __syncwarp();
          valid = min(128, it.lk - j * 128);
          ++n_k;
        }
      }
      if (ok && n_k > 0) {
        const int vt = 2 * n_k - 1;
        ok = v_ready(vt);
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (ok && pv[t]) ok = issue_pv(t, vt);
      }
      if (elect_one()) {  // every product and every arrival of its commits has happened before the CTA exits
        tc_commit(drain);
        mbar_wait_drain(drain, 0);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    PackedSched sched(p);
    PackedItem it;
    // ---- softmax and epilogue: tile t, one row per thread ----
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + C::S_COL(t), t_o = t_lane + C::O_COL(t);
    uint32_t n_s = 0;  // steps done so far (phases of s_full and o_done)
    bool ok = true;
    while (ok && sched.next(it)) {
      const int m = t ? it.m[1] : it.m[0], steps = t ? it.n[1] : it.n[0], head = t ? it.head[1] : it.head[0];
      const int token = m + row;
      // last visible key of this row
      const int limit = min(it.lk - 1, p.causal ? token + it.lk - it.lq : it.lk - 1);
      const int first_limit = min(it.lk - 1, p.causal ? m + it.lk - it.lq : it.lk - 1);
      float m_use = -INFINITY;
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      for (int j = steps - 1; j >= 0; --j) {
        ok = mbar_wait_hot(&s_full[t], n_s & 1u, abort_flag, kTagPacked, 41);
        if (!ok) break;
        tc_fence_after();
        uint32_t r[4][32];
        tmem_ld_32x32b_x32(t_s, r[0]);
        tmem_ld_32x32b_x32(t_s + 32, r[1]);
        tmem_ld_wait();
        tmem_ld_32x32b_x32(t_s + 64, r[2]);
        tmem_ld_32x32b_x32(t_s + 96, r[3]);
        const bool cut = j * 128 + 127 > first_limit;
        const int lim = limit - j * 128;
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // independent chains
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c == 2) tmem_ld_wait();
          if (cut) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i > lim) r[c][i] = 0xff800000u;  // -inf
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            mx4[(i >> 1) & 3] = fmaxf(mx4[(i >> 1) & 3], fmaxf(__uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1])));
        }
        // powers of two of scaled scores; the maximum in use follows when some row of the warp outgrew it
        const float mx =
            fmaxf(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2e, m_use);
        if (__any_sync(0xffffffffu, mx > m_use + 8.f)) {
          const float f = mx == -INFINITY ? 1.f : ex2_approx(m_use - mx);
          m_use = mx;
          sum2[0] = __fmul2_rn(sum2[0], make_float2(f, f));
          sum2[1] = __fmul2_rn(sum2[1], make_float2(f, f));
          if (j != steps - 1) {
            ok = mbar_wait_hot(&o_done[t], (n_s - 1) & 1u, abort_flag, kTagPacked, 42);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(t_o + 32 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st_32x32b_x32(t_o + 32 * c, o);
            }
          }
        }
        const float off = m_use == -INFINITY ? 0.f : -m_use;
        const float2 off2 = make_float2(off, off), scale2 = make_float2(p.scale_log2e, p.scale_log2e);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int c = 2 * h; c < 2 * h + 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 x = __ffma2_rn(
                  make_float2(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])), scale2, off2);
              const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
              sum2[i & 1] = __fadd2_rn(sum2[i & 1], e);
              const __nv_bfloat162 b = __floats2bfloat162_rn(e.x, e.y);
              pk[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            tmem_st_32x32b_x16(t_s + 16 * c, pk);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        ++n_s;
      }
      if (!ok) break;
      const float sum = (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
      const bool live = token < it.lq;
      const long long grow = it.q0 + token;
      __nv_bfloat16* dst = p.out + grow * p.ldo + head * D;
      if (live && p.lse != nullptr)
        p.lse[grow * p.heads + head] = sum > 0.f ? (m_use + log2f(sum)) * 0.69314718055994531f : -INFINITY;
      if (steps == 0) {
        if (live)
#pragma unroll
          for (int c = 0; c < D / 8; ++c) reinterpret_cast<uint4*>(dst)[c] = make_uint4(0u, 0u, 0u, 0u);
        continue;
      }
      ok = mbar_wait_hot(&o_done[t], (n_s - 1) & 1u, abort_flag, kTagPacked, 43);
      if (!ok) break;
      tc_fence_after();
      const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(t_o + 32 * c, o);
        tmem_ld_wait();
        if (live) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[8 * i + e]) * inv;
            reinterpret_cast<uint4*>(dst)[c * 4 + i] = pack8(f);
          }
        }
      }
      tc_fence_before();
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

}  // namespace qib
