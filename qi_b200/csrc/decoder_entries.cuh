// C entry points of the decoder-block operators: residual RMSNorm to 8 bits,
// multi-axis rotary positions with the cache write, packed-prompt attention
// and paged one-token attention.  Included by qi_b200.cu (the kernels share
// that module's device status word).
#pragma once

#include <cfloat>

#include "attn_packed.cuh"
#include "attn_paged.cuh"
#include "rms_quant.cuh"
#include "rope_axes.cuh"

namespace qib {

static inline bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// The kernels take powers of two: scale log2(e) has to be finite as well.
constexpr float kLog2e = 1.4426950408889634f;
static inline bool softmax_scale_ok(float scale) { return scale > 0.0f && scale * kLog2e <= FLT_MAX; }

// Dynamic shared memory above 48 KB, once per kernel and device.
template <auto KERNEL>
static int allow_smem(int bytes) {
  static std::atomic<bool> done[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return QI_B200_ECUDA;
  if (done[dev].load(std::memory_order_acquire)) return QI_B200_OK;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return QI_B200_ECUDA;
  done[dev].store(true, std::memory_order_release);
  return QI_B200_OK;
}

static int launched(cudaError_t e) {
  count_launches(1);
  return e == cudaSuccess ? QI_B200_OK : QI_B200_ECUDA;
}

// Every 16-byte chunk of a head row starts on a 16-byte boundary.
static int check_paged_cache(const qi_b200_paged_cache* c, int kv_heads, int head_dim) {
  if (c->k == nullptr || c->v == nullptr) return QI_B200_EINVAL;
  if (c->pages < 0 || c->page_size <= 0) return QI_B200_ESHAPE;
  if (c->fp8 && (c->scale[0] == nullptr || c->scale[1] == nullptr)) return QI_B200_EINVAL;
  const int unit = c->fp8 ? 16 : 8;
  for (int i = 0; i < 2; ++i) {
    if (c->page_stride[i] < 0 || c->slot_stride[i] < 0 || c->head_stride[i] < 0) return QI_B200_ESHAPE;
    if (c->page_stride[i] % unit || c->slot_stride[i] % unit || c->head_stride[i] % unit) return QI_B200_EALIGN;
    if (kv_heads > 1 && c->head_stride[i] < head_dim) return QI_B200_ESHAPE;
  }
  return aligned16(c->k) && aligned16(c->v) ? QI_B200_OK : QI_B200_EALIGN;
}

template <int FMT>
static int launch_rms_quant(const RmsQuantParams& p, cudaStream_t stream) {
  const int nvec = p.D / 8;
  // chunks per thread: 4, so that a row's loads are in flight together; a few rows
  // spread over more threads instead.  Measured with 1 and 4 (INT8, residual, us):
  // 200 rows of 1024 / 4096 / 8192 2.4, 3.5, 4.7 against 3.7, 4.1, 4.7; 256 rows
  // 2.4, 3.5, 6.1 against 3.8, 4.1, 4.8; 777 rows 2.9, 7.4, 10.8 against 3.8, 6.9,
  // 9.9; 2048 rows 5.0, 15.2, 26.7 against 4.6, 11.2, 25.0 (1024-wide rows alone
  // would gain from 1 up to 1024 rows)
  const int C = p.M < 256 ? 1 : 4;
  int T = std::min(512, (nvec + 32 * C - 1) / (32 * C) * 32);
  int p2 = 32;
  while (p2 < T) p2 *= 2;
  T = p2;  // power of two: rows pack evenly into a CTA
  const int c = (nvec + T - 1) / T;
  const int block = std::max(T, 256);
  const dim3 grid((p.M + block / T - 1) / (block / T));
  if (c <= 1) return launched(launch_pdl(k_rms_quant<1, FMT>, grid, dim3(block), 0, stream, 1, p, T));
  if (c <= 2) return launched(launch_pdl(k_rms_quant<2, FMT>, grid, dim3(block), 0, stream, 1, p, T));
  return launched(launch_pdl(k_rms_quant<4, FMT>, grid, dim3(block), 0, stream, 1, p, T));
}

template <bool IL>
static int launch_rope(const RopeAxesParams& p, int cache, cudaStream_t stream) {
  const dim3 grid((p.M + p.tokens - 1) / p.tokens), block(kRopeThreads);
  if (cache == 0) return launched(launch_pdl(k_rope_axes<IL, 0>, grid, block, 0, stream, 1, p));
  if (cache == 1) return launched(launch_pdl(k_rope_axes<IL, 1>, grid, block, 0, stream, 1, p));
  return launched(launch_pdl(k_rope_axes<IL, 2>, grid, block, 0, stream, 1, p));
}

// Work items of a packed batch, at most: the partial query blocks of the
// sequences are bounded by their number.
static long long packed_items(int n_seq, int total_q, int heads, int kv_heads) {
  const bool pair = heads / kv_heads % 2 == 0;
  return (static_cast<long long>(total_q) / (pair ? 128 : 256) + n_seq) * (pair ? heads / 2 : heads);
}

// Whether a packed batch may profit from cut items (the kernel decides, it
// knows the lengths): with more than 16 items per SM the longest-first order
// is even enough by itself, and below 8 key steps an item is too short.
static size_t packed_workspace(int n_seq, int total_q, int total_k, int heads, int kv_heads, int head_dim, int num_sms) {
  if (packed_items(n_seq, total_q, heads, kv_heads) > 16ll * num_sms || total_k <= 7 * 128) return 0;
  return static_cast<size_t>(num_sms) * 2 *
         ((head_dim == 128 ? packed_part_floats<128>() : packed_part_floats<64>()) * sizeof(float) +
          sizeof(PackedRecord));
}

template <int D>
static int launch_packed(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv,
                         const PackedParams& p, int num_sms, cudaStream_t stream) {
  using C = PackedCfg<D>;
  CUtensorMap tq, tk, tv;
  int rc;
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint64_t wq = static_cast<uint64_t>(p.heads) * D, wk = static_cast<uint64_t>(p.kv_heads) * D;
  if ((rc = make_tmap_2d(&tq, q, bf, wq, p.total_q, ldq * 2, 64, 128))) return rc;
  // without keys nothing is loaded; the maps then only have to be valid
  const bool keys = p.total_k > 0;
  if ((rc = make_tmap_2d(&tk, keys ? k : q, bf, keys ? wk : wq, keys ? p.total_k : p.total_q, (keys ? ldk : ldq) * 2,
                         64, 128)))
    return rc;
  if ((rc = make_tmap_2d(&tv, keys ? v : q, bf, keys ? wk : wq, keys ? p.total_k : p.total_q, (keys ? ldv : ldq) * 2,
                         64, 128)))
    return rc;
  if ((rc = allow_smem<&k_attn_packed<D>>(C::SMEM))) return rc;
  const long long items = packed_items(p.n_seq, p.total_q, p.heads, p.kv_heads);
  if (items > 0x7fff0000ll) return QI_B200_ETOOBIG;  // the kernel counts items in 32 bits
  // with a workspace every SM has a place in it
  const int grid = p.ws != nullptr ? num_sms : static_cast<int>(std::min<long long>(num_sms, std::max(1ll, items)));
  rc = launched(launch_pdl(k_attn_packed<D>, dim3(grid), dim3(C::THREADS), C::SMEM, stream, 1, tq, tk, tv, p));
  if (rc || p.ws == nullptr) return rc;
  return launched(launch_pdl(k_attn_packed_join<D>, dim3(grid, 8), dim3(256), 0, stream, 1, p, grid));
}

// log2 of the most key heads an item may hold: up to 8, evenly.
static int paged_most_teams(int kv_heads) {
  int s = 0;
  while (s < 3 && kv_heads % (2 << s) == 0) ++s;
  return s;
}

template <int D, bool FP8, int HT>
static int launch_paged_tiles(const PagedParams& p, int G, cudaStream_t stream) {
  constexpr int smem = paged_smem<D, FP8, HT>();
  if (int rc = allow_smem<&k_attn_paged<D, FP8, HT>>(smem)) return rc;
  return launched(
      launch_pdl(k_attn_paged<D, FP8, HT>, dim3(G), dim3(PagedCfg<D, FP8>::THREADS), smem, stream, 1, p));
}

template <int D, bool FP8>
static int launch_paged(const PagedParams& p, int G, cudaStream_t stream) {
  int rc = p.group <= 8 ? launch_paged_tiles<D, FP8, 1>(p, G, stream) : launch_paged_tiles<D, FP8, 2>(p, G, stream);
  if (rc) return rc;
  const int heads = std::min(kPagedRows, p.group) << p.team_shift;  // query heads of an item
  return launched(
      launch_pdl(k_attn_paged_join<D>, dim3(G, heads), dim3(kPagedJoinWarps * 32), 0, stream, 1, p, G));
}

}  // namespace qib

extern "C" {

int qi_b200_rms_norm_quant(int kind, const void* x_bf16, long long ldx, const void* y_bf16, long long ldy,
                           void* x_out_bf16, long long ld_out, const void* weight_bf16, void* q, float* scales,
                           void* xn_bf16, int M, int D, float eps, cudaStream_t stream) {
  if (M < 0 || D <= 0 || D % 8 != 0 || D > kRmsMaxDim) return QI_B200_ESHAPE;
  if (kind != QI_B200_KIND_INT8 && kind != QI_B200_KIND_FP8_E4M3 && kind != QI_B200_KIND_BF16) return QI_B200_EINVAL;
  if (M == 0) return QI_B200_OK;
  const bool codes = kind != QI_B200_KIND_BF16;
  if (x_bf16 == nullptr || weight_bf16 == nullptr || (codes && (q == nullptr || scales == nullptr)) ||
      (!codes && xn_bf16 == nullptr) || (y_bf16 != nullptr && x_out_bf16 == nullptr) || !(eps >= 0.f))
    return QI_B200_EINVAL;
  if (ldx < D || ldx % 8 || (y_bf16 != nullptr && (ldy < D || ldy % 8 || ld_out < D || ld_out % 8)))
    return QI_B200_ESHAPE;
  if (!aligned16(x_bf16) || !aligned16(weight_bf16) || (y_bf16 && (!aligned16(y_bf16) || !aligned16(x_out_bf16))) ||
      (xn_bf16 && !aligned16(xn_bf16)) || (codes && !aligned8(q)))
    return QI_B200_EALIGN;
  DeviceInfo* di = nullptr;
  if (int rc = device_info(&di)) return rc;
  RmsQuantParams p;
  p.x = static_cast<const __nv_bfloat16*>(x_bf16);
  p.ldx = ldx;
  p.y = static_cast<const __nv_bfloat16*>(y_bf16);
  p.ldy = ldy;
  p.h = static_cast<__nv_bfloat16*>(x_out_bf16);
  p.ldh = ld_out;
  p.w = static_cast<const __nv_bfloat16*>(weight_bf16);
  p.q = codes ? static_cast<uint8_t*>(q) : nullptr;
  p.s = scales;
  p.xn = static_cast<__nv_bfloat16*>(xn_bf16);
  p.M = M;
  p.D = D;
  p.eps = eps;
  if (kind == QI_B200_KIND_INT8) return launch_rms_quant<1>(p, stream);
  if (kind == QI_B200_KIND_FP8_E4M3) return launch_rms_quant<2>(p, stream);
  return launch_rms_quant<0>(p, stream);
}

int qi_b200_rope_axes(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv,
                      void* q_out, long long ldq_out, void* k_out, long long ldk_out, const void* positions,
                      int positions64, const double* freqs, const int* axes_of, int pairs, int axes, int interleaved,
                      int M, int heads, int kv_heads, int head_dim, const qi_b200_paged_cache* cache,
                      const void* slots, int slots64, cudaStream_t stream) {
  if (M < 0 || heads <= 0 || kv_heads < 0 || head_dim <= 0 || head_dim % 16 || head_dim > 2 * kRopeMaxPairs ||
      pairs <= 0 || pairs % 8 || 2 * pairs > head_dim || axes < 1)
    return QI_B200_ESHAPE;
  if (M == 0) return QI_B200_OK;
  if (q == nullptr || q_out == nullptr || positions == nullptr || freqs == nullptr || axes_of == nullptr)
    return QI_B200_EINVAL;
  if (kv_heads > 0 && (k == nullptr || (cache == nullptr ? k_out == nullptr : (v == nullptr || slots == nullptr))))
    return QI_B200_EINVAL;
  if (cache != nullptr && kv_heads == 0) return QI_B200_EINVAL;
  const long long wq = static_cast<long long>(heads) * head_dim, wk = static_cast<long long>(kv_heads) * head_dim;
  if (ldq < wq || ldq % 8 || ldq_out < wq || ldq_out % 8) return QI_B200_ESHAPE;
  if (!aligned16(q) || !aligned16(q_out)) return QI_B200_EALIGN;
  if (kv_heads > 0) {
    if (ldk < wk || ldk % 8) return QI_B200_ESHAPE;
    if (!aligned16(k)) return QI_B200_EALIGN;
    if (k_out != nullptr && (ldk_out < wk || ldk_out % 8)) return QI_B200_ESHAPE;
    if (k_out != nullptr && !aligned16(k_out)) return QI_B200_EALIGN;
    if (cache != nullptr && (ldv < wk || ldv % 8)) return QI_B200_ESHAPE;
    if (cache != nullptr && !aligned16(v)) return QI_B200_EALIGN;
  }
  if (cache != nullptr)
    if (int rc = check_paged_cache(cache, kv_heads, head_dim)) return rc;
  DeviceInfo* di = nullptr;
  if (int rc = device_info(&di)) return rc;
  RopeAxesParams p = {};
  p.in[0] = static_cast<const __nv_bfloat16*>(q);
  p.in[1] = static_cast<const __nv_bfloat16*>(k);
  p.in[2] = static_cast<const __nv_bfloat16*>(v);
  p.ld_in[0] = ldq;
  p.ld_in[1] = ldk;
  p.ld_in[2] = ldv;
  p.out[0] = static_cast<__nv_bfloat16*>(q_out);
  p.out[1] = static_cast<__nv_bfloat16*>(k_out);
  p.ld_out[0] = ldq_out;
  p.ld_out[1] = ldk_out;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.head_dim = head_dim;
  p.pairs = pairs;
  p.axes = axes;
  p.pos = positions;
  p.pos64 = positions64;
  p.freq = freqs;
  p.axis = axes_of;
  p.M = M;
  int kind = 0;
  if (cache != nullptr) {
    kind = cache->fp8 ? 2 : 1;
    p.cache[0] = cache->k;
    p.cache[1] = cache->v;
    for (int c = 0; c < 2; ++c) {
      p.page_stride[c] = cache->page_stride[c];
      p.slot_stride[c] = cache->slot_stride[c];
      p.head_stride[c] = cache->head_stride[c];
      p.scale[c] = cache->scale[c];
      p.scale_per_head[c] = cache->scale_per_head[c];
    }
    p.slots_total = static_cast<long long>(cache->pages) * cache->page_size;
    p.page_size = cache->page_size;
    p.slots = slots;
    p.slots64 = slots64;
  }
  // tokens per CTA: one where there are few (64 rows 2.9 us against 3.4 with two),
  // two from four CTAs per SM up (3120 rows 16.3 us against 18.4 and 17.1 with one
  // and four), four from eight up (16384 rows 70 us against 77 with two)
  p.tokens = M >= 4 * 8 * di->num_sms ? kRopeMaxTokens : (M >= 2 * 4 * di->num_sms ? 2 : 1);
  const long long units = static_cast<long long>(heads + (cache ? 2 : 1) * kv_heads) * (head_dim / 16);
  if (ldq > kRopeMaxStride || ldk > kRopeMaxStride || ldv > kRopeMaxStride || units > kRopeMaxUnits)
    return QI_B200_ETOOBIG;
  p.inv_token = static_cast<unsigned>(((1ull << 32) + units - 1) / units);
  p.inv_units = static_cast<unsigned>(((1ull << 32) + head_dim / 16 - 1) / (head_dim / 16));
  return interleaved ? launch_rope<true>(p, kind, stream) : launch_rope<false>(p, kind, stream);
}

int qi_b200_attention_packed(const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv,
                             void* out, long long ldo, float* lse, const int* cu_q, const int* cu_k, int n_seq,
                             int total_q, int total_k, int heads, int kv_heads, int head_dim, int flags, float scale,
                             void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (head_dim != 64 && head_dim != 128) return QI_B200_ESHAPE;
  if (n_seq < 0 || total_q < 0 || total_k < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return QI_B200_ESHAPE;
  if (flags & ~(QI_B200_ATTN_CAUSAL | QI_B200_ATTN_ZERO_REST)) return QI_B200_EINVAL;
  const bool zero_rest = (flags & QI_B200_ATTN_ZERO_REST) != 0;
  if (total_q == 0 || (n_seq == 0 && !zero_rest)) return QI_B200_OK;
  if (static_cast<long long>(total_q) + total_k > 0x3fffffff) return QI_B200_ETOOBIG;  // key places in 32 bits
  if (q == nullptr || out == nullptr || cu_q == nullptr || cu_k == nullptr || (total_k > 0 && (!k || !v)))
    return QI_B200_EINVAL;
  if (!softmax_scale_ok(scale)) return QI_B200_EINVAL;
  const long long wq = static_cast<long long>(heads) * head_dim, wk = static_cast<long long>(kv_heads) * head_dim;
  if (ldq < wq || ldo < wq || ldq % 8 || ldo % 8) return QI_B200_ESHAPE;
  if (total_k > 0 && (ldk < wk || ldv < wk || ldk % 8 || ldv % 8)) return QI_B200_ESHAPE;
  if (!aligned16(q) || !aligned16(out) || (total_k > 0 && (!aligned16(k) || !aligned16(v)))) return QI_B200_EALIGN;
  if (workspace != nullptr && !aligned16(workspace)) return QI_B200_EALIGN;
  DeviceInfo* di = nullptr;
  if (int rc = device_info(&di)) return rc;
  if (n_seq == 0)
    return cudaMemset2DAsync(out, ldo * 2, 0, wq * 2, total_q, stream) == cudaSuccess ? QI_B200_OK : QI_B200_ECUDA;
  const size_t need = packed_workspace(n_seq, total_q, total_k, heads, kv_heads, head_dim, di->num_sms);
  PackedParams p = {};
  p.ws = need > 0 && workspace != nullptr && workspace_bytes >= need ? static_cast<float*>(workspace) : nullptr;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.n_seq = n_seq;
  p.total_q = total_q;
  p.total_k = total_k;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.pair_heads = p.group % 2 == 0;
  p.causal = (flags & QI_B200_ATTN_CAUSAL) != 0;
  p.zero_rest = zero_rest;
  p.scale_log2e = scale * kLog2e;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  p.lse = lse;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.ldq = ldq;
  p.ldk = ldk;
  p.ldv = ldv;
  return head_dim == 128 ? launch_packed<128>(q, ldq, k, ldk, v, ldv, p, di->num_sms, stream)
                         : launch_packed<64>(q, ldq, k, ldk, v, ldv, p, di->num_sms, stream);
}

int qi_b200_attention_packed_workspace_bytes(int n_seq, int total_q, int total_k, int heads, int kv_heads, int head_dim,
                                             size_t* bytes) {
  if (bytes == nullptr) return QI_B200_EINVAL;
  if ((head_dim != 64 && head_dim != 128) || n_seq < 0 || total_q < 0 || total_k < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads)
    return QI_B200_ESHAPE;
  DeviceInfo* di = nullptr;
  if (int rc = device_info(&di)) return rc;
  *bytes = packed_workspace(n_seq, total_q, total_k, heads, kv_heads, head_dim, di->num_sms);
  return QI_B200_OK;
}

int qi_b200_attention_paged_workspace_bytes(int kv_heads, int head_dim, size_t* bytes) {
  if (bytes == nullptr) return QI_B200_EINVAL;
  if ((head_dim != 64 && head_dim != 128) || kv_heads <= 0) return QI_B200_ESHAPE;
  DeviceInfo* di = nullptr;
  if (int rc = device_info(&di)) return rc;
  *bytes = (static_cast<size_t>(di->num_sms) * 2 << paged_most_teams(kv_heads)) *
               (head_dim == 128 ? paged_part_floats<128>() : paged_part_floats<64>()) * sizeof(float) +
           di->num_sms * sizeof(PagedRecord);
  return QI_B200_OK;
}

int qi_b200_attention_paged(const void* q, long long ldq, const qi_b200_paged_cache* cache, const int* page_table,
                            long long ld_table, int max_pages, const int* lengths, void* out, long long ldo,
                            float* lse, int B, int heads, int kv_heads, int head_dim, float scale, void* workspace,
                            size_t workspace_bytes, cudaStream_t stream) {
  if (head_dim != 64 && head_dim != 128) return QI_B200_ESHAPE;
  if (B < 0 || B > 65535 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_pages < 0 || ld_table < max_pages)
    return QI_B200_ESHAPE;
  if (B == 0) return QI_B200_OK;
  if (q == nullptr || out == nullptr || lengths == nullptr || cache == nullptr || (max_pages > 0 && !page_table) ||
      workspace == nullptr)
    return QI_B200_EINVAL;
  if (!softmax_scale_ok(scale)) return QI_B200_EINVAL;
  const long long wq = static_cast<long long>(heads) * head_dim;
  if (ldq < wq || ldo < wq || ldq % 8 || ldo % 8) return QI_B200_ESHAPE;
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace)) return QI_B200_EALIGN;
  if (int rc = check_paged_cache(cache, kv_heads, head_dim)) return rc;
  if (static_cast<long long>(max_pages) * cache->page_size > 0x7fff0000ll) return QI_B200_ETOOBIG;
  DeviceInfo* di = nullptr;
  if (int rc = device_info(&di)) return rc;
  size_t need = 0;
  if (int rc = qi_b200_attention_paged_workspace_bytes(kv_heads, head_dim, &need)) return rc;
  if (workspace_bytes < need) return QI_B200_EINVAL;
  PagedParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.ldq = ldq;
  p.cache[0] = static_cast<const uint8_t*>(cache->k);
  p.cache[1] = static_cast<const uint8_t*>(cache->v);
  const int elt = cache->fp8 ? 1 : 2;
  for (int c = 0; c < 2; ++c) {
    p.page_stride[c] = cache->page_stride[c] * elt;
    p.slot_stride[c] = cache->slot_stride[c] * elt;
    p.head_stride[c] = cache->head_stride[c] * elt;
    p.scale[c] = cache->fp8 ? cache->scale[c] : nullptr;
    p.scale_per_head[c] = cache->scale_per_head[c];
  }
  p.pages = page_table;
  p.ld_pages = ld_table;
  p.lengths = lengths;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ldo = ldo;
  p.lse = lse;
  p.ws = static_cast<float*>(workspace);
  p.B = B;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.group = heads / kv_heads;
  p.chunks = (p.group + kPagedRows - 1) / kPagedRows;
  p.page_size = cache->page_size;
  p.page_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (cache->page_size == 1 << s) p.page_shift = s;
  p.max_pages = max_pages;
  p.num_pages = cache->pages;
  p.scale_log2e = scale * kLog2e;
  const int G = di->num_sms;
  // key heads per item: as many as lie next to each other (see the kernel), as
  // long as the longest the lengths may be still gives every SM four units.  The
  // host knows the page table's width, not the lengths: with a table much wider
  // than its sequences a few short ones get items meant for long ones (one
  // sequence of 1000 tokens, 8 key heads: 8.9 us with a table of 63 pages, 16.6
  // with 2048; 8 of about 500 tokens 14.5 and 18.8; 64 of them 38.0 and 38.5)
  // a unit holds a whole number of a warp's blocks (16 tokens of 256-byte rows,
  // else 32), so that blocks keep to multiples of their size and to one page
  const int block_shift = head_dim * elt == 256 ? 4 : 5;
  for (p.team_shift = paged_most_teams(kv_heads); p.team_shift > 0; --p.team_shift) {
    const long long unit = 1ll << std::max(block_shift, kPagedUnitShift - p.team_shift);
    const long long tokens = static_cast<long long>(max_pages) * cache->page_size;
    if (cache->head_stride[0] == head_dim && cache->head_stride[1] == head_dim &&
        B * ((tokens + unit - 1) / unit) * (kv_heads >> p.team_shift) >= 4ll * G)
      break;
  }
  p.groups = kv_heads >> p.team_shift;
  p.unit_shift = std::max(block_shift, kPagedUnitShift - p.team_shift);
  if (head_dim == 128)
    return cache->fp8 ? launch_paged<128, true>(p, G, stream) : launch_paged<128, false>(p, G, stream);
  return cache->fp8 ? launch_paged<64, true>(p, G, stream) : launch_paged<64, false>(p, G, stream);
}

}  // extern "C"
