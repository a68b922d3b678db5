// The decoder-block operators as torch operators (namespace qi_b200), included
// by torch_ops.cpp.  qi_b200.kernels calls them, so there is one place that
// checks arguments: types, shapes and strides first (they hold for tensors of
// any device), then that every tensor lies on one CUDA device.  A refused
// argument is a Python ValueError; a status of the library a RuntimeError.
// Work goes to the current stream of the tensors' own device, which becomes
// the current device for the call; outputs that are not given and workspaces
// come from torch's caching allocator.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "../../include/qi_b200.h"

namespace decoder {

using Opt = std::optional<at::Tensor>;

inline bool given(const Opt& t) { return t.has_value() && t->defined(); }
inline void* ptr(const at::Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }
inline void* ptr(const Opt& t) { return given(t) ? ptr(*t) : nullptr; }

inline void done(int rc, const char* what) {
  TORCH_CHECK(rc == QI_B200_OK, what, " failed with status ", rc, ": ", qi_b200_error_string(rc));
}

// Every tensor of a call, to be checked against the first one's device.
struct SameDevice {
  at::Device dev;
  explicit SameDevice(const at::Tensor& t) : dev(t.device()) {}
  void on(const at::Tensor& t, const char* name) const {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor.");
    TORCH_CHECK_VALUE(t.device() == dev, name, " must be on ", dev.str(), ", got ", t.device().str(), ".");
  }
  void on(const Opt& t, const char* name) const {
    if (given(t)) on(*t, name);
  }
};

// A bf16 [rows, width] block, column slices of wider rows allowed; its row stride.
inline int64_t rows_of(const at::Tensor& t, const char* name, int64_t rows, int64_t width) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 && t.dim() == 2, name, " must be a 2-D bfloat16 tensor.");
  TORCH_CHECK_VALUE(t.size(0) == rows && t.size(1) == width, name, " must be [", rows, ", ", width, "], got ",
                    t.sizes(), ".");
  if (t.numel() == 0) return (width + 7) / 8 * 8;
  const int64_t ld = rows > 1 ? t.stride(0) : (width + 7) / 8 * 8;
  TORCH_CHECK_VALUE((t.stride(1) == 1 || width == 1) && ld >= width && ld % 8 == 0 &&
                        reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
                    name, " must have unit column stride and 16-byte aligned rows that do not overlap.");
  return ld;
}

inline void dense(const at::Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape) {
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type(), ".");
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must be ", shape, ", got ", t.sizes(), ".");
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous.");
}

inline int small(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v >= 0 && v <= 0x7fffffff, name, " is too large: ", v, ".");
  return static_cast<int>(v);
}

// ---------------------------------------------------------------------------

inline std::tuple<Opt, Opt> rms_norm_quant(int64_t kind, const at::Tensor& x, const at::Tensor& weight, const Opt& y,
                                           double eps, const Opt& x_out, const Opt& q, const Opt& s, const Opt& xn) {
  TORCH_CHECK_VALUE(kind == QI_B200_KIND_INT8 || kind == QI_B200_KIND_FP8_E4M3 || kind == QI_B200_KIND_BF16,
                    "unknown kind ", kind, ".");
  TORCH_CHECK_VALUE(x.dim() == 2, "x must be 2-D, got ", x.sizes(), ".");
  const int64_t M = x.size(0), D = x.size(1);
  TORCH_CHECK_VALUE(D > 0 && D % 8 == 0 && D <= 16384, "rms_norm_quant needs D % 8 == 0 and 0 < D <= 16384, got ", D,
                    ".");
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative.");
  const int64_t ldx = rows_of(x, "x", M, D);
  dense(weight, "weight", at::kBFloat16, {D});
  int64_t ldy = 0, ld_out = 0;
  const at::Tensor& h = given(x_out) ? *x_out : x;
  if (given(y)) {
    ldy = rows_of(*y, "y", M, D);
    ld_out = rows_of(h, "x_out", M, D);
  } else {
    TORCH_CHECK_VALUE(!given(x_out), "x_out needs y: without a residual the rows of x do not change.");
  }
  if (given(xn)) dense(*xn, "xn", at::kBFloat16, {M, D});
  const bool codes = kind != QI_B200_KIND_BF16;
  const auto type = kind == QI_B200_KIND_INT8 ? at::kChar : at::kByte;
  TORCH_CHECK_VALUE(codes || (given(xn) && !given(q) && !given(s)), "KIND_BF16 writes xn only.");
  if (given(q)) dense(*q, "q", type, {M, D});
  if (given(s)) dense(*s, "s", at::kFloat, {M});
  SameDevice same(x);
  same.on(x, "x"), same.on(weight, "weight"), same.on(y, "y"), same.on(x_out, "x_out"), same.on(q, "q");
  same.on(s, "s"), same.on(xn, "xn");
  const c10::cuda::CUDAGuard guard(same.dev);
  Opt qo = q, so = s;
  if (codes && !given(q)) qo = at::empty({M, D}, x.options().dtype(type));
  if (codes && !given(s)) so = at::empty({M}, x.options().dtype(at::kFloat));
  done(qi_b200_rms_norm_quant(static_cast<int>(kind), ptr(x), ldx, ptr(y), ldy, given(y) ? ptr(h) : nullptr, ld_out,
                              ptr(weight), ptr(qo), static_cast<float*>(ptr(so)), ptr(xn), small(M, "M"),
                              static_cast<int>(D), static_cast<float>(eps),
                              at::cuda::getCurrentCUDAStream(same.dev.index())),
       "qi_b200_rms_norm_quant");
  return {codes ? qo : std::nullopt, codes ? so : std::nullopt};
}

// ---------------------------------------------------------------------------

inline bool index_type(const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64, got ",
                    t.scalar_type(), ".");
  TORCH_CHECK_VALUE(t.is_contiguous(), name, " must be contiguous.");
  return t.scalar_type() == at::kLong;
}

// A [pages, page_size, kv_heads, head_dim] cache pair with its scales.
inline qi_b200_paged_cache cache_of(const at::Tensor& k, const at::Tensor& v, const Opt& k_scale, const Opt& v_scale,
                                    int64_t kv_heads, int64_t head_dim) {
  qi_b200_paged_cache c = {};
  const auto type = k.scalar_type();
  c.fp8 = type == at::kByte || type == at::kFloat8_e4m3fn;
  TORCH_CHECK_VALUE(c.fp8 || type == at::kBFloat16, "the cache must be bfloat16, uint8 (E4M3 codes) or float8_e4m3fn, got ",
                    type, ".");
  const at::Tensor* t[2] = {&k, &v};
  const Opt* scale[2] = {&k_scale, &v_scale};
  const char* names[2] = {"k_cache", "v_cache"};
  const char* scales[2] = {"k_scale", "v_scale"};
  const int64_t elt = c.fp8 ? 1 : 2;
  for (int i = 0; i < 2; ++i) {
    TORCH_CHECK_VALUE(t[i]->dim() == 4 && t[i]->scalar_type() == type && t[i]->sizes() == k.sizes(), names[i],
                      " must be [pages, page_size, kv_heads, head_dim], both caches alike, got ", t[i]->sizes(), ".");
    TORCH_CHECK_VALUE(t[i]->size(2) == kv_heads && t[i]->size(3) == head_dim, names[i], " must hold ", kv_heads,
                      " heads of ", head_dim, ", got ", t[i]->sizes(), ".");
    TORCH_CHECK_VALUE(t[i]->numel() > 0, names[i], " must hold at least one token.");
    long long st[3];
    bool fine = t[i]->stride(3) == 1 && reinterpret_cast<uintptr_t>(t[i]->data_ptr()) % 16 == 0;
    for (int d = 0; d < 3; ++d) {
      st[d] = t[i]->size(d) > 1 ? t[i]->stride(d) : 0;
      fine = fine && st[d] * elt % 16 == 0;
    }
    TORCH_CHECK_VALUE(fine && (kv_heads == 1 || st[2] >= head_dim), names[i],
                      " must have unit stride inside a head and 16-byte aligned heads that do not overlap.");
    c.page_stride[i] = st[0], c.slot_stride[i] = st[1], c.head_stride[i] = st[2];
    if (!c.fp8) {
      TORCH_CHECK_VALUE(!given(*scale[i]), scales[i], " belongs to an E4M3 cache.");
      continue;
    }
    TORCH_CHECK_VALUE(given(*scale[i]), "an E4M3 cache needs ", scales[i], ".");
    const at::Tensor& s = **scale[i];
    TORCH_CHECK_VALUE(s.scalar_type() == at::kFloat && s.is_contiguous() && (s.numel() == 1 || s.numel() == kv_heads),
                      scales[i], " must be float32 with 1 or ", kv_heads, " values.");
    c.scale[i] = s.data_ptr<float>();
    c.scale_per_head[i] = s.numel() > 1;
  }
  c.k = k.data_ptr(), c.v = v.data_ptr();
  c.pages = small(k.size(0), "the number of pages");
  c.page_size = small(k.size(1), "page_size");
  return c;
}

inline std::tuple<at::Tensor, Opt> rope(const at::Tensor& q, const Opt& k, const Opt& v, const at::Tensor& positions,
                                        const at::Tensor& freqs, const at::Tensor& axes, int64_t D, bool interleaved,
                                        const Opt& out_q, const Opt& out_k, const Opt& k_cache, const Opt& v_cache,
                                        const Opt& slots, const Opt& k_scale, const Opt& v_scale) {
  TORCH_CHECK_VALUE(D > 0 && D % 16 == 0 && D <= 512, "head_dim must be a multiple of 16 up to 512, got ", D, ".");
  TORCH_CHECK_VALUE(q.dim() == 2 && q.size(1) > 0 && q.size(1) % D == 0, "q must be [M, heads * ", D, "], got ",
                    q.sizes(), ".");
  const int64_t M = q.size(0);
  const int64_t ldq = rows_of(q, "q", M, q.size(1));
  const bool pos64 = index_type(positions, "positions");
  TORCH_CHECK_VALUE(positions.dim() >= 1 && positions.dim() <= 2 && positions.size(-1) == M &&
                        (positions.dim() == 1 || positions.size(0) > 0),
                    "positions must be [axes, ", M, "] (or [", M, "] for one axis), got ", positions.sizes(), ".");
  const int64_t P = freqs.numel();
  dense(freqs, "freqs", at::kDouble, {P});
  dense(axes, "axes", at::kInt, {P});
  TORCH_CHECK_VALUE(P > 0 && P % 8 == 0 && 2 * P <= D, "freqs and axes must hold a multiple of 8 pairs, at most ",
                    D / 2, ", got ", P, ".");
  const int64_t ldq_out = given(out_q) ? rows_of(*out_q, "out_q", M, q.size(1)) : q.size(1);
  int64_t ldk = 0, ldv = 0, ldk_out = 0, kv_heads = 0;
  qi_b200_paged_cache cache = {};
  const bool store = given(k_cache);
  bool slots64 = false;
  if (given(k)) {
    TORCH_CHECK_VALUE(k->dim() == 2 && k->size(1) > 0 && k->size(1) % D == 0, "k must be [M, kv_heads * ", D,
                      "], got ", k->sizes(), ".");
    kv_heads = k->size(1) / D;
    ldk = rows_of(*k, "k", M, k->size(1));
    ldk_out = given(out_k) ? rows_of(*out_k, "out_k", M, k->size(1)) : k->size(1);
  } else {
    TORCH_CHECK_VALUE(!given(out_k), "out_k needs k.");
  }
  if (store) {
    TORCH_CHECK_VALUE(given(k) && given(v) && given(v_cache) && given(slots), "the cache needs k, v and slots.");
    ldv = rows_of(*v, "v", M, k->size(1));
    cache = cache_of(*k_cache, *v_cache, k_scale, v_scale, kv_heads, D);
    slots64 = index_type(*slots, "slots");
    TORCH_CHECK_VALUE(slots->dim() == 1 && slots->numel() == M, "slots must be [", M, "], got ", slots->sizes(), ".");
  }
  SameDevice same(q);
  same.on(q, "q"), same.on(k, "k"), same.on(v, "v"), same.on(positions, "positions"), same.on(freqs, "freqs");
  same.on(axes, "axes"), same.on(out_q, "out_q"), same.on(out_k, "out_k"), same.on(k_cache, "k_cache");
  same.on(v_cache, "v_cache"), same.on(slots, "slots"), same.on(k_scale, "k_scale"), same.on(v_scale, "v_scale");
  const c10::cuda::CUDAGuard guard(same.dev);
  at::Tensor oq = given(out_q) ? *out_q : at::empty({M, q.size(1)}, q.options());
  Opt ok = out_k;
  if (given(k) && !store && !given(out_k)) ok = at::empty({M, k->size(1)}, q.options());
  done(qi_b200_rope_axes(ptr(q), ldq, ptr(k), ldk, ptr(v), ldv, ptr(oq), ldq_out, ptr(ok), ldk_out, ptr(positions),
                         pos64, static_cast<const double*>(ptr(freqs)), static_cast<const int*>(ptr(axes)),
                         static_cast<int>(P), positions.dim() == 1 ? 1 : small(positions.size(0), "axes"), interleaved,
                         small(M, "M"), small(q.size(1) / D, "heads"), small(kv_heads, "kv_heads"),
                         static_cast<int>(D), store ? &cache : nullptr, ptr(slots), slots64,
                         at::cuda::getCurrentCUDAStream(same.dev.index())),
       "qi_b200_rope_axes");
  return {oq, ok};
}

inline std::tuple<at::Tensor, Opt> rope_axes(const at::Tensor& q, const Opt& k, const at::Tensor& positions,
                                             const at::Tensor& freqs, const at::Tensor& axes, int64_t head_dim,
                                             bool interleaved, const Opt& out_q, const Opt& out_k) {
  return rope(q, k, {}, positions, freqs, axes, head_dim, interleaved, out_q, out_k, {}, {}, {}, {}, {});
}

inline at::Tensor rope_axes_store(const at::Tensor& q, const Opt& k, const Opt& v, const at::Tensor& positions,
                                  const at::Tensor& freqs, const at::Tensor& axes, int64_t head_dim,
                                  const at::Tensor& k_cache, const at::Tensor& v_cache,
                                  const at::Tensor& slots, bool interleaved, const Opt& k_scale, const Opt& v_scale,
                                  const Opt& out_q, const Opt& out_k) {
  return std::get<0>(rope(q, k, v, positions, freqs, axes, head_dim, interleaved, out_q, out_k, k_cache, v_cache, slots,
                          k_scale, v_scale));
}

// ---------------------------------------------------------------------------

inline float softmax_scale(int64_t head_dim, int64_t heads, int64_t kv_heads, const std::optional<double>& scale,
                           const Opt& lse, int64_t rows) {
  TORCH_CHECK_VALUE(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128, got ", head_dim, ".");
  TORCH_CHECK_VALUE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, heads, " query heads do not share ", kv_heads,
                    " key heads evenly.");
  if (given(lse)) dense(*lse, "lse", at::kFloat, {rows, heads});
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(head_dim));
  const float f = static_cast<float>(s);
  TORCH_CHECK_VALUE(f > 0.f && std::isfinite(f * 1.4426950408889634f),
                    "scale must be positive, and finite times log2(e), got ", s, ".");
  return f;
}

inline at::Tensor attention_packed(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                   const at::Tensor& cu_q, const at::Tensor& cu_k, int64_t heads, int64_t kv_heads,
                                   bool causal, std::optional<double> scale, const Opt& out, const Opt& lse) {
  TORCH_CHECK_VALUE(q.dim() == 2 && heads > 0 && q.size(1) % heads == 0, "q must be [Tq, ", heads,
                    " * head_dim], got ", q.sizes(), ".");
  const int64_t D = q.size(1) / heads, Tq = q.size(0);
  const float f = softmax_scale(D, heads, kv_heads, scale, lse, Tq);
  TORCH_CHECK_VALUE(k.dim() == 2, "k must be 2-D, got ", k.sizes(), ".");
  const int64_t Tk = k.size(0);
  const int64_t ldq = rows_of(q, "q", Tq, heads * D), ldk = rows_of(k, "k", Tk, kv_heads * D);
  const int64_t ldv = rows_of(v, "v", Tk, kv_heads * D);
  dense(cu_q, "cu_q", at::kInt, {cu_q.numel()});
  TORCH_CHECK_VALUE(cu_q.numel() > 0, "cu_q must hold one value more than there are sequences.");
  dense(cu_k, "cu_k", at::kInt, {cu_q.numel()});
  const int64_t ldo = given(out) ? rows_of(*out, "out", Tq, heads * D) : heads * D;
  SameDevice same(q);
  same.on(q, "q"), same.on(k, "k"), same.on(v, "v"), same.on(cu_q, "cu_q"), same.on(cu_k, "cu_k");
  same.on(out, "out"), same.on(lse, "lse");
  const c10::cuda::CUDAGuard guard(same.dev);
  at::Tensor o = given(out) ? *out : at::empty({Tq, heads * D}, q.options());
  const int n_seq = small(cu_q.numel() - 1, "sequences");
  size_t ws_bytes = 0;
  done(qi_b200_attention_packed_workspace_bytes(n_seq, small(Tq, "Tq"), small(Tk, "Tk"), small(heads, "heads"),
                                                small(kv_heads, "kv_heads"), static_cast<int>(D), &ws_bytes),
       "qi_b200_attention_packed_workspace_bytes");
  at::Tensor ws;
  if (ws_bytes) ws = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  // a new output has no contents that its rows outside every sequence could keep
  const int flags = (causal ? QI_B200_ATTN_CAUSAL : 0) | (given(out) ? 0 : QI_B200_ATTN_ZERO_REST);
  done(qi_b200_attention_packed(ptr(q), ldq, ptr(k), ldk, ptr(v), ldv, ptr(o), ldo, static_cast<float*>(ptr(lse)),
                                cu_q.data_ptr<int>(), cu_k.data_ptr<int>(), n_seq, static_cast<int>(Tq),
                                static_cast<int>(Tk), static_cast<int>(heads), static_cast<int>(kv_heads),
                                static_cast<int>(D), flags, f, ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
                                at::cuda::getCurrentCUDAStream(same.dev.index())),
       "qi_b200_attention_packed");
  return o;
}

inline at::Tensor attention_paged(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                  const at::Tensor& pages, const at::Tensor& lengths, std::optional<double> scale,
                                  const Opt& k_scale, const Opt& v_scale, const Opt& out, const Opt& lse) {
  TORCH_CHECK_VALUE(k_cache.dim() == 4, "k_cache must be [pages, page_size, kv_heads, head_dim], got ",
                    k_cache.sizes(), ".");
  const int64_t kv_heads = k_cache.size(2), D = k_cache.size(3);
  TORCH_CHECK_VALUE(q.dim() == 2 && D > 0 && q.size(1) % D == 0, "q must be [B, heads * ", D, "], got ", q.sizes(), ".");
  const int64_t B = q.size(0), heads = q.size(1) / D;
  TORCH_CHECK_VALUE(B <= 65535, "attention_paged takes at most 65535 sequences.");
  const float f = softmax_scale(D, heads, kv_heads, scale, lse, B);
  const int64_t ldq = rows_of(q, "q", B, heads * D);
  const qi_b200_paged_cache cache = cache_of(k_cache, v_cache, k_scale, v_scale, kv_heads, D);
  TORCH_CHECK_VALUE(pages.scalar_type() == at::kInt && pages.dim() == 2 && pages.size(0) == B &&
                        (pages.size(1) <= 1 || pages.stride(1) == 1) && (B <= 1 || pages.stride(0) >= pages.size(1)),
                    "pages must be int32 [", B, ", max_pages] with unit column stride.");
  dense(lengths, "lengths", at::kInt, {B});
  const int64_t ldo = given(out) ? rows_of(*out, "out", B, heads * D) : heads * D;
  SameDevice same(q);
  same.on(q, "q"), same.on(k_cache, "k_cache"), same.on(v_cache, "v_cache"), same.on(pages, "pages");
  same.on(lengths, "lengths"), same.on(k_scale, "k_scale"), same.on(v_scale, "v_scale"), same.on(out, "out");
  same.on(lse, "lse");
  const c10::cuda::CUDAGuard guard(same.dev);
  at::Tensor o = given(out) ? *out : at::empty({B, heads * D}, q.options());
  size_t ws_bytes = 0;
  done(qi_b200_attention_paged_workspace_bytes(small(kv_heads, "kv_heads"), static_cast<int>(D), &ws_bytes),
       "qi_b200_attention_paged_workspace_bytes");
  const at::Tensor ws = at::empty({static_cast<int64_t>(ws_bytes)}, q.options().dtype(at::kByte));
  done(qi_b200_attention_paged(ptr(q), ldq, &cache, static_cast<const int*>(ptr(pages)),
                               B > 1 ? pages.stride(0) : pages.size(1), small(pages.size(1), "max_pages"),
                               static_cast<const int*>(ptr(lengths)), ptr(o), ldo, static_cast<float*>(ptr(lse)),
                               static_cast<int>(B), small(heads, "heads"), small(kv_heads, "kv_heads"),
                               static_cast<int>(D), f, ws.data_ptr(), ws_bytes,
                               at::cuda::getCurrentCUDAStream(same.dev.index())),
       "qi_b200_attention_paged");
  return o;
}

// ---------------------------------------------------------------------------
// The forms that qi_b200.kernels calls: `fresh` returns new tensors only, `out`
// writes given ones and returns nothing, so that what a call writes and what it
// returns never are one tensor (tracers rely on it).  The forms without an
// overload name take either and may return an argument.

inline std::tuple<at::Tensor, at::Tensor> rms_norm_quant_fresh(int64_t kind, const at::Tensor& x,
                                                               const at::Tensor& weight, const Opt& y, double eps,
                                                               const Opt& x_out, const Opt& xn) {
  TORCH_CHECK_VALUE(kind != QI_B200_KIND_BF16, "KIND_BF16 has no codes.");
  TORCH_CHECK_VALUE(!given(y) || given(x_out), "y needs x_out.");
  auto r = rms_norm_quant(kind, x, weight, y, eps, x_out, {}, {}, xn);
  return {*std::get<0>(r), *std::get<1>(r)};
}
inline void rms_norm_quant_out(int64_t kind, const at::Tensor& x, const at::Tensor& weight, const Opt& y, double eps,
                               const Opt& x_out, const Opt& q, const Opt& s, const Opt& xn) {
  TORCH_CHECK_VALUE(!given(y) || given(x_out), "y needs x_out.");
  TORCH_CHECK_VALUE(kind == QI_B200_KIND_BF16 || (given(q) && given(s)), "codes need q and s.");
  rms_norm_quant(kind, x, weight, y, eps, x_out, q, s, xn);
}

inline std::tuple<at::Tensor, at::Tensor> rope_axes_fresh(const at::Tensor& q, const Opt& k, const at::Tensor& positions,
                                                          const at::Tensor& freqs, const at::Tensor& axes,
                                                          int64_t head_dim, bool interleaved) {
  auto r = rope_axes(q, k, positions, freqs, axes, head_dim, interleaved, {}, {});
  const Opt& ok = std::get<1>(r);
  return {std::get<0>(r), given(ok) ? *ok : at::empty({0}, q.options())};
}
inline void rope_axes_out(const at::Tensor& q, const Opt& k, const at::Tensor& positions, const at::Tensor& freqs,
                          const at::Tensor& axes, int64_t head_dim, bool interleaved, const at::Tensor& out_q,
                          const Opt& out_k) {
  TORCH_CHECK_VALUE(given(k) == given(out_k), given(k) ? "k needs out_k." : "out_k needs k.");
  rope_axes(q, k, positions, freqs, axes, head_dim, interleaved, out_q, out_k);
}

inline at::Tensor rope_axes_store_fresh(const at::Tensor& q, const Opt& k, const Opt& v, const at::Tensor& positions,
                                        const at::Tensor& freqs, const at::Tensor& axes, int64_t head_dim,
                                        const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& slots,
                                        bool interleaved, const Opt& k_scale, const Opt& v_scale, const Opt& out_k) {
  return rope_axes_store(q, k, v, positions, freqs, axes, head_dim, k_cache, v_cache, slots, interleaved, k_scale,
                         v_scale, {}, out_k);
}
inline void rope_axes_store_out(const at::Tensor& q, const Opt& k, const Opt& v, const at::Tensor& positions,
                                const at::Tensor& freqs, const at::Tensor& axes, int64_t head_dim,
                                const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& slots,
                                bool interleaved, const Opt& k_scale, const Opt& v_scale, const at::Tensor& out_q,
                                const Opt& out_k) {
  rope_axes_store(q, k, v, positions, freqs, axes, head_dim, k_cache, v_cache, slots, interleaved, k_scale, v_scale,
                  out_q, out_k);
}

inline at::Tensor attention_packed_fresh(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                         const at::Tensor& cu_q, const at::Tensor& cu_k, int64_t heads,
                                         int64_t kv_heads, bool causal, std::optional<double> scale, const Opt& lse) {
  return attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, causal, scale, {}, lse);
}
inline void attention_packed_out(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu_q,
                                 const at::Tensor& cu_k, int64_t heads, int64_t kv_heads, bool causal,
                                 std::optional<double> scale, const at::Tensor& out, const Opt& lse) {
  attention_packed(q, k, v, cu_q, cu_k, heads, kv_heads, causal, scale, out, lse);
}

inline at::Tensor attention_paged_fresh(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                        const at::Tensor& pages, const at::Tensor& lengths,
                                        std::optional<double> scale, const Opt& k_scale, const Opt& v_scale,
                                        const Opt& lse) {
  return attention_paged(q, k_cache, v_cache, pages, lengths, scale, k_scale, v_scale, {}, lse);
}
inline void attention_paged_out(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                const at::Tensor& pages, const at::Tensor& lengths, std::optional<double> scale,
                                const Opt& k_scale, const Opt& v_scale, const at::Tensor& out, const Opt& lse) {
  attention_paged(q, k_cache, v_cache, pages, lengths, scale, k_scale, v_scale, out, lse);
}

}  // namespace decoder

TORCH_LIBRARY_FRAGMENT(qi_b200, m) {
  m.def("rms_norm_quant(int kind, Tensor(a!) x, Tensor weight, Tensor? y=None, float eps=1e-6, Tensor(b!)? x_out=None, "
        "Tensor(c!)? q=None, Tensor(d!)? s=None, Tensor(e!)? xn=None) -> (Tensor(c!)?, Tensor(d!)?)");
  m.def("rms_norm_quant.fresh(int kind, Tensor x, Tensor weight, Tensor? y, float eps, Tensor(a!)? x_out, "
        "Tensor(b!)? xn) -> (Tensor, Tensor)");
  m.def("rms_norm_quant.out(int kind, Tensor x, Tensor weight, Tensor? y, float eps, Tensor(a!)? x_out, "
        "Tensor(b!)? q, Tensor(c!)? s, Tensor(d!)? xn) -> ()");
  m.def("rope_axes(Tensor q, Tensor? k, Tensor positions, Tensor freqs, Tensor axes, int head_dim, "
        "bool interleaved=True, Tensor(a!)? out_q=None, Tensor(b!)? out_k=None) -> (Tensor(a!), Tensor(b!)?)");
  m.def("rope_axes.fresh(Tensor q, Tensor? k, Tensor positions, Tensor freqs, Tensor axes, int head_dim, "
        "bool interleaved) -> (Tensor, Tensor)");
  m.def("rope_axes.out(Tensor q, Tensor? k, Tensor positions, Tensor freqs, Tensor axes, int head_dim, "
        "bool interleaved, Tensor(a!) out_q, Tensor(b!)? out_k) -> ()");
  m.def("rope_axes_store(Tensor q, Tensor? k, Tensor? v, Tensor positions, Tensor freqs, Tensor axes, int head_dim, "
        "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, bool interleaved=True, Tensor? k_scale=None, "
        "Tensor? v_scale=None, Tensor(c!)? out_q=None, Tensor(d!)? out_k=None) -> Tensor(c!)");
  m.def("rope_axes_store.fresh(Tensor q, Tensor? k, Tensor? v, Tensor positions, Tensor freqs, Tensor axes, "
        "int head_dim, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, bool interleaved, Tensor? k_scale, "
        "Tensor? v_scale, Tensor(c!)? out_k) -> Tensor");
  m.def("rope_axes_store.out(Tensor q, Tensor? k, Tensor? v, Tensor positions, Tensor freqs, Tensor axes, "
        "int head_dim, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, bool interleaved, Tensor? k_scale, "
        "Tensor? v_scale, Tensor(c!) out_q, Tensor(d!)? out_k) -> ()");
  m.def("attention_packed(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, int heads, int kv_heads, "
        "bool causal=True, float? scale=None, Tensor(a!)? out=None, Tensor(b!)? lse=None) -> Tensor(a!)");
  m.def("attention_packed.fresh(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, int heads, int kv_heads, "
        "bool causal, float? scale, Tensor(a!)? lse) -> Tensor");
  m.def("attention_packed.out(Tensor q, Tensor k, Tensor v, Tensor cu_q, Tensor cu_k, int heads, int kv_heads, "
        "bool causal, float? scale, Tensor(a!) out, Tensor(b!)? lse) -> ()");
  m.def("attention_paged(Tensor q, Tensor k_cache, Tensor v_cache, Tensor pages, Tensor lengths, float? scale=None, "
        "Tensor? k_scale=None, Tensor? v_scale=None, Tensor(a!)? out=None, Tensor(b!)? lse=None) -> Tensor(a!)");
  m.def("attention_paged.fresh(Tensor q, Tensor k_cache, Tensor v_cache, Tensor pages, Tensor lengths, float? scale, "
        "Tensor? k_scale, Tensor? v_scale, Tensor(a!)? lse) -> Tensor");
  m.def("attention_paged.out(Tensor q, Tensor k_cache, Tensor v_cache, Tensor pages, Tensor lengths, float? scale, "
        "Tensor? k_scale, Tensor? v_scale, Tensor(a!) out, Tensor(b!)? lse) -> ()");
}

// CPU tensors come to the same functions, whose checks refuse them (the checks
// of types and shapes first).  Shapes without data are qi_b200/torch_ops.py's.
namespace decoder {
inline void register_all(torch::Library& m) {
  m.impl("rms_norm_quant", &rms_norm_quant);
  m.impl("rms_norm_quant.fresh", &rms_norm_quant_fresh);
  m.impl("rms_norm_quant.out", &rms_norm_quant_out);
  m.impl("rope_axes", &rope_axes);
  m.impl("rope_axes.fresh", &rope_axes_fresh);
  m.impl("rope_axes.out", &rope_axes_out);
  m.impl("rope_axes_store", &rope_axes_store);
  m.impl("rope_axes_store.fresh", &rope_axes_store_fresh);
  m.impl("rope_axes_store.out", &rope_axes_store_out);
  m.impl("attention_packed", &attention_packed);
  m.impl("attention_packed.fresh", &attention_packed_fresh);
  m.impl("attention_packed.out", &attention_packed_out);
  m.impl("attention_paged", &attention_paged);
  m.impl("attention_paged.fresh", &attention_paged_fresh);
  m.impl("attention_paged.out", &attention_paged_out);
}
}  // namespace decoder

TORCH_LIBRARY_IMPL(qi_b200, CUDA, m) { decoder::register_all(m); }
TORCH_LIBRARY_IMPL(qi_b200, CPU, m) { decoder::register_all(m); }
