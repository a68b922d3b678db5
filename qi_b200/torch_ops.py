"""Torch operators over the C ABI: ``torch.ops.qi_int8_w8a8.linear`` with the
reference's schema (``src/qi/quantization/csrc/int8_w8a8/bindings.cpp:159-165``)
and ``torch.ops.qi_b200.{int8_linear, fp8_linear, w4a16_linear}``, and the
decoder-block operators ``torch.ops.qi_b200.{rms_norm_quant, rope_axes,
rope_axes_store, attention_packed, attention_paged}`` (documented in
``qi_b200.kernels``, which calls them).

They live in the in-tree ``libqi_b200_torch.so`` (``qi_b200/csrc/torch_ops.cpp``,
built by ``python -m qi_b200.build``), which links the in-tree
``libqi_b200.so``.  ``load()`` registers them with torch once, together with
the shapes of the decoder-block operators' results, which tracing (fake and
meta tensors, ``torch.compile``) asks for.  Each of those has three forms:
``fresh`` returns new tensors, ``out`` writes given ones and returns nothing,
the one without an overload name takes either.
"""

from __future__ import annotations

import threading

from .build import TORCH_OPS_LIB

_lock = threading.Lock()
_loaded = False


def load() -> None:
    """Register the operators (idempotent).  Raises ``QiB200Unavailable``
    when the library has not been built."""
    global _loaded
    if _loaded:
        return
    with _lock:
        if _loaded:
            return
        import torch

        from ._lib import QiB200Unavailable, load as load_c_abi

        if not TORCH_OPS_LIB.exists():
            raise QiB200Unavailable(f"{TORCH_OPS_LIB} is missing; build it with `python -m qi_b200.build`.")
        load_c_abi()  # the C ABI library the operators call into
        torch.ops.load_library(str(TORCH_OPS_LIB))
        _register_shapes()
        _loaded = True


def _register_shapes() -> None:
    """Results of the decoder-block operators as empty tensors, from shapes alone.
    Types, strides and devices are checked when the operator runs."""
    import torch

    from ._lib import KIND_BF16, KIND_INT8

    def expect(ok, message):
        if not ok:
            raise ValueError(message)

    def codes(kind, x):
        expect(x.dim() == 2, f"x must be 2-D, got {tuple(x.shape)}.")
        return (x.new_empty(x.shape, dtype=torch.int8 if kind == KIND_INT8 else torch.uint8),
                x.new_empty((x.shape[0],), dtype=torch.float32))

    def norm(kind, x, weight, y=None, eps=1e-6, x_out=None, q=None, s=None, xn=None):
        if kind == KIND_BF16:
            return None, None
        new_q, new_s = codes(kind, x)
        return new_q if q is None else q, new_s if s is None else s

    def norm_fresh(kind, x, weight, y, eps, x_out, xn):
        expect(kind != KIND_BF16, "KIND_BF16 has no codes.")
        return codes(kind, x)

    def like(t, name, head_dim):
        expect(t.dim() == 2 and t.shape[1] % head_dim == 0, f"{name} must be [M, heads * {head_dim}], got {tuple(t.shape)}.")
        return t.new_empty(t.shape)

    def rope(q, k, positions, freqs, axes, head_dim, interleaved=True, out_q=None, out_k=None):
        return (like(q, "q", head_dim) if out_q is None else out_q,
                like(k, "k", head_dim) if k is not None and out_k is None else out_k)

    def rope_fresh(q, k, positions, freqs, axes, head_dim, interleaved):
        return like(q, "q", head_dim), q.new_empty((0,)) if k is None else like(k, "k", head_dim)

    def store(q, k, v, positions, freqs, axes, head_dim, k_cache, v_cache, slots, interleaved=True, k_scale=None,
              v_scale=None, out_q=None, out_k=None):
        return like(q, "q", head_dim) if out_q is None else out_q

    def store_fresh(q, k, v, positions, freqs, axes, head_dim, k_cache, v_cache, slots, interleaved, k_scale, v_scale,
                    out_k):
        return like(q, "q", head_dim)

    def packed(q, k, v, cu_q, cu_k, heads, kv_heads, causal=True, scale=None, out=None, lse=None):
        expect(heads > 0 and q.dim() == 2 and q.shape[1] % heads == 0,
               f"q must be [Tq, {heads} * head_dim], got {tuple(q.shape)}.")
        return q.new_empty(q.shape) if out is None else out

    def paged(q, k_cache, v_cache, pages, lengths, scale=None, k_scale=None, v_scale=None, out=None, lse=None):
        expect(k_cache.dim() == 4, f"k_cache must be [pages, page_size, kv_heads, head_dim], got {tuple(k_cache.shape)}.")
        new = like(q, "q", k_cache.shape[3])
        return new if out is None else out

    for name, fn in {
        "rms_norm_quant": norm, "rms_norm_quant.fresh": norm_fresh, "rope_axes": rope, "rope_axes.fresh": rope_fresh,
        "rope_axes_store": store, "rope_axes_store.fresh": store_fresh, "attention_packed": packed,
        "attention_packed.fresh": lambda q, k, v, cu_q, cu_k, heads, kv_heads, causal, scale, lse:
            packed(q, k, v, cu_q, cu_k, heads, kv_heads),
        "attention_paged": paged,
        "attention_paged.fresh": lambda q, k_cache, v_cache, pages, lengths, scale, k_scale, v_scale, lse:
            paged(q, k_cache, v_cache, pages, lengths),
        **{f"{op}.out": lambda *args: None
           for op in ("rms_norm_quant", "rope_axes", "rope_axes_store", "attention_packed", "attention_paged")},
    }.items():
        torch.library.register_fake("qi_b200::" + name, fn)
