"""Registers the MI355X kernels as one Popcorn backend.

    import popcorn, popcorn.kernels       # or: from popcorn_amd import compat as popcorn
    from popcorn_amd import backend
    backend.register(popcorn)

This is the whole integration: one `declare_backend` (core/sources.py:40-47)
and one `op.register(name, source=..., predicate=..., forward_only=...)` per
op (core/dispatcher.py:324-345), exactly what a backend module under
`popcorn/kernels/` does. Each registration is source-only: the
`popcorn_amd.impls` functions already carry the reference signatures, so
Popcorn calls them directly (core/dispatcher.py:184-201).

The backend's distribution is `popcorn-amd` at `popcorn_amd.__version__`
(setup.py), pinned as both bounds of the version gate; the gate resolves for
an installed copy, and in a source tree once `python -m popcorn_amd.build` (or
`__graft_entry__.build()`) has written the metadata beside the package.

The predicates only describe what the kernels cover -- tensors on a HIP
device, one floating dtype per call, the shapes the kernels implement.
Anything else is declined, and Popcorn serves it with the next eligible
implementation (the torch reference); inside the kernels an unsupported call
raises instead of falling back.
"""

from __future__ import annotations

from types import ModuleType
from typing import Any

import torch

from popcorn_amd import __version__

BACKEND = "mi355x"
DISTRIBUTION = "popcorn-amd"


def _on_hip(*tensors: Any) -> bool:
    ts = [t for t in tensors if t is not None]
    return (
        torch.version.hip is not None
        and all(isinstance(t, torch.Tensor) and t.device.type == "cuda" for t in ts)
        and len({t.device for t in ts}) == 1
    )


_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_HALF = (torch.bfloat16, torch.float16)


def rms_norm_supported(x, weight, bias, eps) -> bool:
    """One float dtype, or a 16-bit x with fp32 weight and bias (the output promotes to fp32)."""
    return (
        _on_hip(x, weight, bias)
        and x.dtype in _FLOATS
        and (weight.dtype == x.dtype or (x.dtype in _HALF and weight.dtype == torch.float32))
        and (bias is None or bias.dtype == weight.dtype)
        and x.shape[-1] > 0
    )


def add_rms_norm_supported(x, residual, weight, eps, offset) -> bool:
    return (
        _on_hip(x, residual, weight)
        and x.dtype == residual.dtype
        and x.dtype in _FLOATS
        and (weight.dtype == x.dtype or (x.dtype in _HALF and weight.dtype == torch.float32))
        and x.shape == residual.shape
        and x.shape[-1] > 0
    )


def swiglu_supported(a, b) -> bool:
    return _on_hip(a, b) and a.dtype == b.dtype and a.dtype in _FLOATS and a.shape == b.shape


def rotary_supported(x, cos, sin, interleaved) -> bool:
    return (
        _on_hip(x, cos, sin)
        and x.dtype in _FLOATS
        and cos.dtype in _FLOATS
        and cos.dtype == sin.dtype
        and x.dim() == 4
        and 2 * cos.shape[-1] <= x.shape[-1]
    )


def rope_supported(q, k, cos, sin) -> bool:
    """q, k one float dtype; cos, sin one float dtype (fp32 tables beside 16-bit q/k promote the outputs)."""
    return (
        _on_hip(q, k, cos, sin)
        and q.dtype in _FLOATS
        and q.dtype == k.dtype
        and cos.dtype in _FLOATS
        and cos.dtype == sin.dtype
        and q.dim() == k.dim() == 4
        and cos.dim() == 3
        and cos.shape == sin.shape
        and q.shape[-1] % 2 == 0
        and k.shape[0] == q.shape[0]
        and k.shape[2:] == q.shape[2:]
        and cos.shape[1:] == q.shape[2:]
        and cos.shape[0] in (1, q.shape[0])
    )


def _norm_rope_head_dim(head_dim: int, dtype: torch.dtype) -> bool:
    """head_dim / 2 = (16-byte pack) * 2^k with at most 64 packs: one row inside one wavefront."""
    pack = 16 // torch.empty((), dtype=dtype).element_size()
    half = head_dim // 2
    if head_dim % 2 or half % pack:
        return False
    packs = half // pack
    return 1 <= packs <= 64 and packs & (packs - 1) == 0


def qk_norm_rope_supported(q, k, q_weight, k_weight, cos, sin, eps) -> bool:
    return (
        _on_hip(q, k, q_weight, k_weight, cos, sin)
        and q.dtype in _FLOATS
        and q.dtype == k.dtype
        and q_weight.dtype == k_weight.dtype
        and (q_weight.dtype == q.dtype or (q.dtype in _HALF and q_weight.dtype == torch.float32))
        and cos.dtype in _FLOATS
        and cos.dtype == sin.dtype
        and q.dim() == k.dim() == 4
        and cos.dim() == 3
        and cos.shape == sin.shape
        and k.shape[0] == q.shape[0]
        and k.shape[2:] == q.shape[2:]
        and q_weight.shape == k_weight.shape == q.shape[-1:]
        and cos.shape[1:] == q.shape[2:]
        and cos.shape[0] in (1, q.shape[0])
        and _norm_rope_head_dim(q.shape[-1], q.dtype)
    )


def _attn_head_dim(head_dim: int) -> bool:
    """head_dim a multiple of 8 up to 256, in every dtype, forward and backward alike (so whether autograd
    records the call does not matter)."""
    return head_dim % 8 == 0 and 8 <= head_dim <= 256


def attn_supported(q, k, v, causal, softmax_scale) -> bool:
    return (
        _on_hip(q, k, v)
        and q.dtype in _FLOATS
        and q.dtype == k.dtype == v.dtype
        and _attn_head_dim(q.shape[-1])
        and k.shape[2] > 0
        and q.shape[2] % k.shape[2] == 0
    )


def attn_varlen_supported(q, k, v, cu_seqlens, causal, softmax_scale) -> bool:
    return (
        _on_hip(q, k, v)
        and isinstance(cu_seqlens, torch.Tensor)
        and not cu_seqlens.is_floating_point()
        and cu_seqlens.dim() == 1
        and q.dtype in _FLOATS
        and q.dtype == k.dtype == v.dtype
        and q.dim() == 3
        and _attn_head_dim(q.shape[-1])
        and k.shape[1] > 0
        and q.shape[1] % k.shape[1] == 0
    )


def _cache_supported(head_dim: int, kv_heads: int, *rows) -> bool:
    """Caches [pages, kv_heads, page_size, row] of one shape, rows contiguous, page_size a multiple of 16."""
    return (
        all(t.dim() == 4 and t.shape == rows[0].shape and t.stride(-1) == 1 for t in rows)
        and rows[0].shape[1] == kv_heads
        and rows[0].shape[2] >= 16
        and rows[0].shape[2] % 16 == 0
        and 8 <= head_dim <= 256
    )


def _mxfp4_supported(head_dim: int, kv_heads: int, codes, scales) -> bool:
    return (
        all(t.dtype == torch.uint8 for t in codes + scales)
        and head_dim % 32 == 0
        and _cache_supported(head_dim, kv_heads, *codes)
        and 2 * codes[0].shape[3] == head_dim
        and all(t.dim() == 4 and t.stride(-1) == 1 for t in scales)
        and all(tuple(t.shape) == (codes[0].shape[0], kv_heads, head_dim // 32, codes[0].shape[2]) for t in scales)
    )


def _append_supported(q, k, v, cos, sin, positions, slots) -> bool:
    integers = (torch.int32, torch.int64)
    return (
        q.dtype in _FLOATS
        and q.dtype == k.dtype == v.dtype
        and cos.dtype in _FLOATS
        and cos.dtype == sin.dtype
        and q.dim() == k.dim() == 3
        and k.shape == v.shape
        and q.shape[0] == k.shape[0]
        and q.shape[2] == k.shape[2]
        and cos.dim() == 2
        and cos.shape == sin.shape
        and cos.shape[0] > 0
        and 1 <= cos.shape[1] <= q.shape[2] // 2
        and positions.dtype in integers
        and slots.dtype in integers
        and positions.shape == slots.shape == q.shape[:1]
    )


def _own_memory(*caches) -> bool:
    return all(stride or size < 2 for t in caches for size, stride in zip(t.shape, t.stride()))


def rope_append_supported(q, k, v, cos, sin, positions, slots, k_cache, v_cache, interleaved) -> bool:
    return (
        _on_hip(q, k, v, cos, sin, positions, slots, k_cache, v_cache)
        and _append_supported(q, k, v, cos, sin, positions, slots)
        and q.dtype == k_cache.dtype == v_cache.dtype
        and q.shape[2] % 8 == 0
        and _cache_supported(q.shape[2], k.shape[1], k_cache, v_cache)
        and k_cache.shape[3] == q.shape[2]
        and _own_memory(k_cache, v_cache)
    )


def rope_append_mxfp4_supported(q, k, v, cos, sin, positions, slots, k_codes, k_scales, v_codes, v_scales,
                                interleaved) -> bool:
    return (
        _on_hip(q, k, v, cos, sin, positions, slots, k_codes, k_scales, v_codes, v_scales)
        and _append_supported(q, k, v, cos, sin, positions, slots)
        and _mxfp4_supported(q.shape[2], k.shape[1], (k_codes, v_codes), (k_scales, v_scales))
        and _own_memory(k_codes, k_scales, v_codes, v_scales)
        and _aligned(4, k_codes, v_codes)
    )


def _table_supported(q, cache, block_table, cache_lens, cu_seqlens) -> bool:
    given = [t for t in (block_table, cache_lens, cu_seqlens) if t is not None]
    seqs = q.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
    return (
        q.dtype in _FLOATS
        and q.dim() == 3
        and cache.dim() == 4
        and cache.shape[1] > 0
        and q.shape[1] % cache.shape[1] == 0
        and all(t.dtype == torch.int32 for t in given)
        and block_table.dim() == 2
        and block_table.shape[0] == seqs
        and tuple(cache_lens.shape) == (seqs,)
        and (cu_seqlens is None or cu_seqlens.dim() == 1)
    )


def _aligned(unit: int, *tensors) -> bool:
    """Every row starts at a multiple of `unit` bytes."""
    return all(t.data_ptr() % unit == 0 and all(n < 2 or s * t.element_size() % unit == 0
                                                for n, s in zip(t.shape[:-1], t.stride())) for t in tensors)


def _alike(a, b) -> bool:
    """The same strides, where a dimension has more than one place."""
    return all(n < 2 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def attn_paged_supported(q, k_cache, v_cache, block_table, cache_lens, cu_seqlens, causal, softmax_scale) -> bool:
    return (
        _on_hip(q, k_cache, v_cache, block_table, cache_lens, cu_seqlens)
        and _table_supported(q, k_cache, block_table, cache_lens, cu_seqlens)
        and q.dtype == k_cache.dtype == v_cache.dtype
        and _attn_head_dim(q.shape[2])
        and _cache_supported(q.shape[2], k_cache.shape[1], k_cache, v_cache)
        and k_cache.shape[3] == q.shape[2]
        and _alike(k_cache, v_cache)
        and _aligned(16, k_cache, v_cache)
    )


def attn_paged_mxfp4_supported(q, k_codes, k_scales, v_codes, v_scales, block_table, cache_lens, cu_seqlens, causal,
                               softmax_scale) -> bool:
    return (
        _on_hip(q, k_codes, k_scales, v_codes, v_scales, block_table, cache_lens, cu_seqlens)
        and _table_supported(q, k_codes, block_table, cache_lens, cu_seqlens)
        and _mxfp4_supported(q.shape[2], k_codes.shape[1], (k_codes, v_codes), (k_scales, v_scales))
        and _alike(k_codes, v_codes)
        and _alike(k_scales, v_scales)
        and _aligned(16, k_codes, v_codes)
        and _aligned(4, k_scales, v_scales)
    )


# (op, source, predicate, forward_only): every op but the paged cache's has its backward kernels.
REGISTRATIONS = (
    ("rms_norm", "popcorn_amd.impls.rms_norm", rms_norm_supported, False),
    ("add_rms_norm", "popcorn_amd.impls.add_rms_norm", add_rms_norm_supported, False),
    ("swiglu", "popcorn_amd.impls.swiglu", swiglu_supported, False),
    ("rotary_embedding", "popcorn_amd.impls.rotary_embedding", rotary_supported, False),
    ("rope", "popcorn_amd.impls.rope", rope_supported, False),
    ("qk_norm_rope", "popcorn_amd.impls.qk_norm_rope", qk_norm_rope_supported, False),
    ("attn", "popcorn_amd.impls.attn", attn_supported, False),
    ("attn_varlen", "popcorn_amd.impls.attn_varlen", attn_varlen_supported, False),
    ("rope_append", "popcorn_amd.impls.rope_append", rope_append_supported, True),
    ("rope_append_mxfp4", "popcorn_amd.impls.rope_append_mxfp4", rope_append_mxfp4_supported, True),
    ("attn_paged", "popcorn_amd.impls.attn_paged", attn_paged_supported, True),
    ("attn_paged_mxfp4", "popcorn_amd.impls.attn_paged_mxfp4", attn_paged_mxfp4_supported, True),
)


def _popcorn() -> ModuleType:
    try:
        import popcorn
        import popcorn.kernels  # noqa: F401  registers Popcorn's ops

        return popcorn
    except ImportError:
        from popcorn_amd import compat

        return compat


def register(popcorn: ModuleType | None = None) -> ModuleType:
    """Declare the backend and register its ops on `popcorn` (default: the real package, else compat)."""
    pc = popcorn if popcorn is not None else _popcorn()
    pc.declare_backend(BACKEND, package=DISTRIBUTION, min_version=__version__, max_version=__version__)
    for op_name, source, predicate, forward_only in REGISTRATIONS:
        op = pc.KERNELS.get(op_name)
        if op is None:  # qk_norm_rope and the paged cache's ops exist once defined (compat ships them)
            continue
        if BACKEND not in op.available_backends():  # registering twice is a no-op, not an error
            op.register(BACKEND, source=source, predicate=predicate, forward_only=forward_only)
    return pc
