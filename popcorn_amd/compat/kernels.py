"""The transformer-block ops, registered with their torch references.

Signatures, shape annotations and test-argument pools are Popcorn's
(kernels/rms_norm.py:16-30, kernels/add_rms_norm.py:8-26, kernels/swiglu.py:9-18,
kernels/rotary_embedding.py:12-40, kernels/rope.py:19-36, kernels/attn.py:10-37,
kernels/attn_varlen.py:15-54); the arithmetic is
the eager-torch restatement in `popcorn_amd.compat.references`.
"""

import torch
from torch import Tensor

from popcorn_amd.compat import references
from popcorn_amd.compat.ops import register_kernel
from popcorn_amd.compat.shapes import Float, Int, Int32, UInt8


@register_kernel(test_args={"eps": [1e-6, 1e-5]})
def rms_norm(
    x: Float[Tensor, "... normalized_shape"],
    weight: Float[Tensor, "normalized_shape"],
    bias: Float[Tensor, "normalized_shape"] | None = None,
    eps: float = 1e-6,
) -> Float[Tensor, "... normalized_shape"]:
    """Root-mean-square normalization: x * rsqrt(mean(x^2) + eps) * weight (+ bias)."""
    return references.rms_norm(x, weight, bias, eps)


@register_kernel(test_args={"eps": [1e-6, 1e-5], "offset": [0.0, 1.0]})
def add_rms_norm(
    x: Float[Tensor, "... hidden"],
    residual: Float[Tensor, "... hidden"],
    weight: Float[Tensor, "hidden"],
    eps: float = 1e-6,
    offset: float = 0.0,
) -> tuple[Tensor, Tensor]:
    """Residual add fused with RMS norm: (rms(x + residual) * (weight + offset), x + residual)."""
    return references.add_rms_norm(x, residual, weight, eps, offset)


@register_kernel
def swiglu(a: Float[Tensor, "... hidden"], b: Float[Tensor, "... hidden"]) -> Float[Tensor, "... hidden"]:
    """SwiGLU gating: silu(a) * b."""
    return references.swiglu(a, b)


@register_kernel
def rotary_embedding(
    x: Float[Tensor, "batch seq heads head_dim"],
    cos: Float[Tensor, "seq half"],
    sin: Float[Tensor, "seq half"],
    interleaved: bool = False,
) -> Float[Tensor, "batch seq heads head_dim"]:
    """Rotary position embedding, GPT-NeoX halves or GPT-J interleaved pairs."""
    return references.rotary_embedding(x, cos, sin, interleaved)


@register_kernel(test_inputs={"cos": references.rope_table(torch.cos), "sin": references.rope_table(torch.sin)},
                 tags={"positional"})
def rope(
    q: Float[Tensor, "batch q_heads seq head_dim"],
    k: Float[Tensor, "batch kv_heads seq head_dim"],
    cos: Float[Tensor, "cos_batch seq head_dim"],
    sin: Float[Tensor, "cos_batch seq head_dim"],
) -> tuple[Tensor, Tensor]:
    """Paired rotary embedding of queries and keys: x*cos + rotate_half(x)*sin."""
    return references.rope(q, k, cos, sin)


@register_kernel(test_args={"eps": [1e-6]},
                 test_inputs={"cos": references.rope_table(torch.cos), "sin": references.rope_table(torch.sin)},
                 tags={"normalization", "positional", "fused"})
def qk_norm_rope(
    q: Float[Tensor, "batch q_heads seq head_dim"],
    k: Float[Tensor, "batch kv_heads seq head_dim"],
    q_weight: Float[Tensor, "head_dim"],
    k_weight: Float[Tensor, "head_dim"],
    cos: Float[Tensor, "cos_batch seq head_dim"],
    sin: Float[Tensor, "cos_batch seq head_dim"],
    eps: float = 1e-6,
) -> tuple[Tensor, Tensor]:
    """Per-head RMS normalization of queries and keys, followed by rotary embedding.

    Not an op Popcorn ships: its kernel-writing notebook defines it
    (examples/03_write_a_kernel.ipynb, cell 3) with this signature and these
    test inputs.
    """
    return references.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, eps)


@register_kernel(test_args={"softmax_scale": [None, 0.25]})
def attn(
    q: Float[Tensor, "batch seq q_heads head_dim"],
    k: Float[Tensor, "batch seq kv_heads head_dim"],
    v: Float[Tensor, "batch seq kv_heads head_dim"],
    causal: bool = False,
    softmax_scale: float | None = None,
) -> Float[Tensor, "batch seq q_heads head_dim"]:
    """Multi-head attention with grouped kv heads (q_heads a multiple of kv_heads)."""
    return references.attn(q, k, v, causal, softmax_scale)


@register_kernel(test_args={"softmax_scale": [None, 0.25]}, test_inputs={"cu_seqlens": references.cuts})
def attn_varlen(
    q: Float[Tensor, "total q_heads head_dim"],
    k: Float[Tensor, "total kv_heads head_dim"],
    v: Float[Tensor, "total kv_heads head_dim"],
    cu_seqlens: Int32[Tensor, "boundaries"],
    causal: bool = False,
    softmax_scale: float | None = None,
) -> Float[Tensor, "total q_heads head_dim"]:
    """Attention over packed variable-length sequences, each attended independently."""
    return references.attn_varlen(q, k, v, cu_seqlens, causal, softmax_scale)


# The paged cache's ops: not Popcorn's, in its manner. They write the cache in place and are forward-only.

@register_kernel(test_inputs={"slots": references.distinct_slots}, tags={"positional", "cache"})
def rope_append(
    q: Float[Tensor, "tokens q_heads head_dim"],
    k: Float[Tensor, "tokens kv_heads head_dim"],
    v: Float[Tensor, "tokens kv_heads head_dim"],
    cos: Float[Tensor, "max_positions half"],
    sin: Float[Tensor, "max_positions half"],
    positions: Int[Tensor, "tokens"],
    slots: Int[Tensor, "tokens"],
    k_cache: Float[Tensor, "pages kv_heads page_size head_dim"],
    v_cache: Float[Tensor, "pages kv_heads page_size head_dim"],
    interleaved: bool = False,
) -> tuple[Tensor, Tensor]:
    """Rotate new queries and keys and append the keys and values to a paged cache: (yq, yk)."""
    return references.rope_append(q, k, v, cos, sin, positions, slots, k_cache, v_cache, interleaved)


@register_kernel(test_inputs={"slots": references.distinct_slots}, tags={"positional", "cache"})
def rope_append_mxfp4(
    q: Float[Tensor, "tokens q_heads head_dim"],
    k: Float[Tensor, "tokens kv_heads head_dim"],
    v: Float[Tensor, "tokens kv_heads head_dim"],
    cos: Float[Tensor, "max_positions half"],
    sin: Float[Tensor, "max_positions half"],
    positions: Int[Tensor, "tokens"],
    slots: Int[Tensor, "tokens"],
    k_codes: UInt8[Tensor, "pages kv_heads page_size packed"],
    k_scales: UInt8[Tensor, "pages kv_heads blocks page_size"],
    v_codes: UInt8[Tensor, "pages kv_heads page_size packed"],
    v_scales: UInt8[Tensor, "pages kv_heads blocks page_size"],
    interleaved: bool = False,
) -> tuple[Tensor, Tensor, Tensor]:
    """`rope_append` into an MXFP4 cache: (yq, yk, yv), the last two what the cache now stands for."""
    return references.rope_append_mxfp4(q, k, v, cos, sin, positions, slots, k_codes, k_scales, v_codes, v_scales,
                                        interleaved)


@register_kernel(test_args={"softmax_scale": [None, 0.25]},
                 test_inputs={"block_table": references.table_entries, "cache_lens": references.cached_lengths,
                              "cu_seqlens": references.cuts},
                 tags={"cache"})
def attn_paged(
    q: Float[Tensor, "total q_heads head_dim"],
    k_cache: Float[Tensor, "pages kv_heads page_size head_dim"],
    v_cache: Float[Tensor, "pages kv_heads page_size head_dim"],
    block_table: Int32[Tensor, "sequences table_pages"],
    cache_lens: Int32[Tensor, "sequences"],
    cu_seqlens: Int32[Tensor, "boundaries"] | None = None,
    causal: bool = True,
    softmax_scale: float | None = None,
) -> Float[Tensor, "total q_heads head_dim"]:
    """Attention of each sequence's new tokens over its pages of a cache of keys and values."""
    return references.attn_paged(q, k_cache, v_cache, block_table, cache_lens, cu_seqlens, causal, softmax_scale)


@register_kernel(test_args={"softmax_scale": [None, 0.25]},
                 test_inputs={"block_table": references.table_entries, "cache_lens": references.cached_lengths,
                              "cu_seqlens": references.cuts},
                 tags={"cache"})
def attn_paged_mxfp4(
    q: Float[Tensor, "total q_heads head_dim"],
    k_codes: UInt8[Tensor, "pages kv_heads page_size packed"],
    k_scales: UInt8[Tensor, "pages kv_heads blocks page_size"],
    v_codes: UInt8[Tensor, "pages kv_heads page_size packed"],
    v_scales: UInt8[Tensor, "pages kv_heads blocks page_size"],
    block_table: Int32[Tensor, "sequences table_pages"],
    cache_lens: Int32[Tensor, "sequences"],
    cu_seqlens: Int32[Tensor, "boundaries"] | None = None,
    causal: bool = True,
    softmax_scale: float | None = None,
) -> Float[Tensor, "total q_heads head_dim"]:
    """`attn_paged` over an MXFP4 cache."""
    return references.attn_paged_mxfp4(q, k_codes, k_scales, v_codes, v_scales, block_table, cache_lens, cu_seqlens,
                                       causal, softmax_scale)
