"""Grouped-query attention decode for a batch that shares a long prefix.

Requests behind one system prompt or one document hold the same keys at their front. ``gqa_decode``
reads them once for every sequence; :func:`prefix_decode` takes them as tensors without a batch
dimension, reads them once for the whole batch, and attends over each sequence's own cache in the same
launch. Head mapping and arithmetic are ``gqa_decode``'s (``docs/research/gqa_decode_model.md``,
"Semantic GQA mapping"; ``flash_attention.py:90-117, 248-264``): scores scaled by ``scale * log2(e)``, P
rounded to the storage dtype before the PV product, base-2 LSE. Inference only: there is no autograd.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from tklab import _hip

_DTYPES = (torch.float16, torch.bfloat16)
_HEAD_DIMS = (64, 128)


def prefix_decode(
    q: torch.Tensor,
    k_prefix: torch.Tensor,
    v_prefix: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cache_seqlens: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of one query token per sequence over a shared prefix and the sequence's own cache.

    Args:
        q: ``[batch, q_heads, head_dim]`` float16/bfloat16.
        k_prefix, v_prefix: ``[kv_heads, prefix_len, head_dim]``, same dtype: the keys and values that
            every sequence sees; at least one. A longer buffer is passed as its first positions
            (``buffer[:, :n]``).
        k_cache, v_cache: ``[batch, kv_heads, max_len, head_dim]``, what follows the prefix in each
            sequence; q_heads a multiple of kv_heads; head_dim 64 or 128. What lies at and past a
            sequence's length is not read.
        cache_seqlens: optional int32 ``[batch]`` lengths of the own caches, clamped to
            ``[0, max_len]`` (0: the sequence sees the prefix alone). ``None``: ``max_len`` each.
        scale: score scale, default ``1 / sqrt(head_dim)``.
        return_lse: also return the float32 base-2 LSE ``[batch, q_heads]``.

    Returns:
        The output, contiguous, in ``q``'s dtype. All tensors may be any strided views whose rows are
        unit-stride and 16-byte aligned.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
    """
    _validate(q, k_prefix, v_prefix, k_cache, v_cache, cache_seqlens, scale)
    batch, q_heads, head_dim = q_shape = q.shape
    _, kv_heads, max_len, _ = k_cache.shape
    prefix_len = k_prefix.shape[1]
    device = q.get_device()
    q_ptr, q_strides = _hip.row_table(q, "q", device, 2, 8)
    kp_ptr, kp_strides = _hip.row_table(k_prefix, "k_prefix", device, 2, 8)
    vp_ptr, vp_strides = _hip.row_table(v_prefix, "v_prefix", device, 2, 8)
    k_ptr, k_strides = _hip.row_table(k_cache, "k_cache", device, 3, 8)
    v_ptr, v_strides = _hip.row_table(v_cache, "v_cache", device, 3, 8)
    if max(kp_strides[1], vp_strides[1], k_strides[2], v_strides[2]) >= 2**24:
        raise ValueError("key strides must be below 2**24 elements")
    slots = _slots(batch, kv_heads, q_heads // kv_heads, prefix_len, max_len, head_dim)
    if slots < 0:
        raise ValueError("prefix_decode: the problem is too large")
    out = torch.empty(q_shape, dtype=q.dtype, device=q.device)
    lse = None
    if return_lse:
        lse = torch.empty((batch, q_heads), dtype=torch.float32, device=q.device)
    # Float32 partial results, as twice as many elements of q's type.
    workspace = q.new_empty(2 * slots * (head_dim + 2))
    _hip.call_on(
        device,
        "tk_prefix_decode",
        _hip.DTYPE_CODES[q.dtype],
        q_ptr,
        kp_ptr,
        vp_ptr,
        k_ptr,
        v_ptr,
        None if cache_seqlens is None else cache_seqlens.data_ptr(),
        out.data_ptr(),
        None if lse is None else lse.data_ptr(),
        workspace.data_ptr(),
        batch,
        q_heads,
        kv_heads,
        prefix_len,
        max_len,
        head_dim,
        q_strides,
        kp_strides,
        vp_strides,
        k_strides,
        v_strides,
        _hip.int64_table((q_heads * head_dim, head_dim)),
        head_dim ** -0.5 if scale is None else float(scale),
        _hip.stream_on(device),
    )
    return (out, lse) if return_lse else out


@lru_cache(maxsize=256)
def _slots(batch: int, kv_heads: int, group: int, prefix_len: int, max_len: int, head_dim: int) -> int:
    """Partial results that the library asks for (a function of the sizes alone)."""
    return _hip.query("tk_prefix_decode_slots", batch, kv_heads, group, prefix_len, max_len, head_dim)


def _validate(q, k_prefix, v_prefix, k_cache, v_cache, cache_seqlens, scale) -> None:
    """Check the contract, up to the rows' layout."""
    q_shape, prefix_shape, cache_shape = q.shape, k_prefix.shape, k_cache.shape
    if len(q_shape) != 3 or len(prefix_shape) != 3 or len(cache_shape) != 4:
        raise ValueError("prefix_decode expects q [batch, q_heads, head_dim], a prefix [kv_heads, "
                         "prefix_len, head_dim] and caches [batch, kv_heads, max_len, head_dim]")
    if v_prefix.shape != prefix_shape or v_cache.shape != cache_shape:
        raise ValueError("keys and values must have identical shapes")
    batch, q_heads, head_dim = q_shape
    kv_heads, prefix_len, prefix_dim = prefix_shape
    if cache_shape[0] != batch or cache_shape[3] != head_dim:
        raise ValueError("q and the caches disagree on batch or head_dim")
    if cache_shape[1] != kv_heads or prefix_dim != head_dim:
        raise ValueError("the prefix and the caches disagree on kv_heads or head_dim")
    if not (batch and q_heads and kv_heads and prefix_len and cache_shape[2] and head_dim):
        raise ValueError("prefix_decode does not support empty dimensions")
    if batch > 65535 or q_heads > 65535:
        raise ValueError("prefix_decode supports at most 65535 sequences and heads")
    if q_heads % kv_heads:
        raise ValueError("q_heads must be a multiple of kv_heads")
    if head_dim not in _HEAD_DIMS:
        raise ValueError("prefix_decode supports head_dim 64 and 128")
    dtype = q.dtype
    if dtype not in _DTYPES or not (
            dtype == k_prefix.dtype == v_prefix.dtype == k_cache.dtype == v_cache.dtype):
        raise ValueError("q, prefix and caches must share a float16 or bfloat16 dtype")
    if scale is not None and not abs(scale) < 2.0**126:
        raise ValueError("scale must be finite and below 2**126")
    if not q.is_cuda:
        raise ValueError("prefix_decode requires CUDA (ROCm/HIP) tensors")
    if cache_seqlens is not None and (
            cache_seqlens.shape != (batch,) or cache_seqlens.dtype != torch.int32
            or cache_seqlens.get_device() != q.get_device() or not cache_seqlens.is_contiguous()):
        raise ValueError("cache_seqlens must be a contiguous int32 [batch] tensor on q's device")
