"""Grouped-query attention decode for a batch that shares a long prefix.

Requests behind one system prompt or one document hold the same keys at their front. ``gqa_decode``
reads them once for every sequence; :func:`prefix_decode` takes them as tensors without a batch
dimension, reads them once for the whole batch, and attends over each sequence's own cache in the same
launch. Head mapping and arithmetic are ``gqa_decode``'s (``docs/research/gqa_decode_model.md``,
"Semantic GQA mapping"; ``flash_attention.py:90-117, 248-264``): scores scaled by ``scale * log2(e)``, P
rounded to the storage dtype before the PV product (in float16 a weight below 2^-21 of the largest is off
by up to 2^-32 of that), base-2 LSE. Inference only: there is no autograd.
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
    if scale is not None and not abs(scale) < 2.0**126:
        raise ValueError("scale must be finite and below 2**126")
    (batch, q_heads, head_dim), kv_heads, prefix_len, max_len, device, slots, tables = _plan(
        q.shape, q.stride(), q.dtype, q.get_device(),
        k_prefix.shape, k_prefix.stride(), k_prefix.dtype, k_prefix.get_device(),
        v_prefix.shape, v_prefix.stride(), v_prefix.dtype, v_prefix.get_device(),
        k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.get_device(),
        v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.get_device(),
        None if cache_seqlens is None else (cache_seqlens.shape, cache_seqlens.stride(),
                                            cache_seqlens.dtype, cache_seqlens.get_device()))
    q_ptr, kp_ptr, vp_ptr = q.data_ptr(), k_prefix.data_ptr(), v_prefix.data_ptr()
    k_ptr, v_ptr = k_cache.data_ptr(), v_cache.data_ptr()
    if (q_ptr | kp_ptr | vp_ptr | k_ptr | v_ptr) & 15:
        _hip.check_aligned(q=q_ptr, k_prefix=kp_ptr, v_prefix=vp_ptr, k_cache=k_ptr, v_cache=v_ptr)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = None
    if return_lse:
        lse = q.new_empty((batch, q_heads), dtype=torch.float32)
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
        *tables,
        head_dim ** -0.5 if scale is None else float(scale),
        _hip.stream_on(device),
    )
    return (out, lse) if return_lse else out


@lru_cache(maxsize=1024)
def _plan(q_shape, q_strides, dtype, device, prefix_shape, kp_strides, kp_dtype, kp_device, vp_shape, vp_strides,
          vp_dtype, vp_device, cache_shape, k_strides, k_dtype, k_device, v_shape, v_strides, v_dtype, v_device,
          seqlens):
    """Check the contract but for addresses and values: sizes, partial results that the library asks
    for, and stride tables, made once for tensors alike."""
    if len(q_shape) != 3 or len(prefix_shape) != 3 or len(cache_shape) != 4:
        raise ValueError("prefix_decode expects q [batch, q_heads, head_dim], a prefix [kv_heads, "
                         "prefix_len, head_dim] and caches [batch, kv_heads, max_len, head_dim]")
    if vp_shape != prefix_shape or v_shape != cache_shape:
        raise ValueError("keys and values must have identical shapes")
    batch, q_heads, head_dim = q_shape
    kv_heads, prefix_len, prefix_dim = prefix_shape
    max_len = cache_shape[2]
    if cache_shape[0] != batch or cache_shape[3] != head_dim:
        raise ValueError("q and the caches disagree on batch or head_dim")
    if cache_shape[1] != kv_heads or prefix_dim != head_dim:
        raise ValueError("the prefix and the caches disagree on kv_heads or head_dim")
    if not (batch and q_heads and kv_heads and prefix_len and max_len and head_dim):
        raise ValueError("prefix_decode does not support empty dimensions")
    if batch > 65535 or q_heads > 65535:
        raise ValueError("prefix_decode supports at most 65535 sequences and heads")
    if q_heads % kv_heads:
        raise ValueError("q_heads must be a multiple of kv_heads")
    if head_dim not in _HEAD_DIMS:
        raise ValueError("prefix_decode supports head_dim 64 and 128")
    if dtype not in _DTYPES or not dtype == kp_dtype == vp_dtype == k_dtype == v_dtype:
        raise ValueError("q, prefix and caches must share a float16 or bfloat16 dtype")
    if device < 0:
        raise ValueError("prefix_decode requires CUDA (ROCm/HIP) tensors")
    for name, other in (("k_prefix", kp_device), ("v_prefix", vp_device), ("k_cache", k_device),
                        ("v_cache", v_device)):
        if other != device:
            raise ValueError(f"{name} must be on q's device")
    if seqlens is not None and (seqlens[0] != (batch,) or seqlens[2] != torch.int32 or seqlens[3] != device
                                or (batch > 1 and seqlens[1][0] != 1)):
        raise ValueError("cache_seqlens must be a contiguous int32 [batch] tensor on q's device")
    tables = (_hip.row_strides("q", q_shape, q_strides, 2, 8),
              _hip.row_strides("k_prefix", prefix_shape, kp_strides, 2, 8),
              _hip.row_strides("v_prefix", prefix_shape, vp_strides, 2, 8),
              _hip.row_strides("k_cache", cache_shape, k_strides, 3, 8),
              _hip.row_strides("v_cache", cache_shape, v_strides, 3, 8),
              _hip.int64_table((q_heads * head_dim, head_dim)))
    if max(tables[1][1], tables[2][1], tables[3][2], tables[4][2]) >= 2**24:
        raise ValueError("key strides must be below 2**24 elements")
    slots = _hip.query("tk_prefix_decode_slots", batch, kv_heads, q_heads // kv_heads, prefix_len, max_len,
                       head_dim)
    if slots < 0:
        raise ValueError("prefix_decode: the problem is too large")
    return tuple(q_shape), kv_heads, prefix_len, max_len, device, slots, tables
