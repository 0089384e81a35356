"""Grouped-query attention decode over a KV cache held in 8 bits.

``gqa_decode`` over the caches of ``quantized_cache``: one query token per sequence, query head ``h``
reads KV head ``h // (q_heads // kv_heads)`` (``docs/research/gqa_decode_model.md``, "Semantic GQA
mapping"), and the arithmetic is the reference attention forward's for one query row
(``flash_attention.py:90-117, 248-264``) on keys and values ``code * scale``: the scales multiply
scores and weights in float32, codes are exact in float16 and bfloat16, and a weight times its value's
scale goes through the second product as two bfloat16 numbers, its rounding and what that left: off by
at most 2^-16 of itself, whatever the other keys' scales and weights. Base-2 LSE. Inference only: there is no autograd.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from tklab import _hip
from tklab.kernels.quantized_cache import cache_meta, check_cache, check_lengths, lengths_meta

_DTYPES = (torch.float16, torch.bfloat16)
_HEAD_DIMS = (64, 128)


def quantized_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    scales: torch.Tensor,
    cache_seqlens: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of one query token per sequence over a grouped 8-bit KV cache.

    Args:
        q: ``[batch, q_heads, head_dim]`` float16/bfloat16; rows unit-stride and 16-byte aligned.
        k_cache, v_cache, scales: as ``append_quantized`` writes them; q_heads a multiple of
            kv_heads; head_dim 64 or 128. What lies at and past a sequence's length is not read.
        cache_seqlens: optional int32 ``[batch]`` context lengths, clamped to ``[0, max_len]`` (a
            length of 0 gives a zero output and an LSE of ``-inf``). ``None``: every sequence has
            ``max_len`` keys.
        scale: score scale, default ``1 / sqrt(head_dim)``.
        return_lse: also return the float32 base-2 LSE ``[batch, q_heads]``.

    Returns:
        The output, contiguous, in ``q``'s dtype.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
    """
    if scale is not None and not abs(scale) < 2.0**126:
        raise ValueError("scale must be finite and below 2**126")
    (batch, q_heads, head_dim), kv_heads, max_len, device, kind, slots, tables = _plan(
        q.shape, q.stride(), q.dtype, q.get_device(), *cache_meta(k_cache, v_cache, scales),
        None if cache_seqlens is None else lengths_meta(cache_seqlens))
    q_ptr, k_ptr, v_ptr, s_ptr = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr()
    if (q_ptr | k_ptr | v_ptr) & 15 or s_ptr & 7:
        _hip.check_aligned(q=q_ptr, k_cache=k_ptr, v_cache=v_ptr)
        raise ValueError("pairs of scales must be 8-byte aligned")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = workspace = None
    if return_lse:
        lse = q.new_empty((batch, q_heads), dtype=torch.float32)
    if slots:
        # Float32 partial results, as twice as many elements of q's type.
        workspace = q.new_empty(2 * slots * (q_heads // kv_heads) * (head_dim + 2))
    _hip.call_on(
        device,
        "tk_quantized_decode",
        _hip.DTYPE_CODES[q.dtype],
        q_ptr,
        k_ptr,
        v_ptr,
        s_ptr,
        None if cache_seqlens is None else cache_seqlens.data_ptr(),
        out.data_ptr(),
        None if lse is None else lse.data_ptr(),
        None if workspace is None else workspace.data_ptr(),
        batch,
        q_heads,
        kv_heads,
        max_len,
        head_dim,
        *tables,
        head_dim ** -0.5 if scale is None else float(scale),
        kind,
        _hip.stream_on(device),
    )
    return (out, lse) if return_lse else out


@lru_cache(maxsize=1024)
def _plan(q_shape, q_strides, dtype, device, k_meta, v_meta, scales_meta, seqlens):
    """Check the contract but for addresses and values: sizes, partial results that the library asks
    for, and stride tables, made once for tensors alike."""
    cache_shape = k_meta[0]
    if len(q_shape) != 3 or len(cache_shape) != 4:
        raise ValueError("quantized_decode expects q [batch, q_heads, head_dim] and caches [batch, "
                         "kv_heads, max_len, head_dim]")
    batch, q_heads, head_dim = q_shape
    _, kv_heads, max_len, _ = cache_shape
    if cache_shape[0] != batch or cache_shape[3] != head_dim:
        raise ValueError("q and the caches disagree on batch or head_dim")
    if not (batch and q_heads and kv_heads and max_len and head_dim):
        raise ValueError("quantized_decode does not support empty dimensions")
    if batch > 65535 or q_heads > 65535:
        raise ValueError("quantized_decode supports at most 65535 sequences and heads")
    if q_heads % kv_heads:
        raise ValueError("q_heads must be a multiple of kv_heads")
    if head_dim not in _HEAD_DIMS:
        raise ValueError("quantized_decode supports head_dim 64 and 128")
    if dtype not in _DTYPES:
        raise ValueError("q must be float16 or bfloat16")
    kind, tables = check_cache(k_meta, v_meta, scales_meta)
    if max(table[2] for table in tables) >= 2**24:
        raise ValueError("key strides must be below 2**24 elements")
    if k_meta[3] != device:
        raise ValueError("q must be on the caches' device")
    if seqlens is not None:
        check_lengths(seqlens, "cache_seqlens", batch, device)
    slots = _hip.query("tk_quantized_decode_slots", batch, kv_heads, q_heads // kv_heads, max_len, head_dim)
    if slots < 0:
        raise ValueError("quantized_decode: the problem is too large")
    tables = (_hip.row_strides("q", q_shape, q_strides, 2, 8), *tables,
              _hip.int64_table((q_heads * head_dim, head_dim)))
    return tuple(q_shape), kv_heads, max_len, device, kind, slots, tables
