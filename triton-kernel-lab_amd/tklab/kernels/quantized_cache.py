"""A KV cache held in 8 bits: tokens quantised as they are written, and the cache read back.

Half the bytes of the 16-bit caches that ``gqa_decode`` reads. Every row, a token's key or value of
one KV head, is 8-bit codes (``torch.float8_e4m3fn`` or ``torch.int8``) and a float32 scale::

    a = max(max |x|, 2**-100);  scale = a / M;  code = round(x * (M * (1 / a)));  M = 448 or 127

Keys and values are two tensors ``[batch, kv_heads, max_len, head_dim]``, their scales one,
``[batch, kv_heads, max_len, 2]`` (the key's, the value's). :func:`append_quantized` writes tokens
behind each sequence's context, :func:`read_quantized` multiplies a cache out, and
``quantized_decode`` attends over it without doing so. There is no counterpart in the reference.
Inference only: autograd does not know of these calls.
"""

from __future__ import annotations

import torch

from tklab import _hip

CACHE_TYPES = {torch.float8_e4m3fn: 0, torch.int8: 1}
_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_MAX_HEAD_DIM = 1024


def append_quantized(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    scales: torch.Tensor,
    cache_seqlens: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    counts: torch.Tensor | None = None,
) -> torch.Tensor:
    """Quantise the tokens of ``k`` and ``v`` behind each sequence's context; return the new lengths.

    Row ``t`` of sequence ``b`` becomes cache row ``cache_seqlens[b] + t``, for ``t < counts[b]``.
    Rows that would lie past the cache's end are not written and not counted; all other rows are
    left as they were. ``cache_seqlens`` is not changed. A row holding an infinity or a NaN gets a
    scale of NaN (and codes of zero): everything read back of it is NaN.

    Args:
        k_cache, v_cache: ``[batch, kv_heads, max_len, head_dim]`` float8_e4m3fn or int8, written in
            place; head_dim a multiple of 16, at most 1024; rows 16-byte aligned.
        scales: float32 ``[batch, kv_heads, max_len, 2]``, written in place; pairs 8-byte aligned.
        cache_seqlens: int32 ``[batch]`` context lengths, clamped to ``[0, max_len]``.
        k, v: ``[batch, kv_heads, tokens, head_dim]`` float16, bfloat16 or float32, any strides whose
            rows are unit-stride and 16-byte aligned; may not overlap the caches.
        counts: optional int32 ``[batch]``, the tokens of each sequence in a padded batch, clamped to
            ``[0, tokens]``; ``None``: all of them.

    Returns:
        int32 ``[batch]``: ``min(cache_seqlens + counts, max_len)``.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
    """
    cache_shape, shape = k_cache.shape, k.shape
    if len(cache_shape) != 4 or len(shape) != 4:
        raise ValueError("append_quantized expects caches [batch, kv_heads, max_len, head_dim] and "
                         "tokens [batch, kv_heads, tokens, head_dim]")
    if v.shape != shape:
        raise ValueError("k and v must have identical shapes")
    if shape[0] != cache_shape[0] or shape[1] != cache_shape[1] or shape[3] != cache_shape[3]:
        raise ValueError("the caches and the tokens disagree on batch, kv_heads or head_dim")
    dtype = k.dtype
    if dtype not in _DTYPES or v.dtype != dtype:
        raise ValueError("k and v must share a float16, bfloat16 or float32 dtype")
    caches = _cache_layout(k_cache, v_cache, scales, written=True)
    batch, kv_heads, tokens, head_dim = shape
    if tokens == 0:
        raise ValueError("append_quantized does not support empty dimensions")
    lanes = min(1 << (head_dim * dtype.itemsize // 16 - 1).bit_length(), 64)
    if batch * kv_heads * tokens * lanes >= 2**31 or tokens > 2**30:
        raise ValueError("append_quantized: the problem is too large")
    device = k_cache.get_device()
    _check_lengths(cache_seqlens, "cache_seqlens", batch, device)
    if counts is not None:
        _check_lengths(counts, "counts", batch, device)
    unit = 16 // dtype.itemsize
    k_ptr, k_strides = _hip.row_table(k, "k", device, 3, unit)
    v_ptr, v_strides = _hip.row_table(v, "v", device, 3, unit)
    lengths = torch.empty_like(cache_seqlens)
    (k_cache_ptr, k_cache_strides), (v_cache_ptr, v_cache_strides), (s_ptr, s_strides), kind = caches
    _hip.call_on(
        device,
        "tk_append_quantized",
        _hip.DTYPE_CODES[dtype],
        k_cache_ptr,
        v_cache_ptr,
        s_ptr,
        cache_seqlens.data_ptr(),
        k_ptr,
        v_ptr,
        None if counts is None else counts.data_ptr(),
        lengths.data_ptr(),
        batch,
        kv_heads,
        cache_shape[2],
        tokens,
        head_dim,
        k_cache_strides,
        v_cache_strides,
        s_strides,
        k_strides,
        v_strides,
        kind,
        _hip.stream_on(device),
    )
    return lengths


def read_quantized(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    scales: torch.Tensor,
    cache_seqlens: torch.Tensor | None = None,
    *,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that an 8-bit cache stands for: ``code * scale`` in ``dtype``.

    Args:
        k_cache, v_cache, scales: as :func:`append_quantized` writes them; slices along the positions
            and other views are taken, so a part of a cache can be read.
        cache_seqlens: optional int32 ``[batch]``; positions from there on are zeros and what the
            cache holds there is not read. ``None``: every position is read.
        dtype: float16, bfloat16 or float32.

    Returns:
        ``(k, v)``, contiguous ``[batch, kv_heads, max_len, head_dim]``; products in float32, rounded
        once.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
    """
    if dtype not in _DTYPES:
        raise ValueError("read_quantized gives float16, bfloat16 or float32")
    if k_cache.ndim != 4:
        raise ValueError("read_quantized expects caches [batch, kv_heads, max_len, head_dim]")
    (k_ptr, k_strides), (v_ptr, v_strides), (s_ptr, s_strides), kind = _cache_layout(
        k_cache, v_cache, scales)
    batch, kv_heads, max_len, head_dim = shape = k_cache.shape
    if max_len * head_dim * dtype.itemsize // 16 > 2**31 - 257:
        raise ValueError("read_quantized: the problem is too large")
    device = k_cache.get_device()
    if cache_seqlens is not None:
        _check_lengths(cache_seqlens, "cache_seqlens", batch, device)
    k, v = (torch.empty(shape, dtype=dtype, device=k_cache.device) for _ in "kv")
    _hip.call_on(
        device,
        "tk_read_quantized",
        _hip.DTYPE_CODES[dtype],
        k_ptr,
        v_ptr,
        s_ptr,
        None if cache_seqlens is None else cache_seqlens.data_ptr(),
        k.data_ptr(),
        v.data_ptr(),
        batch,
        kv_heads,
        max_len,
        head_dim,
        k_strides,
        v_strides,
        s_strides,
        kind,
        _hip.stream_on(device),
    )
    return k, v


def _cache_layout(k_cache, v_cache, scales, *, written: bool = False):
    """(address, strides) of the caches and their scales, checked, and the type's code."""
    shape, kind = k_cache.shape, CACHE_TYPES.get(k_cache.dtype)
    if v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must have identical shapes")
    if kind is None or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must share a float8_e4m3fn or int8 dtype")
    if 0 in shape:
        raise ValueError("a cache may not have empty dimensions")
    batch, kv_heads, max_len, head_dim = shape
    if head_dim % 16 or head_dim > _MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 16, at most {_MAX_HEAD_DIM}")
    if batch > 65535 or kv_heads > 65535 or max_len > 2**30:
        raise ValueError("a cache holds at most 65535 sequences and heads and 2**30 positions")
    if scales.shape != (batch, kv_heads, max_len, 2) or scales.dtype != torch.float32:
        raise ValueError("scales must be a float32 [batch, kv_heads, max_len, 2] tensor")
    if not k_cache.is_cuda:
        raise ValueError("an 8-bit cache requires CUDA (ROCm/HIP) tensors")
    device = k_cache.get_device()
    k = _hip.row_table(k_cache, "k_cache", device, 3, 16)
    v = _hip.row_table(v_cache, "v_cache", device, 3, 16)
    s_ptr, s_strides = scales.data_ptr(), scales.stride()
    if scales.get_device() != device or s_strides[3] != 1:
        raise ValueError("scales must be on the caches' device with a contiguous final dimension")
    if 1 in shape:
        s_strides = tuple(2 if shape[d] == 1 else s_strides[d] for d in range(3))
    if s_ptr & 7 or (s_strides[0] | s_strides[1] | s_strides[2]) & 1:
        raise ValueError("pairs of scales must be 8-byte aligned")
    if written:
        for name, tensor in (("k_cache", k_cache), ("v_cache", v_cache), ("scales", scales)):
            strides = tensor.stride()
            if 0 in strides and any(strides[d] == 0 and shape[d] > 1 for d in range(3)):
                raise ValueError(f"{name} is written: its rows may not share memory")
    return k, v, (s_ptr, _hip.int64_table(s_strides[:3])), kind


def _check_lengths(lengths: torch.Tensor, name: str, batch: int, device: int) -> None:
    if (lengths.shape != (batch,) or lengths.dtype != torch.int32
            or lengths.get_device() != device or not lengths.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 [batch] tensor on the caches' device")
