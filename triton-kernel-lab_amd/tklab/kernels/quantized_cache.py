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

from functools import lru_cache

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
            place; head_dim a multiple of 16, at most 1024; rows 16-byte aligned; they may not overlap
            one another.
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
    device, kind, sizes, tables = _append_plan(
        *cache_meta(k_cache, v_cache, scales), lengths_meta(cache_seqlens),
        (k.shape, k.stride(), k.dtype, k.get_device()), (v.shape, v.stride(), v.dtype, v.get_device()),
        None if counts is None else lengths_meta(counts))
    k_cache_ptr, v_cache_ptr, s_ptr = k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr()
    k_ptr, v_ptr = k.data_ptr(), v.data_ptr()
    if (k_cache_ptr | v_cache_ptr | k_ptr | v_ptr) & 15 or s_ptr & 7:
        _hip.check_aligned(k_cache=k_cache_ptr, v_cache=v_cache_ptr, k=k_ptr, v=v_ptr)
        raise ValueError("pairs of scales must be 8-byte aligned")
    lengths = torch.empty_like(cache_seqlens)
    _hip.call_on(
        device,
        "tk_append_quantized",
        _hip.DTYPE_CODES[k.dtype],
        k_cache_ptr,
        v_cache_ptr,
        s_ptr,
        cache_seqlens.data_ptr(),
        k_ptr,
        v_ptr,
        None if counts is None else counts.data_ptr(),
        lengths.data_ptr(),
        *sizes,
        *tables,
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
    device, kind, sizes, tables = _read_plan(
        dtype, *cache_meta(k_cache, v_cache, scales),
        None if cache_seqlens is None else lengths_meta(cache_seqlens))
    k_ptr, v_ptr, s_ptr = k_cache.data_ptr(), v_cache.data_ptr(), scales.data_ptr()
    if (k_ptr | v_ptr) & 15 or s_ptr & 7:
        _hip.check_aligned(k_cache=k_ptr, v_cache=v_ptr)
        raise ValueError("pairs of scales must be 8-byte aligned")
    k, v = (torch.empty(sizes, dtype=dtype, device=k_cache.device) for _ in "kv")
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
        *sizes,
        *tables,
        kind,
        _hip.stream_on(device),
    )
    return k, v


# Checks of sizes, types and layouts, made once for tensors alike: they see a tensor as (shape, strides,
# dtype, device index).


def cache_meta(k_cache: torch.Tensor, v_cache: torch.Tensor, scales: torch.Tensor):
    """What the checks see of a cache's three tensors."""
    return ((k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.get_device()),
            (v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.get_device()),
            (scales.shape, scales.stride(), scales.dtype, scales.get_device()))


def lengths_meta(lengths: torch.Tensor):
    """What the checks see of a tensor of lengths."""
    return lengths.shape, lengths.stride(), lengths.dtype, lengths.get_device()


def check_cache(k_meta, v_meta, scales_meta):
    """Check a cache; its type's code and the stride tables of its three tensors."""
    shape, k_strides, dtype, device = k_meta
    kind = CACHE_TYPES.get(dtype)
    if v_meta[0] != shape:
        raise ValueError("k_cache and v_cache must have identical shapes")
    if kind is None or v_meta[2] != dtype:
        raise ValueError("k_cache and v_cache must share a float8_e4m3fn or int8 dtype")
    if 0 in shape:
        raise ValueError("a cache may not have empty dimensions")
    batch, kv_heads, max_len, head_dim = shape
    if head_dim % 16 or head_dim > _MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 16, at most {_MAX_HEAD_DIM}")
    if batch > 65535 or kv_heads > 65535 or max_len > 2**30:
        raise ValueError("a cache holds at most 65535 sequences and heads and 2**30 positions")
    scales_shape, s_strides, scales_dtype, scales_device = scales_meta
    if scales_shape != (batch, kv_heads, max_len, 2) or scales_dtype != torch.float32:
        raise ValueError("scales must be a float32 [batch, kv_heads, max_len, 2] tensor")
    if device < 0:
        raise ValueError("an 8-bit cache requires CUDA (ROCm/HIP) tensors")
    if v_meta[3] != device:
        raise ValueError("k_cache and v_cache must be on one device")
    if scales_device != device or s_strides[3] != 1:
        raise ValueError("scales must be on the caches' device with a contiguous final dimension")
    s_strides = tuple(2 if shape[d] == 1 else s_strides[d] for d in range(3))
    if (s_strides[0] | s_strides[1] | s_strides[2]) & 1:
        raise ValueError("pairs of scales must be 8-byte aligned")
    return kind, (_hip.row_strides("k_cache", shape, k_strides, 3, 16),
                  _hip.row_strides("v_cache", shape, v_meta[1], 3, 16), _hip.int64_table(s_strides))


def check_lengths(meta, name: str, batch: int, device: int) -> None:
    """Check a tensor of lengths (of one entry, whose stride addresses nothing, or contiguous)."""
    shape, strides, dtype, where = meta
    if shape != (batch,) or dtype != torch.int32 or where != device or (batch > 1 and strides[0] != 1):
        raise ValueError(f"{name} must be a contiguous int32 [batch] tensor on the caches' device")


@lru_cache(maxsize=1024)
def _append_plan(k_cache, v_cache, scales, seqlens, k, v, counts):
    cache_shape, shape, dtype = k_cache[0], k[0], k[2]
    if len(cache_shape) != 4 or len(shape) != 4:
        raise ValueError("append_quantized expects caches [batch, kv_heads, max_len, head_dim] and "
                         "tokens [batch, kv_heads, tokens, head_dim]")
    if v[0] != shape:
        raise ValueError("k and v must have identical shapes")
    if shape[0] != cache_shape[0] or shape[1] != cache_shape[1] or shape[3] != cache_shape[3]:
        raise ValueError("the caches and the tokens disagree on batch, kv_heads or head_dim")
    if dtype not in _DTYPES or v[2] != dtype:
        raise ValueError("k and v must share a float16, bfloat16 or float32 dtype")
    kind, tables = check_cache(k_cache, v_cache, scales)
    for name, meta in (("k_cache", k_cache), ("v_cache", v_cache), ("scales", scales)):
        if any(meta[1][d] == 0 and cache_shape[d] > 1 for d in range(3)):
            raise ValueError(f"{name} is written: its rows may not share memory")
    batch, kv_heads, tokens, head_dim = shape
    if tokens == 0:
        raise ValueError("append_quantized does not support empty dimensions")
    # Workgroups of 256 lanes, of which a row takes the power of two above its 16-byte parts.
    rows = 256 // min(1 << (head_dim * dtype.itemsize // 16 - 1).bit_length(), 64)
    side_by_side = min(1 << (tokens - 1).bit_length(), rows)
    workgroups = batch * -(-tokens // side_by_side) * -(-kv_heads // (rows // side_by_side))
    if workgroups >= 2**24 or tokens > 2**30:
        raise ValueError("append_quantized: the problem is too large")
    device = k_cache[3]
    if k[3] != device or v[3] != device:
        raise ValueError("k and v must be on the caches' device")
    check_lengths(seqlens, "cache_seqlens", batch, device)
    if counts is not None:
        check_lengths(counts, "counts", batch, device)
    unit = 16 // dtype.itemsize
    tables += (_hip.row_strides("k", shape, k[1], 3, unit), _hip.row_strides("v", shape, v[1], 3, unit))
    return device, kind, (batch, kv_heads, cache_shape[2], tokens, head_dim), tables


@lru_cache(maxsize=1024)
def _read_plan(dtype, k_cache, v_cache, scales, seqlens):
    if dtype not in _DTYPES:
        raise ValueError("read_quantized gives float16, bfloat16 or float32")
    shape, device = tuple(k_cache[0]), k_cache[3]
    if len(shape) != 4:
        raise ValueError("read_quantized expects caches [batch, kv_heads, max_len, head_dim]")
    kind, tables = check_cache(k_cache, v_cache, scales)
    if shape[2] * shape[3] * dtype.itemsize // 16 > 2**31 - 257:
        raise ValueError("read_quantized: the problem is too large")
    if seqlens is not None:
        check_lengths(seqlens, "cache_seqlens", shape[0], device)
    return device, kind, shape, tables
