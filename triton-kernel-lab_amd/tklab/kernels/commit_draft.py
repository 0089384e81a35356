"""Append the accepted nodes of a drafted tree to the KV cache.

``tree_decode`` reads the drafted tokens' keys and values from tensors of their own, so a rejected
draft never touches the cache; this call copies the rows of the branch that ``verify_draft``
accepted behind each sequence's context. There is no counterpart in the reference.
"""

from __future__ import annotations

import torch

from tklab import _hip

_DTYPES = (torch.float16, torch.bfloat16)
_MAX_NODES = 65535


def commit_draft(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cache_seqlens: torch.Tensor,
    k_tree: torch.Tensor,
    v_tree: torch.Tensor,
    path: torch.Tensor,
    count: torch.Tensor,
) -> torch.Tensor:
    """Write rows ``path[b, :count[b]]`` of the tree behind each context; return the new lengths.

    Cache position ``cache_seqlens[b] + i`` of every KV head takes node ``path[b, i]``'s key and
    value, for ``i < count[b]``. Rows that would lie past the cache's end are not written and not
    counted; all other cache rows are left as they were. ``cache_seqlens`` is not changed.

    Args:
        k_cache, v_cache: ``[batch, kv_heads, max_len, head_dim]`` float16 or bfloat16, written
            in place; rows 16-byte aligned.
        cache_seqlens: int32 ``[batch]`` context lengths, clamped to ``[0, max_len]``.
        k_tree, v_tree: ``[batch, kv_heads, nodes, head_dim]``, same dtype; may not overlap the
            caches.
        path: int32 ``[batch, nodes]``, contiguous; an entry outside ``[0, nodes)`` below
            ``count`` leaves its row unwritten.
        count: int32 ``[batch]``, clamped to ``[0, nodes]``.

    Returns:
        int32 ``[batch]``: ``min(cache_seqlens + count, max_len)``.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
    """
    _validate(k_cache, v_cache, cache_seqlens, k_tree, v_tree, path, count)
    batch, kv_heads, max_len, head_dim = k_cache.shape
    lengths = torch.empty_like(cache_seqlens)
    _hip.call_on(
        k_cache,
        "tk_commit_draft",
        _hip.dtype_code(k_cache.dtype),
        k_cache.data_ptr(),
        v_cache.data_ptr(),
        k_tree.data_ptr(),
        v_tree.data_ptr(),
        cache_seqlens.data_ptr(),
        path.data_ptr(),
        count.data_ptr(),
        lengths.data_ptr(),
        batch,
        kv_heads,
        max_len,
        k_tree.shape[2],
        head_dim,
        _hip.int64_array(k_cache.stride()[:3]),
        _hip.int64_array(v_cache.stride()[:3]),
        _hip.int64_array(k_tree.stride()[:3]),
        _hip.int64_array(v_tree.stride()[:3]),
        _hip.stream_of(k_cache),
    )
    return lengths


def _validate(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cache_seqlens: torch.Tensor,
    k_tree: torch.Tensor,
    v_tree: torch.Tensor,
    path: torch.Tensor,
    count: torch.Tensor,
) -> None:
    """Check the contract."""
    if k_cache.ndim != 4 or k_tree.ndim != 4:
        raise ValueError("commit_draft expects caches [batch, kv_heads, max_len, head_dim] and "
                         "drafted keys and values [batch, kv_heads, nodes, head_dim]")
    if v_cache.shape != k_cache.shape or v_tree.shape != k_tree.shape:
        raise ValueError("keys and values must have identical shapes")
    batch, kv_heads, max_len, head_dim = k_cache.shape
    nodes = k_tree.shape[2]
    if (k_tree.shape[0], k_tree.shape[1], k_tree.shape[3]) != (batch, kv_heads, head_dim):
        raise ValueError("the caches and the drafted keys disagree on batch, kv_heads or head_dim")
    if k_cache.numel() == 0 or k_tree.numel() == 0:
        raise ValueError("commit_draft does not support empty dimensions")
    if nodes > _MAX_NODES or batch > 65535 or kv_heads > 65535 or head_dim > 65535:
        raise ValueError("commit_draft supports at most 65535 nodes, sequences, heads and features")
    if max_len >= 2**30:
        raise ValueError("commit_draft supports caches below 2**30 positions")
    if head_dim % 8:
        raise ValueError("commit_draft requires a head_dim that is a multiple of 8")
    if k_cache.dtype not in _DTYPES or any(
            t.dtype != k_cache.dtype for t in (v_cache, k_tree, v_tree)):
        raise ValueError("caches and drafted keys and values must share a float16 or bfloat16 "
                         "dtype")
    if k_cache.device.type != "cuda":
        raise ValueError("commit_draft requires CUDA (ROCm/HIP) tensors")
    for name, tensor in (("k_cache", k_cache), ("v_cache", v_cache), ("k_tree", k_tree),
                         ("v_tree", v_tree)):
        if tensor.device != k_cache.device:
            raise ValueError(f"{name} must be on the caches' device")
        if tensor.stride(-1) != 1:
            raise ValueError(f"{name} requires a contiguous final dimension")
        if tensor.data_ptr() % 16 or any(s % 8 or s < 0 for s in tensor.stride()[:3]):
            raise ValueError(f"{name} rows must be 16-byte aligned (strides multiples of 8)")
    for name, tensor in (("k_cache", k_cache), ("v_cache", v_cache)):
        if any(s == 0 and n > 1 for s, n in zip(tensor.stride(), tensor.shape)):
            raise ValueError(f"{name} is written: its rows may not share memory")
    for name, tensor, shape in (("cache_seqlens", cache_seqlens, (batch,)),
                                ("count", count, (batch,)), ("path", path, (batch, nodes))):
        if (tuple(tensor.shape) != shape or tensor.dtype != torch.int32
                or tensor.device != k_cache.device or not tensor.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous int32 {list(shape)} tensor on the "
                             "caches' device")
