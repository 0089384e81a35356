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
    Inference only: autograd does not know of the write.

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
    device = k_cache.get_device()
    k_ptr, k_strides = _hip.row_layout(k_cache, "k_cache", device)
    v_ptr, v_strides = _hip.row_layout(v_cache, "v_cache", device)
    kt_ptr, kt_strides = _hip.row_layout(k_tree, "k_tree", device)
    vt_ptr, vt_strides = _hip.row_layout(v_tree, "v_tree", device)
    lengths = torch.empty_like(cache_seqlens)
    _hip.call_on(
        device,
        "tk_commit_draft",
        _hip.DTYPE_CODES[k_cache.dtype],
        k_ptr,
        v_ptr,
        kt_ptr,
        vt_ptr,
        cache_seqlens.data_ptr(),
        path.data_ptr(),
        count.data_ptr(),
        lengths.data_ptr(),
        batch,
        kv_heads,
        max_len,
        k_tree.shape[2],
        head_dim,
        k_strides,
        v_strides,
        kt_strides,
        vt_strides,
        _hip.stream_on(device),
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
    """Check the contract, up to the rows' layout."""
    cache_shape, tree_shape = k_cache.shape, k_tree.shape
    if len(cache_shape) != 4 or len(tree_shape) != 4:
        raise ValueError("commit_draft expects caches [batch, kv_heads, max_len, head_dim] and "
                         "drafted keys and values [batch, kv_heads, nodes, head_dim]")
    if v_cache.shape != cache_shape or v_tree.shape != tree_shape:
        raise ValueError("keys and values must have identical shapes")
    batch, kv_heads, max_len, head_dim = cache_shape
    tree_batch, tree_heads, nodes, tree_dim = tree_shape
    if tree_batch != batch or tree_heads != kv_heads or tree_dim != head_dim:
        raise ValueError("the caches and the drafted keys disagree on batch, kv_heads or head_dim")
    if not (batch and kv_heads and max_len and nodes and head_dim):
        raise ValueError("commit_draft does not support empty dimensions")
    if nodes > _MAX_NODES or batch > 65535 or kv_heads > 65535 or head_dim > 65535:
        raise ValueError("commit_draft supports at most 65535 nodes, sequences, heads and features")
    if max_len >= 2**30:
        raise ValueError("commit_draft supports caches below 2**30 positions")
    if head_dim % 8:
        raise ValueError("commit_draft requires a head_dim that is a multiple of 8")
    dtype = k_cache.dtype
    if dtype not in _DTYPES or not dtype == v_cache.dtype == k_tree.dtype == v_tree.dtype:
        raise ValueError("caches and drafted keys and values must share a float16 or bfloat16 "
                         "dtype")
    if not k_cache.is_cuda:
        raise ValueError("commit_draft requires CUDA (ROCm/HIP) tensors")
    device = k_cache.get_device()
    for name, tensor in (("k_cache", k_cache), ("v_cache", v_cache)):
        strides = tensor.stride()
        if 0 in strides and any(strides[d] == 0 and cache_shape[d] > 1 for d in range(3)):
            raise ValueError(f"{name} is written: its rows may not share memory")
    for name, tensor, shape in (("cache_seqlens", cache_seqlens, (batch,)),
                                ("count", count, (batch,)), ("path", path, (batch, nodes))):
        if (tensor.shape != shape or tensor.dtype != torch.int32
                or tensor.get_device() != device or not tensor.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous int32 {list(shape)} tensor on the "
                             "caches' device")
