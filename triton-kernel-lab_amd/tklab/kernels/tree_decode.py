"""Attention of a tree (or chain) of drafted tokens over a grouped KV cache.

The target's pass of speculative decoding: where ``gqa_decode`` answers one query token per
sequence, :func:`tree_decode` answers all of a sequence's drafted tokens at once. Every drafted
token sees the sequence's context in the cache, and those drafted tokens that a mask names (its
ancestors and itself, :func:`tree_mask`). The drafted tokens' keys and values are tensors of their
own, so a rejected draft never enters the cache (``commit_draft`` appends the accepted ones).
Head mapping and arithmetic are ``gqa_decode``'s (``docs/research/gqa_decode_model.md``,
"Semantic GQA mapping"; ``flash_attention.py:90-117, 248-264``): scores scaled by
``scale * log2(e)``, P rounded to the storage dtype before the PV product, base-2 LSE. Inference
only: there is no autograd.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from tklab import _hip

_DTYPES = (torch.float16, torch.bfloat16)
_HEAD_DIMS = (64, 128)
_MAX_NODES = 256


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """The mask of a tree: node ``i`` sees its ancestors and itself.

    ``parents`` is an integer ``[nodes]`` or ``[batch, nodes]`` tensor, every parent before its
    children; a parent outside ``[0, i)`` starts a tree of its own (node 0, padding). Returns bool
    ``[(batch,) nodes, nodes]`` on the same device. Made once per tree shape.
    """
    if parents.ndim not in (1, 2) or parents.numel() == 0 or parents.is_floating_point():
        raise ValueError("parents must be an integer [nodes] or [batch, nodes] tensor")
    nodes = parents.shape[-1]
    index = torch.arange(nodes, device=parents.device)
    # The ancestor `steps` generations back, or the tree's root, and who is reached in fewer.
    ancestor = torch.where((parents >= 0) & (parents < index), parents.long(), index)
    reach = torch.eye(nodes, dtype=torch.bool, device=parents.device).expand(*parents.shape, nodes)
    steps = 1
    while steps <= nodes:
        reach = reach | reach.gather(-2, ancestor[..., None].expand(*parents.shape, nodes))
        ancestor = ancestor.gather(-1, ancestor)
        steps *= 2
    return reach


def tree_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_tree: torch.Tensor,
    v_tree: torch.Tensor,
    mask: torch.Tensor,
    cache_seqlens: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of ``nodes`` drafted tokens per sequence over the cache and each other.

    Args:
        q: ``[batch, q_heads, nodes, head_dim]`` float16/bfloat16; at most 256 nodes.
        k_cache, v_cache: ``[batch, kv_heads, max_len, head_dim]``, same dtype; q_heads a
            multiple of kv_heads; head_dim 64 or 128.
        k_tree, v_tree: ``[batch, kv_heads, nodes, head_dim]``, the drafted tokens' own.
        mask: bool ``[nodes, nodes]`` or ``[batch, nodes, nodes]``: ``mask[i, j]`` lets node
            ``i`` see node ``j``. A key that a node does not see cannot reach its result, whatever
            it holds (infinities and NaN included; cache positions that share memory with a seen
            one must hold finite values).
        cache_seqlens: optional int32 ``[batch]`` context lengths, clamped to ``[0, max_len]``;
            ``None`` means every sequence has ``max_len`` keys.
        scale: score scale, default ``1 / sqrt(head_dim)``.
        return_lse: also return the float32 base-2 LSE ``[batch, q_heads, nodes]``.

    Returns:
        The output in ``q``'s shape and memory order; a node that sees no key at all gives zeros
        and an LSE of ``-inf``. Any strides whose rows are unit-stride and 16-byte aligned.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
    """
    _validate(q, k_cache, v_cache, k_tree, v_tree, mask, cache_seqlens, scale)
    batch, q_heads, nodes, head_dim = q.shape
    _, kv_heads, max_len, _ = k_cache.shape
    device = q.get_device()
    q_ptr, q_strides = _hip.row_layout(q, "q", device)
    k_ptr, k_strides = _hip.row_layout(k_cache, "k_cache", device)
    v_ptr, v_strides = _hip.row_layout(v_cache, "v_cache", device)
    kt_ptr, kt_strides = _hip.row_layout(k_tree, "k_tree", device)
    vt_ptr, vt_strides = _hip.row_layout(v_tree, "v_tree", device)
    group = q_heads // kv_heads
    slots = _slots(batch, kv_heads, group, max_len, nodes, head_dim)
    if slots < 0:
        raise ValueError("tree_decode: the problem is too large")
    out = torch.empty_like(q)
    out_strides = out.stride()
    if out_strides[3] != 1:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        out_strides = out.stride()
    if (out_strides[0] | out_strides[1] | out_strides[2]) & 7:
        out_strides = _hip.row_layout(out, "out", device)[1]
    else:
        out_strides = _hip.int64_bytes(out_strides[:3])
    lse = workspace = None
    if return_lse:
        lse = torch.empty((batch, q_heads, nodes), dtype=torch.float32, device=q.device)
    if slots:
        # Float32 partial results, as twice as many elements of q's type.
        workspace = q.new_empty(2 * slots * nodes * group * (head_dim + 2))
    mask_strides = mask.stride()
    _hip.call_on(
        device,
        "tk_tree_decode",
        _hip.DTYPE_CODES[q.dtype],
        q_ptr,
        k_ptr,
        v_ptr,
        kt_ptr,
        vt_ptr,
        mask.data_ptr(),
        None if cache_seqlens is None else cache_seqlens.data_ptr(),
        out.data_ptr(),
        None if lse is None else lse.data_ptr(),
        None if workspace is None else workspace.data_ptr(),
        batch,
        q_heads,
        kv_heads,
        max_len,
        nodes,
        head_dim,
        q_strides,
        k_strides,
        v_strides,
        kt_strides,
        vt_strides,
        _hip.int64_bytes((0 if len(mask_strides) == 2 else mask_strides[0], mask_strides[-2])),
        out_strides,
        head_dim ** -0.5 if scale is None else float(scale),
        _hip.stream_on(device),
    )
    return (out, lse) if return_lse else out


@lru_cache(maxsize=256)
def _slots(batch: int, kv_heads: int, group: int, max_len: int, nodes: int, head_dim: int) -> int:
    """Partial results per row that the library asks for (a function of the sizes alone)."""
    return _hip.query("tk_tree_decode_slots", batch, kv_heads, group, max_len, nodes, head_dim)


def _validate(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_tree: torch.Tensor,
    v_tree: torch.Tensor,
    mask: torch.Tensor,
    cache_seqlens: torch.Tensor | None,
    scale: float | None,
) -> None:
    """Check the contract, up to the rows' layout."""
    q_shape, cache_shape, tree_shape = q.shape, k_cache.shape, k_tree.shape
    if len(q_shape) != 4 or len(cache_shape) != 4 or len(tree_shape) != 4:
        raise ValueError("tree_decode expects q [batch, q_heads, nodes, head_dim], caches [batch, "
                         "kv_heads, max_len, head_dim] and drafted keys and values [batch, "
                         "kv_heads, nodes, head_dim]")
    if v_cache.shape != cache_shape or v_tree.shape != tree_shape:
        raise ValueError("keys and values must have identical shapes")
    batch, q_heads, nodes, head_dim = q_shape
    cache_batch, kv_heads, max_len, cache_dim = cache_shape
    if cache_batch != batch or cache_dim != head_dim:
        raise ValueError("q and the caches disagree on batch or head_dim")
    if tree_shape != (batch, kv_heads, nodes, head_dim):
        raise ValueError("k_tree and v_tree must be [batch, kv_heads, nodes, head_dim]")
    if not (batch and q_heads and nodes and head_dim and kv_heads and max_len):
        raise ValueError("tree_decode does not support empty dimensions")
    if nodes > _MAX_NODES:
        raise ValueError(f"tree_decode supports at most {_MAX_NODES} nodes")
    if batch > 65535 or q_heads > 65535:
        raise ValueError("tree_decode supports at most 65535 sequences and heads")
    if q_heads % kv_heads:
        raise ValueError("q_heads must be a multiple of kv_heads")
    if head_dim not in _HEAD_DIMS:
        raise ValueError("tree_decode supports head_dim 64 and 128")
    dtype = q.dtype
    if dtype not in _DTYPES or not (
            dtype == k_cache.dtype == v_cache.dtype == k_tree.dtype == v_tree.dtype):
        raise ValueError("q, caches and drafted keys and values must share a float16 or bfloat16 "
                         "dtype")
    mask_shape = mask.shape
    if scale is not None and not abs(scale) < 2.0**126:
        raise ValueError("scale must be finite and below 2**126")
    if mask.dtype != torch.bool or (mask_shape != (nodes, nodes)
                                    and mask_shape != (batch, nodes, nodes)):
        raise ValueError("mask must be a bool [nodes, nodes] or [batch, nodes, nodes] tensor")
    if not q.is_cuda:
        raise ValueError("tree_decode requires CUDA (ROCm/HIP) tensors")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("k_tree", k_tree),
                    ("v_tree", v_tree)):
        if t.stride(2) >= 2**24 and t.shape[2] > 1:
            raise ValueError(f"{name} key strides must be below 2**24 elements")
    device = q.get_device()
    if mask.get_device() != device or (nodes > 1 and mask.stride(-1) != 1):
        raise ValueError("mask must be on q's device with a contiguous final dimension")
    if cache_seqlens is not None and (
            cache_seqlens.shape != (batch,) or cache_seqlens.dtype != torch.int32
            or cache_seqlens.get_device() != device or not cache_seqlens.is_contiguous()):
        raise ValueError("cache_seqlens must be a contiguous int32 [batch] tensor on q's device")
