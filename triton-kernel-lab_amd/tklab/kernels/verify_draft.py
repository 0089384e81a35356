"""Verification of drafted tokens against the target's probabilities.

One step of speculative decoding ends here: the target has scored a chain or a tree of drafted
tokens in one pass (``tree_decode`` and the layers around it, then ``softmax``), and the walk from
the root keeps the branch it agrees with, so that the tokens that come out are distributed as if
the target had been sampled token by token. Random numbers are inputs: the call is deterministic.
There is no counterpart in the reference.
"""

from __future__ import annotations

import torch

from tklab import _hip

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_TOKEN_DTYPES = (torch.int32, torch.int64)
_MAX_NODES = 256
_MAX_VOCABULARY = 2**31 - 65537
_MAX_SPLITS = 64
_CHUNK = 2048
# Workgroups that weigh rows, about: four for each of the 256 CUs. 64 rows of 131072 float32 take
# 14.8 us in 1024 workgroups and 16.9 in 2048 (each repeats the walk); with few bytes to read, more
# and shorter shares are faster (32 rows of 65537 bfloat16: 6.4 us in 1056, 7.2 in 544).
_TARGET_WORKGROUPS = 1024


def verify_draft(
    target_probs: torch.Tensor,
    draft_tokens: torch.Tensor,
    uniforms: torch.Tensor,
    *,
    parents: torch.Tensor | None = None,
    draft_probs: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The accepted branch of each sequence's drafted tokens, and the token drawn behind it.

    Node 0 of a sequence is its last token, node ``i`` a drafted one; ``target_probs[b, i]`` is
    the target's distribution of the token behind node ``i``. From node 0 on, the current node's
    children are tried in order; child ``i`` with token ``x`` is accepted, and becomes the current
    node, if ``uniforms[b, i] * q(x) < p(x)`` where the chain was drawn from ``draft_probs``, or
    if ``uniforms[b, i] * m < p(x)`` with ``m`` the mass that the siblings rejected before have
    left of 1 where the tokens were taken without drawing (an earlier rejected token again is
    rejected). When no child is accepted, the next token is drawn with ``uniforms[b, 0]`` from
    ``max(p - q, 0)`` after a rejection under ``draft_probs``, otherwise from ``p`` without the
    rejected tokens: the first ``v`` whose cumulative weight exceeds ``uniforms[b, 0]`` times the
    total. If these weights have no mass, ``p`` itself is drawn from. All in float64.

    Args:
        target_probs: ``[batch, nodes, vocabulary]`` float16, bfloat16 or float32; rows need not
            sum to 1 for the drawn token. Entries that are not positive and finite weigh nothing.
        draft_tokens: int32 or int64 ``[batch, nodes]``; entry 0 is not read. A token outside the
            vocabulary is no candidate: padding of shorter drafts.
        uniforms: float32 ``[batch, nodes]`` in [0, 1).
        parents: int32 ``[nodes]`` or ``[batch, nodes]``, every parent before its children (entry
            0 is not read; a parent outside ``[0, i)`` leaves node ``i`` out). ``None``: a chain.
        draft_probs: ``[batch, nodes - 1, vocabulary]`` in ``target_probs``' dtype: row ``i - 1``
            is the distribution that node ``i`` was drawn from. Chains only.

    Returns:
        ``(path, count, next_token)``: int32 ``[batch, nodes]`` accepted nodes from node 0 on,
        then -1; int32 ``[batch]`` how many; int64 ``[batch]`` the drawn token (-1 where the
        target's row has no mass at all). At most 256 nodes.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
    """
    _validate(target_probs, draft_tokens, uniforms, parents, draft_probs)
    batch, nodes, vocabulary = target_probs.shape
    device = target_probs.get_device()
    chunk = chunk_length(batch, vocabulary)
    splits = -(-vocabulary // chunk)
    path = torch.empty_like(uniforms, dtype=torch.int32, memory_format=torch.contiguous_format)
    count = path.new_empty(batch)
    if draft_tokens.dtype == torch.int64:
        next_token = draft_tokens.new_empty(batch)
    else:
        next_token = torch.empty(batch, dtype=torch.int64, device=target_probs.device)
    # Words: two float64 sums per split, then four and a list of rejected tokens per sequence.
    workspace = path.new_empty(batch * (4 * splits + 4 + nodes))
    if nodes == 1:
        draft_probs = None
    target_strides = target_probs.stride()
    draft_ptr = draft_strides = parents_ptr = None
    parents_stride = 0
    if draft_probs is not None:
        draft_ptr = draft_probs.data_ptr()
        draft_strides = _hip.int64_bytes(draft_probs.stride()[:2])
    if parents is not None:
        parents_ptr = parents.data_ptr()
        parents_stride = parents.stride(0) if parents.dim() == 2 else 0
    _hip.call_on(
        device,
        "tk_verify_draft",
        _hip.DTYPE_CODES[target_probs.dtype],
        target_probs.data_ptr(),
        draft_ptr,
        draft_tokens.data_ptr(),
        parents_ptr,
        uniforms.data_ptr(),
        path.data_ptr(),
        count.data_ptr(),
        next_token.data_ptr(),
        workspace.data_ptr(),
        batch,
        nodes,
        vocabulary,
        chunk,
        _hip.int64_bytes(target_strides[:2]),
        draft_strides,
        _hip.int64_bytes((draft_tokens.stride(0), parents_stride, uniforms.stride(0))),
        int(draft_tokens.dtype == torch.int64),
        _hip.stream_on(device),
    )
    return path, count, next_token


def chunk_length(batch: int, vocabulary: int) -> int:
    """Row entries per workgroup: a multiple of 2048, at most 64 shares per row, and about
    _TARGET_WORKGROUPS in all once the batch has that much to read (2**30 at most: the library
    counts in 32 bits)."""
    least = -(-vocabulary // (_MAX_SPLITS * _CHUNK))
    share = max(least, batch * vocabulary // (_TARGET_WORKGROUPS * _CHUNK))
    return min(_CHUNK * share, 2**30)


def _validate(
    target_probs: torch.Tensor,
    draft_tokens: torch.Tensor,
    uniforms: torch.Tensor,
    parents: torch.Tensor | None,
    draft_probs: torch.Tensor | None,
) -> None:
    """Check the verification's contract."""
    shape, dtype = target_probs.shape, target_probs.dtype
    if len(shape) != 3:
        raise ValueError("verify_draft expects target_probs [batch, nodes, vocabulary]")
    if 0 in shape:
        raise ValueError("verify_draft does not support empty dimensions")
    batch, nodes, vocabulary = shape
    if nodes > _MAX_NODES:
        raise ValueError(f"verify_draft supports at most {_MAX_NODES} nodes")
    if batch > 65535 or vocabulary > _MAX_VOCABULARY:
        raise ValueError("verify_draft supports at most 65535 sequences and a vocabulary of "
                         f"{_MAX_VOCABULARY}")
    if dtype not in _DTYPES:
        raise ValueError("verify_draft supports float16, bfloat16 and float32 probabilities")
    per_node = (batch, nodes)
    if draft_tokens.shape != per_node or draft_tokens.dtype not in _TOKEN_DTYPES:
        raise ValueError("draft_tokens must be an int32 or int64 [batch, nodes] tensor")
    if uniforms.shape != per_node or uniforms.dtype != torch.float32:
        raise ValueError("uniforms must be a float32 [batch, nodes] tensor")
    if parents is not None:
        if (parents.shape != per_node and parents.shape != (nodes,)) or (
                parents.dtype != torch.int32):
            raise ValueError("parents must be an int32 [nodes] or [batch, nodes] tensor")
        if draft_probs is not None:
            raise ValueError("draft_probs belong to a chain: they cannot be given with parents")
    if draft_probs is not None and (draft_probs.shape != (batch, nodes - 1, vocabulary)
                                    or draft_probs.dtype != dtype):
        raise ValueError("draft_probs must be [batch, nodes - 1, vocabulary] in target_probs' "
                         "dtype")
    if not target_probs.is_cuda:
        raise ValueError("verify_draft requires CUDA (ROCm/HIP) tensors")
    device = target_probs.get_device()
    for name, tensor in (("target_probs", target_probs), ("draft_tokens", draft_tokens),
                         ("uniforms", uniforms), ("parents", parents),
                         ("draft_probs", draft_probs)):
        if tensor is None:
            continue
        if tensor.get_device() != device:
            raise ValueError(f"{name} must be on target_probs' device")
        if tensor.stride(-1) != 1 and tensor.numel() and tensor.shape[-1] > 1:
            raise ValueError(f"{name} requires a contiguous final dimension")
