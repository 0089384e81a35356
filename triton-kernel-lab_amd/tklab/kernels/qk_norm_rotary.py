"""Norms of queries and keys for each head, with the position rotation in the same pass.

A layer that norms its queries and keys runs ``rms_norm`` over every head and then
``rotary_embedding``: two reads and two writes of both. :func:`qk_norm_rotary` is both in one pass,
rounded once, with the arithmetic of each (``rms_norm.py:61-105``, ``rope.py:26-73``; positions and
frequencies as in ``rotary_embedding``), and its gradient is one pass over the inputs and the
outputs' gradients.
"""

from __future__ import annotations

from typing import Any

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from tklab import _hip
from tklab.kernels._norm_common import EPS, validate_epsilon

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_POSITION_DTYPES = (torch.int32, torch.int64)
_MAX_HEAD_DIM = 512
_MAX_HEADS = 65535
_MAX_TOKENS = 2**31 - 65537
_PARTIAL_ROWS = 768


def qk_norm_rotary(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    eps: float = EPS,
    interleaved: bool = False,
    magnitude: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS-norm every head of ``q`` and ``k``, then turn them by their tokens' positions.

    Args:
        q, k: ``[batch, heads, tokens, head_dim]``, or packed ``[tokens, heads, head_dim]``;
            float16, bfloat16 or float32, any strides with a contiguous last dimension, head
            counts of their own. head_dim at most 512, 65535 heads each, 2**31 - 65537 tokens.
        q_weight, k_weight: ``[head_dim]``, same dtype, shared by the heads.
        positions: int32 or int64, ``[batch, tokens]`` or ``[tokens]`` (shared by the batch);
            ``[tokens]`` for packed tensors. Any value, negative ones included.
        frequencies: float64 ``[rotary_dim // 2]`` on the same device
            (:func:`~tklab.kernels.rotary.rotary_frequencies`); they get no gradient; features
            past ``rotary_dim`` are normed but not turned.
        eps: added to a head's mean square; a positive normal float32.
        interleaved: pairs are ``(2i, 2i + 1)``; otherwise ``(i, i + rotary_dim // 2)``.
        magnitude: multiplies cosine and sine (rounded to float32).

    Returns:
        ``(q, k)`` with the inputs' shapes and memory order: statistics and rotation in float32,
        angles in float64, rounded once to the dtype. Differentiable in ``q``, ``k`` and both
        weights, in reverse mode only; the weights' gradients are summed in float32 in a fixed
        order.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
        RuntimeError: on a forward-mode tangent.
    """
    _validate(q, k, q_weight, k_weight, positions, frequencies)
    validate_epsilon(eps)
    if not 2.0**-126 <= eps < 2.0**127:
        raise ValueError("eps must be a normal float32")
    how = (float(eps), float(magnitude), int(interleaved))
    # Within a forward-mode level the inputs may carry tangents, which autograd's function refuses.
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad or q_weight.requires_grad or k_weight.requires_grad):
        return _QkNormRotaryFunction.apply(q, k, q_weight, k_weight, positions, frequencies, how)
    return _forward(q, k, q_weight, k_weight, positions, frequencies, how)


class _QkNormRotaryFunction(torch.autograd.Function):
    """Autograd bridge; the inputs are kept, no statistics."""

    @staticmethod
    def forward(ctx: Any, q, k, q_weight, k_weight, positions, frequencies, how):
        """Norm and turn."""
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, frequencies)
        ctx.how = how
        return _forward(q, k, q_weight, k_weight, positions, frequencies, how)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dq_out, dk_out):
        """Gradients of the sides whose output was given one."""
        q, k, q_weight, k_weight, positions, frequencies = ctx.saved_tensors
        need = ctx.needs_input_grad
        sides = [(0, q, q_weight, dq_out), (1, k, k_weight, dk_out)]
        sides = [s for s in sides if s[3] is not None and (need[s[0]] or need[s[0] + 2])]
        grads: list[torch.Tensor | None] = [None] * 7
        if sides:
            results = _backward([s[1:] for s in sides], positions, frequencies, ctx.how)
            for (which, *_), (dx, dw) in zip(sides, results):
                grads[which] = dx if need[which] else None
                grads[which + 2] = dw if need[which + 2] else None
        return tuple(grads)


def _forward(q, k, q_weight, k_weight, positions, frequencies, how):
    """Allocate the outputs and enqueue the pass over tensors already checked."""
    q_out, q_out_strides = _like(q)
    k_out, k_out_strides = _like(k)
    shape = q.shape
    packed = len(shape) == 3
    device = q.get_device()
    _hip.call_on(
        device,
        "tk_qk_norm_rotary",
        _hip.DTYPE_CODES[q.dtype],
        q.data_ptr(),
        q_out.data_ptr(),
        k.data_ptr(),
        k_out.data_ptr(),
        q_weight.data_ptr(),
        k_weight.data_ptr(),
        positions.data_ptr(),
        frequencies.data_ptr(),
        1 if packed else shape[0],
        shape[0] if packed else shape[2],
        shape[1],
        k.shape[1],
        shape[-1],
        2 * frequencies.shape[0],
        _strides(q.stride()),
        _strides(q_out_strides),
        _strides(k.stride()),
        _strides(k_out_strides),
        _position_strides(positions),
        *how,
        int(positions.dtype == torch.int64),
        _hip.stream_on(device),
    )
    return q_out, k_out


def _backward(sides, positions, frequencies, how):
    """(dx, dweight) of each side (x, weight, dy), one or two of them."""
    arguments, tables, weights, grads = [], [], [], []
    x0 = sides[0][0]
    packed = x0.ndim == 3
    for x, weight, dy in sides:
        if dy.stride(-1) != 1:  # a broadcast gradient has stride 0
            dy = dy.contiguous()
        dx, dx_strides = _like(x)
        dw = torch.empty_like(weight)
        arguments += [x, dy, dx]
        tables += [_strides(x.stride()), _strides(dy.stride()), _strides(dx_strides)]
        weights.append(weight)
        grads.append((dx, dw))
    pad = [None] * (2 - len(sides))
    partials = torch.empty((_PARTIAL_ROWS, x0.shape[-1]), dtype=torch.float32, device=x0.device)
    device = x0.get_device()
    _hip.call_on(
        device,
        "tk_qk_norm_rotary_bwd",
        _hip.DTYPE_CODES[x0.dtype],
        *(t.data_ptr() for t in arguments),
        *(pad * 3),
        *(w.data_ptr() for w in weights),
        *pad,
        *(dw.data_ptr() for _, dw in grads),
        *pad,
        partials.data_ptr(),
        positions.data_ptr(),
        frequencies.data_ptr(),
        1 if packed else x0.shape[0],
        x0.shape[0] if packed else x0.shape[2],
        x0.shape[1],
        0 if pad else sides[1][0].shape[1],
        x0.shape[-1],
        2 * frequencies.shape[0],
        *tables,
        *(pad * 3),
        _position_strides(positions),
        *how,
        int(positions.dtype == torch.int64),
        _hip.stream_on(device),
    )
    return grads


def _like(x: torch.Tensor) -> tuple[torch.Tensor, tuple[int, ...]]:
    """A tensor of x's shape, and order where that leaves the last dimension contiguous, and its
    strides."""
    out = torch.empty_like(x)
    strides = out.stride()
    if strides[-1] != 1:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        strides = out.stride()
    return out, strides


def _strides(strides: tuple[int, ...]):
    """``{batch, head, token}`` strides."""
    return _hip.int64_table((0, strides[1], strides[0]) if len(strides) == 3 else strides[:3])


def _position_strides(positions: torch.Tensor):
    """``{batch, token}`` strides."""
    strides = positions.stride()
    return _hip.int64_table(strides if len(strides) == 2 else (0, strides[0]))


def _validate(q, k, q_weight, k_weight, positions, frequencies) -> None:
    """Check the contract."""
    shape, k_shape, dtype = q.shape, k.shape, q.dtype
    rank = len(shape)
    if rank != 3 and rank != 4:
        raise ValueError("qk_norm_rotary expects q [batch, heads, tokens, head_dim] or packed "
                         "[tokens, heads, head_dim]")
    if len(k_shape) != rank:
        raise ValueError("q and k must both be packed or both be batched")
    if 0 in shape or 0 in k_shape:
        raise ValueError("qk_norm_rotary does not support empty dimensions")
    if k_shape[0] != shape[0] or k_shape[2:] != shape[2:]:
        raise ValueError("q and k may differ only in their head counts")
    if dtype not in _DTYPES:
        raise ValueError("qk_norm_rotary supports float16, bfloat16 and float32 tensors")
    if not dtype == k.dtype == q_weight.dtype == k_weight.dtype:
        raise ValueError("q, k and their weights must share a dtype")
    tokens, dim = shape[0] if rank == 3 else shape[2], shape[-1]
    if q_weight.shape != (dim,) or k_weight.shape != (dim,):
        raise ValueError("q_weight and k_weight must be [head_dim]")
    if dim > 1 and (q_weight.stride(0) != 1 or k_weight.stride(0) != 1):
        raise ValueError("q_weight and k_weight must be contiguous")
    if shape[1] > _MAX_HEADS or k_shape[1] > _MAX_HEADS:
        raise ValueError(f"qk_norm_rotary supports at most {_MAX_HEADS} heads each")
    if tokens * (1 if rank == 3 else shape[0]) > _MAX_TOKENS:
        raise ValueError(f"qk_norm_rotary supports at most {_MAX_TOKENS} tokens")
    wanted, given = (tokens,), positions.shape
    if given != wanted and (rank == 3 or given != (shape[0], *wanted)):
        raise ValueError("positions must be [tokens]" + (" or [batch, tokens]" * (rank == 4)))
    if positions.dtype not in _POSITION_DTYPES:
        raise ValueError("positions must be int32 or int64")
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1:
        raise ValueError("frequencies must be a float64 [rotary_dim // 2] tensor")
    pairs = frequencies.shape[0]
    if pairs == 0 or 2 * pairs > dim:
        raise ValueError("frequencies must cover at least one pair and at most head_dim features")
    if pairs > 1 and frequencies.stride(0) != 1:
        raise ValueError("frequencies must be contiguous")
    if dim > _MAX_HEAD_DIM:
        raise ValueError(f"qk_norm_rotary supports head_dim up to {_MAX_HEAD_DIM}")
    if not q.is_cuda:
        raise ValueError("qk_norm_rotary requires CUDA (ROCm/HIP) tensors")
    device = q.get_device()
    if not (k.get_device() == device == positions.get_device() == frequencies.get_device()
            == q_weight.get_device() == k_weight.get_device()):
        raise ValueError("q, k, their weights, positions and frequencies must be on one device")
    if q.stride(-1) != 1 or k.stride(-1) != 1:
        raise ValueError("q and k require a contiguous final dimension")
