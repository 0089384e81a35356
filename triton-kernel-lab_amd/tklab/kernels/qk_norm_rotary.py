"""Norms of queries and keys for each head, with the position rotation in the same pass.

A layer that norms its queries and keys runs ``rms_norm`` over every head and then
``rotary_embedding``: two reads and two writes of both. :func:`qk_norm_rotary` is both in one pass,
rounded once, with the arithmetic of each (``rms_norm.py:61-105``, ``rope.py:26-73``; positions and
frequencies as in ``rotary_embedding``), and its gradient is one pass over the inputs and the
outputs' gradients.
"""

from __future__ import annotations

from functools import lru_cache
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
        order. As with every autograd function, a backward pass is captured into a graph from leaves
        of which no eager graph is alive.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
        RuntimeError: on a forward-mode tangent.
    """
    plan = _plan_of(q, k, q_weight, k_weight, positions, frequencies)
    validate_epsilon(eps)
    if not 2.0**-126 <= eps < 2.0**127:
        raise ValueError("eps must be a normal float32")
    how = (float(eps), float(magnitude), int(interleaved))
    # Within a forward-mode level the inputs may carry tangents, which autograd's function refuses.
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            q.requires_grad or k.requires_grad or q_weight.requires_grad or k_weight.requires_grad):
        return _QkNormRotaryFunction.apply(q, k, q_weight, k_weight, positions, frequencies, how, plan)
    return _forward(q, k, q_weight, k_weight, positions, frequencies, how, plan)


class _QkNormRotaryFunction(torch.autograd.Function):
    """Autograd bridge; the inputs are kept, no statistics."""

    @staticmethod
    def forward(ctx: Any, q, k, q_weight, k_weight, positions, frequencies, how, plan):
        """Norm and turn."""
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, frequencies)
        ctx.how = how
        return _forward(q, k, q_weight, k_weight, positions, frequencies, how, plan)

    @staticmethod
    def backward(ctx: Any, dq_out, dk_out):
        """Gradients of the sides whose output was given one."""
        if torch.is_grad_enabled():  # create_graph: the result is marked as not differentiable again
            return _once_differentiable(ctx, dq_out, dk_out)
        return _gradients(ctx, dq_out, dk_out)


def _gradients(ctx: Any, dq_out, dk_out):
    """Of all inputs, None where there is none or none is needed."""
    q, k, q_weight, k_weight, positions, frequencies = ctx.saved_tensors
    needs_q, needs_k, needs_q_weight, needs_k_weight, *_ = ctx.needs_input_grad
    # Hooks on saved tensors may give them back with other strides.
    plan = _plan_of(q, k, q_weight, k_weight, positions, frequencies)
    _, sizes, q_strides, k_strides, *_ = plan
    q_side = k_side = None
    dq = dk = dq_weight = dk_weight = None
    if dq_out is not None and (needs_q or needs_q_weight):
        q_side = q, q_weight, dq_out, *q_strides, sizes[2]
    if dk_out is not None and (needs_k or needs_k_weight):
        k_side = k, k_weight, dk_out, *k_strides, sizes[3]
    if q_side is not None:
        dq, dq_weight, dk, dk_weight = _backward(q_side, k_side, positions, frequencies, ctx.how, plan)
    elif k_side is not None:
        dk, dk_weight, *_ = _backward(k_side, None, positions, frequencies, ctx.how, plan)
    return (dq if needs_q else None, dk if needs_k else None, dq_weight if needs_q_weight else None,
            dk_weight if needs_k_weight else None, None, None, None, None)


_once_differentiable = once_differentiable(_gradients)


def _forward(q, k, q_weight, k_weight, positions, frequencies, how, plan):
    """Allocate the outputs and enqueue the pass over tensors already checked."""
    device, sizes, (q_strides, q_out_strides), (k_strides, k_out_strides), position_strides, wide = plan
    q_out, k_out = _like(q), _like(k)
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
        *sizes,
        q_strides,
        q_out_strides,
        k_strides,
        k_out_strides,
        position_strides,
        *how,
        wide,
        _hip.stream_on(device),
    )
    return q_out, k_out


def _backward(first, second, positions, frequencies, how, plan):
    """(dx, dweight) of one side or of both, each (x, weight, dy, strides, strides of dx, heads)."""
    device, (batch, tokens, _, _, *dims), _, _, position_strides, wide = plan
    x, weight, dy, strides, out_strides, heads = first
    dx, dweight = _like(x), torch.empty_like(weight)
    if dy.stride(-1) != 1:  # a broadcast gradient has stride 0
        dy = dy.contiguous()
    tables = (strides, _strides(dy.stride()), out_strides)
    pointers = (x.data_ptr(), dy.data_ptr(), dx.data_ptr())
    if second is None:
        dx2 = dweight2 = None
        more_pointers = more_tables = (None, None, None)
        weights = (weight.data_ptr(), None, dweight.data_ptr(), None)
        heads2 = 0
    else:
        x2, weight2, dy2, strides2, out_strides2, heads2 = second
        dx2, dweight2 = _like(x2), torch.empty_like(weight2)
        if dy2.stride(-1) != 1:
            dy2 = dy2.contiguous()
        more_tables = (strides2, _strides(dy2.stride()), out_strides2)
        more_pointers = (x2.data_ptr(), dy2.data_ptr(), dx2.data_ptr())
        weights = (weight.data_ptr(), weight2.data_ptr(), dweight.data_ptr(), dweight2.data_ptr())
    # Float32, as elements of x's type.
    partials = x.new_empty(_PARTIAL_ROWS * dims[0] * 4 // x.element_size())
    _hip.call_on(
        device,
        "tk_qk_norm_rotary_bwd",
        _hip.DTYPE_CODES[x.dtype],
        *pointers,
        *more_pointers,
        *weights,
        partials.data_ptr(),
        positions.data_ptr(),
        frequencies.data_ptr(),
        batch,
        tokens,
        heads,
        heads2,
        *dims,
        *tables,
        *more_tables,
        position_strides,
        *how,
        wide,
        _hip.stream_on(device),
    )
    return dx, dweight, dx2, dweight2


def _like(x: torch.Tensor) -> torch.Tensor:
    """A tensor of x's shape, and order where that leaves the last dimension contiguous."""
    out = torch.empty_like(x)
    if out.stride(-1) != 1:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    return out


def _strides(strides: tuple[int, ...]):
    """Table of ``{batch, head, token}`` strides."""
    return _hip.int64_table((0, strides[1], strides[0]) if len(strides) == 3 else tuple(strides[:3]))


def _plan_of(q, k, q_weight, k_weight, positions, frequencies):
    """:func:`_plan` of these tensors."""
    return _plan(q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(),
                 q_weight.shape, q_weight.stride(), q_weight.dtype, q_weight.get_device(),
                 k_weight.shape, k_weight.stride(), k_weight.dtype, k_weight.get_device(),
                 positions.shape, positions.stride(), positions.dtype, positions.get_device(),
                 frequencies.shape, frequencies.stride(), frequencies.dtype, frequencies.get_device())


@lru_cache(maxsize=1024)
def _plan(shape, q_strides, dtype, device, k_shape, k_strides, k_dtype, k_device, qw_shape, qw_strides, qw_dtype,
          qw_device, kw_shape, kw_strides, kw_dtype, kw_device, pos_shape, pos_strides, pos_dtype, pos_device,
          freq_shape, freq_strides, freq_dtype, freq_device):
    """Check the contract; device, sizes and stride tables, made once for tensors alike."""
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
    if not dtype == k_dtype == qw_dtype == kw_dtype:
        raise ValueError("q, k and their weights must share a dtype")
    tokens, dim = shape[0] if rank == 3 else shape[2], shape[-1]
    batch = 1 if rank == 3 else shape[0]
    if qw_shape != (dim,) or kw_shape != (dim,):
        raise ValueError("q_weight and k_weight must be [head_dim]")
    if dim > 1 and (qw_strides[0] != 1 or kw_strides[0] != 1):
        raise ValueError("q_weight and k_weight must be contiguous")
    if shape[1] > _MAX_HEADS or k_shape[1] > _MAX_HEADS:
        raise ValueError(f"qk_norm_rotary supports at most {_MAX_HEADS} heads each")
    if tokens * batch > _MAX_TOKENS:
        raise ValueError(f"qk_norm_rotary supports at most {_MAX_TOKENS} tokens")
    if pos_shape != (tokens,) and (rank == 3 or pos_shape != (batch, tokens)):
        raise ValueError("positions must be [tokens]" + (" or [batch, tokens]" * (rank == 4)))
    if pos_dtype not in _POSITION_DTYPES:
        raise ValueError("positions must be int32 or int64")
    if freq_dtype != torch.float64 or len(freq_shape) != 1:
        raise ValueError("frequencies must be a float64 [rotary_dim // 2] tensor")
    pairs = freq_shape[0]
    if pairs == 0 or 2 * pairs > dim:
        raise ValueError("frequencies must cover at least one pair and at most head_dim features")
    if pairs > 1 and freq_strides[0] != 1:
        raise ValueError("frequencies must be contiguous")
    if dim > _MAX_HEAD_DIM:
        raise ValueError(f"qk_norm_rotary supports head_dim up to {_MAX_HEAD_DIM}")
    if device < 0:
        raise ValueError("qk_norm_rotary requires CUDA (ROCm/HIP) tensors")
    if not device == k_device == qw_device == kw_device == pos_device == freq_device:
        raise ValueError("q, k, their weights, positions and frequencies must be on one device")
    if q_strides[-1] != 1 or k_strides[-1] != 1:
        raise ValueError("q and k require a contiguous final dimension")
    outs = [_like(torch.empty_strided(s, t, device="meta")).stride() for s, t in ((shape, q_strides),
                                                                                  (k_shape, k_strides))]
    sizes = (batch, tokens, shape[1], k_shape[1], dim, 2 * pairs)
    position_strides = _hip.int64_table(tuple(pos_strides) if len(pos_strides) == 2 else (0, pos_strides[0]))
    return (device, sizes, (_strides(q_strides), _strides(outs[0])), (_strides(k_strides), _strides(outs[1])),
            position_strides, int(pos_dtype == torch.int64))
