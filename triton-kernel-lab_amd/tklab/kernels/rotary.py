"""Rotary positions from token positions: both pair layouts, part of the head, scaled contexts.

``rope`` takes per-row tables and turns halves of the whole feature dimension, as the reference
does (``rope.py:26-73``). :func:`rotary_embedding` is the form a model's attention layer needs: it
turns the queries and keys of a call in one launch, at positions given per token, over the first
``2 * len(frequencies)`` features of each head, and forms the angles itself in float64, so no
table bounds the context. :func:`rotary_frequencies` makes the frequencies, plain or scaled for
contexts longer than a model was trained on. The gradient is the rotation by the negative angle.
"""

from __future__ import annotations

import math
from typing import Any

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from tklab import _hip

_DTYPES = (torch.float16, torch.bfloat16, torch.float32)
_POSITION_DTYPES = (torch.int32, torch.int64)
_MAX_HEAD_DIM = 1024
_MAX_HEADS = 65535
_MAX_TOKENS = 2**31 - 65537
_SCALINGS = ("none", "linear", "ntk", "yarn")


def rotary_frequencies(
    rotary_dim: int,
    *,
    base: float = 10000.0,
    scaling: str = "none",
    factor: float = 1.0,
    original_length: int | None = None,
    fast_turns: float = 32.0,
    slow_turns: float = 1.0,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, float]:
    """Frequencies (float64 ``[rotary_dim // 2]``, radians per position) and magnitude.

    Pair ``i`` turns by ``base ** (-2 i / rotary_dim)`` radians per position. ``scaling`` stretches
    that for contexts ``factor`` times the original:

    - ``"linear"``: every frequency divided by ``factor``;
    - ``"ntk"``: ``base`` multiplied by ``factor ** (d / (d - 2))``, which divides the slowest
      pair's frequency by ``factor`` and leaves the fastest pair's;
    - ``"yarn"``: pairs that turn more than ``fast_turns`` times over ``original_length`` keep
      their frequency, those below ``slow_turns`` have it divided by ``factor``, with a linear
      ramp over the pairs between; the magnitude is ``0.1 ln(factor) + 1``.

    The magnitude is 1 for the others. Made once for a model and kept.

    Raises:
        ValueError: on an odd or empty ``rotary_dim``, an unknown scaling, a factor below 1, or
            ``"yarn"`` without ``original_length``.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and positive")
    if scaling not in _SCALINGS:
        raise ValueError(f"scaling must be one of {', '.join(_SCALINGS)}")
    if not base > 1.0:
        raise ValueError("base must be greater than 1")
    if not factor >= 1.0:
        raise ValueError("factor must be at least 1")
    half = rotary_dim // 2
    if scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    index = torch.arange(half, dtype=torch.float64, device=device)
    plain = torch.pow(torch.tensor(base, dtype=torch.float64, device=device), -index / half)
    if scaling == "linear":
        return plain / factor, 1.0
    if scaling != "yarn":
        return plain, 1.0
    if original_length is None or original_length <= 0:
        raise ValueError("yarn scaling needs a positive original_length")
    if not fast_turns > slow_turns > 0:
        raise ValueError("yarn scaling needs fast_turns > slow_turns > 0")

    def pair_turning(turns: float) -> float:
        """The (fractional) pair that makes ``turns`` turns over the original length."""
        return half * math.log(original_length / (turns * 2 * math.pi)) / math.log(base)

    low = max(math.floor(pair_turning(fast_turns)), 0)
    # The ramp may end past the last pair, which then turns more than slow_turns times.
    high = min(math.ceil(pair_turning(slow_turns)), rotary_dim - 1)
    if high <= 0:  # no pair turns more than slow_turns times
        ramp = torch.ones_like(index)
    else:
        ramp = ((index - low) / max(high - low, 1e-3)).clamp(0, 1)
    return plain * (1 - ramp) + plain / factor * ramp, 0.1 * math.log(factor) + 1.0


def rotary_embedding(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    interleaved: bool = False,
    magnitude: float = 1.0,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Turn ``q`` (and ``k``) by their tokens' positions.

    Args:
        q, k: ``[batch, heads, tokens, head_dim]``, or packed ``[tokens, heads, head_dim]``;
            float16, bfloat16 or float32, any strides with a contiguous last dimension, head
            counts of their own. ``k`` may be ``None``. head_dim at most 1024, 65535 heads in
            all, 2**31 - 65537 tokens.
        positions: int32 or int64, ``[batch, tokens]`` or ``[tokens]`` (shared by the batch);
            ``[tokens]`` for packed tensors. Any value, negative ones included.
        frequencies: float64 ``[rotary_dim // 2]`` on the same device
            (:func:`rotary_frequencies`), at most 1 where positions reach 2**62 (an angle's
            magnitude is at most 2**63); they get no gradient; features past ``rotary_dim`` are
            copied.
        interleaved: pairs are ``(2i, 2i + 1)``; otherwise ``(i, i + rotary_dim // 2)``.
        magnitude: multiplies cosine and sine (rounded to float32).

    Returns:
        The turned ``q``, or ``(q, k)``, with the inputs' shape and memory order. Angles are
        float64, the rotation float32, rounded once to the dtype. Differentiable in ``q`` and
        ``k``, in reverse mode only.

    Raises:
        ValueError: on an unsupported shape, dtype, layout or device.
        RuntimeError: on a forward-mode tangent.
    """
    _validate(q, k, positions, frequencies)
    # Within a forward-mode level the inputs may carry tangents, which autograd's function refuses.
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (
            q.requires_grad or (k is not None and k.requires_grad)):
        out = _RotaryFunction.apply(q, k, positions, frequencies, interleaved, float(magnitude))
        return out if k is not None else out[0]
    turned_q, turned_k = _launch(q, k, positions, frequencies, interleaved, float(magnitude))
    return turned_q if k is None else (turned_q, turned_k)


class _RotaryFunction(torch.autograd.Function):
    """Autograd bridge: the gradient is the inverse rotation with the same magnitude."""

    @staticmethod
    def forward(ctx: Any, q, k, positions, frequencies, interleaved, magnitude):
        """Turn and keep the positions and frequencies."""
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (interleaved, magnitude)
        return _launch(q, k, positions, frequencies, interleaved, magnitude)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dq, dk):
        """Gradients of the tensors that were given one and need one."""
        positions, frequencies = ctx.saved_tensors
        wanted = [g if need else None for g, need in zip((dq, dk), ctx.needs_input_grad)]
        given = [_unit_stride(g) for g in wanted if g is not None]
        if not given:
            return (None,) * 6
        first, second = given[0], given[1] if len(given) == 2 else None
        turned = list(_launch(first, second, positions, frequencies, *ctx.how, inverse=True))
        grads = [None if g is None else turned.pop(0) for g in wanted]
        return (*grads, None, None, None, None)


def _unit_stride(grad: torch.Tensor) -> torch.Tensor:
    """The gradient with a contiguous last dimension (a broadcast one has stride 0)."""
    return grad if grad.stride(-1) == 1 else grad.contiguous()


def _launch(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    interleaved: bool,
    magnitude: float,
    *,
    inverse: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Allocate the outputs and enqueue the rotation of tensors already checked."""
    q_out = torch.empty_like(q)
    q_strides, q_out_strides = q.stride(), q_out.stride()
    if q_out_strides[-1] != 1:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        q_out_strides = q_out.stride()
    shape, position_strides = q.shape, positions.stride()
    packed = len(shape) == 3
    if k is None:
        k_out = k_ptr = k_out_ptr = k_table = k_out_table = None
        kv_heads = 0
    else:
        k_out = torch.empty_like(k)
        if k_out.stride(-1) != 1:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        kv_heads, k_ptr, k_out_ptr = k.shape[1], k.data_ptr(), k_out.data_ptr()
        k_table, k_out_table = _strides(k.stride(), packed), _strides(k_out.stride(), packed)
    device = q.get_device()
    _hip.call_on(
        device,
        "tk_rotary",
        _hip.DTYPE_CODES[q.dtype],
        q.data_ptr(),
        q_out.data_ptr(),
        k_ptr,
        k_out_ptr,
        positions.data_ptr(),
        frequencies.data_ptr(),
        1 if packed else shape[0],
        shape[0] if packed else shape[2],
        shape[1],
        kv_heads,
        shape[-1],
        2 * frequencies.shape[0],
        _strides(q_strides, packed),
        _strides(q_out_strides, packed),
        k_table,
        k_out_table,
        _hip.int64_bytes(position_strides if len(position_strides) == 2
                         else (0, position_strides[0])),
        magnitude,
        int(interleaved),
        int(positions.dtype == torch.int64),
        int(inverse),
        _hip.stream_on(device),
    )
    return q_out, k_out


def _strides(strides: tuple[int, ...], packed: bool) -> bytes:
    """``{batch, head, token}`` strides."""
    return _hip.int64_bytes((0, strides[1], strides[0]) if packed else strides[:3])


def _validate(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
) -> None:
    """Check the rotation's contract."""
    shape, dtype = q.shape, q.dtype
    rank = len(shape)
    if rank != 3 and rank != 4:
        raise ValueError("rotary_embedding expects q [batch, heads, tokens, head_dim] or packed "
                         "[tokens, heads, head_dim]")
    if 0 in shape:
        raise ValueError("rotary_embedding does not support empty dimensions")
    if k is not None:
        k_shape = k.shape
        if len(k_shape) != rank:
            raise ValueError("q and k must both be packed or both be batched")
        if 0 in k_shape:
            raise ValueError("rotary_embedding does not support empty dimensions")
        if k_shape[0] != shape[0] or k_shape[2:] != shape[2:]:
            raise ValueError("q and k may differ only in their head counts")
        if k.dtype != dtype or k.device != q.device:
            raise ValueError("q and k must share a dtype and a device")
    if dtype not in _DTYPES:
        raise ValueError("rotary_embedding supports float16, bfloat16 and float32 tensors")
    tokens = shape[0] if rank == 3 else shape[2]
    if shape[1] + (0 if k is None else k_shape[1]) > _MAX_HEADS:
        raise ValueError(f"rotary_embedding supports at most {_MAX_HEADS} heads in all")
    if tokens * (1 if rank == 3 else shape[0]) > _MAX_TOKENS:
        raise ValueError(f"rotary_embedding supports at most {_MAX_TOKENS} tokens")
    wanted, given = (tokens,), positions.shape
    if given != wanted and (rank == 3 or given != (shape[0], *wanted)):
        raise ValueError("positions must be [tokens]" + (" or [batch, tokens]" * (rank == 4)))
    if positions.dtype not in _POSITION_DTYPES:
        raise ValueError("positions must be int32 or int64")
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1:
        raise ValueError("frequencies must be a float64 [rotary_dim // 2] tensor")
    pairs = frequencies.shape[0]
    if pairs == 0 or 2 * pairs > shape[-1]:
        raise ValueError("frequencies must cover at least one pair and at most head_dim features")
    if pairs > 1 and frequencies.stride(0) != 1:
        raise ValueError("frequencies must be contiguous")
    if shape[-1] > _MAX_HEAD_DIM:
        raise ValueError(f"rotary_embedding supports head_dim up to {_MAX_HEAD_DIM}")
    if not q.is_cuda:
        raise ValueError("rotary_embedding requires CUDA (ROCm/HIP) tensors")
    device = q.get_device()
    if positions.get_device() != device or frequencies.get_device() != device:
        raise ValueError("q, positions and frequencies must be on one device")
    if q.stride(-1) != 1:
        raise ValueError("q requires a contiguous final dimension")
    if k is not None and k.stride(-1) != 1:
        raise ValueError("k requires a contiguous final dimension")
