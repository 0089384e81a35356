"""qk_norm_rotary against norm and rotation in float64, its gradients, its refusals.

Tolerance, with u = 2^-24 and n = head_dim. The sum of n squares is off by at most n u of itself, so
1 / sqrt(mean + eps) by e = (n / 2 + 4) u. The normed value takes two more products, cosine, sine and
the magnitude are rounded to float32, the rotation makes two products and a sum: an output is off by
at most (e + 8 u) m (|z1| + |z2|) before it is rounded, which adds eps / 2 of it. The gradient of x is
T1 - T2 with |T1| <= r G and |T2| <= |x| r^3 sum(G |x|) / n for G = m (|dy1| + |dy2|) |w|: the first is
off by (e + 10 u), the second by (3 e + n u + 16 u) of that. The weight's is a sum of `rows` products,
off by at most (rows + 16) u + e of the sum of their sizes.
"""

from __future__ import annotations

import pytest
import torch

from tklab.kernels.qk_norm_rotary import qk_norm_rotary
from tklab.kernels.rms_norm import rms_norm
from tklab.kernels.rotary import rotary_embedding, rotary_frequencies

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def _turn(x, cos, sin, interleaved):
    """x with its first features turned; with absolute tables, the sum of both terms' sizes."""
    rotary = 2 * cos.shape[-1]
    part, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), rest), -1)
    a, b = part[..., : rotary // 2], part[..., rotary // 2:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)


def _both(x, rotary, interleaved, magnitude):
    """m (|x1| + |x2|) for each feature of a pair, |x| for the others."""
    one = torch.ones(rotary // 2, dtype=torch.float64, device=x.device)
    x = x.abs()
    sums = _turn(x, one, -one, interleaved)  # (x1 + x2, x2 - x1)
    flipped = _turn(x, one, one, interleaved)  # (x1 - x2, x2 + x1)
    both = torch.maximum(sums, flipped)
    scale = torch.ones_like(both)
    scale[..., :rotary] = abs(magnitude)
    return both * scale


def _rounded(value, bound, dtype):
    info = torch.finfo(dtype)
    return bound + info.eps / 2 * (value.abs() + bound) + info.tiny * info.eps / 2


def _within(got, value, bound):
    off = (got.detach().double() - value).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


class _Side:
    """Value and gradients of one side in float64, with the bounds on their errors."""

    def __init__(self, x, w, positions, frequencies, eps, interleaved, magnitude):
        n, rotary = x.shape[-1], 2 * len(frequencies)
        self.x, self.w, self.dtype, self.how = x.detach().double(), w.detach().double(), x.dtype, (rotary, interleaved)
        angle = positions.double()[..., None] * frequencies
        angle = angle.unsqueeze(1) if x.ndim == 3 or positions.ndim == 2 else angle
        self.cos, self.sin, self.magnitude = magnitude * angle.cos(), magnitude * angle.sin(), magnitude
        self.r = 1 / torch.sqrt(self.x.square().mean(-1, keepdim=True) + eps)
        self.e, self.n = (n / 2 + 4) * U, n

    def value(self):
        z = self.x * self.r * self.w
        y = _turn(z, self.cos, self.sin, self.how[1])
        return y, _rounded(y, (self.e + 8 * U) * _both(z, *self.how, self.magnitude), self.dtype)

    def gradients(self, dy):
        dy = dy.double()
        dz = _turn(dy, self.cos, -self.sin, self.how[1])
        size = _both(dy, *self.how, self.magnitude)
        unit, g, big = self.x * self.r, dz * self.w, size * self.w.abs()
        dx = self.r * (g - unit * (g * unit).mean(-1, keepdim=True))
        second = unit.abs() * self.r * (big * unit.abs()).mean(-1, keepdim=True)
        bound = (self.e + 10 * U) * self.r * big + (3 * self.e + (self.n + 16) * U) * second
        rows = self.x.numel() // self.n
        dw = (dz * unit).flatten(0, -2).sum(0)
        dw_bound = ((rows + 16) * U + self.e) * (size * unit.abs()).flatten(0, -2).sum(0)
        return (dx, _rounded(dx, bound, self.dtype)), (dw, _rounded(dw, dw_bound, self.dtype))


def _make(shape, dtype, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _weights(dim, dtype, seed):
    return tuple((1 + 0.3 * _make((dim,), torch.float32, seed + i)).to(dtype) for i in range(2))


def _check(q, k, qw, kw, positions, frequencies, eps=1e-5, interleaved=False, magnitude=1.0, dq=None, dk=None):
    """Values, and the four gradients where dq and dk are given."""
    leaves = [t.detach().requires_grad_(dq is not None) for t in (q, k, qw, kw)]
    out = qk_norm_rotary(*leaves, positions, frequencies, eps=eps, interleaved=interleaved, magnitude=magnitude)
    sides = [_Side(x, w, positions, frequencies, eps, interleaved, magnitude) for x, w in ((q, qw), (k, kw))]
    for got, x, side in zip(out, (q, k), sides):
        assert got.shape == x.shape and got.dtype == x.dtype
        _within(got, *side.value())
    if dq is None:
        return out
    grads = torch.autograd.grad(out, leaves, (dq, dk))
    for i, (side, dy) in enumerate(zip(sides, (dq, dk))):
        dx, dw = side.gradients(dy)
        assert grads[i].dtype == q.dtype and grads[i + 2].shape == qw.shape
        _within(grads[i], *dx)
        _within(grads[i + 2], *dw)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rotary", [(64, 64), (80, 32), (80, 20), (96, 24), (128, 128), (128, 2), (20, 10), (7, 4),
                                        (2, 2), (66, 34), (256, 64), (512, 512), (511, 510), (300, 150)])
def test_layouts_dtypes_and_parts_of_the_head(interleaved, dtype, dim, rotary) -> None:
    q, k = _make((2, 5, 19, dim), dtype, 1), _make((2, 2, 19, dim), dtype, 2)
    dq, dk = _make((2, 19, 5, dim), dtype, 3).transpose(1, 2), _make((2, 2, 19, dim), dtype, 4)
    freq, _ = rotary_frequencies(rotary, device="cuda")
    pos = torch.arange(38, device="cuda").reshape(2, 19) * 7
    _check(q, k, *_weights(dim, dtype, 5), pos, freq, 1e-6, interleaved, 1.25, dq, dk)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 32, 8), (2, 3, 1), (37, 64, 8), (1000, 7, 7),
                                                   (4099, 16, 2), (3, 300, 5)])
def test_packed_tokens_and_head_counts(tokens, heads, kv_heads) -> None:
    q, k, dq, dk = (_make((tokens, h, 128), torch.bfloat16, 3 + h + i) for i in range(2) for h in (heads, kv_heads))
    freq, _ = rotary_frequencies(128, device="cuda")
    pos = torch.randint(-1000, 100000, (tokens,), device="cuda", dtype=torch.int32)
    _check(q, k, *_weights(128, torch.bfloat16, 9), pos, freq, dq=dq, dk=dk)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1, 2, 4, 8])
def test_views_of_a_joint_projection_at_any_boundary(offset) -> None:
    heads, kv, dim, batch, tokens = 4, 2, 64, 2, 33
    joint = _make((batch, tokens, (heads + 2 * kv) * dim + 9), torch.bfloat16, 7)
    q = joint[..., offset: offset + heads * dim].unflatten(-1, (heads, dim)).transpose(1, 2)
    k = joint[..., offset + heads * dim: offset + (heads + kv) * dim]
    k = k.unflatten(-1, (kv, dim)).transpose(1, 2)
    freq, _ = rotary_frequencies(dim, device="cuda")
    pos = torch.arange(2 * tokens, device="cuda")[::2]
    weights = [w[offset: offset + dim] for w in _weights(dim + offset, torch.bfloat16, 8)]
    before = joint.clone()
    _check(q, k, *weights, pos, freq, dq=_make(q.shape, q.dtype, 9), dk=_make(k.shape, k.dtype, 10))
    assert torch.equal(joint, before)


@pytest.mark.gpu
def test_is_the_norm_and_then_the_rotation() -> None:
    """The two operators after one another, up to the rounding between them (float32)."""
    q, k = _make((29, 6, 128), torch.float32, 11), _make((29, 2, 128), torch.float32, 12)
    qw, kw = _weights(128, torch.float32, 13)
    freq, magnitude = rotary_frequencies(96, scaling="yarn", factor=4.0, original_length=2048, device="cuda")
    pos = torch.arange(29, device="cuda") + 5000
    out = qk_norm_rotary(q, k, qw, kw, pos, freq, eps=1e-5, magnitude=magnitude)
    normed = [rms_norm(x.reshape(-1, 128), w, eps=1e-5).reshape(x.shape) for x, w in ((q, qw), (k, kw))]
    for got, want in zip(out, rotary_embedding(*normed, pos, freq, magnitude=magnitude)):
        torch.testing.assert_close(got, want, rtol=0, atol=2 * (64 + 4 + 8) * U * 2 * magnitude * float(want.abs().max()))


@pytest.mark.gpu
def test_rows_of_zeros_tiny_and_large_rows() -> None:
    scale = torch.tensor([0.0, 1e-30, 1e-4, 1.0, 1e4, 1e15], device="cuda")[:, None, None]
    q = (_make((6, 3, 64), torch.float32, 14) * scale).to(torch.bfloat16)
    k = q[:, :1].contiguous()
    freq, _ = rotary_frequencies(32, device="cuda")
    pos = torch.arange(6, device="cuda")
    out = _check(q, k, *_weights(64, torch.bfloat16, 15), pos, freq, dq=_make(q.shape, q.dtype, 16),
                 dk=_make(k.shape, k.dtype, 17))
    assert not out[0][0].any()


@pytest.mark.gpu
def test_an_infinity_or_nan_stays_in_its_row() -> None:
    q = _make((4, 3, 64), torch.float32, 18)
    q[1, 2, 5], q[2, 0, 40] = torch.inf, torch.nan
    k = _make((4, 1, 64), torch.float32, 19)
    weights = _weights(64, torch.float32, 20)
    freq, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(4, device="cuda")
    out, _ = qk_norm_rotary(q, k, *weights, pos, freq)
    bad = torch.zeros(4, 3, dtype=torch.bool, device="cuda")
    bad[1, 2] = bad[2, 0] = True
    assert bool(out.isnan().any(-1).eq(bad).all())
    clean, _ = qk_norm_rotary(q.nan_to_num(1.0, 1.0), k, *weights, pos, freq)
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.gpu
def test_broadcast_inputs_and_gradients() -> None:
    q = _make((1, 1, 7, 64), torch.float32, 21).expand(3, 4, 7, 64)
    k = _make((3, 2, 7, 64), torch.float32, 22)
    weights = _weights(64, torch.float32, 23)
    freq, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(7, device="cuda").expand(3, 7)
    dq = _make((64,), torch.float32, 24).expand(3, 4, 7, 64)
    dk = torch.ones((), device="cuda").expand(3, 2, 7, 64)
    _check(q, k, *weights, pos, freq, dq=dq, dk=dk)
    # Through the expansion: the leaf's gradient is the sum over its copies.
    leaf = q[:1, :1].detach().requires_grad_()
    out, _ = qk_norm_rotary(leaf.expand(3, 4, 7, 64), k, *weights, pos, freq)
    (got,) = torch.autograd.grad(out, leaf, dq)
    dx, bound = _Side(q, weights[0], pos, freq, 1e-5, False, 1.0).gradients(dq)[0]
    _within(got, dx.sum((0, 1), keepdim=True), (bound + 12 * U * dx.abs()).sum((0, 1), keepdim=True))


@pytest.mark.gpu
def test_gradients_of_one_side_and_of_weights_alone() -> None:
    q, k = _make((5, 4, 64), torch.float32, 25), _make((5, 2, 64), torch.float32, 26)
    qw, kw = _weights(64, torch.float32, 27)
    freq, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(5, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    everything = torch.autograd.grad([o.sum() for o in qk_norm_rotary(*leaves, pos, freq)], leaves)
    q_out, k_out = qk_norm_rotary(*leaves, pos, freq)
    got = torch.autograd.grad(k_out.sum(), leaves, allow_unused=True)
    assert got[0] is None and got[2] is None
    assert torch.equal(got[1], everything[1]) and torch.equal(got[3], everything[3])
    out = qk_norm_rotary(q.detach(), k.detach(), qw, kw.detach(), pos, freq)
    assert out[0].requires_grad
    (got,) = torch.autograd.grad(out[0].sum() + out[1].sum(), qw)
    assert torch.equal(got, everything[2])
    out = qk_norm_rotary(q.detach(), k, qw.detach(), kw.detach(), pos, freq)
    (got,) = torch.autograd.grad(out[0].sum() + out[1].sum(), k)
    assert torch.equal(got, everything[1])


@pytest.mark.gpu
def test_gradients_against_differences() -> None:
    """Central differences of step h are off by h^2 / 6 times the third derivative, below 100 for these
    inputs of size 1, and by the rounding of two sums (float64) of float32 outputs over 2 h: with
    h = 2^-7, at most 2^-14 / 6 * 100 + 60 * 76 * 2^-24 * 8 / (2 h) = 0.14."""
    q, k = _make((2, 3, 10), torch.float32, 28).clamp(-2, 2), _make((2, 1, 10), torch.float32, 29).clamp(-2, 2)
    qw, kw = _weights(10, torch.float32, 30)
    freq, _ = rotary_frequencies(8, device="cuda")
    pos = torch.tensor([3, 50], device="cuda")
    dq, dk = _make(q.shape, torch.float32, 31).clamp(-2, 2), _make(k.shape, torch.float32, 32).clamp(-2, 2)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]

    def loss(*inputs):
        a, b = qk_norm_rotary(*inputs, pos, freq, interleaved=True)
        return (a.double() * dq).sum() + (b.double() * dk).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    for which, index in [(0, (0, 0, 0)), (0, (1, 2, 9)), (1, (1, 0, 3)), (2, (0,)), (2, (9,)), (3, (4,))]:
        ends = []
        for sign in (1, -1):
            moved = [t.detach().clone() for t in leaves]
            moved[which][index] += sign * 2.0 ** -7
            ends.append(loss(*moved))
        change = float(ends[0] - ends[1]) * 2.0 ** 6
        assert abs(change - float(grads[which][index])) <= 0.14


@pytest.mark.gpu
def test_many_rows_and_the_same_bits_again() -> None:
    """More runs than workgroups in the backward: partial sums over several runs, in a fixed order."""
    q, k = _make((3, 12, 3001, 64), torch.bfloat16, 33), _make((3, 3, 3001, 64), torch.bfloat16, 34)
    dq, dk = _make(q.shape, q.dtype, 35), _make(k.shape, k.dtype, 36)
    freq, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(3001, device="cuda")
    weights = _weights(64, torch.bfloat16, 37)
    _check(q, k, *weights, pos, freq, dq=dq, dk=dk)
    leaves = [t.requires_grad_() for t in (q, k, *weights)]
    first, second = (torch.autograd.grad(qk_norm_rotary(*leaves, pos, freq), leaves, (dq, dk)) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(first, second))


@pytest.mark.gpu
def test_offsets_past_32_bits() -> None:
    storage = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device="cuda")
    q = storage.as_strided((2, 2, 3, 128), (2 ** 31, 384, 128, 1))
    q.copy_(_make(q.shape, torch.bfloat16, 38))
    k = _make((2, 1, 3, 128), torch.bfloat16, 39)
    freq, _ = rotary_frequencies(128, device="cuda")
    pos = torch.arange(6, device="cuda").reshape(2, 3)
    _check(q, k, *_weights(128, torch.bfloat16, 40), pos, freq, dq=q.detach(), dk=k.detach())


@pytest.mark.gpu
def test_more_runs_than_one_grid_dimension_holds() -> None:
    """2^24 + 9 workgroups of a token each and more: 16 heads of an odd half, which no vector divides.
    The input is one token's, the output 67 GB."""
    tokens, period = 2 ** 24 + 9, 4096
    q, k = _make((1, 16, 126), torch.bfloat16, 41), _make((1, 1, 126), torch.bfloat16, 42)
    weights = _weights(126, torch.bfloat16, 43)
    freq, _ = rotary_frequencies(126, device="cuda")
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") % period
    want = qk_norm_rotary(q.expand(period, -1, -1), k.expand(period, -1, -1), *weights, positions[:period], freq)
    out = qk_norm_rotary(q.expand(tokens, -1, -1), k.expand(tokens, -1, -1), *weights, positions, freq)
    step = 64 * period
    for got, first in zip(out, want):
        for t in range(0, tokens // step * step, step):
            assert bool((got[t: t + step].view(64, period, *first.shape[1:]) == first).all())
        assert torch.equal(got[-9:], first[:9])


@pytest.mark.gpu
def test_a_captured_training_step_replays() -> None:
    """No eager graph of the captured leaves is alive: they are made for the capture's stream."""
    freq, _ = rotary_frequencies(48, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()

    def step(q, k, qw, kw, pos, dq, dk):
        leaves = (q, k, qw, kw)
        out = qk_norm_rotary(*leaves, pos, freq)
        return (*out, *torch.autograd.grad(out, leaves, (dq, dk)))

    def made(seed):
        q, k = _make((2, 4, 33, 64), torch.bfloat16, seed), _make((2, 2, 33, 64), torch.bfloat16, seed + 1)
        leaves = [t.requires_grad_() for t in (q, k, *_weights(64, torch.bfloat16, seed + 4))]
        return (*leaves, torch.arange(33, device="cuda") * seed, _make(q.shape, torch.bfloat16, seed + 2),
                _make(k.shape, torch.bfloat16, seed + 3))

    with torch.cuda.stream(stream):
        step(*made(1))
        inputs = made(2)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            results = step(*inputs)
    torch.cuda.synchronize()
    for seed in (3, 4, 5):
        other = made(seed)
        eager = step(*other)
        with torch.no_grad():
            for held, new in zip(inputs, other):
                held.copy_(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(results, eager))


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused() -> None:
    q, k = _make((5, 4, 64), torch.float32, 71), _make((5, 2, 64), torch.float32, 72)
    leaves = [t.requires_grad_() for t in (q, k, *_weights(64, torch.float32, 73))]
    freq, pos = rotary_frequencies(64, device="cuda")[0], torch.arange(5, device="cuda")
    dq, dk = _make(q.shape, torch.float32, 74), _make(k.shape, torch.float32, 75)
    want = torch.autograd.grad(qk_norm_rotary(*leaves, pos, freq), leaves, (dq, dk))
    out = qk_norm_rotary(*leaves, pos, freq)
    got = torch.autograd.grad(out, leaves, (dq.requires_grad_(), dk), create_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    for x in got:
        with pytest.raises(RuntimeError, match="once_differentiable"):
            x.sum().backward()


@pytest.mark.gpu
def test_gradients_where_hooks_move_what_is_saved() -> None:
    """A copy to the host and back is dense, whatever the views' strides were."""
    joint = _make((3, 7, 6 * 64 + 40), torch.bfloat16, 61)
    weights, freq = _weights(64, torch.bfloat16, 62), rotary_frequencies(32, device="cuda")[0]
    pos = torch.arange(7, device="cuda").expand(3, 7)
    dq, dk = _make((3, 4, 7, 64), torch.bfloat16, 63), _make((3, 2, 7, 64), torch.bfloat16, 64)

    def gradients():
        leaves = [joint[..., :4 * 64].view(3, 7, 4, 64).transpose(1, 2),
                  joint[..., 4 * 64:6 * 64].view(3, 7, 2, 64).transpose(1, 2), *weights]
        leaves = [t.detach().requires_grad_() for t in leaves]
        return torch.autograd.grad(qk_norm_rotary(*leaves, pos, freq), leaves, (dq, dk))

    want = gradients()
    with torch.autograd.graph.save_on_cpu():
        got = gradients()
    assert all(torch.equal(x, y) for x, y in zip(got, want))

    def whole(t):  # strides of the last dimension other than 1
        return t.movedim(0, -1).contiguous().movedim(-1, 0) if t.ndim == 4 else t

    with torch.autograd.graph.saved_tensors_hooks(whole, lambda t: t), pytest.raises(ValueError, match="contiguous"):
        gradients()


@pytest.mark.gpu
def test_forward_mode_is_refused_not_dropped() -> None:
    from torch.autograd import forward_ad

    q, k = torch.randn(1, 2, 5, 8, device="cuda"), torch.randn(1, 1, 5, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    freq, _ = rotary_frequencies(8, device="cuda")
    positions = torch.arange(5, device="cuda")
    for dual in range(3):
        with torch.no_grad(), forward_ad.dual_level():
            args = [q, k, w]
            args[dual] = forward_ad.make_dual(args[dual], torch.ones_like(args[dual]))
            with pytest.raises(RuntimeError, match="forward mode AD"):
                qk_norm_rotary(*args, w, positions, freq)


# ------------------------------------------------------------------ without a GPU


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("change,message", [
    (dict(q=_meta(4, 64)), "expects q"),
    (dict(q=_meta(2, 0, 5, 64)), "empty"),
    (dict(k=_meta(2, 0, 5, 64)), "empty"),
    (dict(k=_meta(5, 4, 64)), "both"),
    (dict(k=_meta(2, 4, 6, 64)), "head counts"),
    (dict(k=_meta(2, 4, 5, 64, dtype=torch.float16)), "share a dtype"),
    (dict(q_weight=_meta(64, dtype=torch.float32)), "share a dtype"),
    (dict(k_weight=_meta(32)), "weight must be"),
    (dict(k_weight=_meta(128)[::2]), "contiguous"),
    (dict(q=_meta(2, 4, 5, 64, dtype=torch.float64)), "supports float16"),
    (dict(q=_meta(2, 65536, 5, 64)), "65535 heads"),
    (dict(q=_meta(2 ** 16, 1, 2 ** 15, 64), k=_meta(2 ** 16, 1, 2 ** 15, 64)), "tokens"),
    (dict(positions=_meta(4, dtype=torch.int64)), "positions must be"),
    (dict(positions=_meta(5, dtype=torch.float32)), "int32 or int64"),
    (dict(frequencies=_meta(32, dtype=torch.float32)), "float64"),
    (dict(frequencies=_meta(33, dtype=torch.float64)), "cover"),
    (dict(frequencies=_meta(0, dtype=torch.float64)), "cover"),
    (dict(q=_meta(2, 4, 5, 514), k=_meta(2, 4, 5, 514), q_weight=_meta(514), k_weight=_meta(514)), "head_dim up to"),
    (dict(), "requires CUDA"),
])
def test_refusals(change, message) -> None:
    args = dict(q=_meta(2, 4, 5, 64), k=_meta(2, 2, 5, 64), q_weight=_meta(64), k_weight=_meta(64),
                positions=_meta(5, dtype=torch.int64), frequencies=_meta(32, dtype=torch.float64))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        qk_norm_rotary(*args.values())


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [0.0, -1.0, float("nan"), float("inf"), 1e-40, 1e39])
def test_refuses_an_epsilon_that_float32_does_not_hold(eps) -> None:
    q, w = torch.zeros(1, 1, 64, device="cuda"), torch.ones(64, device="cuda")
    freq, _ = rotary_frequencies(64, device="cuda")
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rotary(q, q, w, w, torch.arange(1, device="cuda"), freq, eps=eps)


@pytest.mark.gpu
def test_refuses_rows_without_a_unit_stride() -> None:
    q = torch.zeros(2, 4, 64, 5, device="cuda").transpose(2, 3)
    w = torch.ones(64, device="cuda")
    freq, _ = rotary_frequencies(64, device="cuda")
    with pytest.raises(ValueError, match="contiguous final"):
        qk_norm_rotary(q, q, w, w, torch.arange(5, device="cuda"), freq)
