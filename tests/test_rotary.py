"""rotary_embedding against the rotation in float64, its gradient, its refusals.

Tolerance: cosine, sine and the magnitude are each rounded to float32 and the rotation makes two
products and a sum there, so an output is off by at most 5 * 2^-24 * m * (|x1| + |x2|) before it is
rounded to its dtype, which adds half a step: eps / 2 of the value (and half the smallest
subnormal). float64's own errors (angles up to 10^7 rad: 10^-9) are far below.
"""

from __future__ import annotations

import math

import pytest
import torch

from tklab.kernels.rotary import rotary_embedding, rotary_frequencies

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _pairs(x, rotary, interleaved):
    part = x[..., :rotary]
    if interleaved:
        return part[..., 0::2], part[..., 1::2]
    return part[..., : rotary // 2], part[..., rotary // 2:]


def _join(y1, y2, rest, interleaved):
    turned = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((turned, rest), -1)


def _expected(x, positions, frequencies, interleaved, magnitude, sign=1.0):
    """(value, bound on the difference) in float64."""
    x64, rotary = x.detach().double(), 2 * len(frequencies)
    angle = positions.double()[..., None] * frequencies
    angle = angle.unsqueeze(1) if x.ndim == 3 or positions.ndim == 2 else angle
    c, s = magnitude * angle.cos(), sign * magnitude * angle.sin()
    x1, x2 = _pairs(x64, rotary, interleaved)
    rest = x64[..., rotary:]
    y = _join(x1 * c - x2 * s, x2 * c + x1 * s, rest, interleaved)
    size = abs(magnitude) * (x1.abs() + x2.abs())
    bound = _join(size, size, torch.zeros_like(rest), interleaved) * 5 * 2.0 ** -24
    info = torch.finfo(x.dtype)
    return y, bound + info.eps / 2 * (y.abs() + bound) + info.tiny * info.eps / 2


def _check(out, x, positions, frequencies, interleaved=False, magnitude=1.0, sign=1.0):
    assert out.shape == x.shape and out.dtype == x.dtype
    y, bound = _expected(x, positions, frequencies, interleaved, magnitude, sign)
    off = (out.detach().double() - y).abs()
    assert bool((off <= bound).all()), float((off - bound).max())
    rotary = 2 * len(frequencies)
    assert torch.equal(out[..., rotary:], x[..., rotary:])


def _make(shape, dtype, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rotary", [(64, 64), (80, 32), (80, 20), (96, 24), (128, 128), (128, 2),
                                        (20, 10), (7, 4), (256, 64), (1024, 1024)])
def test_layouts_dtypes_and_parts_of_the_head(interleaved, dtype, dim, rotary) -> None:
    q, k = _make((2, 5, 19, dim), dtype, 1), _make((2, 2, 19, dim), dtype, 2)
    freq, _ = rotary_frequencies(rotary, device="cuda")
    pos = torch.arange(38, device="cuda").reshape(2, 19) * 7
    q_out, k_out = rotary_embedding(q, k, pos, freq, interleaved=interleaved, magnitude=1.25)
    _check(q_out, q, pos, freq, interleaved, 1.25)
    _check(k_out, k, pos, freq, interleaved, 1.25)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (1, 32, 8), (2, 3, 1), (37, 64, 8),
                                                   (1000, 7, 7), (4099, 16, 2)])
def test_packed_tokens_and_head_counts(tokens, heads, kv_heads) -> None:
    q = _make((tokens, heads, 128), torch.bfloat16, 3)
    k = _make((tokens, kv_heads, 128), torch.bfloat16, 4)
    freq, _ = rotary_frequencies(128, device="cuda")
    pos = torch.randint(0, 100000, (tokens,), device="cuda")
    q_out, k_out = rotary_embedding(q, k, pos, freq)
    _check(q_out, q, pos, freq)
    _check(k_out, k, pos, freq)
    assert torch.equal(rotary_embedding(q, None, pos, freq), q_out)


@pytest.mark.gpu
def test_a_call_with_several_blocks_per_token_and_one_with_many_tokens_per_block() -> None:
    freq, _ = rotary_frequencies(256, device="cuda")
    q = _make((3, 200, 2, 256), torch.float32, 5)
    pos = torch.tensor([5, 900], device="cuda", dtype=torch.int32)
    _check(rotary_embedding(q, None, pos, freq), q, pos, freq)
    freq, _ = rotary_frequencies(4, device="cuda")
    q = _make((2, 1, 3001, 8), torch.float16, 6)
    pos = torch.arange(3001, device="cuda", dtype=torch.int32)
    _check(rotary_embedding(q, None, pos, freq, interleaved=True), q, pos, freq, True)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 2, 4, 8])
def test_views_of_a_joint_projection_at_any_boundary(interleaved, offset) -> None:
    """q and k as slices of one [batch, tokens, everything] projection, head-major."""
    heads, kv, dim, batch, tokens = 4, 2, 64, 2, 33
    joint = _make((batch, tokens, (heads + 2 * kv) * dim + 9), torch.bfloat16, 7)
    q = joint[..., offset: offset + heads * dim].unflatten(-1, (heads, dim)).transpose(1, 2)
    k = joint[..., offset + heads * dim: offset + (heads + kv) * dim]
    k = k.unflatten(-1, (kv, dim)).transpose(1, 2)
    freq, _ = rotary_frequencies(dim, device="cuda")
    pos = torch.arange(2 * tokens, device="cuda")[::2]
    before = joint.clone()
    q_out, k_out = rotary_embedding(q, k, pos, freq, interleaved=interleaved)
    _check(q_out, q, pos, freq, interleaved)
    _check(k_out, k, pos, freq, interleaved)
    assert torch.equal(joint, before)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_far_negative_and_expanded_positions(dtype) -> None:
    freq, _ = rotary_frequencies(64, device="cuda")
    q = _make((3, 4, 5, 64), torch.float32, 8)
    pos = torch.tensor([0, -1, -123457, 10 ** 6, 2 ** 31 - 1], device="cuda", dtype=dtype)
    _check(rotary_embedding(q, None, pos, freq), q, pos, freq)
    wide = pos.expand(3, 5)
    _check(rotary_embedding(q, None, wide, freq), q, wide, freq)


@pytest.mark.gpu
def test_positions_whose_angles_pass_53_bits() -> None:
    """Angles are float64, so such a position's is that of its nearest float64; the reference is
    formed from the same one."""
    freq, _ = rotary_frequencies(64, device="cuda")
    q = _make((2, 4, 7, 64), torch.float32, 18)
    pos = torch.tensor([2 ** 50 + 1, -2 ** 52 + 1, 2 ** 53 + 2, 10 ** 17 + 16, -10 ** 18, 2 ** 62 + 4096,
                        -2 ** 63], device="cuda")
    _check(rotary_embedding(q, None, pos, freq), q, pos, freq)


@pytest.mark.gpu
def test_position_zero_is_the_identity_and_quarter_turns_are_exact_swaps() -> None:
    q = _make((6, 2, 8), torch.float32, 9)
    pos = torch.arange(6, device="cuda")
    freq = torch.full((4,), math.pi / 2, dtype=torch.float64, device="cuda")
    out = rotary_embedding(q, None, pos, freq)
    assert torch.equal(out[0], q[0])
    assert torch.allclose(out[1], torch.cat((-q[1, :, 4:], q[1, :, :4]), -1), atol=1e-6)
    assert torch.allclose(out[2], -q[2], atol=1e-6)
    assert torch.allclose(out[4], q[4], atol=1e-6)


@pytest.mark.gpu
def test_offsets_past_32_bits() -> None:
    storage = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device="cuda")
    q = storage.as_strided((2, 2, 3, 128), (2 ** 31, 384, 128, 1))
    q.copy_(_make(q.shape, torch.bfloat16, 10))
    freq, _ = rotary_frequencies(128, device="cuda")
    pos = torch.arange(6, device="cuda").reshape(2, 3)
    _check(rotary_embedding(q, None, pos, freq), q, pos, freq)


@pytest.mark.gpu
def test_broadcast_input() -> None:
    q = _make((1, 1, 7, 64), torch.float32, 11).expand(3, 4, 7, 64).requires_grad_()
    freq, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(7, device="cuda")
    out = rotary_embedding(q, None, pos, freq)
    _check(out, q, pos, freq)
    grad = torch.randn(64, device="cuda").expand(3, 4, 7, 64)
    (dq,) = torch.autograd.grad(out, q, grad)
    _check(dq, grad, pos, freq, sign=-1.0)
    # A gradient that is one number everywhere has no unit stride.
    (dq,) = torch.autograd.grad(rotary_embedding(q, None, pos, freq).sum(), q)
    _check(dq, torch.ones_like(q), pos, freq, sign=-1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,rotary", [(128, 128), (80, 32), (20, 10)])
def test_gradient_is_the_inverse_rotation(interleaved, dtype, dim, rotary) -> None:
    q, k = (_make((2, h, 11, dim), dtype, h).requires_grad_() for h in (6, 2))
    dq, dk = (_make((2, 11, h, dim), dtype, 20 + h).transpose(1, 2) for h in (6, 2))
    freq, _ = rotary_frequencies(rotary, device="cuda")
    pos = torch.arange(11, device="cuda") + 1000
    out = rotary_embedding(q, k, pos, freq, interleaved=interleaved, magnitude=0.75)
    gq, gk = torch.autograd.grad(out, (q, k), (dq, dk))
    _check(gq, dq, pos, freq, interleaved, 0.75, sign=-1.0)
    _check(gk, dk, pos, freq, interleaved, 0.75, sign=-1.0)


@pytest.mark.gpu
def test_gradient_against_differences() -> None:
    """The map is linear, so a central difference is exact up to rounding: with |x|, |dy| <= 4 and a
    step of 1/2, each of the two sums of 2 * 10 products is off by under 2 * 10 * 4 * 4 * 6 * 2^-24,
    which the division by the step doubles at most."""
    q = _make((3, 2, 10), torch.float32, 12).clamp(-4, 4).requires_grad_()
    dy = _make((3, 2, 10), torch.float32, 13).clamp(-4, 4)
    freq, _ = rotary_frequencies(8, device="cuda")
    pos = torch.tensor([3, 50, 700], device="cuda")

    def loss(x):
        return (rotary_embedding(x, None, pos, freq, interleaved=True) * dy).double().sum()

    (grad,) = torch.autograd.grad(loss(q), q)
    for index in [(0, 0, 0), (1, 1, 3), (2, 0, 7), (2, 1, 9)]:
        up, down = q.detach().clone(), q.detach().clone()
        up[index] += 0.25
        down[index] -= 0.25
        change = float((loss(up) - loss(down)) / (up[index] - down[index]))
        assert abs(change - float(grad[index])) <= 2 * 2 * 2 * 10 * 4 * 4 * 6 * 2.0 ** -24


@pytest.mark.gpu
def test_gradient_of_one_output_alone() -> None:
    q, k = (_make((2, h, 5, 64), torch.float32, h).requires_grad_() for h in (4, 2))
    freq, _ = rotary_frequencies(64, device="cuda")
    pos = torch.arange(5, device="cuda")
    _, k_out = rotary_embedding(q, k, pos, freq)
    dk = _make(k.shape, torch.float32, 14)
    got, none = torch.autograd.grad(k_out, (k, q), dk, allow_unused=True)
    assert none is None
    _check(got, dk, pos, freq, sign=-1.0)
    q_out, k_out = rotary_embedding(q.detach(), k, pos, freq)
    (got,) = torch.autograd.grad((q_out.sum() + (k_out * dk).sum()), k)
    _check(got, dk, pos, freq, sign=-1.0)


@pytest.mark.gpu
def test_matches_rope_with_tables_of_the_same_angles() -> None:
    from tklab.kernels.rope import rope

    x = _make((40, 128), torch.float32, 15)
    freq, _ = rotary_frequencies(128, device="cuda")
    pos = torch.arange(40, device="cuda")
    angle = pos.double()[:, None] * freq
    expected = rope(x, angle.cos().float(), angle.sin().float())
    got = rotary_embedding(x[:, None], None, pos, freq)[:, 0]
    # Both round the tables to float32 and make the same two products: 3 * 2^-24 of the pair each.
    size = x[:, :64].abs() + x[:, 64:].abs()
    assert bool(((got - expected).abs() <= 6 * 2.0 ** -24 * torch.cat((size, size), 1)).all())


@pytest.mark.gpu
def test_a_captured_call_replays_with_new_positions_on_another_stream() -> None:
    q, k = _make((1, 8, 4, 128), torch.bfloat16, 16), _make((1, 2, 4, 128), torch.bfloat16, 17)
    freq, _ = rotary_frequencies(128, device="cuda")
    pos = torch.arange(4, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        rotary_embedding(q, k, pos, freq)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            q_out, k_out = rotary_embedding(q, k, pos, freq)
    torch.cuda.synchronize()
    for step in range(4):
        pos.fill_(37 * step).add_(torch.arange(4, device="cuda"))
        eager = rotary_embedding(q, k, pos, freq)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q_out, eager[0]) and torch.equal(k_out, eager[1])


@pytest.mark.gpu
def test_a_captured_forward_and_backward_replays() -> None:
    """No eager graph of the captured leaves is alive: they are made for the capture's stream."""
    freq, _ = rotary_frequencies(48, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()

    def step(q, k, pos, dq, dk):
        return torch.autograd.grad(rotary_embedding(q, k, pos, freq), (q, k), (dq, dk))

    def made(seed):
        q, k = _make((2, 4, 33, 64), torch.bfloat16, seed), _make((2, 2, 33, 64), torch.bfloat16, seed + 1)
        return (q.requires_grad_(), k.requires_grad_(), torch.arange(33, device="cuda") * seed,
                _make(q.shape, torch.bfloat16, seed + 2), _make(k.shape, torch.bfloat16, seed + 3))

    with torch.cuda.stream(stream):
        step(*made(1))
        inputs = made(2)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            grads = step(*inputs)
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
        assert all(torch.equal(x, y) for x, y in zip(grads, eager))


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
    (dict(q=_meta(2, 4, 5, 64, dtype=torch.float64), k=None), "supports float16"),
    (dict(positions=_meta(4, dtype=torch.int64)), "positions must be"),
    (dict(positions=_meta(1, 5, dtype=torch.int64)), "positions must be"),
    (dict(positions=_meta(5, dtype=torch.float32)), "int32 or int64"),
    (dict(frequencies=_meta(32, dtype=torch.float32)), "float64"),
    (dict(frequencies=_meta(33, dtype=torch.float64)), "cover"),
    (dict(frequencies=_meta(0, dtype=torch.float64)), "cover"),
    (dict(q=_meta(2, 4, 5, 1026), k=None), "head_dim up to"),
    (dict(), "requires CUDA"),
])
def test_refusals(change, message) -> None:
    args = dict(q=_meta(2, 4, 5, 64), k=_meta(2, 2, 5, 64), positions=_meta(5, dtype=torch.int64),
                frequencies=_meta(32, dtype=torch.float64))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        rotary_embedding(args["q"], args["k"], args["positions"], args["frequencies"])


@pytest.mark.gpu
def test_refuses_rows_without_a_unit_stride() -> None:
    q = torch.zeros(2, 4, 64, 5, device="cuda").transpose(2, 3)
    freq, _ = rotary_frequencies(64, device="cuda")
    with pytest.raises(ValueError, match="contiguous final"):
        rotary_embedding(q, None, torch.arange(5, device="cuda"), freq)


@pytest.mark.gpu
@pytest.mark.parametrize("dual", ["q", "k"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused_not_dropped(dual, grad) -> None:
    """A tangent is an error, as it is for ``rope``, whether or not anything requires a gradient."""
    from torch.autograd import forward_ad

    x = {name: torch.randn(1, 2, 5, 8, device="cuda") for name in "qk"}
    freq, _ = rotary_frequencies(8, device="cuda")
    positions = torch.arange(5, device="cuda")
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        plain = rotary_embedding(x["q"], x["k"], positions, freq)
        x[dual] = forward_ad.make_dual(x[dual], torch.ones_like(x[dual]))
        with pytest.raises(RuntimeError, match="forward mode AD"):
            rotary_embedding(x["q"], x["k"], positions, freq)
    again = rotary_embedding(x["q"], x["k"], positions, freq)
    assert all(torch.equal(a, b) for a, b in zip(plain, again))


@pytest.mark.gpu
def test_more_token_runs_than_one_grid_dimension_holds() -> None:
    """2^24 + 9 workgroups of a token each: rows of odd halves, which no vector divides. The input is
    one token's row, the output 34 GB."""
    tokens, period = 2 ** 24 + 9, 4096
    q = torch.randn(1, 2, 514, device="cuda").bfloat16()
    freq, _ = rotary_frequencies(514, device="cuda")
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") % period
    want = rotary_embedding(q.expand(period, -1, -1), None, positions[:period], freq)
    out = rotary_embedding(q.expand(tokens, -1, -1), None, positions, freq)
    assert out.shape == (tokens, 2, 514)
    step = 64 * period
    for t in range(0, tokens // step * step, step):
        assert bool((out[t: t + step].view(64, period, 2, 514) == want).all())
    assert torch.equal(out[-9:], want[:9])


def test_plain_and_linear_frequencies() -> None:
    freq, magnitude = rotary_frequencies(8, base=10000.0)
    assert freq.dtype == torch.float64 and magnitude == 1.0
    expected = torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64)
    torch.testing.assert_close(freq, expected, rtol=1e-14, atol=0)
    slower, magnitude = rotary_frequencies(8, scaling="linear", factor=4.0)
    torch.testing.assert_close(slower, expected / 4, rtol=1e-14, atol=0)
    assert magnitude == 1.0


def test_ntk_frequencies_keep_the_fastest_pair_and_slow_the_slowest_by_the_factor() -> None:
    plain, _ = rotary_frequencies(64)
    scaled, magnitude = rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert float(scaled[0]) == 1.0 and magnitude == 1.0
    assert float(plain[-1] / scaled[-1]) == pytest.approx(8.0, rel=1e-12)


def test_yarn_frequencies_keep_fast_pairs_and_slow_the_slow_ones() -> None:
    plain, _ = rotary_frequencies(128)
    scaled, magnitude = rotary_frequencies(128, scaling="yarn", factor=16.0, original_length=8192)
    assert magnitude == pytest.approx(0.1 * math.log(16.0) + 1.0)
    turns = 8192 * plain / (2 * math.pi)
    ratio = plain / scaled
    assert bool((ratio[turns > 40] == 1).all())
    torch.testing.assert_close(ratio[turns < 0.8], torch.full_like(ratio[turns < 0.8], 16.0))
    assert bool((ratio[1:] >= ratio[:-1]).all())


@pytest.mark.parametrize("kwargs,message", [
    (dict(rotary_dim=7), "even"),
    (dict(rotary_dim=0), "even"),
    (dict(rotary_dim=8, scaling="other"), "one of"),
    (dict(rotary_dim=8, factor=0.5), "factor"),
    (dict(rotary_dim=8, base=1.0), "base"),
    (dict(rotary_dim=2, scaling="ntk", factor=2.0), "above 2"),
    (dict(rotary_dim=8, scaling="yarn", factor=2.0), "original_length"),
    (dict(rotary_dim=8, scaling="yarn", original_length=64, fast_turns=1.0), "fast_turns"),
])
def test_refused_frequencies(kwargs, message) -> None:
    with pytest.raises(ValueError, match=message):
        rotary_frequencies(**kwargs)


@pytest.mark.parametrize("q,k,positions,message", [
    ((1, 65536, 1, 64), None, (1,), "65535 heads"),
    ((1, 65000, 1, 64), (1, 600, 1, 64), (1,), "65535 heads"),
    ((2, 65536, 64), None, (2,), "65535 heads"),
    ((2 ** 31 - 65536, 1, 64), None, (2 ** 31 - 65536,), "tokens"),
    ((2 ** 16, 1, 2 ** 15, 64), None, (2 ** 15,), "tokens"),
])
def test_sizes_past_the_librarys_counters_are_value_errors(q, k, positions, message) -> None:
    def meta(shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")

    with pytest.raises(ValueError, match=message):
        rotary_embedding(meta(q), None if k is None else meta(k), meta(positions, torch.int32),
                         meta((32,), torch.float64))
