"""quantized_decode against attention in float64 over the multiplied-out cache.

Tolerance. With A = sum_j p_j |v_j| / sum_j p_j: rounding a weight times its scale to the storage
dtype moves a result by at most eps / 2 * A, rounding the result by eps / 2 of it. A score is a
float32 sum of head_dim products times two factors, off by delta = (head_dim + 8) 2^-24 scale sum|q k|,
which moves the weights' numerator and denominator by that share each, as do the hardware exponential
(2^-22) and its argument's rounding (2^-24 of up to |s| + |m|); sums of n keys add (n + 64) 2^-24. In
float16 a weight below 2^-14 of the unit (at most 2 max |vs|) is a subnormal, off by 2^-25 of it.
"""

from __future__ import annotations

import math

import pytest
import torch

from tklab.kernels.gqa_decode import gqa_decode
from tklab.kernels.quantized_cache import append_quantized, read_quantized
from tklab.kernels.quantized_decode import quantized_decode

HALF = [torch.bfloat16, torch.float16]
KINDS = [torch.float8_e4m3fn, torch.int8]


def _problem(batch, heads, kv, max_len, dim, dtype, kind, seed, spread=3):
    gen = torch.Generator("cuda").manual_seed(seed)
    q = torch.randn(batch, heads, dim, generator=gen, device="cuda").to(dtype)
    shape = (batch, kv, max_len, dim)
    size = torch.exp2(torch.randint(-spread, spread + 1, (2, *shape[:3], 1), generator=gen, device="cuda").float())
    k = torch.randn(shape, generator=gen, device="cuda") * size[0].clamp(max=1)
    v = torch.randn(shape, generator=gen, device="cuda") * size[1]
    caches = [torch.zeros(shape, dtype=kind, device="cuda") for _ in "kv"]
    scales = torch.zeros(batch, kv, max_len, 2, device="cuda")
    append_quantized(*caches, scales, torch.zeros(batch, dtype=torch.int32, device="cuda"), k, v)
    return q, *caches, scales


def _check(q, k_cache, v_cache, scales, lens=None, scale=None):
    out, lse = quantized_decode(q, k_cache, v_cache, scales, lens, scale=scale, return_lse=True)
    batch, heads, dim = q.shape
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    assert lse.shape == (batch, heads) and lse.dtype == torch.float32
    group, factor = heads // k_cache.shape[1], dim ** -0.5 if scale is None else scale
    half = torch.finfo(q.dtype).eps / 2
    for b in range(batch):
        n = k_cache.shape[2] if lens is None else min(max(int(lens[b]), 0), k_cache.shape[2])
        for g in range(k_cache.shape[1]):
            rows = slice(g * group, (g + 1) * group)
            if n == 0:
                assert not out[b, rows].any() and bool((lse[b, rows] == -math.inf).all())
                continue
            s = scales[b, g, :n].double()
            keys = k_cache[b, g, :n].double() * s[:, :1]
            codes = v_cache[b, g, :n].double()
            values = codes * s[:, 1:]
            x = q[b, rows].double()
            scores = x @ keys.t() * factor
            delta = (dim + 8) * 2.0 ** -24 * (x.abs() @ keys.abs().t() * abs(factor)).amax(1, keepdim=True)
            delta = delta + 2.0 ** -22 + 2.0 ** -23 * (scores.abs().amax(1, keepdim=True) * 1.45 + 8)
            log = torch.logsumexp(scores, 1, keepdim=True)
            p = torch.exp(scores - log)
            want, size = p @ values, p @ values.abs()
            bound = half * size + (2 * delta + (n + 64) * 2.0 ** -24) * (size + want.abs())
            if q.dtype == torch.float16:
                bound = bound + 2.0 ** -25 * 2 * s[:, 1].abs().amax() * codes.abs().sum(0)
            info = torch.finfo(q.dtype)
            bound = bound + half * (want.abs() + bound) + info.tiny * info.eps
            off = (out[b, rows].double() - want).abs()
            assert bool((off <= bound).all()), float((off / bound).max())
            lse_off = (lse[b, rows].double() - log[:, 0] / math.log(2)).abs()
            lse_bound = (delta[:, 0] + (n + 64) * 2.0 ** -24) * 1.45 + 2.0 ** -22 * (log[:, 0].abs() * 1.45 + 1)
            assert bool((lse_off <= lse_bound).all()), float((lse_off / lse_bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (8, 2), (7, 1), (24, 2), (32, 2), (34, 2), (64, 1), (100, 1)])
def test_types_heads_and_groups(heads, kv, dtype, kind, dim) -> None:
    _check(*_problem(2, heads, kv, 77, dim, dtype, kind, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("max_len", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 160, 1000, 4100])
def test_cache_sizes(max_len, dtype, kind) -> None:
    _check(*_problem(1, 8, 2, max_len, 128, dtype, kind, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", HALF)
def test_ragged_lengths_and_lengths_out_of_range(dtype, dim) -> None:
    problem = _problem(9, 8, 2, 700, dim, dtype, torch.float8_e4m3fn, 3)
    lens = torch.tensor([0, 1, 31, 32, 33, 699, 700, 5000, -7], dtype=torch.int32, device="cuda")
    _check(*problem, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [64, 65, 130, 300])
def test_more_sequences_than_lanes(batch) -> None:
    problem = _problem(batch, 4, 1, 300, 64, torch.bfloat16, torch.int8, 4)
    gen = torch.Generator("cuda").manual_seed(5)
    lens = torch.randint(0, 301, (batch,), generator=gen, device="cuda", dtype=torch.int32)
    _check(*problem, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", HALF)
def test_a_long_context_of_one_sequence(dtype, kind) -> None:
    _check(*_problem(1, 4, 1, 70001, 128, dtype, kind, 6))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("kind", KINDS)
def test_scales_of_any_size_and_sign(dtype, kind) -> None:
    """Value scales over a wide range, growing and falling along the cache, of both signs and zero."""
    q, k, v, scales = _problem(2, 4, 2, 200, 64, dtype, kind, 7)
    steps = torch.linspace(-1, 1, 200, device="cuda")
    for shape in (steps, -steps, steps.abs()):
        # float16 results hold values of up to 448 * 2^6.
        scales[..., 1] = torch.exp2(shape * 20 - 16)
        scales[:, 1, ::3, 1] *= -1
        scales[:, 0, 50:90, 1] = 0
        scales[..., 0] = torch.exp2(steps * 3 - 8) * torch.where(torch.arange(200, device="cuda") % 2 == 0, 1.0, -1.0)
        _check(q, k, v, scales)
    scales[..., 1] = 0
    _check(q, k, v, scales)
    scales[..., 1] = 2.0 ** -120
    if dtype == torch.bfloat16:
        _check(q, k, v, scales)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0, 1e-30])
@pytest.mark.parametrize("dtype", HALF)
def test_score_scales(scale, dtype) -> None:
    problem = _problem(2, 8, 2, 150, 64, dtype, torch.float8_e4m3fn, 8, spread=1)
    _check(*problem, torch.tensor([150, 40], dtype=torch.int32, device="cuda"), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_growing_and_falling_scores(dtype) -> None:
    """The running maximum moves at every tile, or is set by the first key."""
    q, k, v, scales = _problem(1, 4, 1, 640, 64, dtype, torch.int8, 9)
    q.copy_(q.abs())
    k.copy_(k.abs().clamp(min=1))
    ramp = torch.linspace(0.001, 0.5, 640, device="cuda")
    for order in (ramp, ramp.flip(0)):
        scales[0, 0, :, 0] = order
        _check(q, k, v, scales)


@pytest.mark.gpu
def test_what_lies_past_a_length_cannot_reach_a_result() -> None:
    q, k, v, scales = _problem(3, 8, 2, 300, 128, torch.bfloat16, torch.float8_e4m3fn, 10)
    lens = torch.tensor([0, 45, 290], dtype=torch.int32, device="cuda")
    want = quantized_decode(q, k, v, scales, lens)
    for b, n in enumerate(lens.tolist()):
        for x in (k, v):
            x.view(torch.uint8)[b, :, n:] = 0x7F
        scales[b, :, n:] = torch.nan
    assert torch.equal(quantized_decode(q, k, v, scales, lens), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
def test_a_row_without_a_number_reaches_its_head_alone(dtype) -> None:
    q, k, v, scales = _problem(2, 8, 2, 100, 64, dtype, torch.int8, 11)
    want = quantized_decode(q, k, v, scales)
    scales[1, 0, 37, 1] = torch.nan
    got = quantized_decode(q, k, v, scales)
    assert bool(got[1, :4].isnan().all())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, 4:], want[1, 4:])


@pytest.mark.gpu
def test_is_gqa_decode_of_the_cache_read_back() -> None:
    """Codes and scales are exact in float16 where the scales are powers of two: then both see the same
    cache, and differ by the rounding of their weights and results."""
    q, k, v, scales = _problem(4, 16, 4, 500, 128, torch.float16, torch.int8, 12)
    scales.copy_(torch.exp2(scales.log2().round().clamp(-12, 4)))
    lens = torch.tensor([500, 0, 77, 300], dtype=torch.int32, device="cuda")
    keys, values = read_quantized(k, v, scales, lens, dtype=torch.float16)
    want, want_lse = gqa_decode(q, keys, values, lens, return_lse=True)
    got, lse = quantized_decode(q, k, v, scales, lens, return_lse=True)
    size = values.abs().float().amax()
    assert float((got.float() - want.float()).abs().amax()) <= 4 * 2.0 ** -11 * float(size)
    torch.testing.assert_close(lse, want_lse, rtol=1e-5, atol=1e-4)


@pytest.mark.gpu
def test_views_of_queries_and_caches() -> None:
    gen = torch.Generator("cuda").manual_seed(13)
    q, k, v, scales = _problem(3, 8, 2, 90, 128, torch.bfloat16, torch.float8_e4m3fn, 14)
    want = quantized_decode(q, k, v, scales)
    joint = torch.randn(3, 12, 128, generator=gen, device="cuda").bfloat16()
    joint[:, 2:10] = q
    turned = [x.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(x.dtype) for x in (k, v)]
    wide = torch.randn(3, 2, 200, 6, generator=gen, device="cuda")
    wide[:, :, 55:145, 2:4] = scales
    assert not turned[0].is_contiguous()
    assert torch.equal(quantized_decode(joint[:, 2:10], *turned, wide[:, :, 55:145, 2:4]), want)
    # One sequence, one head, one position: strides that address nothing.
    one = [x.view(torch.uint8)[:1, :1, :1].as_strided((1, 1, 1, 128), (3, 5, 7, 1)).view(x.dtype) for x in (k, v)]
    got = quantized_decode(q[:1, :4].as_strided((1, 4, 128), (1, 128, 1)), *one, scales[:1, :1, :1])
    assert torch.equal(got, quantized_decode(q[:1, :4].contiguous(), *(x[:1, :1, :1] for x in (k, v)), scales[:1, :1, :1]))


@pytest.mark.gpu
def test_offsets_past_32_bits() -> None:
    q, k, v, scales = _problem(2, 4, 1, 65, 128, torch.bfloat16, torch.int8, 15)
    far = 2 ** 32 + 4096
    room = torch.zeros(2, far + 65 * 128, dtype=torch.int8, device="cuda")
    k_far, v_far = (r.as_strided((2, 1, 65, 128), (far, 128, 128, 1)) for r in room)
    k_far.copy_(k)
    v_far.copy_(v)
    assert torch.equal(quantized_decode(q, k_far, v_far, scales), quantized_decode(q, k, v, scales))
    # Positions far apart: 65 rows of 2^23 bytes.
    long = torch.zeros(2 ** 30, dtype=torch.int8, device="cuda").as_strided((1, 1, 65, 128), (0, 0, 2 ** 23, 1))
    long.copy_(k[:1])
    got = quantized_decode(q[:1], long, v[:1], scales[:1])
    assert torch.equal(got, quantized_decode(q[:1], k[:1], v[:1], scales[:1]))


@pytest.mark.gpu
def test_captured_calls_replay_with_other_lengths_on_another_stream() -> None:
    q, k, v, scales = _problem(4, 8, 2, 500, 64, torch.bfloat16, torch.float8_e4m3fn, 16)
    lens = torch.full((4,), 500, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        quantized_decode(q, k, v, scales, lens)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            held = quantized_decode(q, k, v, scales, lens, return_lse=True)
    torch.cuda.synchronize()
    for new in ([1, 0, 499, 32], [500, 100, 3, 250], [0, 0, 0, 0], [77, 500, 500, 1]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        q.copy_(q.flip(0).contiguous())
        want = quantized_decode(q, k, v, scales, lens, return_lse=True)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, want))


# ------------------------------------------------------------------ without a GPU


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("change,message", [
    (dict(q=_meta(2, 8, 1, 64)), "expects q"),
    (dict(q=_meta(3, 8, 64)), "disagree"),
    (dict(q=_meta(2, 8, 128)), "disagree"),
    (dict(q=_meta(2, 0, 64)), "empty"),
    (dict(q=_meta(2, 7, 64)), "multiple of kv_heads"),
    (dict(q=_meta(2, 65536, 64)), "65535"),
    (dict(q=_meta(2, 8, 64, dtype=torch.float32)), "float16 or bfloat16"),
    (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"),
    (dict(k_cache=_meta(2, 2, 10, 64)), "share a float8"),
    (dict(v_cache=_meta(2, 2, 9, 64, dtype=F8)), "identical"),
    (dict(scales=_meta(2, 2, 2, 10, dtype=torch.float32)), "scales must be"),
    (dict(), "requires CUDA"),
])
def test_refusals(change, message) -> None:
    args = dict(q=_meta(2, 8, 64), k_cache=_meta(2, 2, 10, 64, dtype=F8), v_cache=_meta(2, 2, 10, 64, dtype=F8),
                scales=_meta(2, 2, 10, 2, dtype=torch.float32))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        quantized_decode(**args)


def test_refused_head_dim() -> None:
    with pytest.raises(ValueError, match="64 and 128"):
        quantized_decode(_meta(2, 8, 96), *[_meta(2, 2, 10, 96, dtype=F8)] * 2, _meta(2, 2, 10, 2, dtype=torch.float32))


def test_slots_of_sizes_that_are_not_taken() -> None:
    from tklab import _hip

    assert _hip.query("tk_quantized_decode_slots", 1, 8, 4, 2000, 128) > 0
    assert _hip.query("tk_quantized_decode_slots", 1, 8, 4, 32, 128) == 0
    for sizes in [(0, 8, 4, 2000, 128), (1, 8, 4, 2000, 96), (1, 8, -4, 2000, 128), (70000, 8, 4, 2000, 128),
                  (1, 8, 9000, 2000, 128), (1, 8, 4, 2 ** 31, 128), (60000, 1, 4, 2 ** 30, 128)]:
        assert _hip.query("tk_quantized_decode_slots", *sizes) == -1


# ------------------------------------------------------------------ weights of very different sizes


def _near(q, codes_k, codes_v, scales, factor):
    """What one KV head's rows are in float64, and how far off a result may be whose weights go through
    the second product as a bfloat16 and the bfloat16 of what that leaves.

    Each of the two is off by at most 2^-8 of what it rounds, so both together by 2^-16 of a weight times
    its scale, whatever the scales of other keys; the other terms are this module's.
    """
    s = scales.double()
    keys, values = codes_k.double() * s[:, :1], codes_v.double() * s[:, 1:]
    x, dim, n = q.double(), q.shape[-1], s.shape[0]
    scores = x @ keys.t() * factor
    delta = (dim + 8) * 2.0 ** -24 * (x.abs() @ keys.abs().t() * abs(factor)).amax(1, keepdim=True)
    delta = delta + 2.0 ** -22 + 2.0 ** -23 * (scores.abs().amax(1, keepdim=True) * 1.45 + 8)
    p = scores.softmax(1)
    want, size = p @ values, p @ values.abs()
    bound = 2.0 ** -16 * size + (2 * delta + (n + 64) * 2.0 ** -24) * (size + want.abs())
    info = torch.finfo(q.dtype)
    return want, bound + info.eps / 2 * (want.abs() + bound) + info.tiny * info.eps


def _check_near(q, k, v, scales, some):
    """Some (sequence, KV head)."""
    out = quantized_decode(q, k, v, scales)
    group = q.shape[1] // k.shape[1]
    for b, g in some:
        rows = slice(g * group, (g + 1) * group)
        want, bound = _near(q[b, rows], k[b, g], v[b, g], scales[b, g], q.shape[-1] ** -0.5)
        off = (out[b, rows].double() - want).abs()
        assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("larger", [0, 5, 13, 20, 30])
@pytest.mark.parametrize("above", [0, 14])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", HALF)
def test_keys_beside_a_large_value_without_weight(dtype, kind, above, larger) -> None:
    """One key whose value is 2^larger times the others' and whose weight is negligible, before or behind
    them; and, `above` nats over the others, a key without a value. So many sequences that each is one run."""
    q, k, v, scales = _problem(16, 128, 64, 1000, 64, dtype, kind, 20, spread=0)
    # The first feature alone makes the difference: 8 times 1/8 times the key's.
    q[..., 0] = 8
    scales[..., 1] *= 64  # (results of normal float16 numbers)
    k.view(torch.uint8)[..., 0] = 0
    k.view(torch.uint8)[:, :, [3, 700, 40], :] = 0
    one = torch.ones((), device="cuda").to(kind)
    scales[:, :, [3, 700], 0], scales[:, :, 40, 0] = -40.0, float(above)
    k.view(torch.uint8)[:, :, [3, 700, 40], 0] = one.view(torch.uint8)
    scales[:8, :, 3, 1] *= 2.0 ** larger
    scales[8:, :, 700, 1] *= 2.0 ** larger
    v.view(torch.uint8)[:, :, 40] = 0
    _check_near(q, k, v, scales, [(0, 0), (1, 63), (8, 5), (15, 31)])


def _few_keys(dtype, kind, device):
    """Values of both signs under weights of some size each: results below the sizes that were summed."""
    gen = torch.Generator(device).manual_seed(21)
    q = (0.3 * torch.randn(4, 8, 64, generator=gen, device=device)).to(dtype)
    codes = [(50 * torch.randn(4, 2, 5, 64, generator=gen, device=device)).round().clamp(-120, 120).to(kind) for _ in "kv"]
    return q, *codes, torch.rand(4, 2, 5, 2, generator=gen, device=device) * 0.01 + 0.01


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", HALF)
def test_weights_keep_what_their_rounding_left(dtype, kind) -> None:
    _check_near(*_few_keys(dtype, kind, "cuda"), [(b, g) for b in range(4) for g in range(2)])


@pytest.mark.parametrize("dtype", HALF)
def test_the_bound_is_passed_by_weights_rounded_once(dtype) -> None:
    """The same problem with weights of one rounding, on the CPU: what the bound has to notice."""
    q, k, v, scales = _few_keys(dtype, torch.int8, "cpu")

    def worst(parts):
        most = 0.0
        for b in range(4):
            for g in range(2):
                x, s = q[b, 4 * g: 4 * g + 4], scales[b, g]
                want, bound = _near(x, k[b, g], v[b, g], s, 64 ** -0.5)
                scores = x.double() @ (k[b, g].double() * s[:, :1]).t() * 64 ** -0.5
                p = torch.exp(scores - scores.amax(1, keepdim=True))
                weights = p * s[:, 1]
                rounded = sum(parts(weights.float()))
                got = ((rounded @ v[b, g].double()) / p.sum(1, keepdim=True)).to(dtype)
                most = max(most, float(((got.double() - want).abs() / bound).max()))
        return most

    def pair(w):
        first = w.bfloat16().float()
        return first.double(), (w - first).bfloat16().double()

    assert worst(lambda w: [w.to(dtype).double()]) > 1 and worst(pair) <= 1
