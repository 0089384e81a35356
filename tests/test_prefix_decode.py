"""prefix_decode against attention in float64 over the prefix and each sequence's own keys.

Tolerance, as for the other decodes. With A = sum_j p_j |v_j| / sum_j p_j: rounding P to the storage
dtype moves a result by at most eps / 2 * A, rounding the result by eps / 2 of it. A score is a float32
sum of head_dim products, off by delta = (head_dim + 4) 2^-24 scale sum|q k|, which moves the weights'
numerator and denominator by that share each, as do the hardware exponential (2^-22) and its argument's
rounding (2^-24 of up to |s| + |m|); sums of n keys add (n + 64) 2^-24. Below 2^-14 a float16 P is a
subnormal, off by 2^-25 of the largest P, at most 2^-25 sum|v| in all.
"""

from __future__ import annotations

import math

import pytest
import torch

from tklab.kernels.gqa_decode import gqa_decode
from tklab.kernels.prefix_decode import prefix_decode

HALF = [torch.bfloat16, torch.float16]


def _problem(batch, heads, kv, prefix, max_len, dim, dtype, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    return (normal(batch, heads, dim), normal(kv, prefix, dim), normal(kv, prefix, dim),
            normal(batch, kv, max_len, dim), normal(batch, kv, max_len, dim))


def _check(q, kp, vp, k, v, lens=None, scale=None, some=None):
    """All sequences, or `some` of them."""
    out, lse = prefix_decode(q, kp, vp, k, v, lens, scale=scale, return_lse=True)
    batch, heads, dim = q.shape
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    assert lse.shape == (batch, heads) and lse.dtype == torch.float32
    group, factor = heads // k.shape[1], dim ** -0.5 if scale is None else scale
    half, info = torch.finfo(q.dtype).eps / 2, torch.finfo(q.dtype)
    for b in range(batch) if some is None else some:
        n = k.shape[2] if lens is None else min(max(int(lens[b]), 0), k.shape[2])
        keys = torch.cat((kp, k[b, :, :n]), 1).double()
        values = torch.cat((vp, v[b, :, :n]), 1).double()
        x = q[b].double().reshape(k.shape[1], group, dim)
        scores = x @ keys.transpose(1, 2).contiguous() * factor
        size = x.abs() @ keys.abs().transpose(1, 2).contiguous() * abs(factor)
        delta = (dim + 4) * 2.0 ** -24 * size.amax(-1, keepdim=True)
        delta = delta + 2.0 ** -22 + 2.0 ** -23 * (scores.abs().amax(-1, keepdim=True) * 1.45 + 8)
        log = torch.logsumexp(scores, -1, keepdim=True)
        p = torch.exp(scores - log)
        want, spread = p @ values, p @ values.abs()
        count = (keys.shape[1] + 64) * 2.0 ** -24
        bound = half * spread + (2 * delta + count) * (spread + want.abs())
        if q.dtype == torch.float16:
            bound = bound + 2.0 ** -25 * values.abs().sum(1, keepdim=True)
        bound = bound + half * (want.abs() + bound) + info.tiny * info.eps
        off = (out[b].double().reshape(want.shape) - want).abs()
        assert bool((off <= bound).all()), float((off / bound).max())
        lse_off = (lse[b].double().reshape(log.shape) - log / math.log(2)).abs()
        lse_bound = (delta + count) * 1.45 + 2.0 ** -22 * (log.abs() * 1.45 + 1)
        assert bool((lse_off <= lse_bound).all()), float((lse_off / lse_bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("batch,heads,kv", [(1, 1, 1), (3, 4, 4), (4, 8, 2), (5, 7, 1), (2, 24, 2), (3, 32, 2),
                                            (8, 34, 2), (1, 64, 1), (3, 100, 1), (20, 12, 2), (33, 8, 2)])
def test_types_heads_and_groups(batch, heads, kv, dtype, dim) -> None:
    """From one row per KV head to several blocks of rows, groups of more than 16 heads."""
    _check(*_problem(batch, heads, kv, 203, 77, dim, dtype, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("batch", [1, 8, 16, 40])
@pytest.mark.parametrize("prefix,max_len", [(1, 1), (1, 200), (31, 32), (32, 33), (33, 1), (129, 128), (160, 31),
                                            (1000, 17), (4100, 300), (20001, 5)])
def test_prefix_and_cache_sizes(prefix, max_len, batch, dtype) -> None:
    _check(*_problem(batch, 4, 2, prefix, max_len, 128, dtype, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("heads", [2, 8, 32])
def test_ragged_lengths_and_lengths_out_of_range(heads, dtype, dim) -> None:
    problem = _problem(9, heads, 2, 500, 700, dim, dtype, 3)
    lens = torch.tensor([0, 1, 31, 32, 33, 699, 700, 5000, -7], dtype=torch.int32, device="cuda")
    _check(*problem, lens)
    _check(*problem, torch.zeros_like(lens))


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [64, 65, 130, 300])
@pytest.mark.parametrize("heads", [1, 4])
def test_more_sequences_than_lanes(batch, heads) -> None:
    problem = _problem(batch, heads, 1, 700, 300, 64, torch.bfloat16, 4)
    gen = torch.Generator("cuda").manual_seed(5)
    lens = torch.randint(0, 301, (batch,), generator=gen, device="cuda", dtype=torch.int32)
    _check(*problem, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch", [2, 16, 64])
def test_long_prefixes(batch, dim) -> None:
    """Runs longer than the ring, one very long own cache among short ones."""
    problem = _problem(batch, 8, 1, 70001, 5000, dim, torch.bfloat16, 6)
    lens = torch.arange(batch, dtype=torch.int32, device="cuda") * 7
    lens[batch // 2] = 5000
    _check(*problem, lens, some=[0, 1, batch // 2, batch - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0, 1e-30])
@pytest.mark.parametrize("dtype", HALF)
def test_score_scales(scale, dtype) -> None:
    problem = _problem(5, 8, 2, 150, 60, 64, dtype, 7)
    _check(*problem, torch.tensor([60, 40, 0, 1, 33], dtype=torch.int32, device="cuda"), scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("batch", [2, 24])
def test_growing_and_falling_scores(batch, dtype) -> None:
    """The running maximum moves at every tile, or is set by the first key; the parts' maxima are far
    apart."""
    q, kp, vp, k, v = _problem(batch, 4, 1, 640, 320, 64, dtype, 8)
    q.copy_(q.abs())
    ramp = torch.linspace(0.01, 4, 640, device="cuda")[:, None]
    for order in (ramp, ramp.flip(0)):
        kp.copy_((kp.float().abs().clamp(0.5, 1) * order).to(dtype))
        k.copy_((k.float().abs().clamp(0.5, 1) * order[::2]).to(dtype))
        _check(q, kp, vp, k, v)
        kp.copy_(torch.randn_like(kp))
        _check(q, kp, vp, k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [3, 24])
def test_what_lies_past_a_length_cannot_reach_a_result(batch) -> None:
    q, kp, vp, k, v = _problem(batch, 8, 2, 300, 100, 128, torch.bfloat16, 9)
    lens = torch.tensor([0, 45, 99], dtype=torch.int32, device="cuda").repeat(batch // 3)
    longer = [torch.full((2, 340, 128), torch.nan, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    for into, x in zip(longer, (kp, vp)):
        into[:, :300] = x
    want = prefix_decode(q, kp, vp, k, v, lens)
    for b, n in enumerate(lens.tolist()):
        k[b, :, n:], v[b, :, n:] = torch.nan, torch.inf
    assert torch.equal(prefix_decode(q, *(x[:, :300] for x in longer), k, v, lens), want)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [2, 24])
def test_a_value_without_a_number_reaches_who_sees_it(batch) -> None:
    q, kp, vp, k, v = _problem(batch, 8, 2, 300, 100, 64, torch.float16, 10)
    want = prefix_decode(q, kp, vp, k, v)
    v[1, 0, 50, 3] = torch.nan
    got = prefix_decode(q, kp, vp, k, v)
    bad = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    bad[1, :4, 3] = True
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad])
    vp[1, 7, 5] = torch.inf
    got = prefix_decode(q, kp, vp, k, v)
    bad[:, 4:, 5] = True
    assert torch.equal(~got.isfinite(), bad) and torch.equal(got[~bad], want[~bad])


@pytest.mark.gpu
def test_is_gqa_decode_of_the_joined_keys() -> None:
    q, kp, vp, k, v = _problem(6, 16, 4, 500, 300, 128, torch.float16, 11)
    joined = [torch.cat((p.expand(6, -1, -1, -1), x), 2) for p, x in ((kp, k), (vp, v))]
    want, want_lse = gqa_decode(q, *joined, return_lse=True)
    got, lse = prefix_decode(q, kp, vp, k, v, return_lse=True)
    # Each rounds its weights and its result to float16.
    assert float((got.float() - want.float()).abs().amax()) <= 4 * 2.0 ** -11 * float(v.abs().float().amax())
    torch.testing.assert_close(lse, want_lse, rtol=1e-5, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [3, 20])
def test_views_of_queries_prefixes_and_caches(batch) -> None:
    gen = torch.Generator("cuda").manual_seed(12)
    q, kp, vp, k, v = _problem(batch, 8, 2, 90, 40, 128, torch.bfloat16, 13)
    want = prefix_decode(q, kp, vp, k, v)
    joint = torch.randn(batch, 12, 128, generator=gen, device="cuda").bfloat16()
    joint[:, 2:10] = q
    kp, vp = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (kp, vp))
    k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    assert not kp.is_contiguous() and not k.is_contiguous()
    assert torch.equal(prefix_decode(joint[:, 2:10], kp, vp, k, v), want)
    # One of everything: strides that address nothing.
    one = q[:1, :1].as_strided((1, 1, 128), (3, 5, 1))
    keys = kp[:1, :1].as_strided((1, 1, 128), (7, 9, 1))
    cache = k[:1, :1, :1].as_strided((1, 1, 1, 128), (3, 5, 7, 1))
    got = prefix_decode(one, keys, keys, cache, cache)
    plain = [x.contiguous() for x in (q[:1, :1], kp[:1, :1], kp[:1, :1], k[:1, :1, :1], k[:1, :1, :1])]
    assert torch.equal(got, prefix_decode(*plain))
    # Sequences that share an own cache.
    shared = [x[:1].expand(batch, -1, -1, -1) for x in (k, v)]
    assert torch.equal(prefix_decode(q, kp, vp, *shared), prefix_decode(q, kp, vp, *(x.contiguous() for x in shared)))


@pytest.mark.gpu
def test_offsets_past_32_bits() -> None:
    q, kp, vp, k, v = _problem(2, 4, 2, 65, 40, 128, torch.bfloat16, 14)
    want = prefix_decode(q, kp, vp, k, v)
    far = 2 ** 31 + 4096
    room = torch.empty(far + 65 * 128, dtype=torch.bfloat16, device="cuda")
    other = torch.empty(far + 65 * 128 + 4096, dtype=torch.bfloat16, device="cuda")
    kp_far, k_far = room.as_strided((2, 65, 128), (far, 128, 1)), other.as_strided((2, 2, 40, 128), (far, 5120, 128, 1))
    kp_far.copy_(kp)
    k_far.copy_(k)
    assert torch.equal(prefix_decode(q, kp_far, vp, k_far, v), want)
    # Positions far apart: 65 rows of 2^23 elements.
    long = torch.empty(2 ** 30, dtype=torch.bfloat16, device="cuda").as_strided((1, 65, 128), (0, 2 ** 23, 1))
    long.copy_(kp[:1])
    got = prefix_decode(q[:, :2], long, vp[:1], k[:, :1], v[:, :1])
    assert torch.equal(got, prefix_decode(q[:, :2], kp[:1], vp[:1], k[:, :1], v[:, :1]))


@pytest.mark.gpu
def test_captured_calls_replay_with_other_lengths_on_another_stream() -> None:
    """Two graphs of one stream, replayed in turn, each with a workspace of its own."""
    problems = [_problem(4, 8, 2, 400, 300, 64, torch.bfloat16, 15), _problem(24, 8, 2, 700, 300, 64, torch.bfloat16, 16)]
    lens = [torch.full((n,), 300, dtype=torch.int32, device="cuda") for n in (4, 24)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, held = [torch.cuda.CUDAGraph() for _ in lens], []
    with torch.cuda.stream(stream):
        for problem, n, graph in zip(problems, lens, graphs):
            prefix_decode(*problem, n)
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                held.append(prefix_decode(*problem, n, return_lse=True))
    torch.cuda.synchronize()
    gen = torch.Generator("cuda").manual_seed(17)
    for most in (301, 40, 1, 301):
        for problem, n in zip(problems, lens):
            n.copy_(torch.randint(0, most, n.shape, generator=gen, device="cuda", dtype=torch.int32))
            problem[0].copy_(problem[0].flip(0).contiguous())
        want = [prefix_decode(*problem, n, return_lse=True) for problem, n in zip(problems, lens)]
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip(held, want):
            assert all(torch.equal(x, y) for x, y in zip(got, expected))


# ------------------------------------------------------------------ without a GPU


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("change,message", [
    (dict(q=_meta(2, 8, 1, 64)), "expects q"),
    (dict(k_prefix=_meta(1, 2, 9, 64)), "expects q"),
    (dict(v_prefix=_meta(2, 8, 64)), "identical"),
    (dict(v_cache=_meta(2, 2, 9, 64)), "identical"),
    (dict(q=_meta(3, 8, 64)), "disagree on batch"),
    (dict(q=_meta(2, 8, 128)), "disagree on batch"),
    (dict(k_prefix=_meta(4, 9, 64), v_prefix=_meta(4, 9, 64)), "disagree on kv_heads"),
    (dict(k_prefix=_meta(2, 0, 64), v_prefix=_meta(2, 0, 64)), "empty"),
    (dict(k_cache=_meta(2, 2, 0, 64), v_cache=_meta(2, 2, 0, 64)), "empty"),
    (dict(q=_meta(2, 7, 64)), "multiple of kv_heads"),
    (dict(q=_meta(2, 65536, 64)), "65535"),
    (dict(q=_meta(2, 8, 64, dtype=torch.float16)), "share a float16"),
    (dict(k_cache=_meta(2, 2, 10, 64, dtype=torch.int8), v_cache=_meta(2, 2, 10, 64, dtype=torch.int8)), "share a float16"),
    (dict(scale=float("nan")), "finite"),
    (dict(), "requires CUDA"),
])
def test_refusals(change, message) -> None:
    args = dict(q=_meta(2, 8, 64), k_prefix=_meta(2, 9, 64), v_prefix=_meta(2, 9, 64), k_cache=_meta(2, 2, 10, 64),
                v_cache=_meta(2, 2, 10, 64))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        prefix_decode(**args)


def test_refused_head_dim() -> None:
    with pytest.raises(ValueError, match="64 and 128"):
        prefix_decode(_meta(2, 8, 96), *[_meta(2, 9, 96)] * 2, *[_meta(2, 2, 10, 96)] * 2)


def test_slots_of_sizes_that_are_not_taken() -> None:
    from tklab import _hip

    assert _hip.query("tk_prefix_decode_slots", 4, 8, 4, 2000, 200, 128) > 0
    for sizes in [(0, 8, 4, 2000, 200, 128), (4, 8, 4, 0, 200, 128), (4, 8, 4, 2000, 200, 96),
                  (70000, 8, 4, 2000, 200, 128), (4, 8, 9000, 2000, 200, 128), (4, 8, 4, 2 ** 31, 200, 128),
                  (60000, 1, 1, 2000, 2 ** 30, 128), (60000, 1, 60000, 200, 200, 128)]:
        assert _hip.query("tk_prefix_decode_slots", *sizes) == -1


@pytest.mark.gpu
def test_refused_layouts() -> None:
    q, kp, vp, k, v = _problem(2, 4, 2, 10, 10, 64, torch.bfloat16, 18)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    odd = torch.zeros(2 * 10 * 68, dtype=torch.bfloat16, device="cuda")
    for args, message in [
        ((q, odd.as_strided((2, 10, 64), (680, 68, 1)), vp, k, v), "k_prefix rows must be 16-byte"),
        ((q, kp, odd[1:].as_strided((2, 10, 64), (640, 64, 1)), k, v), "v_prefix rows must be 16-byte"),
        ((q, kp, vp, k, v.transpose(2, 3).contiguous().transpose(2, 3)), "v_cache requires a contiguous"),
        ((q, kp, vp, k, v, lens.long()), "cache_seqlens must be"),
        ((q, kp, vp, k, v, lens.cpu()), "cache_seqlens must be"),
        ((q, kp.cpu(), vp, k, v), "k_prefix must be on"),
    ]:
        with pytest.raises(ValueError, match=message):
            prefix_decode(*args)


def test_lengths_of_another_batch_are_refused() -> None:
    """One length for several sequences, several for one, on whatever device the check sees."""
    from tklab.kernels.prefix_decode import _plan

    def alike(*shape):
        x = _meta(*shape)
        return x.shape, x.stride(), x.dtype, 0

    def plan(batch, lengths, strides=(1,), dtype=torch.int32, device=0):
        return _plan(*alike(batch, 8, 64), *alike(2, 9, 64), *alike(2, 9, 64), *alike(batch, 2, 10, 64),
                     *alike(batch, 2, 10, 64), ((lengths,), strides, dtype, device))

    assert plan(4, 4)[0] == (4, 8, 64) and plan(1, 1, strides=(7,))[0] == (1, 8, 64)
    for wrong in (dict(batch=4, lengths=1), dict(batch=1, lengths=4), dict(batch=4, lengths=4, strides=(2,)),
                  dict(batch=4, lengths=4, dtype=torch.int64), dict(batch=4, lengths=4, device=1)):
        with pytest.raises(ValueError, match="cache_seqlens must be"):
            plan(**wrong)


# ------------------------------------------------------------------ weights of very different sizes


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [1, 2, 4, 8])
@pytest.mark.parametrize("dtype", HALF)
def test_keys_far_below_keys_without_values(dtype, heads) -> None:
    """Every 512th key has no value and is 17 nats above the others, which are all there is to a result:
    over runs of a thousand keys of the prefix and of the own caches, in each of the workgroups' shapes.

    This module's tolerance, but for float16's subnormals: a weight is held in units of at most 2^-7 of its
    run's largest, so one below 2^-14 of such a unit is off by 2^-32 of the largest weight at most.
    """
    batch, kv, dim = 16, 64, 64
    q, kp, vp, k, v = _problem(batch, heads * kv, kv, 8192, 1024, dim, dtype, 30)
    q[..., 0] = 8
    for keys, values in ((kp, vp), (k, v)):
        keys[..., 0] = 0
        keys[..., 40::512, :] = 0
        keys[..., 40::512, 0] = 17
        values.copy_(values.abs() * 1024)  # of one sign, and results of normal float16 numbers
        values[..., 40::512, :] = 0
    out, lse = prefix_decode(q, kp, vp, k, v, return_lse=True)
    half, info = torch.finfo(dtype).eps / 2, torch.finfo(dtype)
    for b, g in ((0, 0), (7, 21), (15, 63)):
        rows = slice(g * heads, (g + 1) * heads)
        keys, values = torch.cat((kp[g], k[b, g])).double(), torch.cat((vp[g], v[b, g])).double()
        x = q[b, rows].double()
        scores = x @ keys.t() * dim ** -0.5
        delta = (dim + 4) * 2.0 ** -24 * (x.abs() @ keys.abs().t() * dim ** -0.5).amax(1, keepdim=True)
        delta = delta + 2.0 ** -22 + 2.0 ** -23 * (scores.abs().amax(1, keepdim=True) * 1.45 + 8)
        log = torch.logsumexp(scores, 1, keepdim=True)
        p = torch.exp(scores - log)
        want, spread = p @ values, p @ values.abs()
        count = (keys.shape[0] + 64) * 2.0 ** -24
        bound = half * spread + (2 * delta + count) * (spread + want.abs())
        if dtype == torch.float16:
            bound = bound + 2.0 ** -32 * p.amax(1, keepdim=True) * values.abs().sum(0)
        bound = bound + half * (want.abs() + bound) + info.tiny * info.eps
        off = (out[b, rows].double() - want).abs()
        assert bool((off <= bound).all()), float((off / bound).max())
        lse_off = (lse[b, rows].double() - log[:, 0] / math.log(2)).abs()
        lse_bound = (delta[:, 0] + count) * 1.45 + 2.0 ** -22 * (log[:, 0].abs() * 1.45 + 1)
        assert bool((lse_off <= lse_bound).all()), float((lse_off / lse_bound).max())


def test_more_work_than_a_share_counts_is_refused() -> None:
    """Tiles of a workgroup's share are counted in 32 bits: views that repeat positions or heads reach
    sizes at which that would overflow (a prefix of 2^30 keys and 32600 heads), calls of many minutes."""
    from tklab import _hip

    for sizes in [(128, 32600, 1, 2 ** 30, 32, 64), (1, 65535, 1, 2 ** 30, 32, 64), (31, 2040, 1, 32, 2 ** 30, 64),
                  (30, 65535, 1, 33, 2 ** 30, 128), (65535, 16, 64, 2 ** 30, 32, 64)]:
        assert _hip.query("tk_prefix_decode_slots", *sizes) == -1
    for sizes in [(128, 8, 4, 2 ** 30, 32, 64), (31, 8, 4, 32, 2 ** 30, 128), (1, 4096, 1, 2 ** 30, 32, 64)]:
        assert _hip.query("tk_prefix_decode_slots", *sizes) > 0
