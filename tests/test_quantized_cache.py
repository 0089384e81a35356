"""append_quantized and read_quantized: codes, scales, places, refusals.

Codes are compared bit by bit with the same float32 steps in torch (a reciprocal, two products, a
rounding to nearest even), and with the definition in float64: x and code * scale differ by at most
half a step of the code plus the roundings of these steps and of the scale (4 * 2^-24 of x). A value read back is one float32 product, rounded to its dtype.
"""

from __future__ import annotations

import pytest
import torch

from tklab.kernels.quantized_cache import append_quantized, read_quantized

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
KINDS = [torch.float8_e4m3fn, torch.int8]
MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def _rows(gen, *shape, dtype):
    """Rows whose sizes differ by powers of ten."""
    x = torch.randn(shape, generator=gen, device="cuda")
    size = 10.0 ** torch.randint(-4, 4, (*shape[:-1], 1), generator=gen, device="cuda").float()
    return (x * size).to(dtype)


def _cache(batch, kv, length, dim, kind, fill=3):
    return (*(torch.full((batch, kv, length, dim), fill, dtype=torch.uint8, device="cuda").view(kind) for _ in "kv"),
            torch.full((batch, kv, length, 2), -7.0, device="cuda"))


def _bytes(x):
    return x.view(torch.uint8)


def _encoded(x, kind):
    """Codes as bytes, and scales, of rows in float32."""
    x = x.float()
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    most = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    codes = (x * (most.reciprocal() * MOST[kind])).masked_fill(bad, 0)
    codes = codes.to(kind) if kind == torch.float8_e4m3fn else codes.round().to(kind)
    return _bytes(codes), (most / torch.full_like(most, MOST[kind])).masked_fill(bad, torch.nan)[..., 0]


def _check_append(k_cache, v_cache, scales, lens, k, v, counts=None):
    before = [t.clone() for t in (k_cache, v_cache, scales, lens)]
    got = append_quantized(k_cache, v_cache, scales, lens, k, v, counts)
    max_len, tokens = k_cache.shape[2], k.shape[2]
    want_k, want_v, want_s = _bytes(before[0]).clone(), _bytes(before[1]).clone(), before[2].clone()
    ends = []
    for b in range(k.shape[0]):
        start = min(max(int(lens[b]), 0), max_len)
        n = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        n = min(n, max_len - start)
        ends.append(start + n)
        for i, (want, x) in enumerate(((want_k, k), (want_v, v))):
            codes, scale = _encoded(x[b, :, :n], k_cache.dtype)
            want[b, :, start: start + n] = codes
            want_s[b, :, start: start + n, i] = scale
    assert int((_bytes(k_cache) != want_k).sum()) == 0 and int((_bytes(v_cache) != want_v).sum()) == 0
    assert int((scales.nan_to_num(-1.5) != want_s.nan_to_num(-1.5)).sum()) == 0
    assert got.dtype == torch.int32 and got.tolist() == ends
    assert torch.equal(lens, before[3])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128, 240, 512, 1024])
def test_types_and_head_sizes(kind, dtype, dim) -> None:
    gen = torch.Generator("cuda").manual_seed(1)
    cache = _cache(3, 2, 40, dim, kind)
    k, v = (_rows(gen, 3, 2, 11, dim, dtype=dtype) for _ in "kv")
    _check_append(*cache, torch.tensor([0, 17, 29], dtype=torch.int32, device="cuda"), k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_codes_are_the_nearest(kind) -> None:
    """Against the definition in float64, over values that meet many codes and their borders."""
    gen = torch.Generator("cuda").manual_seed(2)
    x = _rows(gen, 1, 1, 3000, 64, dtype=torch.float32)
    # Rows whose scale is 1 and whose entries lie on halves of the codes' steps.
    steps = torch.arange(64, device="cuda").float()
    x[0, 0, :8, 1:] = (steps[1:] * 0.5 if kind == torch.int8 else (16 + steps[1:] % 16) * 2.0 ** -7)
    x[0, 0, :8, 0] = MOST[kind]
    k_cache, v_cache, scales = _cache(1, 1, 3000, 64, kind)
    append_quantized(k_cache, v_cache, scales, torch.zeros(1, dtype=torch.int32, device="cuda"), x, x)
    assert bool((scales[0, 0, :8] == 1).all())
    scale = scales[..., 0:1].double()
    code = k_cache.double() if kind == torch.float8_e4m3fn else k_cache.to(torch.float64)
    if kind == torch.int8:
        half = torch.full_like(code, 0.5)
    else:
        half = torch.exp2(torch.frexp(x.double().abs() / scale)[1].clamp(min=-5).double() - 5)
    off = (code * scale - x.double()).abs()
    assert bool((off <= half * scale + 4 * 2.0 ** -24 * x.double().abs()).all())
    assert torch.equal(_bytes(k_cache), _bytes(v_cache)) and torch.equal(scales[..., 0], scales[..., 1])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_padded_batches_full_caches_and_lengths_out_of_range(kind) -> None:
    gen = torch.Generator("cuda").manual_seed(3)
    cache = _cache(7, 3, 33, 64, kind)
    k, v = (_rows(gen, 7, 9, 3, 64, dtype=torch.bfloat16).transpose(1, 2) for _ in "kv")
    lens = torch.tensor([0, 33, 30, -4, 100, 24, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    counts = torch.tensor([0, 9, 9, 5, 3, 100, -2 ** 31], dtype=torch.int32, device="cuda")
    _check_append(*cache, lens, k, v, counts)
    _check_append(*cache, lens, k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_zeros_tiny_large_and_not_finite(kind, dtype) -> None:
    gen = torch.Generator("cuda").manual_seed(4)
    x = _rows(gen, 1, 1, 12, 64, dtype=torch.float32)
    info = torch.finfo(dtype)
    x[0, 0, 0] = 0
    x[0, 0, 1] = -0.0
    x[0, 0, 2] *= info.tiny / x[0, 0, 2].abs().amax()
    x[0, 0, 3] *= (info.max / 2) / x[0, 0, 3].abs().amax()
    x[0, 0, 4, 63], x[0, 0, 5, 0], x[0, 0, 6, 31] = torch.inf, -torch.inf, torch.nan
    x[0, 0, 7, :] = torch.nan
    k = x.to(dtype)
    k[0, 0, 8, 5] = info.max
    k[0, 0, 9] = info.smallest_normal * info.eps
    cache = _cache(1, 1, 20, 64, kind)
    lens = torch.tensor([3], dtype=torch.int32, device="cuda")
    _check_append(*cache, lens, k, k.flip(2).contiguous())
    back, _ = read_quantized(*cache, dtype=torch.float32)
    # Rows of numbers give numbers (the fourth row's factor leaves float32 for some types).
    sound = k[0, 0].isfinite().all(-1)
    assert not sound[4:8].any() and bool(sound[[0, 1, 2, 8, 9, 10, 11]].all())
    assert int((back[0, 0, 3: 3 + 12].isnan() != ~sound[:, None]).sum()) == 0
    assert not back[0, 0, 3: 3 + 2].any()


@pytest.mark.gpu
def test_one_token_of_many_sequences_and_many_tokens_of_one() -> None:
    gen = torch.Generator("cuda").manual_seed(5)
    cache = _cache(300, 8, 5, 128, torch.float8_e4m3fn)
    lens = torch.randint(0, 6, (300,), generator=gen, device="cuda", dtype=torch.int32)
    k, v = (_rows(gen, 300, 1, 8, 128, dtype=torch.bfloat16).transpose(1, 2) for _ in "kv")
    _check_append(*cache, lens, k, v)
    cache = _cache(1, 1, 5001, 64, torch.int8)
    k, v = (_rows(gen, 1, 1, 5001, 64, dtype=torch.float16) for _ in "kv")
    _check_append(*cache, torch.zeros(1, dtype=torch.int32, device="cuda"), k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_caches_and_tokens_as_views(kind) -> None:
    """Position-major caches, keys and values as slices of one projection, scales inside another
    tensor; memory around the views stays as it was."""
    gen = torch.Generator("cuda").manual_seed(6)
    batch, kv, dim, tokens = 2, 3, 64, 5
    room = torch.full((2, batch, 20, kv + 1, dim), 9, dtype=torch.uint8, device="cuda")
    k_cache, v_cache = (r[:, :, :kv].transpose(1, 2).view(kind) for r in room)
    inside = torch.full((batch, 20, kv, 6), 5.0, device="cuda")
    scales = inside[..., 2:4].transpose(1, 2)
    joint = _rows(gen, batch, tokens, 2 * kv + 2, dim, dtype=torch.bfloat16)
    k, v = joint[:, :, 1: kv + 1].transpose(1, 2), joint[:, :, kv + 2:].transpose(1, 2)
    assert not k_cache.is_contiguous()
    lens = torch.tensor([16, 4], dtype=torch.int32, device="cuda")
    _check_append(k_cache, v_cache, scales, lens, k, v)
    assert bool((room[:, :, :, kv] == 9).all()) and bool((inside[..., [0, 1, 4, 5]] == 5).all())
    _check_read(k_cache, v_cache, scales, lens, torch.float16)


def _check_read(k_cache, v_cache, scales, lens, dtype):
    got = read_quantized(k_cache, v_cache, scales, lens, dtype=dtype)
    there = torch.ones(k_cache.shape[:3], dtype=torch.bool, device="cuda")
    if lens is not None:
        there &= torch.arange(k_cache.shape[2], device="cuda") < lens[:, None, None]
    for i, (out, cache) in enumerate(zip(got, (k_cache, v_cache))):
        want = (cache.float() * scales[..., i: i + 1]).to(dtype).masked_fill(~there[..., None], 0)
        assert out.is_contiguous() and out.dtype == dtype and out.shape == cache.shape
        assert int((out.float().nan_to_num(1.5, 2.5, -2.5) != want.float().nan_to_num(1.5, 2.5, -2.5)).sum()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 80, 128, 1024])
def test_every_code_read_back(kind, dtype, dim) -> None:
    """Every bit pattern (NaN codes among them), behind scales of both signs and of no number."""
    length = 37
    codes = torch.arange(2 * length * dim, device="cuda").reshape(1, 2, length, dim).remainder(256).to(torch.uint8)
    k_cache, v_cache = codes.view(kind), codes.flip(3).contiguous().view(kind)
    scales = torch.exp2(torch.arange(-37, 37, device="cuda").float() / 4).reshape(1, 1, length, 2).repeat(1, 2, 1, 1)
    scales[0, 0, 5, 0], scales[0, 1, 6, 1], scales[0, 0, 7, 1] = -0.3, torch.nan, 0.0
    _check_read(k_cache, v_cache, scales, None, dtype)
    for n in (0, 1, 36, 100, -3):
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        _check_read(k_cache, v_cache, scales, lens, dtype)
    _check_read(k_cache[:, :, 4:19], v_cache[:, :, 4:19], scales[:, :, 4:19], None, dtype)


@pytest.mark.gpu
def test_what_lies_past_a_length_is_not_read_into_the_result() -> None:
    k_cache, v_cache, scales = _cache(2, 2, 10, 64, torch.float8_e4m3fn, fill=0x7F)
    scales.fill_(torch.nan)
    lens = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    for x in (k_cache, v_cache):
        _bytes(x)[1, :, :3] = 0x38  # 1.0
    scales[1, :, :3] = 2.0
    for out in read_quantized(k_cache, v_cache, scales, lens):
        assert not out[0].any() and bool((out[1, :, :3] == 2).all()) and not out[1, :, 3:].any()


@pytest.mark.gpu
def test_offsets_past_32_bits() -> None:
    gen = torch.Generator("cuda").manual_seed(7)
    far = 2 ** 32 + 4096
    room = torch.zeros(2, far + 4096, dtype=torch.uint8, device="cuda")
    k_cache, v_cache = (r.as_strided((2, 2, 5, 128), (far, 1024, 128, 1)).view(torch.float8_e4m3fn) for r in room)
    scales = torch.zeros(2, 2, 5, 2, device="cuda")
    k, v = (_rows(gen, 2, 2, 3, 128, dtype=torch.bfloat16) for _ in "kv")
    lens = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    _check_append(k_cache, v_cache, scales, lens, k, v)
    _check_read(k_cache, v_cache, scales, lens + 3, torch.bfloat16)


@pytest.mark.gpu
def test_captured_steps_replay_on_another_stream() -> None:
    gen = torch.Generator("cuda").manual_seed(8)
    kind = torch.float8_e4m3fn
    held, eager = _cache(2, 2, 12, 64, kind), _cache(2, 2, 12, 64, kind)
    k, v = (_rows(gen, 2, 2, 1, 64, dtype=torch.bfloat16) for _ in "kv")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        append_quantized(*held, lens, k, v)
        read_quantized(*held, lens)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            lens.copy_(append_quantized(*held, lens, k, v))
            read = read_quantized(*held, lens)
    torch.cuda.synchronize()
    at = torch.zeros(2, dtype=torch.int32, device="cuda")
    for step in range(4):
        k.copy_(_rows(gen, *k.shape, dtype=k.dtype))
        v.copy_(_rows(gen, *v.shape, dtype=v.dtype))
        at = append_quantized(*eager, at, k, v)
        want = read_quantized(*eager, at)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert lens.tolist() == [step + 1] * 2
        assert all(torch.equal(x, y) for x, y in zip(read, want))


# ------------------------------------------------------------------ without a GPU


def _meta(*shape, dtype):
    return torch.empty(shape, dtype=dtype, device="meta")


F8, BF, I32 = torch.float8_e4m3fn, torch.bfloat16, torch.int32


@pytest.mark.parametrize("change,message", [
    (dict(k_cache=_meta(2, 3, 64, dtype=F8)), "expects caches"),
    (dict(v=_meta(2, 4, 4, 64, dtype=BF)), "identical"),
    (dict(k=_meta(2, 4, 5, 64, dtype=BF), v=_meta(2, 4, 5, 64, dtype=BF)), "disagree"),
    (dict(v=_meta(2, 3, 5, 64, dtype=torch.float16)), "share a float16"),
    (dict(v_cache=_meta(2, 3, 11, 64, dtype=F8)), "identical"),
    (dict(v_cache=_meta(2, 3, 10, 64, dtype=torch.int8)), "share a float8"),
    (dict(k_cache=_meta(2, 3, 10, 64, dtype=BF), v_cache=_meta(2, 3, 10, 64, dtype=BF)), "share a float8"),
    (dict(k_cache=_meta(2, 3, 0, 64, dtype=F8), v_cache=_meta(2, 3, 0, 64, dtype=F8)), "empty"),
    (dict(scales=_meta(2, 3, 10, dtype=torch.float32)), "scales must be"),
    (dict(scales=_meta(2, 3, 10, 2, dtype=BF)), "scales must be"),
    (dict(), "requires CUDA"),
])
def test_refused_appends(change, message) -> None:
    args = dict(k_cache=_meta(2, 3, 10, 64, dtype=F8), v_cache=_meta(2, 3, 10, 64, dtype=F8),
                scales=_meta(2, 3, 10, 2, dtype=torch.float32), cache_seqlens=_meta(2, dtype=I32),
                k=_meta(2, 3, 5, 64, dtype=BF), v=_meta(2, 3, 5, 64, dtype=BF))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        append_quantized(**args)


@pytest.mark.parametrize("dim", [8, 72, 1040])
def test_refused_head_sizes(dim) -> None:
    caches = [_meta(2, 3, 10, dim, dtype=F8)] * 2
    scales = _meta(2, 3, 10, 2, dtype=torch.float32)
    with pytest.raises(ValueError, match="multiple of 16"):
        append_quantized(*caches, scales, _meta(2, dtype=I32), *[_meta(2, 3, 5, dim, dtype=BF)] * 2)
    with pytest.raises(ValueError, match="multiple of 16"):
        read_quantized(*caches, scales)


def test_refused_reads() -> None:
    cache, scales = _meta(2, 3, 10, 64, dtype=F8), _meta(2, 3, 10, 2, dtype=torch.float32)
    with pytest.raises(ValueError, match="gives float16"):
        read_quantized(cache, cache, scales, dtype=torch.float64)
    with pytest.raises(ValueError, match="expects caches"):
        read_quantized(cache[0], cache[0], scales)
    with pytest.raises(ValueError, match="requires CUDA"):
        read_quantized(cache, cache, scales)


@pytest.mark.gpu
def test_refused_layouts() -> None:
    k_cache, v_cache, scales = _cache(2, 2, 10, 64, F8)
    lens = torch.zeros(2, dtype=I32, device="cuda")
    k = torch.zeros(2, 2, 5, 64, dtype=BF, device="cuda")
    off = torch.zeros(2 * 2 * 5 * 64 + 1, dtype=BF, device="cuda")[1:].view(2, 2, 5, 64)
    one = scales.new_zeros(2 * 2 * 10 * 2 + 1)[1:].view(2, 2, 10, 2)
    for args, message in [
        ((k_cache, v_cache, scales, lens, off, k), "k rows must be 16-byte"),
        ((k_cache, v_cache, scales, lens, k, k.transpose(2, 3).contiguous().transpose(2, 3)), "v requires a contiguous"),
        ((k_cache, v_cache, one, lens, k, k), "8-byte"),
        ((k_cache, v_cache, scales, lens.long(), k, k), "cache_seqlens must be"),
        ((k_cache, v_cache, scales, lens[:1], k, k), "cache_seqlens must be"),
        ((k_cache, v_cache, scales, lens, k, k, lens.cpu()), "counts must be"),
        ((k_cache[:1].expand(2, 2, 10, 64), v_cache, scales, lens, k, k), "share memory"),
        ((k_cache, v_cache, scales[:, :1].expand(2, 2, 10, 2), lens, k, k), "share memory"),
    ]:
        with pytest.raises(ValueError, match=message):
            append_quantized(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 80)])
def test_many_tokens_of_many_sequences(kind, dtype, dim) -> None:
    """Several tokens a lane: calls of more workgroups than that needs, counts that end inside one."""
    gen = torch.Generator("cuda").manual_seed(9)
    batch, kv, tokens = 9, 5, 1203
    cache = _cache(batch, kv, 1300, dim, kind)
    k, v = (_rows(gen, batch, tokens, kv, dim, dtype=dtype).transpose(1, 2) for _ in "kv")
    lens = torch.tensor([0, 97, 98, 500, 1299, 1300, 3, 64, 1], dtype=torch.int32, device="cuda")
    counts = torch.tensor([1203, 1203, 1203, 7, 9, 9, 0, 1025, 17], dtype=torch.int32, device="cuda")
    _check_append(*cache, lens, k, v, counts)
    _check_append(*cache, lens, k, v)


def test_append_refuses_more_rows_than_a_launch_holds() -> None:
    from tklab.kernels.quantized_cache import _append_plan

    def alike(*shape, dtype):
        x = _meta(*shape, dtype=dtype)
        return x.shape, x.stride(), x.dtype, 0

    def plan(batch, kv, tokens, dim):
        cache = alike(batch, kv, 64, dim, dtype=F8)
        one = alike(batch, kv, tokens, dim, dtype=torch.float32)
        return _append_plan(cache, cache, alike(batch, kv, 64, 2, dtype=torch.float32), alike(batch, dtype=I32), one,
                            one, None)

    assert plan(65535, 1024, 1, 64)[2] == (65535, 1024, 64, 1, 64)
    for sizes in [(65535, 8192, 1, 64), (60000, 1, 60000, 1024), (1, 1, 2 ** 30 + 1, 16), (65535, 65535, 1, 16)]:
        with pytest.raises(ValueError, match="too large"):
            plan(*sizes)
