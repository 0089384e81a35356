"""A layer of a serving batch, step by step through the operators as a program uses them.

Prompts of different lengths join an 8-bit cache; then every step norms and turns the new token's queries
and keys, appends its key and value, and attends, over the quantised cache or over a shared prefix and
the sequence's own 16-bit cache. Each step is compared with the same step in float64 from the same
projections: the norm and the rotation are formed there again, the quantised cache is read back (its own
tests say how near it is to what was appended).
"""

from __future__ import annotations

import pytest
import torch

from tklab.kernels.commit_draft import commit_draft
from tklab.kernels.matmul import matmul_fp32acc
from tklab.kernels.prefix_decode import prefix_decode
from tklab.kernels.qk_norm_rotary import qk_norm_rotary
from tklab.kernels.quantized_cache import append_quantized, read_quantized
from tklab.kernels.quantized_decode import quantized_decode
from tklab.kernels.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, BATCH, MAX_LEN, EPS = 256, 8, 2, 64, 5, 160, 1e-5
DTYPE = torch.bfloat16


class _Layer:
    def __init__(self, seed):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.qkv = (torch.randn(HIDDEN, (HEADS + 2 * KV) * DIM, generator=gen, device="cuda") * HIDDEN ** -0.5).to(DTYPE)
        self.q_weight, self.k_weight = ((1 + 0.3 * torch.randn(DIM, generator=gen, device="cuda")).to(DTYPE)
                                        for _ in "qk")
        self.frequencies, _ = rotary_frequencies(DIM // 2, device="cuda")

    def project(self, x, positions):
        """[batch, tokens, hidden] -> normed and turned q and k, and v, head-major; and the raw q and k."""
        batch, tokens, _ = x.shape
        joint = matmul_fp32acc(x.reshape(batch * tokens, HIDDEN), self.qkv)
        joint = joint.reshape(batch, tokens, HEADS + 2 * KV, DIM).transpose(1, 2)
        q, k, v = joint.split((HEADS, KV, KV), 1)
        turned = qk_norm_rotary(q, k, self.q_weight, self.k_weight, positions, self.frequencies, eps=EPS)
        for got, raw, w in zip(turned, (q, k), (self.q_weight, self.k_weight)):
            self._check(got, raw, w, positions)
        return *turned, v

    def _check(self, got, x, w, positions):
        z = x.double()
        z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS) * w.double()
        half = DIM // 4
        angle = (positions.double()[..., None] * self.frequencies).unsqueeze(1)
        a, b = z[..., :half], z[..., half: 2 * half]
        want = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), z[..., 2 * half:]), -1)
        # Half a step of bfloat16, and float32's errors (below 2^-17 of the pair).
        size = torch.cat((a.abs() + b.abs(), a.abs() + b.abs(), z[..., 2 * half:].abs()), -1)
        assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -16 * size).all())


def _attend64(q, keys, values):
    """[heads, dim] over [kv, n, dim]."""
    x = q.double().reshape(KV, HEADS // KV, DIM)
    p = (x @ keys.double().transpose(1, 2).contiguous() * DIM ** -0.5).softmax(-1)
    out = p @ values.double()
    spread = p @ values.double().abs()
    return out.reshape(HEADS, DIM), spread.reshape(HEADS, DIM)


def _close(got, want, spread):
    # The weights' and the result's rounding, 2^-8 each of what they round, and float32's errors.
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * (1.01 * spread + want.abs()) + 2.0 ** -14 * spread).all())


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
def test_prompts_and_answers_over_a_quantised_cache(kind) -> None:
    layer, gen = _Layer(1), torch.Generator("cuda").manual_seed(2)
    k_cache, v_cache = (torch.full((BATCH, KV, MAX_LEN, DIM), 0x7F, dtype=torch.uint8, device="cuda").view(kind)
                        for _ in "kv")
    scales = torch.full((BATCH, KV, MAX_LEN, 2), torch.nan, device="cuda")
    lengths = torch.zeros(BATCH, dtype=torch.int32, device="cuda")
    prompts = torch.tensor([150, 1, 0, 37, 64], dtype=torch.int32, device="cuda")
    tokens = int(prompts.max())
    x = torch.randn(BATCH, tokens, HIDDEN, generator=gen, device="cuda").to(DTYPE)
    _, k, v = layer.project(x, torch.arange(tokens, device="cuda").expand(BATCH, tokens))
    lengths = append_quantized(k_cache, v_cache, scales, lengths, k, v, prompts)
    assert torch.equal(lengths, prompts)
    held = read_quantized(k_cache, v_cache, scales, lengths, dtype=torch.float32)
    step = 2.0 ** -4 if kind == torch.float8_e4m3fn else 0.5 / 127
    for back, kept in zip(held, (k, v)):
        for b, n in enumerate(prompts.tolist()):
            most = kept[b, :, :n].float().abs().amax(-1, keepdim=True)
            # e4m3 is off by 2^-4 of a value, or, where steps end, by 2^-10 of scale = most / 448.
            size = kept[b, :, :n].float().abs() + most / 448 if kind == torch.float8_e4m3fn else most
            assert bool(((back[b, :, :n] - kept[b, :, :n].float()).abs() <= 1.001 * step * size).all())
            assert not back[b, :, n:].any()
    for _ in range(12):  # the first sequence fills its cache and stays there
        x = torch.randn(BATCH, 1, HIDDEN, generator=gen, device="cuda").to(DTYPE)
        q, k, v = layer.project(x, lengths[:, None])
        lengths = append_quantized(k_cache, v_cache, scales, lengths, k, v)
        out = quantized_decode(q[:, :, 0], k_cache, v_cache, scales, lengths)
        keys, values = read_quantized(k_cache, v_cache, scales, lengths, dtype=torch.float32)
        for b, n in enumerate(lengths.tolist()):
            _close(out[b], *_attend64(q[b, :, 0], keys[b, :, :n], values[b, :, :n]))
    assert lengths.tolist() == [160, 13, 12, 49, 76]


def test_answers_behind_a_shared_prefix() -> None:
    layer, gen = _Layer(3), torch.Generator("cuda").manual_seed(4)
    prefix = 203
    x = torch.randn(1, prefix, HIDDEN, generator=gen, device="cuda").to(DTYPE)
    _, k, v = layer.project(x, torch.arange(prefix, device="cuda")[None])
    # The prefix lies in a buffer with room behind it.
    k_room, v_room = (torch.full((KV, 256, DIM), torch.nan, dtype=DTYPE, device="cuda") for _ in "kv")
    k_room[:, :prefix], v_room[:, :prefix] = k[0], v[0]
    k_cache, v_cache = (torch.full((BATCH, KV, 20, DIM), torch.nan, dtype=DTYPE, device="cuda") for _ in "kv")
    lengths = torch.tensor([0, 3, 0, 1, 0], dtype=torch.int32, device="cuda")
    for cache in (k_cache, v_cache):
        cache[1, :, :3] = torch.randn(KV, 3, DIM, generator=gen, device="cuda").to(DTYPE)
        cache[3, :, :1] = torch.randn(KV, 1, DIM, generator=gen, device="cuda").to(DTYPE)
    one = torch.ones(BATCH, dtype=torch.int32, device="cuda")
    for _ in range(10):
        x = torch.randn(BATCH, 1, HIDDEN, generator=gen, device="cuda").to(DTYPE)
        q, k, v = layer.project(x, prefix + lengths[:, None])
        lengths = commit_draft(k_cache, v_cache, lengths, k, v, torch.zeros_like(one)[:, None], one)
        out = prefix_decode(q[:, :, 0], k_room[:, :prefix], v_room[:, :prefix], k_cache, v_cache, lengths)
        for b, n in enumerate(lengths.tolist()):
            keys, values = (torch.cat((room[:, :prefix], cache[b, :, :n]), 1)
                            for room, cache in ((k_room, k_cache), (v_room, v_cache)))
            _close(out[b], *_attend64(q[b, :, 0], keys, values))
    assert lengths.tolist() == [10, 13, 10, 11, 10]


def test_a_captured_step_replays() -> None:
    """Append and attention of one token, captured once and replayed with the lengths on the device."""
    layer, gen = _Layer(5), torch.Generator("cuda").manual_seed(6)
    caches, want = [], []
    for _ in range(2):
        k_cache, v_cache = (torch.zeros((BATCH, KV, MAX_LEN, DIM), dtype=torch.float8_e4m3fn, device="cuda") for _ in "kv")
        caches.append((k_cache, v_cache, torch.zeros(BATCH, KV, MAX_LEN, 2, device="cuda")))
    inputs = [torch.randn(BATCH, 1, HIDDEN, generator=gen, device="cuda").to(DTYPE) for _ in range(5)]
    lengths = torch.tensor([0, 1, 2, 3, 158], dtype=torch.int32, device="cuda")
    at = lengths.clone()

    def step(x, cache, n):
        joint = matmul_fp32acc(x.reshape(BATCH, HIDDEN), layer.qkv).reshape(BATCH, 1, HEADS + 2 * KV, DIM).transpose(1, 2)
        q, k, v = joint.split((HEADS, KV, KV), 1)
        q, k = qk_norm_rotary(q, k, layer.q_weight, layer.k_weight, n[:, None], layer.frequencies, eps=EPS)
        n = append_quantized(*cache, n, k, v)
        return quantized_decode(q[:, :, 0], *cache, n), n

    x, n = inputs[0].clone(), lengths.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step(x, caches[0], n)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out, after = step(x, caches[0], n)
            n.copy_(after)
    torch.cuda.synchronize()
    for t in inputs:
        want, at = step(t, caches[1], at)
        x.copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(n, at)
    assert at.tolist() == [5, 6, 7, 8, 160]


def test_two_batches_on_two_streams_at_once() -> None:
    """Steps of two batches, sent for in turns: each call's workspace is its own."""
    gen = torch.Generator("cuda").manual_seed(7)
    batches = []
    for heads, length in ((8, 3000), (32, 900)):
        cache = [torch.randint(-100, 101, (BATCH, KV, length, DIM), generator=gen, device="cuda", dtype=torch.int8)
                 for _ in "kv"]
        scales = torch.rand(BATCH, KV, length, 2, generator=gen, device="cuda") * 0.02
        prefix = [torch.randn(KV, 4 * length, DIM, generator=gen, device="cuda").to(DTYPE) for _ in "kv"]
        own = [torch.randn(BATCH, KV, length, DIM, generator=gen, device="cuda").to(DTYPE) for _ in "kv"]
        lens = torch.randint(1, length + 1, (BATCH,), generator=gen, device="cuda", dtype=torch.int32)
        queries = [torch.randn(BATCH, heads, DIM, generator=gen, device="cuda").to(DTYPE) for _ in range(8)]
        batches.append((queries, (*cache, scales, lens), (*prefix, *own, lens)))

    def step(batch, i):
        queries, cache, shared = batch
        return (*quantized_decode(queries[i], *cache, return_lse=True), *prefix_decode(queries[i], *shared, return_lse=True))

    want = [[step(batch, i) for i in range(8)] for batch in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    got = [[], []]
    for i in range(8):
        for batch, stream, into in zip(batches, streams, got):
            with torch.cuda.stream(stream):
                into.append(step(batch, i))
    torch.cuda.synchronize()
    for one, other in zip(got, want):
        assert all(torch.equal(x, y) for a, b in zip(one, other) for x, y in zip(a, b))
