"""One layer's speculative decoding, the operators one after the other as a program uses them.

A target of one attention layer decodes drafted trees step by step: projections, rotary positions
by depth, tree attention over the cache and the tree, output head, softmax, verification, and the
accepted nodes' move into the cache. Each step is compared with the same step in float64 from the
same cache and the same drafts; at the end the cache holds exactly the keys and values of the
tokens that came out.
"""

from __future__ import annotations

import pytest
import torch

from tklab.kernels.commit_draft import commit_draft
from tklab.kernels.fused_softmax import softmax
from tklab.kernels.gqa_decode import gqa_decode
from tklab.kernels.matmul import matmul_fp32acc
from tklab.kernels.rotary import rotary_embedding, rotary_frequencies
from tklab.kernels.tree_decode import tree_decode, tree_mask
from tklab.kernels.verify_draft import verify_draft

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, DIM, VOCABULARY, MAX_LEN = 256, 8, 2, 64, 512, 96
PARENTS = [-1, 0, 0, 0, 1, 1, 2, 4, 4]


class _Layer:
    """Weights of a one-layer target; the residual stream is the token's embedding."""

    def __init__(self, seed, dtype=torch.bfloat16):
        gen = torch.Generator("cuda").manual_seed(seed)

        def weight(n, k, std):
            return (torch.randn(n, k, generator=gen, device="cuda") * std).to(dtype)

        self.embedding = weight(VOCABULARY, HIDDEN, 1.0)
        self.qkv = weight(HIDDEN, (HEADS + 2 * KV) * DIM, HIDDEN ** -0.5)
        self.head = weight(HEADS * DIM, VOCABULARY, 0.3)
        self.frequencies, self.magnitude = rotary_frequencies(DIM // 2, scaling="linear", factor=2.0,
                                                              device="cuda")

    def project(self, tokens, positions):
        """Rotated q and k, and v, of [batch, n] tokens, head-major."""
        batch, n = tokens.shape
        x = self.embedding[tokens].reshape(batch * n, HIDDEN)
        joint = matmul_fp32acc(x, self.qkv).reshape(batch, n, HEADS + 2 * KV, DIM).transpose(1, 2)
        q, k, v = joint.split((HEADS, KV, KV), 1)
        q, k = rotary_embedding(q, k, positions, self.frequencies, interleaved=True,
                                magnitude=self.magnitude)
        return q, k, v

    def probabilities(self, attended):
        """[batch, heads, n, dim] attention outputs -> [batch, n, vocabulary]."""
        batch, _, n, _ = attended.shape
        rows = attended.transpose(1, 2).reshape(batch * n, HEADS * DIM)
        return softmax(matmul_fp32acc(rows, self.head)).reshape(batch, n, VOCABULARY)


def _attend64(q, k, v, sees):
    group = HEADS // KV
    k, v = (t.double().repeat_interleave(group, 1) for t in (k, v))
    scores = torch.matmul(q.double(), k.transpose(2, 3).contiguous()) * DIM ** -0.5
    return torch.matmul(scores.masked_fill(~sees[:, None], -torch.inf).softmax(-1), v)


@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_steps_of_speculative_decoding(kind) -> None:
    layer, gen = _Layer(1), torch.Generator("cuda").manual_seed(2)
    batch = 3
    parents = PARENTS if kind == "tree" else list(range(-1, 8))
    nodes = len(parents)
    up = torch.tensor(parents, dtype=torch.int32, device="cuda")
    mask = tree_mask(up)
    depth = mask.sum(1) - 1
    k_cache, v_cache = (torch.full((batch, KV, MAX_LEN, DIM), torch.nan, dtype=torch.bfloat16, device="cuda")
                        for _ in "kv")
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    last = torch.randint(0, VOCABULARY, (batch,), generator=gen, device="cuda")
    out = [[] for _ in range(batch)]
    accepted = 0
    for _ in range(6):
        tokens = torch.randint(0, VOCABULARY, (batch, nodes), generator=gen, device="cuda")
        tokens[:, 0] = last
        # Draft what the target itself finds likely behind each node, so that some is accepted.
        for i in range(1, nodes):
            path = [j for j in range(i) if mask[parents[i], j]]
            q, k, v = layer.project(tokens[:, path], lengths[:, None] + depth[path])
            p = layer.probabilities(tree_decode(q, k_cache, v_cache, k, v, tree_mask(torch.arange(
                -1, len(path) - 1, device="cuda")), lengths))
            tokens[:, i] = p[:, -1].topk(3, -1).indices[:, i % 3]
        q, k, v = layer.project(tokens, lengths[:, None] + depth)
        attended, lse = tree_decode(q, k_cache, v_cache, k, v, mask, lengths, return_lse=True)
        sees = torch.cat(((torch.arange(MAX_LEN, device="cuda") < lengths[:, None])[:, None].expand(
            -1, nodes, -1), mask.expand(batch, nodes, nodes)), 2)
        want = _attend64(q, torch.cat((k_cache.nan_to_num(), k), 2), torch.cat((v_cache.nan_to_num(), v), 2), sees)
        # P and the result are rounded to bfloat16 (2^-8 each) and |v| here stays below 8.
        assert bool(((attended.double() - want).abs() <= 2 * 2.0 ** -8 * 8).all())
        probabilities = layer.probabilities(attended)
        uniforms = torch.rand(batch, nodes, generator=gen, device="cuda")
        path, count, drawn = verify_draft(probabilities, tokens, uniforms,
                                          parents=up if kind == "tree" else None)
        before = lengths
        lengths = commit_draft(k_cache, v_cache, lengths, k, v, path, count)
        assert torch.equal(lengths, before + count)
        for b in range(batch):
            for node in path[b, : int(count[b])].tolist():
                out[b].append(int(tokens[b, node]))
        accepted += int(count.sum()) - batch
        last = drawn
    assert accepted > 0
    # The cache against one pass over the tokens that came out.
    for b in range(batch):
        n = len(out[b])
        assert n == int(lengths[b])
        row = torch.tensor(out[b], device="cuda")[None]
        q, k, v = layer.project(row, torch.arange(n, device="cuda"))
        assert torch.equal(k_cache[b: b + 1, :, :n], k) and torch.equal(v_cache[b: b + 1, :, :n], v)
        assert bool(k_cache[b, :, n:].isnan().all()) and bool(v_cache[b, :, n:].isnan().all())
        # The last token's attention, as the one-token decode computes it.
        one = gqa_decode(q[:, :, -1].contiguous(), k_cache[b: b + 1], v_cache[b: b + 1], lengths[b: b + 1])
        want = _attend64(q[:, :, -1:], k, v, torch.ones(1, 1, n, dtype=torch.bool, device="cuda"))
        assert bool(((one.double() - want[:, :, 0]).abs() <= 2 * 2.0 ** -8 * 8).all())


def test_a_training_step_through_rotary_positions_and_attention() -> None:
    """Rotation of part of the head under grouped-query attention: gradients against float64's."""
    from tklab.kernels.flash_attention import grouped_query_attention

    gen = torch.Generator("cuda").manual_seed(3)
    q, k, v = (torch.randn(2, h, 70, 64, generator=gen, device="cuda").bfloat16().requires_grad_()
               for h in (8, 2, 2))
    freq, magnitude = rotary_frequencies(32, scaling="yarn", factor=4.0, original_length=64, device="cuda")
    pos = torch.arange(70, device="cuda")
    dout = torch.randn(2, 8, 70, 64, generator=gen, device="cuda").bfloat16()
    q_turned, k_turned = rotary_embedding(q, k, pos, freq, magnitude=magnitude)
    out = grouped_query_attention(q_turned, k_turned, v, causal=True)
    grads = torch.autograd.grad(out, (q, k, v), dout)

    leaves = [t.detach().cpu().double().requires_grad_() for t in (q, k, v)]
    angle = pos.cpu().double()[:, None] * freq.cpu()
    c, s = magnitude * angle.cos(), magnitude * angle.sin()

    def turn(x):
        a, b = x[..., :16], x[..., 16:32]
        return torch.cat((a * c - b * s, b * c + a * s, x[..., 32:]), -1)

    rows = torch.ones(70, 70, dtype=torch.bool).tril()
    keys, values = (t.repeat_interleave(4, 1) for t in (turn(leaves[1]), leaves[2]))
    scores = (turn(leaves[0]) @ keys.transpose(2, 3) * 64 ** -0.5).masked_fill(~rows, -torch.inf)
    want = torch.autograd.grad(scores.softmax(-1) @ values, leaves, dout.cpu().double())
    for got, ref in zip(grads, want):
        # A handful of bfloat16 roundings on the way (q, k, P, dS, the gradient), 2^-8 each at most.
        assert float((got.cpu().double() - ref).norm() / ref.norm()) <= 5 * 2.0 ** -8
