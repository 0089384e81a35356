"""tree_decode against attention in float64, its masks, layouts and refusals.

Tolerance. With A = sum_j p_j |v_j| / sum_j p_j: rounding P to the storage dtype moves a result by
at most eps / 2 * A, rounding the result by eps / 2 of it. A score is a float32 sum of head_dim
products, off by delta = (head_dim + 4) 2^-24 scale sum|q k|, which moves the weights' numerator and
denominator by that share each, as does the hardware exponential (2^-22); sums of n keys add
(n + 64) 2^-24. Below 2^-14 a float16 P is a subnormal, off by 2^-25 of the largest P, at most
2^-25 sum|v| in all.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from tklab.kernels.gqa_decode import gqa_decode
from tklab.kernels.tree_decode import tree_decode, tree_mask

HALF = [torch.bfloat16, torch.float16]


def _rows(gen, *shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _problem(batch, heads, kv_heads, nodes, max_len, dim, dtype, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    q = _rows(gen, batch, nodes, heads, dim, dtype=dtype).transpose(1, 2)
    k, v = (_rows(gen, batch, kv_heads, max_len, dim, dtype=dtype) for _ in "kv")
    kt, vt = (_rows(gen, batch, nodes, kv_heads, dim, dtype=dtype).transpose(1, 2) for _ in "kv")
    return q, k, v, kt, vt


def _tree(nodes, seed=0, reach=4):
    rng = random.Random(seed)
    return torch.tensor([-1] + [rng.randint(max(0, i - reach), i - 1) for i in range(1, nodes)])


def _check(q, k, v, kt, vt, mask, lens=None, scale=None):
    out, lse = tree_decode(q, k, v, kt, vt, mask, lens, scale=scale, return_lse=True)
    batch, heads, nodes, dim = q.shape
    assert out.shape == q.shape and out.dtype == q.dtype
    assert lse.shape == (batch, heads, nodes) and lse.dtype == torch.float32
    group, factor = heads // k.shape[1], dim ** -0.5 if scale is None else scale
    half = torch.finfo(q.dtype).eps / 2
    masks = mask.expand(batch, nodes, nodes)
    for b in range(batch):
        n = k.shape[2] if lens is None else min(max(int(lens[b]), 0), k.shape[2])
        sees = torch.cat((torch.ones(nodes, n, dtype=torch.bool, device="cuda"), masks[b]), 1)
        for g in range(k.shape[1]):
            keys = torch.cat((k[b, g, :n], kt[b, g])).double()
            values = torch.cat((v[b, g, :n], vt[b, g])).double()
            used = sees.any(0)
            keys, values, seen = keys[used], values[used], sees[:, used]
            rows = q[b, g * group: (g + 1) * group].double()
            scores = (rows @ keys.t() * factor).masked_fill(~seen, -math.inf)
            sizes = (rows.abs() @ keys.abs().t() * abs(factor)).masked_fill(~seen, 0)
            log = torch.logsumexp(scores, -1, keepdim=True)
            share = torch.exp(scores - log).masked_fill(~seen, 0)
            some = seen.any(-1)[None, :, None]
            want = torch.where(some, share @ values, 0.0)
            spread = share @ values.abs()
            delta = (dim + 4) * 2.0 ** -24 * sizes.amax(-1, keepdim=True) if seen.shape[1] else 0.0
            sums = 2 * delta + 2.0 ** -21 + (seen.shape[1] + 64) * 2.0 ** -24
            bound = spread * (half + sums)
            if q.dtype == torch.float16 and seen.shape[1]:
                bound = bound + 2.0 ** -25 * values.abs().sum(0)
            bound = bound + half * (want.abs() + bound) + 2.0 ** -25
            got = out[b, g * group: (g + 1) * group].double()
            assert bool(((got - want).abs() <= bound).all()), (b, g, float(((got - want).abs() / bound).max()))
            want_lse = (log / math.log(2))[..., 0]
            got_lse = lse[b, g * group: (g + 1) * group].double()
            finite = some[..., 0].expand_as(want_lse)
            off = (got_lse - want_lse).abs()[finite]
            limit = (1.5 * sums + 2.0 ** -22 * (1 + want_lse.abs())[..., None])[..., 0][finite]
            assert bool((off <= limit).all()), float((off - limit).max())
            assert bool(torch.isneginf(got_lse[~finite]).all())
    return out, lse


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nodes,group", [(1, 1), (1, 8), (5, 3), (16, 1), (8, 4), (17, 2), (16, 4),
                                         (33, 3), (32, 4), (43, 3), (64, 4), (64, 5), (64, 8),
                                         (255, 1), (256, 2)])
def test_row_counts_of_every_workgroup_shape(dtype, dim, nodes, group) -> None:
    q, k, v, kt, vt = _problem(2, 2 * group, 2, nodes, 777, dim, dtype, nodes * 10 + group)
    _check(q, k, v, kt, vt, tree_mask(_tree(nodes).cuda()), _ints([777, 130]))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nodes,group", [(3, 4), (8, 8), (40, 8)])
@pytest.mark.parametrize("length", [1, 31, 32, 33, 63, 64, 65, 95, 127, 128, 129, 1000, 4096])
def test_lengths_and_tile_edges(dim, nodes, group, length) -> None:
    q, k, v, kt, vt = _problem(2, 2 * group, 2, nodes, length, dim, torch.bfloat16, length)
    _check(q, k, v, kt, vt, tree_mask(_tree(nodes).cuda()))


@pytest.mark.gpu
def test_ragged_batch_with_empty_clamped_and_full_contexts() -> None:
    q, k, v, kt, vt = _problem(7, 8, 2, 9, 3000, 128, torch.bfloat16, 1)
    lens = _ints([3000, 0, 1, -7, 9999, 1537, 32])
    _check(q, k, v, kt, vt, tree_mask(_tree(9).cuda()), lens)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [65, 130, 300])
def test_batches_past_one_wave_of_lengths(batch) -> None:
    q, k, v, kt, vt = _problem(batch, 2, 1, 3, 700, 64, torch.bfloat16, 2)
    rng = random.Random(batch)
    _check(q, k, v, kt, vt, tree_mask(_tree(3).cuda()), _ints([rng.randint(0, 700) for _ in range(batch)]))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,nodes", [(128, 9), (64, 70)])
def test_whole_and_split_sequences_in_one_batch(dim, nodes) -> None:
    """128 pairs of a sequence and a KV head: up to 40 tiles are one run, longer sequences several."""
    q, k, v, kt, vt = _problem(16, 16, 8, nodes, 2900, dim, torch.bfloat16, 4)
    edge = (40 - -(-nodes // 32)) * 32
    lens = [0, 1, edge - 1, edge, edge + 1, 2900, 33, 640, edge + 32, 1, 2899, 500, edge, 31, 32, 1700]
    _check(q, k, v, kt, vt, tree_mask(_tree(nodes).cuda()), _ints(lens))


@pytest.mark.gpu
@pytest.mark.parametrize("batch,tiles", [(1, 10), (4, 10), (16, 18), (64, 40)])
@pytest.mark.parametrize("more", [0, 1])
def test_caches_at_the_limit_of_unsplit_calls(batch, tiles, more) -> None:
    length = (tiles - 1) * 32 + more
    q, k, v, kt, vt = _problem(batch, 4, 2, 7, length, 64, torch.float16, 5)
    _check(q, k, v, kt, vt, tree_mask(_tree(7).cuda()))


@pytest.mark.gpu
def test_one_long_sequence_among_short_ones() -> None:
    q, k, v, kt, vt = _problem(6, 4, 1, 5, 40000, 64, torch.float16, 3)
    _check(q, k, v, kt, vt, tree_mask(_tree(5).cuda()), _ints([3, 40000, 0, 77, 32, 900]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("nodes,group", [(7, 1), (20, 4), (70, 4)])
def test_random_masks_with_rows_that_see_nothing(dtype, nodes, group) -> None:
    q, k, v, kt, vt = _problem(4, 2 * group, 2, nodes, 200, 128, dtype, 4)
    gen = torch.Generator("cuda").manual_seed(5)
    mask = torch.rand(4, nodes, nodes, generator=gen, device="cuda") < 0.3
    mask[:, 2] = False
    mask[3] = False
    out, lse = _check(q, k, v, kt, vt, mask, _ints([0, 0, 200, 0]))
    assert bool((out[0, :, 2] == 0).all()) and bool((out[3] == 0).all())
    assert bool(torch.isneginf(lse[3]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nodes,group", [(6, 2), (40, 4), (64, 8)])
def test_what_a_node_does_not_see_cannot_reach_it(bad, dtype, dim, nodes, group) -> None:
    """Cache rows past the length and hidden nodes' rows hold infinities or NaN; a node that sees
    a NaN value gets it, its neighbours stay what they were."""
    q, k, v, kt, vt = _problem(2, 2 * group, 2, nodes, 100, dim, dtype, 6)
    mask = tree_mask(_tree(nodes).cuda())
    lens = _ints([77, 0])
    clean, clean_lse = tree_decode(q, k, v, kt, vt, mask, lens, return_lse=True)
    k[0, :, 77:], v[0, :, 77:], k[1], v[1] = bad, bad, bad, bad
    hidden = nodes - 1
    mask = mask.clone()
    mask[:, hidden] = False  # no node sees it, itself included
    kt[:, :, hidden], vt[:, :, hidden, 3] = bad, bad
    out, lse = _check(q, k, v, kt, vt, mask, lens)
    assert bool((lse[:, :, :hidden] == clean_lse[:, :, :hidden]).all())
    # One node sees it: that node's row alone changes.
    kt[:, :, hidden] = 0
    mask[1, hidden] = True
    vt[:, :, hidden] = bad
    got = tree_decode(q, k, v, kt, vt, mask, lens)
    assert not bool(torch.isfinite(got[:, :, 1]).any())
    others = [i for i in range(nodes) if i != 1]
    assert bool(torch.isfinite(got[:, :, others]).all())
    half = torch.finfo(dtype).eps
    near = (got[:, :, others].float() - out[:, :, others].float()).abs()
    assert bool((near <= 2 * half * (out[:, :, others].float().abs() + vt[:, :, :hidden].float().abs().max())).all())


@pytest.mark.gpu
def test_large_scores_and_a_given_scale() -> None:
    q, k, v, kt, vt = _problem(2, 8, 2, 6, 500, 128, torch.float16, 7)
    mask = tree_mask(_tree(6).cuda())
    _check(q * 8, k, v, kt, vt, mask, scale=0.5)
    _check(q, k, v, kt, vt, mask, scale=0.0)
    _check(q, k, v, kt, vt, mask, scale=-0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,group", [(5, 4), (24, 4)])
def test_views(nodes, group) -> None:
    """[batch, max_len, heads, dim] caches, drafted keys and queries out of one joint projection,
    and one context shared by the whole batch."""
    gen = torch.Generator("cuda").manual_seed(8)
    kv, dim, batch = 2, 64, 3
    heads = kv * group
    k, v = (_rows(gen, batch, 300, kv, dim, dtype=torch.bfloat16).transpose(1, 2) for _ in "kv")
    joint = _rows(gen, batch, nodes, (heads + 2 * kv) * dim + 8, dtype=torch.bfloat16)
    cut = [joint[..., a * dim: b * dim].unflatten(-1, (-1, dim)).transpose(1, 2)
           for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv))]
    mask = tree_mask(torch.stack([_tree(nodes, s) for s in range(batch)]).cuda())
    wide = torch.zeros(batch, nodes + 2, 2 * nodes, dtype=torch.bool, device="cuda")
    wide[:, 1: nodes + 1, 3: nodes + 3] = mask
    mask = wide[:, 1: nodes + 1, 3: nodes + 3]
    out, _ = _check(cut[0], k, v, cut[1], cut[2], mask, _ints([300, 0, 41]))
    assert out.transpose(1, 2).is_contiguous()  # the queries' memory order
    shared = [t[:1].expand(batch, kv, 300, dim) for t in (k, v)]
    _check(cut[0], *shared, cut[1], cut[2], mask, _ints([300, 10, 41]))


@pytest.mark.gpu
def test_offsets_past_32_bits() -> None:
    """4100 keys 2^20 elements apart."""
    storage = torch.empty(4100 * 2 ** 20 + 512, dtype=torch.bfloat16, device="cuda")
    k = storage.as_strided((1, 2, 4100, 64), (0, 64, 2 ** 20, 1))
    v = storage[128:].as_strided((1, 2, 4100, 64), (0, 64, 2 ** 20, 1))
    q, kc, vc, kt, vt = _problem(1, 8, 2, 5, 4100, 64, torch.bfloat16, 9)
    k.copy_(kc)
    v.copy_(vc)
    _check(q, k, v, kt, vt, tree_mask(_tree(5).cuda()))


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 4, 8])
def test_one_node_agrees_with_the_one_token_decode(group) -> None:
    q, k, v, kt, vt = _problem(3, 2 * group, 2, 1, 1000, 128, torch.bfloat16, 10)
    lens = _ints([999, 0, 431])
    mask = torch.ones(1, 1, dtype=torch.bool, device="cuda")
    out, lse = _check(q, k, v, kt, vt, mask, lens)
    for b, n in enumerate(lens.tolist()):
        k[b, :, n], v[b, :, n] = kt[b, :, 0], vt[b, :, 0]
    want, want_lse = gqa_decode(q[:, :, 0].contiguous(), k, v, lens + 1, return_lse=True)
    torch.testing.assert_close(out[:, :, 0], want, rtol=2 ** -7, atol=2 ** -8)
    torch.testing.assert_close(lse[:, :, 0], want_lse, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_results_are_bitwise_reproducible() -> None:
    q, k, v, kt, vt = _problem(3, 32, 8, 12, 5000, 128, torch.bfloat16, 11)
    mask, lens = tree_mask(_tree(12).cuda()), _ints([5000, 17, 2500])
    a = tree_decode(q, k, v, kt, vt, mask, lens, return_lse=True)
    b = tree_decode(q, k, v, kt, vt, mask, lens, return_lse=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
def test_captured_calls_replay_with_other_lengths_on_another_stream() -> None:
    q, k, v, kt, vt = _problem(3, 8, 2, 6, 2000, 128, torch.bfloat16, 12)
    mask, lens = tree_mask(_tree(6).cuda()), _ints([1, 2, 3])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        tree_decode(q, k, v, kt, vt, mask, lens)
        stream.synchronize()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(tree_decode(q, k, v, kt, vt, mask, lens, return_lse=True))
            graphs.append(graph)
    torch.cuda.synchronize()
    for values in ([0, 0, 0], [2000, 5, 700], [1, 2000, 2000], [31, 33, 0]):
        lens.copy_(_ints(values))
        eager = tree_decode(q, k, v, kt, vt, mask, lens, return_lse=True)
        torch.cuda.synchronize()
        for graph, out in zip(graphs, outs):
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(x, y) for x, y in zip(out, eager))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-60, 2.0 ** -149, 2.0 ** -103, -(2.0 ** -103), 2.0 ** -100])
@pytest.mark.parametrize("dim,nodes,group", [(64, 6, 2), (128, 6, 2), (128, 40, 4)])
def test_scales_of_nothing_and_next_to_nothing(scale, dim, nodes, group) -> None:
    """Products of 2^100 and a scale that takes them to nothing, or to a handful."""
    q, k, v, kt, vt = _problem(2, 2 * group, 2, nodes, 150, dim, torch.bfloat16, 14)
    far = 2.0 ** 50
    mask = tree_mask(_tree(nodes).cuda())
    mask[nodes - 2] = False
    _check(q * far, k * far, v, kt * far, vt, mask, _ints([150, 0]), scale=scale)


def _single(x, dim):
    """x with an odd stride in a dimension of one entry, which no address uses."""
    strides = list(x.stride())
    assert x.shape[dim] == 1
    strides[dim] = 2 ** 24 + 1027
    return x.as_strided(x.shape, strides)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_strides_of_single_entries_do_not_matter(dim) -> None:
    """One sequence, one head and one node, as slices of wider tensors leave them."""
    mask = torch.ones(1, 1, dtype=torch.bool, device="cuda")
    q, k, v, kt, vt = _problem(1, 4, 1, 1, 70, dim, torch.bfloat16, 15)
    want, want_lse = _check(q, k, v, kt, vt, mask)
    odd = [q, k, v, kt, vt]
    for d in range(3):
        odd = [_single(x, d) if x.shape[d] == 1 else x for x in odd]
    out, lse = _check(*odd, mask)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    q, k, v, kt, vt = _problem(2, 4, 2, 3, 1, dim, torch.float16, 16)
    _check(q, _single(k, 2), _single(v, 2), kt, vt, torch.ones(3, 3, dtype=torch.bool, device="cuda"), _ints([1, 0]))
    # The output's memory order is still the queries'.
    q, k, v, kt, vt = _problem(1, 4, 2, 3, 40, dim, torch.float16, 17)
    out = tree_decode(_single(q, 0), k, v, kt, vt, torch.ones(3, 3, dtype=torch.bool, device="cuda"))
    assert out.stride()[1:] == q.stride()[1:]


def _run_tiles(lengths, max_len, kv_heads, group, nodes, dim):
    """Tiles of a run where one round of workgroups makes at least 8, from the library's plan."""
    from tklab import _hip

    batch = len(lengths)
    slots = _hip.query("tk_tree_decode_slots", batch, kv_heads, group, max_len, nodes, dim)
    runs = slots // kv_heads - batch
    total = sum(-(-n // 32) + -(-nodes // 32) for n in lengths)
    tiles = -(-total // runs)
    assert tiles >= 8
    return tiles


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("dim,nodes,group,lengths,kv_heads,tiles", [
    # 256 rows at head_dim 128: two tiles a step, four steps in LDS.
    (128, 64, 4, [9000], 8, 9),
    (128, 64, 4, [11990], 8, 12),
    (128, 64, 4, [17003], 8, 17),
    (128, 64, 4, [33001], 8, 33),
    # Waves without rows, and a second block with some.
    (128, 33, 4, [20000], 8, 20),
    (128, 48, 3, [14001], 8, 14),
    (128, 65, 4, [9002], 8, 18),
    # Runs that end a sequence, begin in its drafted tiles or hold nothing else.
    (128, 64, 4, [30000, 0, 70000], 1, 13),
    (128, 256, 1, [20001, 31, 40000, 1], 2, 16),
    # The other shapes, past what their rings hold.
    (64, 64, 4, [33001], 8, 17),
    (64, 20, 4, [33001], 8, 17),
    (64, 12, 4, [33001], 8, 17),
    (128, 20, 4, [33001], 8, 17),
    (128, 12, 4, [17003], 8, 9),
    (128, 6, 4, [17003], 8, 9),
    (128, 3, 4, [17003], 8, 9),
])
def test_runs_longer_than_the_ring(dtype, dim, nodes, group, lengths, kv_heads, tiles) -> None:
    """Every slot of the ring in LDS is read, filled again and read again."""
    max_len = max(lengths) + 5
    assert _run_tiles(lengths, max_len, kv_heads, group, nodes, dim) == tiles
    q, k, v, kt, vt = _problem(len(lengths), kv_heads * group, kv_heads, nodes, max_len, dim, dtype, 18)
    k[0, :, lengths[0]:], v[0, :, lengths[0]:] = math.nan, math.nan
    # A key of weight in every tile, so that a stale or missing tile shows.
    v[:, :, ::32] += 4
    _check(q, k, v, kt, vt, tree_mask(_tree(nodes).cuda()), _ints(lengths))


# ------------------------------------------------------------------ without a GPU


def test_tree_mask_names_ancestors() -> None:
    mask = tree_mask(torch.tensor([-1, 0, 0, 1, 3, -1, 9, 2], dtype=torch.int32))
    want = {0: {0}, 1: {0, 1}, 2: {0, 2}, 3: {0, 1, 3}, 4: {0, 1, 3, 4}, 5: {5}, 6: {6}, 7: {0, 2, 7}}
    assert {i: {j for j in range(8) if mask[i, j]} for i in range(8)} == want
    chain = tree_mask(torch.arange(-1, 99))
    assert torch.equal(chain, torch.ones(100, 100, dtype=torch.bool).tril())
    both = tree_mask(torch.tensor([[-1, 0, 1], [-1, 0, 0]]))
    assert both.shape == (2, 3, 3) and bool(both[0, 2, 1]) and not bool(both[1, 2, 1])
    for wrong in (torch.zeros(2, 2, 2, dtype=torch.int32), torch.zeros(3), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="parents"):
            tree_mask(wrong)


@pytest.mark.parametrize("nodes", [1, 2, 3, 31, 100, 256])
def test_tree_mask_is_the_closure_of_the_parents(nodes) -> None:
    gen = torch.Generator().manual_seed(nodes)
    parents = torch.randint(-2, nodes + 2, (3, nodes), generator=gen, dtype=torch.int32)
    mask = tree_mask(parents)
    for b in range(3):
        for i in range(nodes):
            seen, at = {i}, i
            while 0 <= int(parents[b, at]) < at:
                at = int(parents[b, at])
                seen.add(at)
            assert set(mask[b, i].nonzero().flatten().tolist()) == seen
    assert torch.equal(tree_mask(parents[1]), mask[1])


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("change,message", [
    (dict(q=_meta(2, 8, 64)), "expects"),
    (dict(v_cache=_meta(2, 2, 99, 64)), "identical"),
    (dict(v_tree=_meta(2, 2, 4, 64)), "identical"),
    (dict(k_cache=_meta(3, 2, 100, 64), v_cache=_meta(3, 2, 100, 64)), "disagree"),
    (dict(k_tree=_meta(2, 2, 4, 64), v_tree=_meta(2, 2, 4, 64)), "k_tree and v_tree"),
    (dict(k_cache=_meta(2, 2, 0, 64), v_cache=_meta(2, 2, 0, 64)), "empty"),
    (dict(q=_meta(2, 7, 5, 64)), "multiple of kv_heads"),
    (dict(q=_meta(2, 8, 257, 64), k_tree=_meta(2, 2, 257, 64), v_tree=_meta(2, 2, 257, 64)), "at most 256"),
    (dict(q=_meta(2, 8, 5, 32), k_cache=_meta(2, 2, 100, 32), v_cache=_meta(2, 2, 100, 32),
          k_tree=_meta(2, 2, 5, 32), v_tree=_meta(2, 2, 5, 32)), "head_dim 64"),
    (dict(q=_meta(2, 8, 5, 64, dtype=torch.float32)), "share"),
    (dict(v_tree=_meta(2, 2, 5, 64, dtype=torch.float16)), "share"),
    (dict(mask=_meta(5, 5, dtype=torch.uint8)), "mask must be a bool"),
    (dict(mask=_meta(1, 5, 5, dtype=torch.bool)), "mask must be a bool"),
    (dict(scale=math.nan), "scale must be"),
    (dict(scale=-math.inf), "scale must be"),
    (dict(scale=1e300), "scale must be"),
    (dict(), "requires CUDA"),
])
def test_refusals(change, message) -> None:
    args = dict(q=_meta(2, 8, 5, 64), k_cache=_meta(2, 2, 100, 64), v_cache=_meta(2, 2, 100, 64),
                k_tree=_meta(2, 2, 5, 64), v_tree=_meta(2, 2, 5, 64), mask=_meta(5, 5, dtype=torch.bool))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        tree_decode(**args)


@pytest.mark.gpu
def test_refuses_layouts_the_kernel_cannot_read() -> None:
    q, k, v, kt, vt = _problem(2, 4, 2, 4, 50, 64, torch.bfloat16, 13)
    mask = torch.ones(4, 4, dtype=torch.bool, device="cuda")
    with pytest.raises(ValueError, match="aligned"):
        tree_decode(q, torch.zeros(2, 2, 50, 65, device="cuda").bfloat16()[..., 1:], v, kt, vt, mask)
    with pytest.raises(ValueError, match="contiguous final"):
        tree_decode(q, k.transpose(2, 3).contiguous().transpose(2, 3), v, kt, vt, mask)
    with pytest.raises(ValueError, match="2\\*\\*24"):
        tree_decode(q, torch.empty(2 ** 24 * 49 + 256, device="cuda", dtype=torch.bfloat16).as_strided(
            (2, 2, 50, 64), (64, 128, 2 ** 24, 1)), v, kt, vt, mask)
    with pytest.raises(ValueError, match="mask must be on"):
        tree_decode(q, k, v, kt, vt, torch.ones(4, 8, dtype=torch.bool, device="cuda")[:, ::2])
    with pytest.raises(ValueError, match="cache_seqlens"):
        tree_decode(q, k, v, kt, vt, mask, torch.zeros(2, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("sizes", [
    (65535, 128, 1, 32, 1, 64),        # 2^23 workgroups
    (1, 1, 1, 64, 257, 64),            # nodes
    (65536, 1, 1, 64, 1, 64),          # sequences
    (1, 65536, 1, 64, 1, 64),          # heads
    (1, 2, 32768, 64, 1, 64),
    (1, 1, 1, 2 ** 31 - 1, 1, 64),     # positions
    (60000, 1, 1, 2 ** 21, 1, 64),     # tiles in all
    (1, 1, 1, 64, 1, 96),              # head_dim
    (0, 1, 1, 64, 1, 64),
])
def test_sizes_the_library_does_not_take_have_no_plan(sizes) -> None:
    from tklab import _hip

    assert _hip.query("tk_tree_decode_slots", *sizes) == -1


@pytest.mark.gpu
def test_too_many_workgroups_are_a_value_error() -> None:
    def wide(*shape):
        return torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda").expand(shape)

    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="too large"):
        tree_decode(wide(65535, 128, 1, 64), *(wide(65535, 128, 1, 64) for _ in range(4)),
                    torch.ones(1, 1, dtype=torch.bool, device="cuda"))
    assert torch.cuda.memory_allocated() <= before + 4096  # refused before the output is made
