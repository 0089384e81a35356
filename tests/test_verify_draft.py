"""verify_draft against the walk written out in float64, node by node.

Whole numbers have to be equal. The kernel and the oracle add the same float64 weights in another
order, so they could disagree only where a cumulative sum lies within about 10^-15 of the goal;
the inputs are continuous draws (or exact binary fractions, whose sums are exact in any order).
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from tklab.kernels.verify_draft import chunk_length, verify_draft

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _oracle(target, tokens, uniforms, parents=None, draft=None):
    """(path, count, next_token) as lists, from the definition."""
    batch, nodes, vocabulary = target.shape

    def row(t, b, i):
        p = t[b, i].double().cpu()
        return torch.where((p > 0) & (p < math.inf), p, torch.zeros(()).double())

    tokens, uniforms = tokens.tolist(), uniforms.double().cpu().tolist()
    if parents is None:
        up = [list(range(-1, nodes - 1))] * batch
    else:
        up = parents.expand(batch, nodes).tolist()
    paths, counts, drawn = [], [], []
    for b in range(batch):
        path, weights = [0], row(target, b, 0)
        while True:
            node = path[-1]
            p = row(target, b, node)
            weights, mass, gone = p.clone(), 1.0, set()
            kept = None
            for i in range(node + 1, nodes):
                token = tokens[b][i]
                if up[b][i] != node or not 0 <= token < vocabulary:
                    continue
                if draft is not None:
                    q = row(draft, b, i - 1)
                    if uniforms[b][i] * float(q[token]) < float(p[token]):
                        kept = i
                    else:
                        weights = (p - q).clamp(min=0)
                elif token not in gone:
                    if uniforms[b][i] * mass < float(p[token]):
                        kept = i
                    else:
                        mass = max(mass - float(p[token]), 0.0)
                        gone.add(token)
                        weights[token] = 0
                if kept is not None:
                    break
            if kept is None:
                break
            path.append(kept)
        if not float(weights.sum()) > 0:
            weights = row(target, b, path[-1])
        sums = weights.cumsum(0)
        u = uniforms[b][0]
        u = min(max(u, 0.0), 1 - 2.0 ** -53) if u == u else 0.0
        if not float(sums[-1]) > 0:
            token = -1
        else:
            past = (sums > u * sums[-1]) & (weights > 0)
            token = int(past.to(torch.int8).argmax()) if bool(past.any()) else int(weights.nonzero()[-1])
        paths.append(path + [-1] * (nodes - len(path)))
        counts.append(len(path))
        drawn.append(token)
    return paths, counts, drawn


def _check(target, tokens, uniforms, **kwargs):
    path, count, token = verify_draft(target, tokens, uniforms, **kwargs)
    assert (path.dtype, count.dtype, token.dtype) == (torch.int32, torch.int32, torch.int64)
    draft, parents = kwargs.get("draft_probs"), kwargs.get("parents")
    expected = _oracle(target, tokens, uniforms, parents, draft)
    assert (path.tolist(), count.tolist(), token.tolist()) == expected
    return expected


def _problem(batch, nodes, vocabulary, dtype, seed, sampled=False, likely=False):
    gen = torch.Generator("cuda").manual_seed(seed)
    logits = 2 * torch.randn(batch, nodes, vocabulary, generator=gen, device="cuda")
    target = torch.softmax(logits, -1).to(dtype)
    uniforms = torch.rand(batch, nodes, generator=gen, device="cuda")
    tokens = torch.randint(0, vocabulary, (batch, nodes), generator=gen, device="cuda")
    draft = None
    if sampled and nodes > 1:
        noise = torch.randn(batch, nodes - 1, vocabulary, generator=gen, device="cuda")
        draft = torch.softmax(logits[:, :-1] + 0.5 * noise, -1).to(dtype)
        picks = torch.multinomial(draft.float().flatten(0, 1), 1, generator=gen)
        tokens[:, 1:] = picks.reshape(batch, nodes - 1)
    elif likely:
        best = logits.topk(min(4, vocabulary), -1).indices
        pick = torch.randint(0, best.shape[-1], (batch, nodes, 1), generator=gen, device="cuda")
        tokens[:, 1:] = best.gather(2, pick)[:, :-1, 0]
    return target, tokens, uniforms, draft


def _tree(nodes, seed, reach=5):
    rng = random.Random(seed)
    return [-1] + [rng.randint(max(0, i - reach), i - 1) for i in range(1, nodes)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [1, 2, 7, 8, 100, 2047, 2048, 2049, 8193, 32001])
def test_sampled_chains(dtype, vocabulary) -> None:
    target, tokens, uniforms, draft = _problem(9, 6, vocabulary, dtype, vocabulary, sampled=True)
    _check(target, tokens, uniforms, draft_probs=draft)


@pytest.mark.gpu
def test_a_chain_without_drafts_takes_draft_probs_without_rows() -> None:
    target, tokens, uniforms, _ = _problem(3, 1, 500, torch.float32, 11)
    _check(target, tokens, uniforms)
    given = verify_draft(target, tokens, uniforms, draft_probs=target[:, 1:])
    assert all(torch.equal(x, y) for x, y in zip(given, verify_draft(target, tokens, uniforms)))


@pytest.mark.gpu
def test_sampled_chains_end_everywhere() -> None:
    target, tokens, uniforms, draft = _problem(64, 5, 1000, torch.float32, 1, sampled=True)
    _, counts, _ = _check(target, tokens, uniforms, draft_probs=draft)
    assert set(counts) == {1, 2, 3, 4, 5}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nodes", [1, 2, 3, 17, 64, 65, 128, 130, 256])
def test_trees_of_any_size(dtype, nodes) -> None:
    target, tokens, uniforms, _ = _problem(7, nodes, 500, dtype, nodes, likely=True)
    parents = torch.tensor(_tree(nodes, nodes), dtype=torch.int32, device="cuda")
    best = target.float().topk(4, -1).indices
    for i in range(1, nodes):
        tokens[:, i] = best[:, int(parents[i]), i % 4]
    # Small random numbers walk deep: several 64-node groups are passed.
    _check(target, tokens, uniforms * 0.3, parents=parents)
    each = torch.stack([torch.tensor(_tree(nodes, b, 2 + b), dtype=torch.int32) for b in range(7)])
    _check(target, tokens, uniforms, parents=each.cuda())


@pytest.mark.gpu
def test_chains_of_tokens_taken_without_drawing() -> None:
    target, tokens, uniforms, _ = _problem(33, 8, 4000, torch.bfloat16, 2, likely=True)
    _, counts, _ = _check(target, tokens, uniforms * 0.05)
    assert max(counts) > 2
    _check(target, tokens.int(), uniforms)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,vocabulary", [(1, 131072), (1, 262147), (40, 70001)])
def test_many_splits(batch, vocabulary) -> None:
    assert -(-vocabulary // chunk_length(batch, vocabulary)) > 1
    target, tokens, uniforms, draft = _problem(batch, 3, vocabulary, torch.bfloat16, 3, sampled=True)
    _check(target, tokens, uniforms, draft_probs=draft)
    _check(target, tokens, uniforms)


@pytest.mark.gpu
def test_split_rows_longer_than_one_pass_of_the_draw() -> None:
    target, tokens, uniforms, _ = _problem(2, 1, 2 ** 21 + 3, torch.float32, 4)
    assert chunk_length(2, 2 ** 21 + 3) > 3 * 8192
    for u in (0.0, 0.37, 0.999999):
        uniforms[:, 0] = u
        _check(target, tokens, uniforms)


@pytest.mark.gpu
@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, math.nan])
def test_borders_of_exact_weights(u) -> None:
    """Binary fractions add up exactly: the goal can lie on a border, which belongs to the next."""
    target = torch.full((3, 1, 4096), 2.0 ** -12, device="cuda")
    target[1, 0, 1::2] = 0
    target[2, 0] = 0
    target[2, 0, 4000] = 1.0
    uniforms = torch.full((3, 1), u, device="cuda")
    _, _, drawn = _check(target, torch.zeros(3, 1, dtype=torch.int64, device="cuda"), uniforms)
    assert drawn[2] == 4000
    if u == 0.5:
        assert drawn[:2] == [2048, 2048]
    if u >= 1.0:
        assert drawn[:2] == [4095, 4094]


@pytest.mark.gpu
@pytest.mark.parametrize("sampled", [False, True])
def test_entries_that_are_no_probabilities_weigh_nothing(sampled) -> None:
    target, tokens, uniforms, draft = _problem(16, 3, 300, torch.float32, 5, sampled=True)
    target[:, :, 10] = math.nan
    target[:, :, 20] = math.inf
    target[:, :, 30] = -1.0
    target[0] = math.nan
    target[1, 1:] = 0.0
    tokens[2:6, 1] = torch.tensor([10, 20, 30, 299], device="cuda")
    if sampled:
        draft[:, :, 40] = math.nan
        draft[:, :, 50] = math.inf
        tokens[6, 1], tokens[7, 1] = 40, 50
    _, counts, drawn = _check(target, tokens, uniforms, draft_probs=draft if sampled else None)
    assert drawn[0] == -1 and counts[0] == 1


@pytest.mark.gpu
def test_a_rejection_that_leaves_no_mass_draws_from_the_target() -> None:
    """q >= p everywhere (sums above 1 by rounding): a rejected token leaves nothing to draw."""
    target = torch.full((1, 2, 4), 0.25, device="cuda")
    draft = torch.full((1, 1, 4), 0.5, device="cuda")
    tokens = torch.tensor([[0, 2]], device="cuda")
    uniforms = torch.tensor([[0.6, 0.9]], device="cuda")
    expected = _check(target, tokens, uniforms, draft_probs=draft)
    assert expected == ([[0, -1]], [1], [2])
    # The only likely token of a distribution, rejected by a random number of 1 minus a little.
    target = torch.tensor([[[0.0, 0.5, 0.0, 0.0]] * 2], device="cuda")
    expected = _check(target, torch.tensor([[0, 1]], device="cuda"), uniforms)
    assert expected == ([[0, -1]], [1], [1])


@pytest.mark.gpu
def test_repeated_and_absent_siblings_and_unattached_nodes() -> None:
    target = torch.tensor([[[0.1, 0.2, 0.3, 0.4]] * 7], device="cuda")
    parents = torch.tensor([-1, 0, 0, 0, 5, -3, 0], dtype=torch.int32, device="cuda")
    tokens = torch.tensor([[0, 1, 1, -1, 3, 3, 2]], device="cuda")
    for last, seen in ((0.3, [0, 6]), (0.9, [0])):
        uniforms = torch.tensor([[0.5, 0.9, 0.0, 0.0, 0.0, 0.0, last]], device="cuda")
        path, _, _ = _check(target, tokens, uniforms, parents=parents)
        assert [i for i in path[0] if i >= 0] == seen
    tokens[0, 6] = 4  # past the vocabulary
    path, _, _ = _check(target, tokens, uniforms, parents=parents)
    assert path[0][:2] == [0, -1]


@pytest.mark.gpu
def test_shorter_drafts_are_padded_with_tokens_outside_the_vocabulary() -> None:
    target, tokens, uniforms, draft = _problem(6, 5, 64, torch.float16, 6, sampled=True)
    lengths = torch.arange(6, device="cuda").clamp(max=4)[:, None]
    tokens = torch.where(torch.arange(5, device="cuda") > lengths, -1, tokens)
    uniforms[:, 1:] = 0
    _, counts, _ = _check(target, tokens, uniforms, draft_probs=draft)
    assert counts == [1, 2, 3, 4, 5, 5]


@pytest.mark.gpu
def test_strided_inputs() -> None:
    """Rows inside wider tensors, at any element boundary, and one target for every sequence."""
    gen = torch.Generator("cuda").manual_seed(7)
    wide = torch.softmax(torch.randn(10, 8, 1203, generator=gen, device="cuda"), -1).to(torch.bfloat16)
    target, draft = wide[::2, 1:6, 1:1002], wide[1::2, 3:7, 5:1006]
    tokens = torch.randint(0, 1001, (5, 9), generator=gen, device="cuda")[:, 2:7]
    uniforms = torch.rand(5, 11, generator=gen, device="cuda")[:, 3:8]
    _check(target, tokens, uniforms, draft_probs=draft)
    shared = target[:1].expand(5, 5, 1001)
    parents = torch.tensor(_tree(5, 8), dtype=torch.int32, device="cuda").expand(5, 5)
    _check(shared, tokens, uniforms, parents=parents)


@pytest.mark.gpu
def test_offsets_past_32_bits() -> None:
    storage = torch.zeros(2 ** 31 + 4096, dtype=torch.float16, device="cuda")
    target = storage.as_strided((2, 2, 1000), (2 ** 31, 1000, 1))
    small, tokens, uniforms, _ = _problem(2, 2, 1000, torch.float16, 8, likely=True)
    target.copy_(small)
    _check(target, tokens, uniforms)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 40])
def test_the_last_entry_of_the_longest_row(batch) -> None:
    """The last share's end, counted from its start in whole shares, lies past 32 bits."""
    vocabulary = 2 ** 31 - 65537
    row = torch.zeros(vocabulary, dtype=torch.float16, device="cuda")
    row[-1] = 0.5
    target = row.expand(batch, 1, vocabulary)
    tokens = torch.zeros(batch, 1, dtype=torch.int64, device="cuda")
    path, count, token = verify_draft(target, tokens, torch.full((batch, 1), 0.5, device="cuda"))
    assert bool((token == vocabulary - 1).all())
    assert bool((path == 0).all()) and bool((count == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("sampled", [False, True])
def test_what_comes_out_is_distributed_like_the_target(sampled) -> None:
    """Over a grid of random numbers, the first token that comes out follows p: each of its
    border lines in the unit square crosses at most 2 * 128 cells of 128^2 per node and token."""
    steps, p = 128, torch.tensor([0.1, 0.2, 0.3, 0.4], device="cuda")
    q = torch.tensor([0.4, 0.3, 0.2, 0.1], device="cuda")
    centre = (torch.arange(steps, device="cuda") + 0.5) / steps
    u = torch.cartesian_prod(centre, centre)
    total = torch.zeros(4, dtype=torch.float64)
    for x in range(4):
        n = len(u)
        tokens = torch.tensor([0, x], device="cuda").expand(n, 2)
        target = p.expand(n, 2, 4)
        draft = q.expand(n, 1, 4) if sampled else None
        _, count, token = verify_draft(target, tokens, u.contiguous(), draft_probs=draft)
        first = torch.where(count > 1, x, token).cpu()
        share = torch.bincount(first, minlength=4).double() / n
        total += share * (float(q[x]) if sampled else 0.25)
    assert bool(((total - p.cpu().double()).abs() < 4 * 2 / steps).all())


@pytest.mark.gpu
def test_a_captured_call_replays_on_another_stream() -> None:
    target, tokens, uniforms, draft = _problem(4, 4, 5000, torch.float32, 9, sampled=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        verify_draft(target, tokens, uniforms, draft_probs=draft)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = verify_draft(target, tokens, uniforms, draft_probs=draft)
    torch.cuda.synchronize()
    for step in range(4):
        uniforms.copy_(torch.rand(4, 4, generator=torch.Generator().manual_seed(step)))
        eager = verify_draft(target, tokens, uniforms, draft_probs=draft)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


# ------------------------------------------------------------------ without a GPU


def _meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("change,message", [
    (dict(target_probs=_meta(2, 100)), "expects"),
    (dict(target_probs=_meta(2, 0, 100)), "empty"),
    (dict(target_probs=_meta(2, 257, 100)), "at most 256"),
    (dict(target_probs=_meta(65536, 4, 100)), "65535"),
    (dict(target_probs=_meta(2, 4, 100, dtype=torch.float64)), "float16"),
    (dict(draft_tokens=_meta(2, 3, dtype=torch.int64)), "draft_tokens"),
    (dict(draft_tokens=_meta(2, 4)), "draft_tokens"),
    (dict(uniforms=_meta(2, 3)), "uniforms"),
    (dict(uniforms=_meta(2, 4, dtype=torch.float64)), "uniforms"),
    (dict(parents=_meta(3, dtype=torch.int32), draft_probs=None), "parents"),
    (dict(parents=_meta(4, dtype=torch.int64), draft_probs=None), "parents"),
    (dict(parents=_meta(4, dtype=torch.int32)), "chain"),
    (dict(draft_probs=_meta(2, 4, 100)), "draft_probs"),
    (dict(draft_probs=_meta(2, 3, 100, dtype=torch.float16)), "draft_probs"),
    (dict(), "requires CUDA"),
])
def test_refusals(change, message) -> None:
    args = dict(target_probs=_meta(2, 4, 100), draft_tokens=_meta(2, 4, dtype=torch.int64),
                uniforms=_meta(2, 4), parents=None, draft_probs=_meta(2, 3, 100))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        verify_draft(args["target_probs"], args["draft_tokens"], args["uniforms"],
                     parents=args["parents"], draft_probs=args["draft_probs"])


@pytest.mark.gpu
def test_refuses_rows_without_a_unit_stride() -> None:
    target = torch.zeros(2, 10, 4, device="cuda").transpose(1, 2)
    tokens = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="contiguous final"):
        verify_draft(target, tokens, torch.zeros(2, 4, device="cuda"))


def test_chunks_cover_the_row_in_at_most_64_splits() -> None:
    for batch in (1, 3, 64, 65535):
        for vocabulary in (1, 2048, 2049, 131072, 2 ** 31 - 65537):
            chunk = chunk_length(batch, vocabulary)
            assert chunk % 8 == 0 and -(-vocabulary // chunk) <= 64


def test_shares_stay_within_what_the_library_counts() -> None:
    for batch in (1, 40, 1024, 65535):
        assert chunk_length(batch, 2 ** 31 - 65537) <= 2 ** 30
