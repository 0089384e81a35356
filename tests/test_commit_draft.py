"""commit_draft: the accepted rows land behind each context, everything else stays."""

from __future__ import annotations

import pytest
import torch

from tklab.kernels.commit_draft import commit_draft


def _expected(k, v, lengths, k_tree, v_tree, path, count):
    k, v, ends = k.clone(), v.clone(), []
    max_len, nodes = k.shape[2], k_tree.shape[2]
    for b, (n, c) in enumerate(zip(lengths.tolist(), count.tolist())):
        n, c = min(max(n, 0), max_len), min(max(c, 0), nodes)
        for i, node in enumerate(path[b].tolist()[:c]):
            if n + i < max_len and 0 <= node < nodes:
                k[b, :, n + i], v[b, :, n + i] = k_tree[b, :, node], v_tree[b, :, node]
        ends.append(min(n + c, max_len))
    return k, v, torch.tensor(ends, dtype=torch.int32, device=k.device)


def _check(k, v, lengths, k_tree, v_tree, path, count):
    expected = _expected(k, v, lengths, k_tree, v_tree, path, count)
    before = lengths.clone()
    ends = commit_draft(k, v, lengths, k_tree, v_tree, path, count)
    assert torch.equal(k, expected[0]) and torch.equal(v, expected[1])
    assert torch.equal(ends, expected[2]) and ends.dtype == torch.int32
    assert torch.equal(lengths, before)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _problem(batch, kv_heads, max_len, nodes, dim, dtype, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def rows(n):
        return torch.randn(batch, kv_heads, n, dim, generator=gen, device="cuda").to(dtype)

    return rows(max_len), rows(max_len), rows(nodes), rows(nodes)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 64, 80, 128])
@pytest.mark.parametrize("nodes", [1, 2, 33, 256])
def test_branches_of_any_length(dtype, dim, nodes) -> None:
    k, v, k_tree, v_tree = _problem(4, 3, 600, nodes, dim, dtype, nodes + dim)
    path = torch.argsort(torch.rand(4, nodes, device="cuda"), 1).to(torch.int32)
    count = _ints([0, 1, nodes, (nodes + 1) // 2])
    _check(k, v, _ints([0, 599, 300, 17]), k_tree, v_tree, path, count)


@pytest.mark.gpu
def test_full_caches_and_values_out_of_range() -> None:
    k, v, k_tree, v_tree = _problem(6, 2, 40, 8, 64, torch.bfloat16, 1)
    path = _ints([[0, 2, 5, 7, -1, -1, -1, -1]] * 6)
    path[5] = _ints([0, 8, -1, 3, 2 ** 30, 1, 6, 5])
    _check(k, v, _ints([40, 38, 1000, -5, 36, 10]), k_tree, v_tree, path, _ints([4, 4, 4, 4, -1, 100]))


@pytest.mark.gpu
def test_sequence_major_caches_and_views() -> None:
    """[batch, max_len, kv_heads, dim] caches and the keys of a joint projection, head-major."""
    k, v = (torch.randn(3, 50, 4, 64, device="cuda").half().transpose(1, 2) for _ in "kv")
    joint = torch.randn(3, 6, 2 * 4 * 64 + 8, device="cuda").half()
    k_tree, v_tree = (joint[..., o: o + 256].unflatten(-1, (4, 64)).transpose(1, 2) for o in (8, 264))
    _check(k, v, _ints([0, 10, 44]), k_tree, v_tree, _ints([[0, 1, 3, 5, -1, -1]] * 3), _ints([4, 2, 4]))


@pytest.mark.gpu
def test_offsets_past_32_bits() -> None:
    storage = torch.zeros(2 ** 31 + 2 ** 16, dtype=torch.bfloat16, device="cuda")
    k = storage.as_strided((2, 2, 100, 64), (2 ** 31, 6400, 64, 1))
    v, _, k_tree, v_tree = _problem(2, 2, 100, 4, 64, torch.bfloat16, 2)
    _check(k, v, _ints([5, 90]), k_tree, v_tree, _ints([[0, 1, 3, -1]] * 2), _ints([3, 2]))


@pytest.mark.gpu
def test_a_captured_call_replays() -> None:
    k, v, k_tree, v_tree = _problem(2, 2, 64, 4, 64, torch.bfloat16, 3)
    lengths, count = _ints([3, 7]), _ints([2, 3])
    path = _ints([[0, 2, -1, -1], [0, 1, 3, -1]])
    graph = torch.cuda.CUDAGraph()
    commit_draft(k, v, lengths, k_tree, v_tree, path, count)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ends = commit_draft(k, v, lengths, k_tree, v_tree, path, count)
    for step in range(4):
        k_tree.normal_()
        lengths.add_(step)
        expected = _expected(k, v, lengths, k_tree, v_tree, path, count)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, expected[0]) and torch.equal(v, expected[1])
        assert torch.equal(ends, expected[2])


@pytest.mark.gpu
def test_strides_of_single_entries_do_not_matter() -> None:
    """One sequence, head and node, as slices of wider tensors leave them."""
    k, v, k_tree, v_tree = _problem(1, 1, 20, 1, 64, torch.bfloat16, 5)
    odd = [t.as_strided(t.shape, (1027, 3, 64 if t.shape[2] > 1 else 77, 1)) for t in (k, v, k_tree, v_tree)]
    _check(odd[0], odd[1], _ints([7]), odd[2], odd[3], _ints([[0]]), _ints([1]))


# ------------------------------------------------------------------ without a GPU


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("change,message", [
    (dict(k_cache=_meta(2, 4, 64)), "expects"),
    (dict(v_cache=_meta(2, 4, 99, 64)), "identical"),
    (dict(v_tree=_meta(2, 4, 7, 64)), "identical"),
    (dict(k_tree=_meta(2, 3, 8, 64), v_tree=_meta(2, 3, 8, 64)), "disagree"),
    (dict(k_tree=_meta(2, 4, 0, 64), v_tree=_meta(2, 4, 0, 64)), "empty"),
    (dict(k_cache=_meta(2, 4, 2 ** 30, 64), v_cache=_meta(2, 4, 2 ** 30, 64)), "positions"),
    (dict(k_cache=_meta(2, 4, 100, 64, dtype=torch.float32)), "dtype"),
    (dict(k_tree=_meta(2, 4, 8, 64, dtype=torch.float16)), "dtype"),
    (dict(), "requires CUDA"),
])
def test_refusals(change, message) -> None:
    args = dict(k_cache=_meta(2, 4, 100, 64), v_cache=_meta(2, 4, 100, 64),
                cache_seqlens=_meta(2, dtype=torch.int32), k_tree=_meta(2, 4, 8, 64),
                v_tree=_meta(2, 4, 8, 64), path=_meta(2, 8, dtype=torch.int32),
                count=_meta(2, dtype=torch.int32))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        commit_draft(**args)


@pytest.mark.gpu
def test_refuses_layouts_the_kernel_cannot_write() -> None:
    k, v, k_tree, v_tree = _problem(2, 2, 20, 4, 64, torch.bfloat16, 4)
    ints = _ints([0, 0])
    path = _ints([[0, 1, 2, 3]] * 2)
    with pytest.raises(ValueError, match="share memory"):
        commit_draft(k[:, :1].expand(2, 2, 20, 64), v, ints, k_tree, v_tree, path, ints)
    with pytest.raises(ValueError, match="aligned"):
        commit_draft(k, v, ints, torch.zeros(2, 2, 4, 65, device="cuda").bfloat16()[..., 1:], v_tree, path, ints)
    with pytest.raises(ValueError, match="cache_seqlens"):
        commit_draft(k, v, ints.long(), k_tree, v_tree, path, ints)
    with pytest.raises(ValueError, match="path"):
        commit_draft(k, v, ints, k_tree, v_tree, path.t().contiguous().t(), ints)
    with pytest.raises(ValueError, match="multiple of 8"):
        commit_draft(*(t[..., :4] for t in (k, v)), ints, *(t[..., :4] for t in (k_tree, v_tree)), path, ints)
