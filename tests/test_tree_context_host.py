"""What a drafted-tree step does to the cache's bookkeeping, on the CPU (the kernels' calls replaced)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from engine import paged_ops
from engine.kv_cache import PagedKVCache


@pytest.fixture
def host(monkeypatch):
    """Tree contexts on host tensors: the index is blank, and the pool's moves and copies are noted instead of made."""
    noted = SimpleNamespace(moves=[], copies=[])

    def index(parents, cu_q, ctx_start, tables, max_q_len, block_size):
        n = parents.shape[0]
        return torch.zeros(n, dtype=torch.int64), torch.zeros(n, dtype=torch.int64), torch.zeros(n, 1, dtype=torch.int64)

    monkeypatch.setattr(paged_ops, "_require_device", lambda *tensors: None)
    monkeypatch.setattr(paged_ops, "tree_index", index)
    monkeypatch.setattr(paged_ops, "tree_commit", lambda *args: noted.moves.append(args))
    monkeypatch.setattr(paged_ops, "copy_blocks", lambda k, v, pairs: noted.copies.extend(pairs))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: SimpleNamespace(synchronize=lambda: None))
    return noted


def make_cache(num_blocks=4, max_len=64):
    return PagedKVCache(1, 2, 16, num_blocks=num_blocks, block_size=4, max_seqs=6, max_len=max_len, dtype=torch.float32,
                        device="cpu")


def sequence(cache, tokens):
    slot = cache.allocate(tokens)
    cache.lengths[slot] = tokens
    return slot


def state(cache):
    return ({s: list(t) for s, t in cache.block_tables.items()}, dict(cache.lengths), list(cache._free_blocks),
            list(cache._ref_counts), cache.cow_copies, None if cache._journal is None else list(cache._journal))


def chain(n):
    return list(range(1, n + 1)), list(range(-1, n - 1))


@pytest.mark.parametrize("mirror", [False, True])
def test_a_refused_step_takes_no_blocks(host, mirror):
    """Two sequences whose trees fit one at a time: the refusal leaves the blocks, and a decode step for both fits."""
    cache = make_cache()
    a, b = sequence(cache, 4), sequence(cache, 4)
    if mirror:
        cache.enable_device_tables()
    before = state(cache)
    tokens, parents = chain(8)
    with pytest.raises(ValueError, match="no room"):
        cache.tree_context([a, b], [tokens, tokens], [parents, parents])
    assert state(cache) == before
    assert cache.ensure_capacity(a, 5) and cache.ensure_capacity(b, 5)


def test_a_step_refused_by_the_length_limit_takes_no_blocks(host):
    cache = make_cache(num_blocks=8, max_len=12)
    a, b = sequence(cache, 4), sequence(cache, 8)
    before = state(cache)
    with pytest.raises(ValueError, match="no room"):
        cache.tree_context([a, b], [chain(8)[0], chain(5)[0]], [chain(8)[1], chain(5)[1]])
    assert state(cache) == before


def test_a_step_refused_for_its_copies_takes_no_blocks(host):
    """The nodes' own blocks are there, those of the shared partial block's copy are not."""
    cache = make_cache(num_blocks=4)
    a = sequence(cache, 6)
    child = cache.fork(a)
    before = state(cache)
    tokens, parents = chain(10)  # two blocks beside the shared one, which takes a third
    with pytest.raises(RuntimeError, match="copy-on-write"):
        cache.tree_context([child], [tokens], [parents])
    assert state(cache) == before and not host.copies
    ctx = cache.tree_context([child], [tokens[:6]], [parents[:6]])
    assert len(host.copies) == cache.cow_copies == 1 and cache.num_free_blocks == 0
    assert ctx.starts == [6] and len(cache.block_tables[child]) == 3


def test_a_token_that_no_index_holds_takes_no_blocks(host):
    cache = make_cache()
    a = sequence(cache, 4)
    before = state(cache)
    with pytest.raises(OverflowError):
        cache.tree_context([a], [[1, 1 << 70]], [[-1, 0]])
    assert state(cache) == before


I32 = dict(dtype=torch.int32)
#      0
#    1   2
#   3   4 5
TREE = [1, 2, 3, 4, 5, 6], [-1, 0, 0, 1, 2, 2]


def tree_step(cache):
    slot = sequence(cache, 6)
    return slot, cache.tree_context([slot], [TREE[0]], [TREE[1]])


@pytest.mark.parametrize("path,count", [
    ([0, 1, 2], 3),      # two siblings
    ([0, 3], 2),         # a node without its parent
    ([0, 1, 4], 3),      # a child of another branch
    ([0, 2, 5], -1),     # no such count
    ([0, 2, 5], 4),      # more nodes than the path has
    ([0, 2, 5], 0), ([0, 2, 6], 3), ([0, 0], 2), ([2, 5], 2), ([0, -1], 2)])
def test_what_is_not_a_path_is_not_committed(host, path, count):
    cache = make_cache(num_blocks=8)
    slot, ctx = tree_step(cache)
    with pytest.raises(ValueError, match="not a path"):
        ctx.commit(torch.tensor([path], **I32), torch.tensor([count], **I32))
    assert cache.lengths[slot] == 6 and not host.moves
    assert ctx.commit(torch.tensor([[0, 2, 5]], **I32), torch.tensor([3], **I32)) == [[0, 2, 5]]  # it can still be settled
    assert cache.lengths[slot] == 9 and len(host.moves) == 1


@pytest.mark.parametrize("path", [[0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], [0, 2, 5]])
def test_every_path_from_the_root_is_committed(host, path):
    cache = make_cache(num_blocks=8)
    slot, ctx = tree_step(cache)
    padded = path + [-1] * (6 - len(path))
    assert ctx.commit(torch.tensor([padded], **I32), torch.tensor([len(path)], **I32)) == [path]
    assert cache.lengths[slot] == 6 + len(path)
    assert len(host.moves) == (path not in ([0], [0, 1]))  # those lie in place


def test_counts_and_paths_of_other_batches_are_refused(host):
    cache = make_cache(num_blocks=8)
    _, ctx = tree_step(cache)
    for path, counts in (([[0], [0]], [1]), ([[0]], [1, 1]), ([[0], [0]], [1, 1])):
        with pytest.raises(ValueError, match="paths for"):
            ctx.commit(torch.tensor(path, **I32), torch.tensor(counts, **I32))


def stale_length(cache, slot):
    cache.ensure_capacity(slot, 7)
    cache.lengths[slot] += 1


def freed(cache, slot):
    cache.free(slot)


def reused(cache, slot):
    cache.free(slot)
    other = sequence(cache, 12)
    assert sequence(cache, 6) == slot or other == slot
    cache.lengths[slot] = 6


def forked_and_written(cache, slot):
    cache.fork(slot)
    cache.prepare_writes([slot], [6], [2])


@pytest.mark.parametrize("change", [stale_length, freed, reused, forked_and_written])
def test_a_step_made_before_the_sequence_changed_is_not_committed(host, change):
    """Its rows lie where the nodes were appended, which is not behind the sequence's tokens any more."""
    cache = make_cache(num_blocks=8)
    slot, ctx = tree_step(cache)
    change(cache, slot)
    before = state(cache)
    with pytest.raises(RuntimeError, match="changed since"):
        ctx.commit(torch.tensor([[0, 2, 5]], **I32), torch.tensor([3], **I32))
    assert state(cache) == before and not host.moves


def test_a_fork_made_before_the_commit_leaves_it_valid(host):
    cache = make_cache(num_blocks=8)
    slot, ctx = tree_step(cache)
    child = cache.fork(slot)
    assert ctx.commit(torch.tensor([[0, 2, 5]], **I32), torch.tensor([3], **I32)) == [[0, 2, 5]]
    assert cache.lengths[slot] == 9 and cache.lengths[child] == 6


def test_a_tree_context_follows_what_is_assigned_to_it(host):
    """A mask, tables or slots put in the place of the step's own reach the layer calls, also after the first of them."""
    cache = make_cache(num_blocks=8)
    _, ctx = tree_step(cache)
    kept = ctx.calls
    assert ctx.calls is kept
    ctx.other = 1
    assert ctx.calls is kept
    for name in ("block_tables", "cu_q", "ctx_start", "mask", "slot_mapping"):
        setattr(ctx, name, getattr(ctx, name).clone())
        assert ctx.calls is not kept and getattr(ctx.calls, name) is getattr(ctx, name), name
        kept = ctx.calls
    ctx.max_q_len = 7
    assert ctx.calls.max_q_len == 7
