"""Copy-on-write either happens for every block of a call or for none (host bookkeeping, on the CPU)."""

from __future__ import annotations

import pytest
import torch

from engine.kv_cache import PagedKVCache


@pytest.fixture
def cache(monkeypatch):
    """Blocks of 4 tokens; copies noted instead of made."""
    c = PagedKVCache(1, 2, 16, num_blocks=6, block_size=4, max_seqs=6, max_len=64, dtype=torch.float32, device="cpu")
    c.copied = []
    monkeypatch.setattr(c, "copy_blocks", lambda pairs: c.copied.extend(pairs))
    return c


def state(c):
    return ({s: list(t) for s, t in c.block_tables.items()}, dict(c.lengths), list(c._free_blocks), list(c._ref_counts),
            c.cow_copies, list(c.copied), None if c._journal is None else list(c._journal))


def sequence(c, tokens):
    s = c.allocate(tokens)
    c.lengths[s] = tokens
    return s


@pytest.mark.parametrize("mirror", [False, True])
def test_two_forks_and_one_free_block(cache, mirror):
    a, b = sequence(cache, 6), sequence(cache, 6)
    forks = [cache.fork(a), cache.fork(b)]
    sequence(cache, 4)
    assert cache.num_free_blocks == 1
    if mirror:
        cache.enable_device_tables()
    before = state(cache)
    with pytest.raises(RuntimeError, match="copy-on-write"):
        cache.prepare_writes(forks, [6, 6], [1, 1])
    assert state(cache) == before
    pairs = cache.prepare_writes(forks[:1], [6], [1])  # one still fits
    assert pairs == cache.copied == [(before[0][a][1], cache.block_tables[forks[0]][1])]
    assert cache.ref_count(pairs[0][0]) == cache.ref_count(pairs[0][1]) == 1


def test_one_fork_over_several_shared_blocks(cache):
    a = sequence(cache, 14)  # four blocks, the last two about to be written
    cache.lengths[a] = 9
    child = cache.fork(a)
    sequence(cache, 4)
    before = state(cache)
    with pytest.raises(RuntimeError, match="copy-on-write"):
        cache.prepare_writes([child], [9], [5])
    assert state(cache) == before


def test_the_last_of_several_sharers_needs_no_copy(cache):
    """Three sequences of one block written in one call: two copies, the third keeps the block, so two free ones do."""
    a = sequence(cache, 2)
    forks = [cache.fork(a), cache.fork(a)]
    sequence(cache, 12)
    assert cache.num_free_blocks == 2
    shared = cache.block_tables[a][0]
    pairs = cache.prepare_writes([*forks, a], [2, 2, 2], [1, 1, 1])
    assert [old for old, _ in pairs] == [shared, shared] and cache.copied == pairs
    assert cache.block_tables[a] == [shared] and cache.num_free_blocks == 0
    assert sorted(cache.ref_count(cache.block_tables[s][0]) for s in (a, *forks)) == [1, 1, 1]


def test_a_sequence_named_twice_is_copied_once(cache):
    a = sequence(cache, 2)
    child = cache.fork(a)
    assert len(cache.prepare_writes([child, child], [2, 2], [1, 1])) == 1
    assert cache.block_tables[child] != cache.block_tables[a] and cache.cow_copies == 1
