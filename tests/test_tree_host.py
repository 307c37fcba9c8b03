"""Drafted trees on the host: refused calls, the C entries' checks, and the plain forms that the kernels are tested
against (all on the CPU; nothing is launched)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from engine import _native, paged_ops
from engine.kv_cache import PagedKVCache
from oracle import tree_ref as ref


def attend_args(n=5, s=2, hq=4, hkv=2, d=64, bs=16, width=3, dtype=torch.float16):
    return dict(q=torch.zeros(n, hq, d, dtype=dtype), k_cache=torch.zeros(9, hkv, bs, d, dtype=dtype),
                v_cache=torch.zeros(9, hkv, bs, d, dtype=dtype), block_tables=torch.zeros(s, width, dtype=torch.int32),
                cu_q=torch.tensor([0, 2, n], dtype=torch.int32), ctx_start=torch.zeros(s, dtype=torch.int32),
                mask=torch.zeros(n, 1, dtype=torch.int64), max_q_len=3)


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(5, 4, 32, dtype=torch.float16)), ValueError),
    (dict(q=torch.zeros(5, 3, 64, dtype=torch.float16)), ValueError),
    (dict(q=torch.zeros(5, 4, 64)), TypeError),
    (dict(q=torch.zeros(5, 64, 4, dtype=torch.float16).transpose(1, 2)), ValueError),
    (dict(v_cache=torch.zeros(9, 2, 16, 64)), TypeError),
    (dict(v_cache=torch.zeros(8, 2, 16, 64, dtype=torch.float16)), ValueError),
    (dict(k_cache=torch.zeros(9, 16, 2, 64, dtype=torch.float16).transpose(1, 2)), ValueError),
    (dict(block_tables=torch.zeros(2, 3)), TypeError),
    (dict(block_tables=torch.zeros(1, 3, dtype=torch.int32)), ValueError),
    (dict(block_tables=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError),
    (dict(cu_q=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(cu_q=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(cu_q=torch.zeros(6, dtype=torch.int32)[::2]), ValueError),
    (dict(ctx_start=torch.zeros(4, dtype=torch.int32)[::2]), ValueError),
    (dict(mask=torch.zeros(4, 1, dtype=torch.int64)), ValueError),
    (dict(mask=torch.zeros(5, 1, dtype=torch.int32)), ValueError),
    (dict(mask=torch.zeros(5, 4, dtype=torch.int64)[:, ::2]), ValueError),
    (dict(mask=torch.zeros(5, 1, dtype=torch.int64), max_q_len=65), ValueError),
    (dict(max_q_len=-1), ValueError),
    (dict(max_blocks=4), ValueError),
    (dict(max_blocks=0), ValueError),
    (dict(scale=0.0), ValueError),
    (dict(scale=-1.0), ValueError),
    (dict(scale=math.nan), ValueError),
    (dict(scale=math.inf), ValueError),
    (dict(out=torch.zeros(5, 4, 64)), ValueError),
    (dict(out=torch.zeros(4, 4, 64, dtype=torch.float16)), ValueError),
    ({}, RuntimeError),  # a good call, but on the CPU
])
def test_attention_refuses(change, error):
    with pytest.raises(error):
        paged_ops.paged_tree(**{**attend_args(), **change})


def test_attention_refuses_other_types():
    with pytest.raises((TypeError, RuntimeError)):
        paged_ops.paged_tree(**attend_args(dtype=torch.float64))


@pytest.mark.parametrize("change,error", [
    (dict(parents=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(parents=torch.zeros(10, dtype=torch.int32)[::2]), ValueError),
    (dict(ctx_start=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(cu_q=torch.zeros(3)), TypeError),
    (dict(max_blocks=9), ValueError),
    (dict(max_q_len=-2), ValueError),
    ({}, RuntimeError),
])
def test_index_refuses(change, error):
    args = dict(parents=torch.zeros(5, dtype=torch.int32), cu_q=torch.tensor([0, 2, 5], dtype=torch.int32),
                ctx_start=torch.zeros(2, dtype=torch.int32), block_tables=torch.zeros(2, 3, dtype=torch.int32), max_q_len=3,
                block_size=16)
    with pytest.raises(error):
        paged_ops.tree_index(**{**args, **change})


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(5)), ValueError),
    (dict(logits=torch.zeros(5, 0)), ValueError),
    (dict(logits=torch.zeros(7, 5).t()), ValueError),
    (dict(logits=torch.zeros(5, 7, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(1, 7).expand(5, 7)), ValueError),
    (dict(tokens=torch.zeros(5, dtype=torch.int32)), ValueError),
    (dict(tokens=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(parents=torch.zeros(4, dtype=torch.int32)), ValueError),
    (dict(cu_q=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(cu_q=torch.zeros(0, dtype=torch.int32)), ValueError),
    (dict(max_q_len=-1), ValueError),
    ({}, RuntimeError),
])
def test_verify_refuses(change, error):
    args = dict(logits=torch.zeros(5, 7), tokens=torch.zeros(5, dtype=torch.int64), parents=torch.zeros(5, dtype=torch.int32),
                cu_q=torch.tensor([0, 2, 5], dtype=torch.int32), max_q_len=3)
    with pytest.raises(error):
        paged_ops.tree_verify(**{**args, **change})


@pytest.mark.parametrize("change,error", [
    (dict(k_pool=torch.zeros(9, 2, 16, 64)), ValueError),
    (dict(v_pool=torch.zeros(2, 9, 2, 16, 64).half()), TypeError),
    (dict(v_pool=torch.zeros(3, 9, 2, 16, 64)), ValueError),
    (dict(path=torch.zeros(2, 3, dtype=torch.int64)), TypeError),
    (dict(path=torch.zeros(3, 3, dtype=torch.int32)), ValueError),
    (dict(path=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError),
    (dict(path=torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)), ValueError),
    (dict(counts=torch.zeros(4, dtype=torch.int32)[::2]), ValueError),
    (dict(ctx_start=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(block_tables=torch.zeros(1, 3, dtype=torch.int32)), ValueError),
    (dict(max_blocks=4), ValueError),
    ({}, RuntimeError),
])
def test_commit_refuses(change, error):
    args = dict(k_pool=torch.zeros(2, 9, 2, 16, 64), v_pool=torch.zeros(2, 9, 2, 16, 64),
                block_tables=torch.zeros(2, 3, dtype=torch.int32), ctx_start=torch.zeros(2, dtype=torch.int32),
                path=torch.zeros(2, 3, dtype=torch.int32), counts=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(error):
        paged_ops.tree_commit(**{**args, **change})


def test_c_entries_check_before_they_launch():
    """Empty work returns OK, rejected arguments their status (addresses that would fault if anything read them)."""
    lib = _native.load()
    p, ok, bad, no = 256, _native.MIP_OK, _native.MIP_EINVAL, _native.MIP_EUNSUPPORTED

    def attend(out=p, q=p, k=p, bt_stride=4, mask=p, mask_stride=1, words=1, s=1, m=3, hq=4, hkv=2, d=64, bs=16, mb=4,
               scale=0.1, ws=None, ws_bytes=0, dt=_native.MIP_F16, q_stride=256):
        return lib.mip_paged_tree(out, 256, 64, q, q_stride, 64, k, p, 9, p, bt_stride, p, p, mask, mask_stride, words, s,
                                  m, hq, hkv, d, bs, mb, scale, ws, ws_bytes, dt, None)

    assert attend(s=0) == ok and attend(m=0) == ok
    for kw in (dict(dt=7), dict(s=-1), dict(m=-1), dict(hq=3), dict(hkv=0), dict(d=0), dict(bs=12), dict(bs=8192), dict(mb=0),
               dict(bt_stride=3), dict(scale=0.0), dict(scale=math.nan), dict(out=None), dict(q=None), dict(mask=None),
               dict(words=0), dict(mask_stride=0), dict(m=65), dict(k=p + 8), dict(q=p + 1), dict(mb=1 << 26, bt_stride=1 << 26)):
        assert attend(**kw) == bad, kw
    assert attend(mb=1024, bt_stride=1024, s=8, m=3) == bad  # cut contexts need a workspace
    assert attend(mb=1024, bt_stride=1024, s=8, m=3, ws=p + 8, ws_bytes=1 << 40) == bad
    assert attend(d=96) == no and attend(d=512) == no
    size = lib.mip_paged_tree_workspace
    assert size(8, 3, 4, 2, 64, 16, 1024, _native.MIP_F16) > 0
    large = size(1024, 3, 4, 2, 64, 16, 1024, _native.MIP_F16)
    assert large > 0 and size(5000, 3, 4, 2, 64, 16, 1024, _native.MIP_F16) == large
    assert attend(mb=1024, bt_stride=1024, s=5000, ws=p, ws_bytes=large - 1) == bad
    assert size(0, 3, 4, 2, 64, 16, 1024, _native.MIP_F16) == 0 and size(1, 3, 3, 2, 64, 16, 4, _native.MIP_F16) == 0

    def index(words=1, n=3, s=1, m=3, bs=16, mb=4, parents=p, tables=p):
        return lib.mip_tree_index(p, p, p, words, parents, n, p, p, tables, 4, s, m, bs, mb, None)

    assert index(n=0) == ok
    assert index(m=1025) == no and index(s=1 << 24) == no
    for kw in (dict(words=0), dict(words=17), dict(s=-1), dict(n=-1), dict(bs=3), dict(mb=5), dict(mb=0), dict(parents=None),
               dict(tables=None), dict(m=65)):
        assert index(**kw) == bad, kw

    def verify(n=3, vocab=100, stride=100, s=1, m=3, ws=p, ws_bytes=1 << 20, dt=_native.MIP_F32, logits=p):
        return lib.mip_tree_verify(p, p, p, p, logits, stride, n, vocab, p, p, p, s, m, ws, ws_bytes, dt, None)

    assert verify(n=0, s=0) == ok
    assert verify(m=1025) == no
    for kw in (dict(vocab=0), dict(stride=99), dict(n=-1), dict(ws=None), dict(ws_bytes=8), dict(ws=p + 4), dict(dt=3),
               dict(logits=None), dict(logits=p + 2)):
        assert verify(**kw) == bad, kw
    assert lib.mip_tree_verify_workspace(3, 151936, _native.MIP_BF16) >= 3 * 8

    def commit(layers=2, hkv=2, d=64, bs=16, mb=4, stride=3, width=3, s=1, k=p, dt=_native.MIP_F16):
        return lib.mip_tree_commit(k, p, layers, 9, hkv, d, bs, p, 4, mb, p, p, stride, width, p, s, dt, None)

    assert commit(s=0) == ok and commit(width=0) == ok
    for kw in (dict(layers=0), dict(hkv=0), dict(d=0), dict(bs=6), dict(mb=5), dict(stride=2), dict(k=None), dict(k=p + 1), dict(dt=9)):
        assert commit(**kw) == bad, kw
    assert commit(s=65536) == no
    assert lib.mip_tree_step_attend(None, p, p, p, p, None) == bad


def small_cache(max_len=64):
    return PagedKVCache(1, 2, 16, num_blocks=12, block_size=4, max_seqs=4, max_len=max_len, dtype=torch.float32, device="cpu")


@pytest.mark.parametrize("slots,tokens,parents,match", [
    ([], [], [], "at least one sequence"),
    ([0, 0], [[1], [2]], [[-1], [-1]], "twice"),
    ([0], [[1], [2]], [[-1]], "lists of tokens"),
    ([0], [[1, 2]], [[-1]], "a token and a parent"),
    ([0], [[]], [[]], "needs a root"),
    ([0], [[1, 2]], [[0, -1]], "node 0 is the root"),
    ([0], [[1, 2]], [[-1, -1]], "node 0 is the root"),
    ([0], [[1, 2, 3]], [[-1, 2, 0]], "comes before"),
    ([0], [[1, 2, -1]], [[-1, 0, 1]], "negative"),
    ([0], [[0] * 1025], [[-1] + [0] * 1024], "at most 1024"),
])
def test_tree_context_refuses(slots, tokens, parents, match):
    cache = small_cache()
    for _ in range(2):
        cache.allocate(5)
    free = cache.num_free_blocks
    with pytest.raises(ValueError, match=match):
        cache.tree_context(slots, tokens, parents)
    assert cache.num_free_blocks == free


def test_tree_context_needs_the_gpu_and_takes_no_blocks_without():
    cache = small_cache()
    slot = cache.allocate(4)
    free = cache.num_free_blocks
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache.tree_context([slot], [[1, 2, 3]], [[-1, 0, 0]])
    assert cache.num_free_blocks == free


def test_step_struct_fields_follow_the_header():
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parent.parent / "include" / "mipaged.h").read_text()
    body = re.search(r"typedef struct mip_tree_step \{(.*?)\}", text, re.S).group(1)
    names = [n.strip(" *") for decl in body.split(";") if decl.strip() for n in re.sub(r"^.*?(?:_t|void|float)\*? ", "", " ".join(decl.split())).split(",")]
    assert names == [f[0] for f in _native.TreeStep._fields_]


# ---------------------------------------------------------------------------------- the plain forms
def test_plain_index_of_a_known_tree():
    #      0
    #    1   2
    #   3 4    5
    pos, slots, mask = ref.index([[-1, 0, 0, 1, 1, 2]], [6], [[3, 1, 0]], 4, 3, 1)
    assert pos.tolist() == [6, 7, 7, 8, 8, 8]
    assert slots.tolist() == [6, 7, 0, 1, 2, 3]
    assert [bin(x) for x in mask[:, 0]] == ["0b1", "0b11", "0b101", "0b1011", "0b10011", "0b100101"]


def test_plain_attention_of_a_chain_is_causal_attention():
    from oracle import paged_ref

    rng = np.random.default_rng(0)
    k, v = rng.standard_normal((2, 6, 2, 4, 8)).astype(np.float32)
    q = rng.standard_normal((5, 4, 8)).astype(np.float32)
    tables, starts, counts = [[4, 0, 2]], [6], [5]
    mask = ref.index([[-1, 0, 1, 2, 3]], starts, tables, 4, 3, 1)[2]
    got, spread, _ = ref.attention(q, k, v, tables, starts, counts, mask, 4, 1 / math.sqrt(8))
    want = paged_ref.prefill_attention_f64(q, k, v, tables, starts, counts, 4)
    assert np.abs(got - want).max() < 1e-12 and (spread >= np.abs(got) - 1e-12).all()


def test_plain_attention_of_siblings_is_that_of_two_chains():
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((2, 4, 1, 4, 8))
    q = rng.standard_normal((3, 2, 8))
    mask = ref.index([[-1, 0, 0]], [5], [[0, 2]], 4, 2, 1)[2]
    both, _, _ = ref.attention(q, k, v, [[0, 2]], [5], [3], mask, 4, 0.3)
    k[2, :, 2], v[2, :, 2] = k[2, :, 3], v[2, :, 3]  # the second sibling in the first one's place
    chain = ref.index([[-1, 0]], [5], [[0, 2]], 4, 2, 1)[2]
    alone, _, _ = ref.attention(q[[0, 2]], k, v, [[0, 2]], [5], [2], chain, 4, 0.3)
    assert np.abs(both[2] - alone[1]).max() < 1e-12


def test_plain_verify_takes_the_first_child_and_stops_where_none_agrees():
    logits = np.full((6, 10), -1.0)
    for r, t in enumerate([3, 5, 7, 1, 1, 9]):
        logits[r, t] = 2.0
    logits[0, 8] = 2.0  # a tie: the lower index stands
    target, paths, following = ref.verify(logits, [[0, 4, 3, 3, 7, 2]], [[-1, 0, 0, 0, 2, 4]])
    assert target == [3, 5, 7, 1, 1, 9] and paths == [[0, 2, 4]] and following == [1]
