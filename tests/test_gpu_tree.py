"""The drafted-tree operators on the GPU against their plain 64-bit forms (oracle/tree_ref.py).

Bound of an attention output element, from the arithmetic: a score is a sum of D products in fp32, off by at
most (D + 2) 2^-24 times its sum of absolute products (``reach``), and exp2 by 2^-22, so a weight is off by a
relative delta = (D + 2) 2^-24 reach + 2^-21; 16-bit calls round it to fp16 (2^-11, or 2^-25 on fp16's
subnormal grid where the largest weight is at least 1). Weights enter the sum and the normaliser, hence
twice; fp32 sums over n keys add n 2^-23. Times the weighted mean of |v| (``spread``), and half a step of
the output type on top. Index, verification and move are exact.
"""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

from conftest import announce
from oracle import tree_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def random_tree(n, rng, chain=False):
    return [-1 if i == 0 else i - 1 if chain else max(rng.randrange(i), rng.randrange(i)) // 2 for i in range(n)]


class Step:
    """A pool, tables, packed q and masks of sequences with ``starts`` cached tokens and ``nodes`` drafted ones."""

    def __init__(self, dtype, d, hq, hkv, bs, starts, nodes, seed=0, kind="tree", scale=None):
        rng = random.Random(seed)
        self.dtype, self.bs, self.starts, self.nodes, self.hq, self.hkv, self.d = dtype, bs, starts, nodes, hq, hkv, d
        need = [max(1, -(-(a + n) // bs)) for a, n in zip(starts, nodes)]
        ids = list(range(sum(need) + 3))
        rng.shuffle(ids)
        self.tables, at = [], 0
        for k in need:
            self.tables.append(ids[at:at + k])
            at += k
        gen = torch.Generator().manual_seed(seed)
        dt = DTYPES[dtype]
        self.k, self.v = (torch.randn(len(ids) + 1, hkv, bs, d, generator=gen).to(dt) for _ in range(2))
        n = sum(nodes)
        self.qkv = (torch.randn(n, (hq + 2 * hkv) * d, generator=gen) * 2).to(dt)
        self.most = max(nodes)
        self.words = max(1, -(-self.most // 64))
        self.parents = [random_tree(m, rng, kind == "chain") for m in nodes]
        if kind == "free":
            bits = [[sum(1 << j for j in range(m) if rng.random() < 0.4) for _ in range(m)] for m in nodes]
            rows = [[(x >> (64 * w)) & (2**64 - 1) for w in range(self.words)] for t in bits for x in t]
            self.mask = np.array(rows, np.uint64).reshape(n, self.words).view(np.int64)
        else:
            self.mask = ref.index(self.parents, starts, self.tables, bs, 1 << 30, self.words)[2]
        self.scale = scale

    def width(self):
        return max(map(len, self.tables))

    def to(self, gpu):
        tab = torch.full((len(self.tables), self.width() + 1), -1, dtype=torch.int32)
        for i, t in enumerate(self.tables):
            tab[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        cu = np.concatenate([[0], np.cumsum(self.nodes)]).astype(np.int32)
        n = sum(self.nodes)
        return dict(q=self.qkv.to(gpu)[:, :self.hq * self.d].view(n, self.hq, self.d), k_cache=self.k.to(gpu),
                    v_cache=self.v.to(gpu), block_tables=tab.to(gpu), cu_q=torch.from_numpy(cu).to(gpu),
                    ctx_start=torch.tensor(self.starts, dtype=torch.int32).to(gpu),
                    mask=torch.from_numpy(self.mask).to(gpu), max_q_len=self.most, scale=self.scale)

    def want(self, max_blocks=None):
        n = sum(self.nodes)
        q = self.qkv[:, :self.hq * self.d].view(n, self.hq, self.d).double().numpy()
        scale = self.scale or 1.0 / math.sqrt(self.d)
        with np.errstate(invalid="ignore", over="ignore"):
            return ref.attention(q, self.k.double().numpy(), self.v.double().numpy(), self.tables, self.starts,
                                 self.nodes, self.mask, self.bs, scale, max_blocks)

    def check(self, got, max_blocks=None):
        out, spread, reach = self.want(max_blocks)
        got = got.double().cpu().numpy()
        half_step = torch.finfo(DTYPES[self.dtype]).eps / 2
        keys = max(a + n for a, n in zip(self.starts, self.nodes))
        delta = (self.d + 2) * 2.0**-24 * reach + 2.0**-21 + keys * 2.0**-23
        vmax = float(self.v.double().abs().nan_to_num(0, 0, 0).max())
        floor = 0.0
        if self.dtype != "float32":
            delta = delta + 2.0**-11
            floor = keys * 2.0**-24 * vmax
        finite = np.isfinite(out)
        assert np.array_equal(finite, np.isfinite(got))
        assert np.array_equal(np.isnan(out), np.isnan(got))
        assert np.array_equal(out[np.isinf(out)], got[np.isinf(out)])
        err = np.abs(got - out)[finite]
        tiny = torch.finfo(DTYPES[self.dtype]).smallest_normal * half_step * 2
        bound = (half_step * 1.01 * np.abs(out) + 2.05 * delta[..., None] * spread + floor + tiny)[finite]
        assert (err <= bound).all(), float((err / bound).max())


def run(gpu, step, **kw):
    from engine import paged_ops

    out = paged_ops.paged_tree(**{**step.to(gpu), **kw})
    torch.cuda.synchronize()
    return out


SHAPES = [(64, 14, 2, 16), (128, 28, 4, 32), (64, 8, 8, 16), (64, 6, 3, 1), (128, 16, 1, 4), (64, 40, 2, 64)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,hq,hkv,bs", SHAPES)
@pytest.mark.parametrize("starts,nodes,kind", [
    ([37], [5], "chain"), ([0, 3, 64], [1, 2, 1], "tree"), ([130, 0, 31, 512], [9, 4, 0, 17], "tree"),
    ([63, 65, 1], [33, 64, 20], "tree"), ([0, 17], [70, 130], "free"), ([700], [3], "free")])
def test_tree_attention_matches_f64(gpu, dtype, d, hq, hkv, bs, starts, nodes, kind):
    announce(f"paged_tree {dtype} d={d} hq={hq} hkv={hkv} bs={bs} starts={starts} nodes={nodes} {kind}")
    step = Step(dtype, d, hq, hkv, bs, starts, nodes, seed=len(starts), kind=kind)
    step.check(run(gpu, step))


@pytest.mark.parametrize("dtype,d,hq,hkv,bs", [
    ("float32", 64, 14, 2, 16), ("float32", 128, 8, 2, 32), ("float32", 8, 4, 4, 4), ("float32", 256, 4, 2, 16),
    ("float16", 32, 8, 2, 16), ("bfloat16", 256, 4, 2, 16), ("float16", 16, 5, 1, 2), ("bfloat16", 8, 3, 3, 8),
    ("float32", 64, 40, 2, 16), ("float32", 128, 7, 1, 8), ("float32", 16, 2, 1, 16)])
@pytest.mark.parametrize("starts,nodes,kind", [([37], [5], "chain"), ([130, 0, 31], [9, 4, 0], "tree"),
                                               ([0, 17], [70, 30], "free")])
def test_tree_attention_other_types_and_head_sizes(gpu, dtype, d, hq, hkv, bs, starts, nodes, kind):
    announce(f"paged_tree {dtype} d={d} hq={hq} hkv={hkv} bs={bs} starts={starts} nodes={nodes} {kind}")
    step = Step(dtype, d, hq, hkv, bs, starts, nodes, seed=7, kind=kind)
    step.check(run(gpu, step))


@pytest.mark.parametrize("dtype,d,hq,hkv,bs,starts,nodes", [
    ("bfloat16", 64, 14, 2, 16, [6000], [5]), ("float16", 64, 7, 1, 16, [9001], [2]),
    ("bfloat16", 128, 4, 1, 32, [5001, 40, 700], [3, 8, 1]), ("float16", 64, 4, 2, 16, [3000, 1], [40, 64]),
    ("bfloat16", 128, 14, 2, 16, [2500], [20]), ("float32", 64, 4, 1, 16, [3000], [4])])
def test_tree_attention_long_contexts_in_pieces(gpu, dtype, d, hq, hkv, bs, starts, nodes):
    announce(f"paged_tree long {dtype} d={d} hq={hq} hkv={hkv} starts={starts} nodes={nodes}")
    step = Step(dtype, d, hq, hkv, bs, starts, nodes, seed=3)
    step.check(run(gpu, step))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 8)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_has_no_influence(gpu, dtype, d, bs, bad):
    """NaN and infinities in the keys and values of other branches and behind the last key, and an infinite value
    that some rows do see: those rows alone become infinite."""
    announce(f"paged_tree masked {bad} {dtype} d={d} bs={bs}")
    step = Step(dtype, d, 8, 2, bs, [45, 300], [20, 9], seed=11)
    leaf = 19  # the last node of the first tree: nobody but itself sees it
    p = 45 + leaf
    step.k[step.tables[0][p // bs], :, p % bs] = bad
    step.v[step.tables[0][p // bs], :, p % bs] = bad
    last = step.tables[1][-1]
    used = 309 - (len(step.tables[1]) - 1) * bs
    step.k[last, :, used:] = bad
    step.v[last, :, used:] = bad
    step.v[step.tables[1][7 // bs], 0, 7 % bs, 3] = math.inf  # a cached key of the second sequence: all its rows see it
    got = run(gpu, step).double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        out, _, _ = step.want()
    own = np.zeros(29, bool)
    own[leaf] = True
    assert np.isfinite(got[:leaf]).all()
    assert np.array_equal(np.isinf(got[20:]), np.isinf(out[20:])) and np.isinf(got[20:, :4, 3]).all()
    fine = np.isfinite(out) & ~own[:, None, None]
    tol = {"float16": 4e-3, "bfloat16": 2e-2, "float32": 1e-5}[dtype]  # 8 half steps of values of order one
    assert np.abs(got - out)[fine].max() <= tol


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("nodes", [[4], [40]])
def test_large_values(gpu, dtype, nodes):
    """Values that fp16 cannot hold (bf16), and the largest that it can."""
    announce(f"paged_tree large values {dtype} nodes={nodes}")
    step = Step(dtype, 64, 4, 2, 16, [200], nodes, seed=5)
    step.v[step.tables[0][2], :, 5] = 3e5 if dtype == "bfloat16" else 65504.0
    step.v[step.tables[0][12], :, 8] = -2e38 if dtype == "bfloat16" else -65504.0
    step.check(run(gpu, step))


def widened(step, args):
    """``args`` with tables so wide (their further entries are no blocks) that the call is taken for a large one: its rows
    of more than 64 then run on wavefronts that share their keys."""
    rows = step.most * (step.hq // step.hkv)
    assert rows > 64 and step.bs >= 8
    width = -(-(32 << 20) // (len(step.nodes) * step.hkv * rows * step.bs)) + step.width()
    tab = torch.full((len(step.nodes), width), -1, dtype=torch.int32, device=args["block_tables"].device)
    tab[:, :args["block_tables"].shape[1]] = args["block_tables"]
    return {**args, "block_tables": tab}


LARGE = [(64, 14, 2, 16), (128, 28, 4, 32), (64, 8, 1, 8), (128, 16, 1, 8), (64, 40, 2, 64)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,hq,hkv,bs", LARGE)
@pytest.mark.parametrize("starts,nodes,kind", [
    ([300], [20], "tree"), ([0, 3, 64], [20, 1, 33], "tree"), ([130, 0, 31, 512, 257], [30, 20, 0, 17, 2], "tree"),
    ([0, 17], [70, 130], "free"), ([2222], [40], "chain")])
def test_large_calls_match_f64(gpu, dtype, d, hq, hkv, bs, starts, nodes, kind):
    announce(f"paged_tree large call {dtype} d={d} hq={hq} hkv={hkv} bs={bs} starts={starts} nodes={nodes} {kind}")
    step = Step(dtype, d, hq, hkv, bs, starts, nodes, seed=len(starts) + 20, kind=kind)
    step.check(run(gpu, step, **widened(step, step.to(gpu))))


@pytest.mark.parametrize("d,hq,hkv,bs", [(64, 14, 2, 8), (128, 28, 4, 16)])
def test_large_calls_at_every_end(gpu, d, hq, hkv, bs):
    """Contexts that end at every place of a step of 32 keys and of a block, in one batch."""
    announce(f"paged_tree large call, every end d={d}")
    step = Step("bfloat16", d, hq, hkv, bs, list(range(40, 74)), [12] * 34, seed=31)
    step.check(run(gpu, step, **widened(step, step.to(gpu))))


@pytest.mark.parametrize("d,bs", [(64, 16), (128, 8)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_large_calls_what_a_row_does_not_see_has_no_influence(gpu, d, bs, bad):
    announce(f"paged_tree large call masked {bad} d={d}")
    step = Step("bfloat16", d, 28, 4, bs, [45, 300], [20, 9], seed=11)
    step.tables[1][3] = -7  # a block outside the pool
    leaf = 19
    for x in (step.k, step.v):
        x[step.tables[0][(45 + leaf) // bs], :, (45 + leaf) % bs] = bad
        x[step.tables[1][-1], :, 309 - (len(step.tables[1]) - 1) * bs:] = bad
    got = run(gpu, step, **widened(step, step.to(gpu))).double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        out, _, _ = step.want()
    keep = [i for i in range(29) if i != leaf]
    assert np.isfinite(out[keep]).all() and np.abs(got[keep] - out[keep]).max() <= 2e-2  # 8 half steps of values of order one


@pytest.mark.parametrize("d,hq,hkv", [(64, 14, 2), (128, 28, 4)])
@pytest.mark.parametrize("scale", [2.0**-30, 1.0, 2.0**100])
def test_large_calls_with_small_and_large_values(gpu, d, hq, hkv, scale):
    """bf16 values that fp16 does not hold: everywhere, and in one dim of ordinary ones."""
    announce(f"paged_tree large call values of {scale} d={d}")
    step = Step("bfloat16", d, hq, hkv, 16, [300, 50], [12, 20], seed=33)
    step.v *= scale
    step.v[..., 9] *= 2.0**-30
    got = run(gpu, step, **widened(step, step.to(gpu))).double().cpu().numpy()
    out, spread, reach = step.want()
    delta = (d + 2) * 2.0**-24 * reach + 2.0**-21 + 400 * 2.0**-23 + 2.0**-11
    bound = 2.0**-8 * 1.01 * np.abs(out) + 2.05 * delta[..., None] * spread + 400 * 2.0**-31 * spread
    assert (np.abs(got - out) <= bound)[..., 9].all()
    if scale != 1.0:
        assert (np.abs(got - out) <= bound).all()
    step.check(torch.from_numpy(got))


def test_a_tree_of_a_thousand_nodes(gpu):
    announce("paged_tree 1024 nodes")
    for dtype, d, hq in (("bfloat16", 64, 4), ("float32", 64, 2)):
        step = Step(dtype, d, hq, 2, 16, [21], [1024], seed=34)
        step.check(run(gpu, step))


@pytest.mark.parametrize("dtype,d,hq,hkv,nodes", [
    ("bfloat16", 64, 14, 2, [3, 12]), ("bfloat16", 64, 14, 2, [40, 5]), ("bfloat16", 128, 28, 4, [12]), ("bfloat16", 64, 14, 2, [2]),
    ("float32", 64, 14, 2, [12]), ("bfloat16", 32, 14, 2, [12])])
@pytest.mark.parametrize("where", ["all", "one dim", "one sequence"])
def test_values_below_fp16(gpu, dtype, d, hq, hkv, nodes, where):
    """Values of about 2^-30, everywhere or beside ordinary ones, keep their relative accuracy."""
    announce(f"paged_tree small values {dtype} d={d} nodes={nodes} {where}")
    step = Step(dtype, d, hq, hkv, 16, [300] * len(nodes), nodes, seed=15)
    if where == "all":
        step.v *= 2.0**-30
    elif where == "one dim":
        step.v[..., 7] *= 2.0**-30
    else:
        step.v[torch.tensor(step.tables[0])] *= 2.0**-30
    got = run(gpu, step).double().cpu().numpy()
    out, spread, reach = step.want()
    half_step = torch.finfo(DTYPES[dtype]).eps / 2
    delta = (d + 2) * 2.0**-24 * reach + 2.0**-21 + 400 * 2.0**-23 + (0 if dtype == "float32" else 2.0**-11)
    small = np.zeros(out.shape, bool)
    if where == "all":
        small[:] = True
    elif where == "one dim":
        small[..., 7] = True
    else:
        small[:nodes[0]] = True
    bound = half_step * 1.01 * np.abs(out) + 2.05 * delta[..., None] * spread + 400 * 2.0**-31 * spread
    assert (np.abs(got - out) <= bound)[small].all()
    step.check(torch.from_numpy(got))


def test_a_long_tail_of_small_weights(gpu):
    """One key far above 30000 others whose weights (2^-25.5 of its own) fp16 alone would round by half: each is held to
    2^-32 of the largest."""
    announce("paged_tree tail of small weights")
    step = Step("float16", 64, 2, 1, 16, [30000], [40], seed=16, scale=1.0)
    step.qkv.zero_()
    step.k.zero_()
    step.qkv[:, 0] = step.qkv[:, 64] = 1.0
    step.k[step.tables[0][3], 0, 5, 0] = 25.5 * math.log(2.0)
    step.v.fill_(1.0)
    step.v[step.tables[0][3], 0, 5] = 0.0
    out, _, _ = step.want()
    got = run(gpu, step).double().cpu().numpy()
    assert 5e-4 < out.min() and np.abs(got - out).max() <= 30040 * 2.0**-32 + 2.0**-11 * out.max() * 3


@pytest.mark.parametrize("dtype,d,start", [("float16", 64, 600), ("float16", 64, 20), ("float32", 64, 900), ("float32", 32, 900),
                                           ("bfloat16", 128, 600), ("float32", 64, 20)])
def test_trees_longer_than_max_q_len_end_there(gpu, dtype, d, start):
    """Nodes from max_q_len on are no rows and no keys; their output rows stay as they were."""
    announce(f"paged_tree clipped trees {dtype} d={d} start={start}")
    step = Step(dtype, d, 4, 2, 16, [start, 8, start], [10, 3, 7], seed=17, kind="free")
    args = step.to(gpu)
    out = torch.full((20, 4, d), 7.0, dtype=DTYPES[dtype], device=gpu)
    run(gpu, step, max_q_len=4, out=out)
    assert (out[4:10] == 7).all() and (out[17:] == 7).all()
    keep = [0, 1, 2, 3, 10, 11, 12, 13, 14, 15, 16]
    step.nodes, step.mask, step.qkv = [4, 3, 4], step.mask[keep], step.qkv[keep]
    step.check(out[keep])
    del args


@pytest.mark.parametrize("dtype,d", [("float16", 64), ("bfloat16", 128), ("float32", 64), ("float16", 32)])
def test_rows_that_see_nothing_and_rows_of_nobody(gpu, dtype, d):
    announce(f"paged_tree empty rows {dtype} d={d}")
    step = Step(dtype, d, 4, 2, 16, [0, 20, 0], [6, 3, 0], seed=9, kind="free")
    step.mask[2] = 0
    step.mask[4] = 0
    args = step.to(gpu)
    # Two rows ahead of the first sequence and three behind the last belong to nobody and stay as they are.
    pad = [torch.cat([torch.full_like(args[x][:1], fill).expand(2, *args[x].shape[1:]), args[x],
                      torch.full_like(args[x][:1], fill).expand(3, *args[x].shape[1:])]).contiguous()
           for x, fill in (("q", math.nan), ("mask", -1))]
    out = torch.full((14, 4, d), 7.0, dtype=DTYPES[dtype], device=gpu)
    got = run(gpu, step, q=pad[0], mask=pad[1], cu_q=args["cu_q"] + 2, out=out)
    assert got is out
    assert (out[:2] == 7).all() and (out[11:] == 7).all()
    assert (out[4] == 0).all() and (out[6] == 0).all()
    step.check(out[2:11])


def test_block_ids_outside_the_pool_hide_their_keys(gpu):
    for dtype, d, nodes in (("bfloat16", 64, [5, 9]), ("float16", 128, [30, 2]), ("float32", 64, [5, 9])):
        announce(f"paged_tree bad blocks {dtype} d={d}")
        step = Step(dtype, d, 4, 2, 16, [100, 250], nodes, seed=2)
        step.tables[0][1] = -3
        step.tables[1][0] = step.k.shape[0]
        step.tables[1][6] = 1 << 30
        step.check(run(gpu, step))


def test_keys_past_the_table_are_never_read(gpu):
    for dtype, d in (("bfloat16", 64), ("float32", 64), ("float16", 128)):
        announce(f"paged_tree short table {dtype} d={d}")
        step = Step(dtype, d, 4, 2, 16, [100, 60], [9, 9], seed=4)
        step.check(run(gpu, step, max_blocks=4), max_blocks=4)


def test_strides_alignment_and_wide_masks(gpu):
    from engine import paged_ops

    for dtype, shift in (("bfloat16", 8), ("float16", 1), ("float32", 1)):
        announce(f"paged_tree strides {dtype} shift={shift}")
        step = Step(dtype, 64, 6, 2, 16, [77, 20], [8, 21], seed=6)
        args = step.to(gpu)
        n = 29
        wide = torch.zeros(n, 6, 64 + 16, dtype=DTYPES[dtype], device=gpu)
        wide[:, :, shift:shift + 64] = args["q"]
        mask = torch.full((n, 5), -1, dtype=torch.int64, device=gpu)
        mask[:, 0] = args["mask"][:, 0]
        mask[:, 1:] = 0
        out = torch.zeros(6, n, 64 + 8, dtype=DTYPES[dtype], device=gpu).transpose(0, 1)[:, :, shift:shift + 64]
        paged_ops.paged_tree(**{**args, "q": wide[:, :, shift:shift + 64], "mask": mask[:, :3], "out": out,
                                "block_tables": torch.cat([args["block_tables"]] * 2, 1)}, max_blocks=step.width())
        torch.cuda.synchronize()
        step.check(out)


def test_scale_and_peaked_scores(gpu):
    for scale in (0.02, 3.0):
        announce(f"paged_tree scale {scale}")
        step = Step("bfloat16", 64, 7, 1, 16, [333], [12], seed=8, scale=scale)
        step.check(run(gpu, step))


def test_many_sequences(gpu):
    rng = random.Random(1)
    for count in (300, 1024, 1030):
        announce(f"paged_tree {count} sequences")
        starts = [rng.randrange(40) for _ in range(count)]
        step = Step("float16", 64, 2, 1, 8, starts, [rng.randrange(4) for _ in range(count)], seed=count)
        step.check(run(gpu, step))


def test_row_offsets_past_32_bits(gpu):
    """A pool of more than 2^32 bytes (and 2^31 elements) a side, its last blocks in use."""
    from engine import paged_ops

    announce("paged_tree pool of 2^31 elements")
    blocks, hkv, bs, d = (1 << 31) // (8 * 64 * 128) + 40, 8, 64, 128
    k, v = (torch.zeros(blocks, hkv, bs, d, dtype=torch.float16, device=gpu) for _ in range(2))
    step = Step("float16", d, 16, hkv, bs, [200], [5], seed=12)
    args = step.to(gpu)
    ids = [blocks - 1 - i for i in range(len(step.tables[0]))]
    for new, old in zip(ids, step.tables[0]):
        k[new], v[new] = args["k_cache"][old], args["v_cache"][old]
    tab = torch.tensor([ids], dtype=torch.int32, device=gpu)
    out = paged_ops.paged_tree(**{**args, "k_cache": k, "v_cache": v, "block_tables": tab})
    torch.cuda.synchronize()
    step.check(out)
    path, counts = torch.tensor([[0, 2, 4]], dtype=torch.int32, device=gpu), torch.tensor([3], dtype=torch.int32, device=gpu)
    want = [k[ids[3], :, 8 + i].clone() for i in (0, 2, 4)]
    paged_ops.tree_commit(k[None], v[None], tab, args["ctx_start"], path, counts)
    torch.cuda.synchronize()
    assert all(torch.equal(k[ids[3], :, 8 + i], w) for i, w in enumerate(want))


@pytest.mark.parametrize("parents", [
    [[-1]], [[-1, 0, 1, 2, 3]], [[-1, 0, 0, 1, 1, 2, 2], [], [-1, 0]], [[-1, 5, 1, 3, -7, 0, 100, 6]],
    [list(range(-1, 63))], [list(range(-1, 64)), [-1, 0, 0]], [list(range(-1, 299)), [-1] * 70],
    [list(range(-1, 1023))]])
@pytest.mark.parametrize("bs,max_blocks", [(16, None), (1, None), (64, 2)])
def test_tree_index(gpu, parents, bs, max_blocks):
    from engine import paged_ops

    announce(f"tree_index nodes={[len(t) for t in parents]} bs={bs} max_blocks={max_blocks}")
    rng = random.Random(3)
    starts = [rng.randrange(100) for _ in parents]
    most = max(map(len, parents))
    width = -(-(max(starts) + most) // bs)
    tables = [[rng.randrange(1 << 20) for _ in range(max(width, 3))] for _ in parents]
    limit = width if max_blocks is None else max_blocks
    words = -(-most // 64)
    want = ref.index(parents, starts, tables, bs, limit, words)
    cu = np.concatenate([[0], np.cumsum([len(t) for t in parents])]).astype(np.int32)
    got = paged_ops.tree_index(torch.tensor([p for t in parents for p in t], dtype=torch.int32, device=gpu),
                               torch.from_numpy(cu).to(gpu), torch.tensor(starts, dtype=torch.int32, device=gpu),
                               torch.tensor(tables, dtype=torch.int32, device=gpu), most, bs, max_blocks=limit)
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert np.array_equal(x.cpu().numpy(), y)


def verify_inputs(dtype, vocab, sizes, seed):
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    n = sum(sizes)
    logits = torch.randn(n, vocab, generator=gen).to(DTYPES[dtype])
    parents = [random_tree(m, rng) for m in sizes]
    tokens = [[rng.randrange(vocab) for _ in t] for t in parents]
    at = 0
    for toks, tree in zip(tokens, parents):
        for i, p in enumerate(tree):
            if p >= 0 and rng.random() < 0.7:
                toks[i] = int(torch.where(logits[at + p] == logits[at + p].max())[0][0])
        at += len(tree)
    return logits, tokens, parents


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("vocab,sizes", [(151936, [5]), (1, [3, 1]), (7, [4, 0, 30]), (1001, [70, 2, 130]),
                                         (32003, [9, 16]), (4096, [1] * 300), (257, [64])])
def test_tree_verify(gpu, dtype, vocab, sizes):
    from engine import paged_ops

    announce(f"tree_verify {dtype} vocab={vocab} sizes={sizes[:4]}")
    logits, tokens, parents = verify_inputs(dtype, vocab, sizes, 5)
    if vocab > 64:
        logits[0, 60] = logits[0, 5] = 50.0  # a tie
        logits[-1, 40:44] = math.nan         # the first of several NaN, ahead of infinity
        logits[-1, 3] = math.inf
    if len(logits) > 2:
        logits[1] = -math.inf
    check_verify(gpu, logits.to(gpu), tokens, parents)


def check_verify(gpu, logits, tokens, parents, lead=0, tail=0):
    from engine import paged_ops

    flat_p, flat_t = [p for t in parents for p in t], [x for t in tokens for x in t]
    target, paths, following = ref.verify(logits[lead:len(logits) - tail].float().cpu().numpy(), tokens, parents)
    most = max(map(len, parents))
    cu = np.concatenate([[0], np.cumsum([len(t) for t in parents])]).astype(np.int32) + lead
    got = paged_ops.tree_verify(logits, torch.tensor([0] * lead + flat_t + [0] * tail, device=gpu),
                                torch.tensor([-1] * lead + flat_p + [-1] * tail, dtype=torch.int32, device=gpu),
                                torch.from_numpy(cu).to(gpu), most)
    torch.cuda.synchronize()
    assert got[0][lead:len(logits) - tail].tolist() == target
    assert got[1].tolist() == [p + [-1] * (most - len(p)) for p in paths]
    assert got[2].tolist() == [len(p) for p in paths]
    assert got[3].tolist() == following
    return got


def test_tree_verify_rows_of_nobody_strides_and_odd_starts(gpu):
    announce("tree_verify strided rows")
    for dtype, vocab, shift in (("bfloat16", 1000, 3), ("float32", 517, 1), ("float16", 2048, 5)):
        logits, tokens, parents = verify_inputs(dtype, vocab, [6, 3], 8)
        wide = torch.zeros(9 + 5, vocab + 11, dtype=DTYPES[dtype], device=gpu)
        wide[2:11, shift:shift + vocab] = logits.to(gpu)
        wide[0, shift + 17] = wide[13, shift + 400] = 3.0
        got = check_verify(gpu, wide[:, shift:shift + vocab], tokens, parents, lead=2, tail=3)
        assert got[0][[0, 1, 11, 12, 13]].tolist() == [17, 0, 0, 0, 400]  # every row has its target


def test_tree_verify_many_rows_is_the_same_every_time(gpu):
    announce("tree_verify repeated")
    logits, tokens, parents = verify_inputs("bfloat16", 5000, [40, 17, 1], 2)
    first = check_verify(gpu, logits.to(gpu), tokens, parents)
    again = check_verify(gpu, logits.to(gpu), tokens, parents)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def commit_want(pool, tables, starts, paths, bs):
    out = pool.clone()
    for table, start, path in zip(tables, starts, paths):
        for d, i in enumerate(path):
            a, b = start + i, start + d
            out[:, table[b // bs], :, b % bs] = pool[:, table[a // bs], :, a % bs]
    return out


@pytest.mark.parametrize("dtype,d", [("float16", 64), ("bfloat16", 128), ("float32", 64), ("float16", 5), ("float16", 6)])
@pytest.mark.parametrize("bs", [16, 1, 4])
def test_tree_commit(gpu, dtype, d, bs):
    from engine import paged_ops

    announce(f"tree_commit {dtype} d={d} bs={bs}")
    starts = [0, 7, 30, 15, 3, 50]
    paths = [[0], [0, 2, 3, 4, 9], [0, 1, 5, 6, 7, 8, 9, 10, 11, 12, 13, 20, 21, 39], list(range(30)),
             list(range(0, 60, 2)), []]
    step = Step("float16", 8, 1, 1, bs, starts, [64] * 6, seed=1)
    gen = torch.Generator().manual_seed(4)
    pools = [torch.randn(3, step.k.shape[0], 2, bs, d, generator=gen).to(DTYPES[dtype]) for _ in range(2)]
    for p in pools:
        p[1, ::3] = math.nan
    k, v = (p.to(gpu) for p in pools)
    path = torch.tensor([p + [-1] * (30 - len(p)) for p in paths], dtype=torch.int32, device=gpu)
    counts = torch.tensor([len(p) for p in paths], dtype=torch.int32, device=gpu)
    paged_ops.tree_commit(k, v, step.to(gpu)["block_tables"], torch.tensor(starts, dtype=torch.int32, device=gpu), path,
                          counts)
    torch.cuda.synchronize()
    raw = torch.int32 if dtype == "float32" else torch.int16
    for got, pool in zip((k, v), pools):
        assert torch.equal(got.cpu().view(raw), commit_want(pool, step.tables, starts, paths, bs).view(raw))


def test_tree_commit_ends_at_a_bad_entry(gpu):
    """An entry that does not rise, or whose place lies outside the table or the pool, ends its path."""
    from engine import paged_ops

    announce("tree_commit bad entries")
    bs, starts = 4, [0, 0, 0, 2, 0]
    tables = [[0, 1, 2], [3, 4, 5], [6, 7, 8], [9, 10, 11], [12, 99, 13]]
    given = [[0, 2, 1, 5], [0, 3, -1, 6], [1, 2, 1, 4], [0, 3, 11, 5], [0, 2, 4, 9]]
    done = [[0, 2], [0, 3], [1, 2], [0, 3], [0, 2]]
    pool = torch.randn(2, 15, 1, bs, 8).half()
    k, v = pool.to(gpu), (-pool).to(gpu)
    i32 = dict(dtype=torch.int32, device=gpu)
    paged_ops.tree_commit(k, v, torch.tensor(tables, **i32), torch.tensor(starts, **i32), torch.tensor(given, **i32),
                          torch.full((5,), 4, **i32))
    torch.cuda.synchronize()
    assert torch.equal(k.cpu(), commit_want(pool, tables, starts, done, bs))
    assert torch.equal(v.cpu(), commit_want(-pool, tables, starts, done, bs))


def test_two_streams_with_their_own_scratch(gpu):
    from engine import paged_ops

    announce("paged_tree and tree_verify on two streams")
    steps = [Step("bfloat16", 64, 14, 2, 16, [4000, 50], [5, 12], seed=s) for s in (1, 2)]
    args = [s.to(gpu) for s in steps]
    need = paged_ops.tree_workspace_bytes(2, 12, 14, 2, 64, 16, args[0]["block_tables"].shape[1], torch.bfloat16)
    assert need > 0
    want = [paged_ops.paged_tree(**a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    work = [torch.empty(need, dtype=torch.uint8, device=gpu) for _ in args]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for a, s, ws in zip(args, streams, work):
            with torch.cuda.stream(s):
                got.append(paged_ops.paged_tree(**a, workspace=ws))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, want[i % 2])


def test_calls_on_two_streams_and_two_graphs_do_not_meet(gpu):
    """Without ``workspace`` every call has scratch memory of its own: calls in flight on two streams, and two captured
    graphs replayed on two streams, give what each gives alone."""
    from engine import paged_ops

    announce("paged_tree and tree_verify on two streams, eager and captured")
    args = [Step("bfloat16", 64, 14, 2, 16, [4000, 50], [5, 12], seed=s).to(gpu) for s in (1, 2)]
    logits = [torch.randn(17, 50000, device=gpu) for _ in args]
    tokens, parents = torch.zeros(17, dtype=torch.int64, device=gpu), torch.zeros(17, dtype=torch.int32, device=gpu)

    def work(i):
        return (paged_ops.paged_tree(**args[i]), *paged_ops.tree_verify(logits[i], tokens, parents, args[i]["cu_q"], 12))

    want = [work(i) for i in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = []
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, work(i)))
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in args], []
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            outs.append(work(i))
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        got += [(i, [x.clone() for x in o]) for i, o in enumerate(outs)]
        torch.cuda.synchronize()
    for i, out in got:
        assert all(torch.equal(x, y) for x, y in zip(out, want[i]))


def test_index_of_a_padded_batch(gpu):
    """Rows of no node (ahead of the first tree, behind the last, past max_q_len) get slot -1 and no bits."""
    from engine import paged_ops

    announce("tree_index padded")
    i32 = dict(dtype=torch.int32, device=gpu)
    for most, sizes in ((3, [5, 2]), (70, [90, 3])):
        n = 2 + sum(sizes) + 4
        parents = torch.tensor([9, 9] + [p for k in sizes for p in range(-1, k - 1)] + [9] * 4, **i32)
        cu = torch.tensor([2, 2 + sizes[0], 2 + sum(sizes)], **i32)
        tables = torch.tensor([[4] * 8, [6] * 8], **i32)
        pos, slots, mask = paged_ops.tree_index(parents, cu, torch.tensor([10, 3], **i32), tables, most, 16)
        live = [2 + i for i in range(most)] + [2 + sizes[0] + i for i in range(sizes[1])]
        want = ref.index([range(-1, most - 1), range(-1, sizes[1] - 1)], [10, 3], [[4] * 8, [6] * 8], 16, 8, mask.shape[1])
        for got, full, blank in zip((pos, slots, mask), want, (0, -1, 0)):
            got = got.cpu().numpy()
            assert np.array_equal(got[live], full)
            assert (np.delete(got, live, axis=0) == blank).all()
    pos, slots, mask = paged_ops.tree_index(torch.zeros(3, **i32), torch.zeros(1, **i32), torch.zeros(0, **i32),
                                            torch.zeros(0, 1, **i32), 0, 16)
    assert pos.tolist() == [0] * 3 and slots.tolist() == [-1] * 3 and mask.shape == (3, 0)


def test_a_captured_step_replays_on_new_inputs(gpu):
    """Index, attention, verification and move in one graph: every replay equals the eager calls on what the
    buffers hold then, eager work between the replays."""
    from engine import paged_ops

    announce("tree operators captured")
    step = Step("float16", 64, 14, 2, 16, [3000, 20, 90], [5, 12, 8], seed=3)
    a = step.to(gpu)
    parents = torch.tensor([p for t in step.parents for p in t], dtype=torch.int32, device=gpu)
    logits = torch.randn(25, 3000, device=gpu)
    tokens = torch.randint(0, 3000, (25,), device=gpu)
    pools = [a["k_cache"][None], a["v_cache"][None]]

    def work():
        pos, slots, mask = paged_ops.tree_index(parents, a["cu_q"], a["ctx_start"], a["block_tables"], 12, 16)
        out = paged_ops.paged_tree(**{**a, "mask": mask})
        target, path, counts, following = paged_ops.tree_verify(logits, tokens, parents, a["cu_q"], 12)
        paged_ops.tree_commit(*pools, a["block_tables"], a["ctx_start"], path, counts)
        return pos, slots, mask, out, target, path, counts, following

    keep = [p.clone() for p in pools]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for i in range(4):
        gen = torch.Generator(device=gpu).manual_seed(i)
        logits.normal_(generator=gen)
        best = logits.argmax(1)
        rows = torch.arange(25, device=gpu)
        up = rows - torch.arange(25, device=gpu) + torch.repeat_interleave(a["cu_q"][:-1].long(), torch.tensor(step.nodes, device=gpu))
        tokens.copy_(best[(up + parents).clamp(min=0)])
        a["ctx_start"].copy_(torch.tensor([3000 - 700 * i, 20 + i, 90], dtype=torch.int32))
        a["q"].normal_(generator=gen)
        for p, k in zip(pools, keep):
            p.copy_(k)
        graph.replay()
        torch.cuda.synchronize()
        got, moved = [x.clone() for x in outs], [p.clone() for p in pools]
        for p, k in zip(pools, keep):
            p.copy_(k)
        want = work()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert all(torch.equal(x, y) for x, y in zip(moved, pools))
        assert int(got[6].max()) > 1


def test_refusals(gpu):
    from engine import _native, paged_ops

    announce("tree operators: refused calls")
    step = Step("float16", 96, 4, 2, 16, [20], [3])
    with pytest.raises(_native.NativeError, match="unsupported shape"):
        paged_ops.paged_tree(**step.to(gpu))
    step = Step("float16", 64, 4, 2, 16, [5000], [3])
    a = step.to(gpu)
    for kw in (dict(workspace=torch.empty(64, dtype=torch.uint8, device=gpu)), dict(cu_q=a["cu_q"].cpu()),
               dict(mask=a["mask"].cpu())):
        with pytest.raises(ValueError):
            paged_ops.paged_tree(**{**a, **kw})
    with pytest.raises(_native.NativeError, match="unsupported shape"):
        paged_ops.tree_index(torch.zeros(3, dtype=torch.int32, device=gpu), a["cu_q"], a["ctx_start"], a["block_tables"],
                             1025, 16)
    with pytest.raises(_native.NativeError, match="invalid"):
        paged_ops.tree_index(torch.zeros(3, dtype=torch.int32, device=gpu), a["cu_q"], a["ctx_start"], a["block_tables"],
                             3, 24)
