"""Drafted-tree attention where rounding or the range of fp32 shows, against the plain 64-bit form.

Bound of an output element (see test_gpu_tree.py for the scores): a weight is off by a relative
delta = (D + 2) 2^-24 reach + 2^-21 (score, exp2) and, on the 16-bit matrix cores, by what is left of it beside its two
16-bit parts: a part rounds to half a step h (fp16 2^-11, bf16 2^-8), so two leave h^2 of it at most, fp16 parts 2^-32
of the row's largest weight besides. Weights enter the sum and the normaliser; fp32 sums over n keys add n 2^-23. Times
the weighted mean of |v|, and half a step of the output on top, nothing absolute.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from conftest import announce
from test_gpu_tree import DTYPES, Step, run, widened

pytestmark = pytest.mark.gpu


def bound_of(step, out, spread, reach, keys):
    half_step = torch.finfo(DTYPES[step.dtype]).eps / 2
    delta = (step.d + 2) * 2.0**-24 * reach + 2.0**-21 + keys * 2.0**-23
    if step.dtype != "float32":
        delta = delta + half_step**2 + keys * 2.0**-32
    least = torch.finfo(DTYPES[step.dtype]).smallest_normal * half_step
    return 1.01 * half_step * np.abs(out) + 2.05 * delta[..., None] * spread + least


def wide(step, gpu, large):
    """The call's arguments; large False: as they are, None: with tables of 2000 tokens, at which the matrix cores are taken
    for short contexts too, True: with tables at which a call of more than 64 rows is a large one."""
    args = step.to(gpu)
    if large is None:
        tab = torch.full((len(step.nodes), max(2000 // step.bs, step.width())), -1, dtype=torch.int32, device=gpu)
        tab[:, :args["block_tables"].shape[1]] = args["block_tables"]
        return {**args, "block_tables": tab}
    return widened(step, args) if large else args


@pytest.mark.parametrize("dtype,d,hq,hkv,bs,nodes,large", [
    ("float32", 32, 4, 2, 16, [3], False), ("bfloat16", 32, 4, 2, 16, [3], False), ("float16", 256, 2, 1, 16, [3], False),
    ("bfloat16", 64, 4, 2, 16, [3], False), ("float32", 64, 4, 2, 16, [3], False), ("float32", 128, 28, 4, 16, [30], False),
    ("float16", 64, 14, 2, 16, [9], None), ("bfloat16", 128, 28, 4, 16, [40], None), ("bfloat16", 64, 14, 2, 16, [40], True), ("bfloat16", 128, 28, 4, 16, [40], True)])
def test_scores_below_fp32_weigh_nothing(gpu, dtype, d, hq, hkv, bs, nodes, large):
    """A product within fp32 whose score passes its range: -inf, in the first keys that are met and among later ones."""
    announce(f"paged_tree scores below fp32 {dtype} d={d} nodes={nodes} large={large}")
    step = Step(dtype, d, hq, hkv, bs, [150], nodes, seed=41, kind="free", scale=2.0**125)
    step.qkv.zero_()
    step.qkv[:, 0:hq * d:d] = 1.0
    step.k.zero_()
    for key in [*range(64), 70, 99, 140]:
        step.k[step.tables[0][key // bs], :, key % bs, 0] = -16.0  # score -2^129
    got = run(gpu, step, **wide(step, gpu, large)).double().cpu().numpy()
    out, spread, reach = step.want()
    assert np.isfinite(got).all()
    assert (np.abs(got - out) <= bound_of(step, out, spread, 0 * reach, 200)).all()  # the seen scores are 0, exactly


def cancelling(dtype, d, hq, hkv, bs, nodes, mean, keys=9, seed=42):
    """Cached keys with scores of 0 to 1, and values whose weighted mean is about ``mean`` / 9 in every dim: what a weight is
    off by shows in the output, whose own rounding is small. The nodes are seen by nobody."""
    step = Step(dtype, d, hq, hkv, bs, [keys], nodes, seed=seed, kind="free", scale=1.0)
    step.mask[:] = 0
    step.qkv.zero_()
    step.qkv[:, 0:hq * d:d] = 1.0
    gen = torch.Generator().manual_seed(seed)
    at = [(step.tables[0][p // bs], p % bs) for p in range(keys)]
    for h in range(hkv):
        score = torch.rand(keys, generator=gen).to(DTYPES[dtype])
        w = torch.exp(score.double())
        v = torch.randn(keys, d, generator=gen).to(DTYPES[dtype])
        v[-1] = (-(w[:-1, None] * v[:-1].double()).sum(0) / w[-1] + mean).to(v.dtype)
        for (b, o), s, row in zip(at, score, v):
            step.k[b, h, o] = 0
            step.k[b, h, o, 0] = s
            step.v[b, h, o] = row
    return step


SIZES = [(d, hq, hkv, bs, [n], False, 0.0) for d, hq, hkv, bs in ((64, 14, 2, 16), (128, 28, 4, 32)) for n in (2, 4, 9, 40)]
LARGE_SIZES = [(d, hq, hkv, bs, [40], True, mean) for d, hq, hkv, bs in ((64, 14, 2, 16), (128, 28, 4, 32)) for mean in (0.0, 0.02)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,hq,hkv,bs,nodes,large,mean", SIZES + LARGE_SIZES)
def test_weights_keep_their_bits(gpu, dtype, d, hq, hkv, bs, nodes, large, mean):
    announce(f"paged_tree cancelling values {dtype} d={d} nodes={nodes} large={large}")
    step = cancelling(dtype, d, hq, hkv, bs, nodes, mean)
    got = run(gpu, step, **wide(step, gpu, large or None)).double().cpu().numpy()
    out, spread, reach = step.want()
    assert np.abs(out).max() < 0.02 * spread.max()
    err, bound = np.abs(got - out), bound_of(step, out, spread, reach, 9)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("d,hq,hkv", [(64, 14, 2), (128, 28, 4)])
@pytest.mark.parametrize("small", [2.0**-19, 2.0**-26, 2.0**-60])
@pytest.mark.parametrize("zeros", [False, True])
def test_a_row_of_small_values_beside_ordinary_ones(gpu, d, hq, hkv, small, zeros):
    """Nothing cached: a root that sees itself alone, a node that sees it and another small one; with and without a dim of zeros."""
    announce(f"paged_tree large call, one row of {small} d={d}")
    step = Step("bfloat16", d, hq, hkv, 16, [0, 31], [40, 12], seed=43, kind="free")
    step.mask[0], step.mask[7] = 1, (1 << 7) | 1
    for node in (0, 7):
        step.v[step.tables[0][node // 16], :, node % 16] *= small
    if zeros:
        step.v[..., 5] = 0
    got = run(gpu, step, **wide(step, gpu, True)).double().cpu().numpy()
    out, spread, reach = step.want()
    err, bound = np.abs(got - out), bound_of(step, out, spread, reach, 52)
    assert (err <= bound).all(), float((err / bound).max())
    assert np.abs(got[[0, 7]]).max() > 0 and (got[..., 5] == 0).all() == zeros


def test_of_siblings_with_one_token_the_first_is_taken(gpu):
    """Whatever follows the others, in kernel and plain form alike; the tokens are the greedy ones in any case."""
    from oracle import tree_ref as ref
    from test_gpu_tree import check_verify

    announce("tree_verify equal siblings")
    logits = np.full((6, 10), -1.0)
    for r, t in enumerate([5, 7, 7, 2, 3, 0]):
        logits[r, t] = 1.0
    tokens, parents = [[1, 5, 5, 7, 7, 2]], [[-1, 0, 0, 2, 2, 3]]
    _, paths, following = ref.verify(logits, tokens, parents)
    assert paths == [[0, 1]] and following == [7]
    check_verify(gpu, torch.from_numpy(logits).float().to(gpu), tokens, parents)


@torch.inference_mode()
def test_layer_calls_of_a_step_on_two_streams(gpu):
    """A step's later layer calls, in flight on two streams at once, give what each gives alone (a long context, whose
    pieces meet in scratch memory)."""
    from engine.kv_cache import PagedKVCache

    announce("tree layer calls on two streams")
    cache = PagedKVCache(2, 2, 64, num_blocks=300, block_size=16, max_seqs=2, max_len=4600, dtype=torch.bfloat16, device=gpu)
    slot = cache.allocate(4500)
    cache.lengths[slot] = 4500
    cache.k.normal_()
    cache.v.normal_()
    ctx = cache.tree_context([slot], [[1] * 9], [[-1, 0, 0, 1, 1, 2, 3, 4, 4]])
    q = [torch.randn(1, 9, 14, 64, device=gpu).bfloat16().transpose(1, 2) for _ in range(2)]
    want = [ctx.calls.attend(layer, q[layer], cache.k, cache.v) for layer in range(2)]
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(6):
        for layer, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((layer, ctx.calls.attend(layer, q[layer], cache.k, cache.v)))
    torch.cuda.synchronize()
    for layer, out in got:
        assert torch.equal(out, want[layer])
