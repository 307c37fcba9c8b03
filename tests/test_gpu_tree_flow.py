"""A model decoding with drafted trees on the GPU: the tokens and the cache are those of one token a step."""

from __future__ import annotations

import random

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

BS = 16


def make_model(gpu, dtype, heads=14, kv=2, head_dim=64):
    from engine.model import Qwen2Config, Qwen2ForCausalLM, random_init_

    cfg = Qwen2Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_layers=2, num_heads=heads,
                      num_kv_heads=kv, head_dim=head_dim)
    with torch.device(gpu):
        model = Qwen2ForCausalLM(cfg)
    return cfg, random_init_(model.to(gpu, dtype), seed=1, std=0.08)


def make_cache(cfg, dtype, gpu, **kw):
    from engine.kv_cache import PagedKVCache

    return PagedKVCache.for_model(cfg, num_blocks=96, block_size=BS, max_seqs=8, max_len=256, dtype=dtype, device=gpu, **kw)


def prefill(model, cache, slots, prompts, gpu):
    ctx = cache.packed_prefill_context(slots, [len(p) for p in prompts])
    ids = torch.tensor([t for p in prompts for t in p], device=gpu)[None]
    logits = model.compute_logits(model(ids, ctx.positions[None], ctx)[0, ctx.last_index])
    ctx.commit()
    return logits


def decode(model, cache, slots, tokens, gpu):
    for s in slots:
        assert cache.ensure_capacity(s, cache.lengths[s] + 1)
    ctx = cache.decode_context(slots)
    logits = model.compute_logits(model(torch.tensor(tokens, device=gpu)[:, None], ctx.positions[:, None], ctx)[:, -1])
    ctx.commit()
    return logits


def rows_of(cache, slot):
    n = cache.lengths[slot]
    table = torch.tensor(cache.block_tables[slot][:cache.blocks_for(n)], device=cache.k.device)
    return [x[:, table].transpose(1, 2).reshape(x.shape[0], x.shape[2], -1, x.shape[4])[:, :, :n] for x in (cache.k, cache.v)]


def draft(truth, at, rng, vocab, widths=(2, 2, 1)):
    """A tree under the last token whose branches hold the true continuation among wrong ones, at random places."""
    tokens, parents, true_node = [truth[at]], [-1], 0
    frontier = [0]
    for depth, width in enumerate(widths):
        nxt, right = [], rng.randrange(width)
        for node in frontier:
            for w in range(width):
                tokens.append(rng.randrange(vocab))
                parents.append(node)
                if node == true_node and w == right and rng.random() < 0.8:
                    tokens[-1] = truth[at + depth + 1]
                    hit = len(tokens) - 1
                    nxt.append(hit)
                else:
                    nxt.append(len(tokens) - 1)
        true_node = next((i for i in nxt if parents[i] == true_node and tokens[i] == truth[at + depth + 1]), -1)
        frontier = nxt
    return tokens, parents


@pytest.mark.parametrize("heads,kv,head_dim", [(14, 2, 64), (4, 4, 32), (4, 2, 128)])
@torch.inference_mode()
def test_trees_give_the_tokens_and_the_cache_of_plain_decoding(gpu, heads, kv, head_dim):
    """fp32: the accepted tokens are the greedy ones (the top two logits differ by far more than rounding), every step's
    logits on the path match decoding's, and so do the cached rows."""
    announce(f"tree decoding {heads}q/{kv}kv d{head_dim}")
    cfg, model = make_model(gpu, torch.float32, heads, kv, head_dim)
    rng = random.Random(3)
    prompts = [[rng.randrange(512) for _ in range(n)] for n in (5, 33, 16)]
    plain = make_cache(cfg, torch.float32, gpu)
    slots = [plain.allocate(len(p)) for p in prompts]
    logits = prefill(model, plain, slots, prompts, gpu)
    truth, seen = [[] for _ in prompts], []
    for _ in range(30):
        top = logits.topk(2, dim=-1).values
        assert float((top[:, 0] - top[:, 1]).min()) > 1e-3
        for t, x in zip(truth, logits.argmax(-1).tolist()):
            t.append(x)
        seen.append(logits)
        logits = decode(model, plain, slots, [t[-1] for t in truth], gpu)

    cache = make_cache(cfg, torch.float32, gpu)
    mine = [cache.allocate(len(p)) for p in prompts]
    first = prefill(model, cache, mine, prompts, gpu).argmax(-1).tolist()
    out = [[x] for x in first]
    steps = accepted = 0
    while min(map(len, out)) < 24:
        live = [i for i in range(3) if len(out[i]) < 24]
        trees = [draft(truth[i], len(out[i]) - 1, rng, 512, rng.choice([(2, 2, 1), (3,), (1, 1, 1, 1), ()])) for i in live]
        ctx = cache.tree_context([mine[i] for i in live], [t for t, _ in trees], [p for _, p in trees])
        hidden = model(ctx.input_ids[None], ctx.positions[None], ctx)
        logits = model.compute_logits(hidden[0])
        scale = float(logits.abs().max())
        row = 0
        for i, (toks, _) in zip(live, trees):  # the root's logits are decoding's for that token
            assert float((logits[row] - seen[len(out[i])][i]).abs().max()) < 1e-4 * scale
            row += len(toks)
        new = ctx.accept(logits)
        for i, got in zip(live, new):
            assert got and got == truth[i][len(out[i]):len(out[i]) + len(got)]
            out[i] += got
            accepted += len(got)
        steps += len(live)
    assert accepted > 1.3 * steps  # drafts were accepted, not roots alone
    for i, slot in enumerate(mine):
        n = cache.lengths[slot]
        assert n == len(prompts[i]) + len(out[i]) - 1  # the last token is not cached
        for got, want in zip(rows_of(cache, slot), rows_of(plain, slots[i])):
            assert float((got - want[:, :, :n]).abs().max()) < 1e-4 * float(want.abs().max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@torch.inference_mode()
def test_a_path_of_a_tree_is_a_chain(gpu, dtype):
    """The logits of the nodes on one path equal those of the same tokens as a packed prefill's, and accepting the path
    leaves the same rows (16 bits: what differs is the order of sums, a few roundings of the activations)."""
    announce(f"tree path against prefill {dtype}")
    cfg, model = make_model(gpu, dtype)
    rng = random.Random(4)
    prompt, path = [rng.randrange(512) for _ in range(50)], [rng.randrange(512) for _ in range(4)]
    a, b = make_cache(cfg, dtype, gpu), make_cache(cfg, dtype, gpu)
    sa, sb = a.allocate(50), b.allocate(50)
    for c, s in ((a, sa), (b, sb)):
        prefill(model, c, [s], [prompt], gpu)
    ctx = a.packed_prefill_context([sa], [4])
    want = model.compute_logits(model(torch.tensor([path], device=gpu), ctx.positions[None], ctx)[0])
    ctx.commit()
    tokens = [path[0], 9, path[1], 8, 7, path[2], 6, path[3]]
    tree = b.tree_context([sb], [tokens], [[-1, 0, 0, 1, 2, 2, 3, 5]])
    got = model.compute_logits(model(tree.input_ids[None], tree.positions[None], tree)[0])
    nodes = [0, 2, 5, 7]
    tol = 2e-2 if dtype == torch.bfloat16 else 4e-3
    assert float((got[nodes].float() - want.float()).abs().max()) < tol * float(want.float().abs().max())
    assert tree.commit(torch.tensor([nodes], dtype=torch.int32, device=gpu), torch.tensor([4], dtype=torch.int32, device=gpu)) == [nodes]
    assert b.lengths[sb] == 54
    for x, y in zip(rows_of(b, sb), rows_of(a, sa)):
        assert float((x.float() - y.float()).abs().max()) < tol * float(y.float().abs().max())
    with pytest.raises(RuntimeError, match="have been committed"):
        tree.commit(torch.tensor([nodes], dtype=torch.int32, device=gpu), torch.tensor([4], dtype=torch.int32, device=gpu))


@torch.inference_mode()
def test_a_forked_sequence_keeps_its_rows(gpu):
    """A tree on a fork writes into private copies: the parent's rows stay, in the shared partial block too."""
    announce("tree on a fork")
    cfg, model = make_model(gpu, torch.bfloat16)
    cache = make_cache(cfg, torch.bfloat16, gpu)
    rng = random.Random(5)
    slot = cache.allocate(40)
    prefill(model, cache, [slot], [[rng.randrange(512) for _ in range(40)]], gpu)
    before = [x.clone() for x in rows_of(cache, slot)]
    child = cache.fork(slot)
    ctx = cache.tree_context([child], [[1, 2, 3, 4]], [[-1, 0, 0, 2]])
    logits = model.compute_logits(model(ctx.input_ids[None], ctx.positions[None], ctx)[0])
    new = ctx.accept(logits)
    assert cache.cow_copies == 1 and cache.lengths[child] == 40 + len(new[0])
    for x, y in zip(rows_of(cache, slot), before):
        assert torch.equal(x, y)
    assert cache.block_tables[slot][2] != cache.block_tables[child][2]


def test_trees_that_do_not_fit_are_refused(gpu):
    from engine.kv_cache import PagedKVCache

    announce("tree context refusals")
    cache = PagedKVCache(1, 2, 64, num_blocks=4, block_size=4, max_seqs=2, max_len=14, dtype=torch.float16, device=gpu)
    slot = cache.allocate(10)
    cache.lengths[slot] = 10
    with pytest.raises(ValueError, match="no room"):
        cache.tree_context([slot], [[1] * 5], [[-1, 0, 0, 0, 0]])
    ctx = cache.tree_context([slot], [[1] * 4], [[-1, 0, 0, 0]])
    i32 = dict(dtype=torch.int32, device=gpu)
    for path, count in (([[1, 2]], [2]), ([[0, 2, 1]], [3]), ([[0, 4]], [2]), ([[0]], [0])):
        with pytest.raises(ValueError, match="not a path"):
            ctx.commit(torch.tensor(path, **i32), torch.tensor(count, **i32))
    with pytest.raises(ValueError, match="paths for"):
        ctx.commit(torch.zeros(2, 1, **i32), torch.ones(2, **i32))
    assert ctx.commit(torch.tensor([[0, 3]], **i32), torch.tensor([2], **i32)) == [[0, 3]]
    assert cache.lengths[slot] == 12


@torch.inference_mode()
def test_layer_calls_that_change_layout_are_checked_again(gpu):
    """The step's cached layer call serves calls of one layout; others run their own full call, with the same result."""
    from engine import paged_ops

    announce("tree layer calls")
    from engine.kv_cache import PagedKVCache

    cache = PagedKVCache(3, 2, 64, num_blocks=20, block_size=16, max_seqs=2, max_len=200, dtype=torch.float16, device=gpu)
    slot = cache.allocate(100)
    cache.lengths[slot] = 100
    cache.k.normal_()
    cache.v.normal_()
    ctx = cache.tree_context([slot], [[1, 2, 3]], [[-1, 0, 0]])
    for layer in range(3):
        q = torch.randn(1, 6, 3, 64, device=gpu).half()
        if layer == 2:
            q = torch.randn(1, 3, 6, 64, device=gpu).half().transpose(1, 2)
        k, v = (torch.randn(1, 2, 3, 64, device=gpu).half() for _ in range(2))
        out = ctx.attend(layer, q, k, v)
        want = paged_ops.paged_tree(q[0].transpose(0, 1), cache.k[layer], cache.v[layer], ctx.block_tables, ctx.cu_q,
                                    ctx.ctx_start, ctx.mask, 3)
        torch.cuda.synchronize()
        assert out.shape == (1, 6, 3, 64) and torch.equal(out[0].transpose(0, 1), want)


@torch.inference_mode()
def test_captured_layer_calls_replay_on_new_inputs(gpu):
    """A step's layer calls in a graph (long context: scratch memory in use): every replay equals the eager calls on
    what the buffers hold then, eager calls of the same step between the replays."""
    from engine.kv_cache import PagedKVCache

    announce("captured tree layer calls")
    cache = PagedKVCache(2, 2, 64, num_blocks=300, block_size=16, max_seqs=2, max_len=4600, dtype=torch.bfloat16, device=gpu)
    slot = cache.allocate(4500)
    cache.lengths[slot] = 4500
    cache.k.normal_()
    cache.v.normal_()
    ctx = cache.tree_context([slot], [[1] * 9], [[-1, 0, 0, 1, 1, 2, 3, 4, 4]])
    q = torch.randn(2, 1, 9, 14, 64, device=gpu).bfloat16().transpose(2, 3)
    k, v = (torch.randn(2, 1, 9, 2, 64, device=gpu).bfloat16().transpose(2, 3) for _ in range(2))

    def work():
        return [ctx.attend(layer, q[layer], k[layer], v[layer]) for layer in range(2)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for seed in range(4):
        gen = torch.Generator(device=gpu).manual_seed(seed)
        for x in (q, k, v):
            x.normal_(generator=gen)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs]
        want = work()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert float(got[0].float().abs().max()) > 0
