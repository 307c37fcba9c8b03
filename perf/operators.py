"""Operators of speculative decoding over the paged KV cache, with their plain forms and what they cost.

A step of speculative decoding verifies, for each sequence, a small tree of drafted tokens in one pass
of the model: node 0 is the sequence's last token, every other node a drafted token that continues its
parent. Four operators make up the step beside the model's own layers:

``attend``   attention of every node over its sequence's cached keys and the nodes on its path to the
             root, read in place from the pool (``paged_ops.paged_tree``).
``index``    from the trees' parents and the sequences' lengths and block tables: every node's position,
             pool slot and the bit set of the nodes it sees (``paged_ops.tree_index``).
``verify``   the model's choice after every node, and the longest drafted path that agrees with it
             (``paged_ops.tree_verify``).
``commit``   the accepted nodes' keys and values moved to the consecutive places that a cache of the
             accepted tokens has them in, all layers (``paged_ops.tree_commit``).

``listed()`` names the cases and ``draw(rng)`` gives more of the same ranges. A case's lengths come from
the case alone (``mix`` seeds them); values, trees and block placement come from the seed. With ``own``
false, ``run`` computes the plain forms in elementary torch operations, in 32 bits.
"""

from __future__ import annotations

import math
import random
import sys
from functools import reduce
from pathlib import Path

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, dtype, seqs, lo, hi, n_lo, n_hi, heads=14, kv_heads=2, head_dim=64, block=16, layers=1,
          vocab=151936, tree="wide", log=False, mix=0):
    c = {"op": op, "dtype": dtype, "seqs": seqs, "lo": lo, "hi": hi, "n_lo": n_lo, "n_hi": n_hi, "heads": heads,
         "kv_heads": kv_heads, "head_dim": head_dim, "block": block, "layers": layers, "vocab": vocab, "tree": tree,
         "log": log, "mix": mix}
    return {"name": name, **c} if name else c


def listed():
    big = {"heads": 28, "kv_heads": 4, "head_dim": 128, "block": 32}  # the 7B-class head shape
    return [
        # One user, a chat turn just begun, four tokens drafted in a row: nothing but latency.
        _case("attend_bf16_one", "attend", "bf16", 1, 37, 37, 5, 5, tree="chain"),
        # A lightly loaded server, trees of 8 to 24 nodes.
        _case("attend_fp16_b32", "attend", "fp16", 32, 128, 1024, 8, 24),
        # A full server with large trees: the case with the most products for each key read.
        _case("attend_bf16_b64", "attend", "bf16", 64, 128, 4096, 33, 64, log=True),
        # One user on a long document: the keys of few rows, to be split over the chip.
        _case("attend_bf16_long", "attend", "bf16", 1, 32000, 32000, 61, 61, **big),
        # A full batch of long contexts, short drafts: the most keys and values read.
        _case("attend_bf16_d128_b128", "attend", "bf16", 128, 512, 8192, 4, 8, log=True, **big),
        # A numerics run in fp32.
        _case("attend_fp32_b8", "attend", "fp32", 8, 16, 256, 2, 7),
        # The indexes of one user's step, and of a full batch's.
        _case("index_one", "index", "bf16", 1, 37, 37, 5, 5, tree="chain"),
        _case("index_b256", "index", "bf16", 256, 128, 4096, 17, 64, log=True),
        # Verification over the vocabulary of the 0.5B configuration: one user; a batch with fp32 logits.
        _case("verify_bf16_one", "verify", "bf16", 1, 37, 37, 5, 5, tree="chain"),
        _case("verify_fp32_b64", "verify", "fp32", 64, 128, 1024, 9, 16),
        # The accepted tokens of one user (24 layers), and of a batch at the 7B-class shape (28 layers).
        _case("commit_fp16_one", "commit", "fp16", 1, 100, 100, 16, 16, layers=24),
        _case("commit_bf16_b64", "commit", "bf16", 64, 64, 512, 17, 64, layers=28, **big),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: the same operators, head shapes, types and ranges of lengths."""
    op = rng.choice(("attend", "attend", "attend", "attend", "index", "verify", "verify", "commit"))
    mix = rng.randrange(1, 1 << 20)
    tree = rng.choice(("wide", "wide", "chain", "free" if op == "attend" else "wide"))
    dtype = rng.choice(("fp16", "bf16", "fp16", "bf16", "fp32"))
    n_hi = _log_int(rng, 1, 128 if op in ("attend", "index") else 48)
    n_lo = rng.randint(max(1, n_hi // 3), n_hi)
    if op == "attend":
        kv, group, d = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 6, 7, 8)), rng.choice((64, 64, 128))
        hi = _log_int(rng, 8, 2048 if dtype == "fp32" else 16384)
        # Within the largest listed case: so many keys, and so many products.
        most = min((1 << 27) // (hi * kv * d), (1 << 32) // (hi * n_hi * kv * group * d), 128)
        seqs = _log_int(rng, 1, max(1, most))
        return _case("", op, dtype, seqs, rng.choice((0, 1 + hi // 16, hi)), hi, n_lo, n_hi, kv * group, kv, d,
                     rng.choice((16, 32, 64, 8)), tree=tree, mix=mix)
    if op == "index":
        return _case("", op, "bf16", _log_int(rng, 1, 256), 0, _log_int(rng, 16, 8192), n_lo, n_hi,
                     block=rng.choice((8, 16, 32)), tree=tree, mix=mix)
    if op == "verify":
        vocab = rng.choice((151936, 152064, _log_int(rng, 1000, 160000)))
        seqs = _log_int(rng, 1, max(1, min(64, 800 // n_hi)))
        return _case("", op, dtype, seqs, 1, 64, n_lo, n_hi, vocab=vocab, tree=tree, mix=mix)
    kv, d = rng.choice(((2, 64), (4, 128), (8, 64)))
    return _case("", op, dtype, _log_int(rng, 1, 64), 0, _log_int(rng, 16, 512), n_lo, n_hi, 7 * kv, kv, d,
                 rng.choice((16, 32)), layers=rng.randint(1, 28) if dtype != "fp32" else rng.randint(1, 12), mix=mix)


# ---------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Cached tokens and drafted nodes (the root among them) of each sequence."""
    rng = random.Random(case["mix"] * 1009 + case["seqs"])
    log = case["log"]
    ctx = [_log_int(rng, case["lo"], case["hi"]) if log else rng.randint(case["lo"], case["hi"])
           for _ in range(case["seqs"])]
    return ctx, [rng.randint(case["n_lo"], case["n_hi"]) for _ in ctx]


def _paths(case):
    """The nodes that each sequence accepts. The first lie in place already, the others behind all the places that
    are written, so that the same pass can be made again."""
    rng, paths = random.Random(case["mix"] + 5), []
    for n in _lengths(case)[1]:
        c = rng.randint(1, min(n, 8))
        keep = max(rng.randint(1, min(c, 2)), 2 * c - n)
        paths.append(list(range(keep)) + sorted(rng.sample(range(c, n), c - keep)))
    return paths


def _parents(kind, n, rng):
    """A tree of n nodes, parents before children: a chain, or one that thins out with depth, as drafting makes them."""
    if kind == "chain":
        return [i - 1 for i in range(n)]
    return [-1] + [max(0, min(rng.randrange(i), rng.randrange(i))) for i in range(1, n)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tables(case, ctx, nodes, rng):
    """Block tables of sequences whose blocks lie anywhere in the pool (a few blocks are nobody's)."""
    need = [max(1, -(-(a + n) // case["block"])) for a, n in zip(ctx, nodes)]
    ids = list(range(sum(need) + 8))
    rng.shuffle(ids)
    rows, at = torch.zeros(len(need), max(need), dtype=torch.int32), 0
    for i, k in enumerate(need):
        rows[i, :k] = torch.tensor(ids[at:at + k], dtype=torch.int32)
        at += k
    return rows.cuda(), len(ids)


def _bit_words(seen, words):
    """Sets of node numbers as rows of 64-bit words (two's complement)."""
    rows = []
    for s in seen:
        x = sum(1 << j for j in s)
        rows.append([((x >> (64 * w)) + (1 << 63)) % (1 << 64) - (1 << 63) for w in range(words)])
    return torch.tensor(rows, dtype=torch.int64).reshape(len(seen), words)


def _seen(parents):
    """The nodes on each node's path to its root, itself among them."""
    out = []
    for i, p in enumerate(parents):
        out.append(([] if p < 0 else out[p]) + [i])
    return out


def prepare(case, seed):
    rng = random.Random(seed * 7919 + 13)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ctx, nodes = _lengths(case)
    total, most, dtype = sum(nodes), max(nodes), DTYPES[case["dtype"]]
    trees = [_parents(case["tree"], n, rng) for n in nodes]
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    st = {"case": case, "ctx": ctx, "nodes": nodes, "trees": trees, "most": most, "cu_q": _i32(cu),
          "ctx_start": _i32(ctx), "parents": _i32([p for t in trees for p in t])}
    st["tables"], blocks = _tables(case, ctx, nodes, rng)
    hq, hkv, d, bs = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    if case["op"] == "attend":
        words = -(-most // 64)
        if case["tree"] == "free":  # any mask at all, rows that see no node among them
            seen = [[j for j in range(n) if rng.random() < 0.4] for n in nodes for _ in range(n)]
        else:
            seen = [s for t in trees for s in _seen(t)]
        st["mask"] = _bit_words(seen, words).cuda()
        st["k"], st["v"] = (torch.randn(blocks + 1, hkv, bs, d, generator=gen, device="cuda", dtype=dtype)
                            for _ in range(2))
        # q as a view of a projection's output rows, as an attention layer has it; scores of some spread.
        qkv = torch.randn(total, (hq + 2 * hkv) * d, generator=gen, device="cuda", dtype=dtype) * 2
        st["q"] = qkv[:, :hq * d].view(total, hq, d)
    elif case["op"] == "verify":
        logits = torch.randn(total, case["vocab"], generator=gen, device="cuda", dtype=torch.float32) * 3
        logits = logits.to(dtype)
        best = [rng.randrange(case["vocab"]) for _ in range(total)]
        rows, cols = torch.arange(total, device="cuda"), torch.tensor(best, device="cuda")
        logits[rows, cols] = 24.0
        logits[rows[::3], (cols[::3] + case["vocab"] // 2) % case["vocab"]] = 24.0  # ties
        first = [min(b, (b + case["vocab"] // 2) % case["vocab"]) if r % 3 == 0 else b for r, b in enumerate(best)]
        tokens = [rng.randrange(case["vocab"]) for _ in range(total)]
        for at, tree in zip(cu, trees):  # drafts that the model agrees with more often than not
            for i, p in enumerate(tree):
                if p >= 0 and rng.random() < 0.6:
                    tokens[at + i] = first[at + p]
        st["logits"], st["tokens"] = logits, torch.tensor(tokens, device="cuda")
    elif case["op"] == "commit":
        st["k"], st["v"] = (torch.randn(case["layers"], blocks + 1, hkv, bs, d, generator=gen, device="cuda",
                                        dtype=dtype) for _ in range(2))
        paths = _paths(case)
        st["path"], st["counts"] = _i32([p + [-1] * (most - len(p)) for p in paths]), _i32([len(p) for p in paths])
    return st


# ---------------------------------------------------------------------------------- plain forms
def _rows(st):
    """Each sequence's rows padded to the largest tree: their places in the packed rows, which are real, and each
    packed row's sequence."""
    cu = st["cu_q"].long()
    i = torch.arange(st["most"], device="cuda")
    real = i[None] < (cu[1:] - cu[:-1])[:, None]
    return torch.where(real, cu[:-1, None] + i, 0), real


def _packed(st, x):
    """Rows padded by sequence ``[S, m, ..]`` back in packed order ``[N, ..]``."""
    cu = st["cu_q"].long()
    r = torch.arange(st["parents"].shape[0], device="cuda")
    s = (r[:, None] >= cu[None, 1:]).sum(1)
    return x[s, r - cu[s]]


def _plain_attend(st):
    case, q, bs = st["case"], st["q"], st["case"]["block"]
    at, real = _rows(st)
    ctx, n = st["ctx_start"].long(), real.sum(1)
    pos = torch.arange(max(a + b for a, b in zip(st["ctx"], st["nodes"])), device="cuda")
    blk = st["tables"].long()[:, pos // bs]
    k, v = (st[x][blk, :, pos % bs].transpose(1, 2).float() for x in ("k", "v"))  # [S, hkv, keys, D]
    s_n, m, hq, hkv, d = at.shape[0], at.shape[1], case["heads"], case["kv_heads"], case["head_dim"]
    qp = q[at].float().transpose(1, 2).reshape(s_n, hkv, hq // hkv * m, d)
    # Key e nodes behind the cached ones is seen where bit e of the row's words is set.
    e = pos[None] - ctx[:, None]
    bits = ((st["mask"][at].unsqueeze(-1) >> torch.arange(64, device="cuda")) & 1).flatten(2)
    node = bits.gather(2, e.clamp(0, bits.shape[2] - 1)[:, None].expand(-1, m, -1)) == 1
    sees = (e < 0)[:, None] | ((e >= 0) & (e < n[:, None]))[:, None] & node
    scores = (qp @ k.transpose(-1, -2)).view(s_n, hkv, hq // hkv, m, -1) * (1.0 / math.sqrt(d))
    scores.masked_fill_(~sees[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p.view(s_n, hkv, -1, p.shape[-1]) @ v).view(s_n, hkv, hq // hkv, m, d)
    out = torch.where(total > 0, out / total, 0.0)
    return _packed(st, out.reshape(s_n, hq, m, d).transpose(1, 2)).to(q.dtype)


def _reach(st):
    """``[S, m, m]``: 1 where the column's node lies on the row's node's path to its root."""
    at, real = _rows(st)
    parent = torch.where(real, st["parents"].long()[at], -1)
    node = torch.arange(st["most"], device="cuda")
    step = ((parent[:, :, None] == node) | torch.eye(st["most"], dtype=torch.bool, device="cuda")).float()
    doublings = max(1, (st["most"] - 1).bit_length())
    return parent, real, at, reduce(lambda r, _: (r @ r).clamp_(max=1.0), range(doublings), step)


def _plain_index(st):
    bs = st["case"]["block"]
    _, _, _, reach = _reach(st)
    words = -(-st["most"] // 64)
    bits = torch.nn.functional.pad(reach, (0, 64 * words - st["most"])).long().unflatten(2, (words, 64))
    mask = (bits << torch.arange(64, device="cuda")).sum(-1)
    ctx, node = st["ctx_start"].long()[:, None], torch.arange(st["most"], device="cuda")[None]
    place = (ctx + node).clamp(max=st["tables"].shape[1] * bs - 1)
    slots = st["tables"].long().gather(1, place // bs) * bs + place % bs
    return _packed(st, ctx + reach.sum(-1).long() - 1), _packed(st, slots), _packed(st, mask)


def _plain_verify(st):
    x = st["logits"]
    col = torch.arange(x.shape[1], device="cuda", dtype=torch.int32)
    target = torch.where(x == x.amax(1, keepdim=True), col, x.shape[1]).amin(1).long()
    parent, real, at, reach = _reach(st)
    token, m = st["tokens"][at], st["most"]
    node = torch.arange(m, device="cuda")
    agrees = real & (parent >= 0) & (token == target[at].gather(1, parent.clamp(min=0)))
    twin = (parent[:, :, None] == parent[:, None, :]) & agrees[:, None, :] & (node[None, :] < node[:, None])
    good = (agrees & ~twin.any(-1)) | ((node == 0) & real)  # the first child that agrees; node 0 stands
    accepted = real & ((reach @ (~good).float().unsqueeze(-1)).squeeze(-1) == 0)
    counts = accepted.sum(1)
    path = torch.where(accepted, node, m).sort(1).values
    last = path.gather(1, (counts - 1).clamp(min=0)[:, None])
    following = torch.where(counts > 0, target[at].gather(1, last.clamp(max=m - 1)).squeeze(1), -1)
    return target, torch.where(path < m, path, -1).int(), counts.int(), following


def _plain_commit(st):
    bs, ctx, tables = st["case"]["block"], st["ctx_start"].long()[:, None], st["tables"].long()
    place = torch.arange(st["path"].shape[1], device="cuda")[None]
    moves = place < st["counts"][:, None]
    src, dst = (ctx + torch.where(moves, x, 0) for x in (st["path"].long(), place))
    # Where nothing is to move, row 0 of a sequence stands for both, which is a move of its own.
    (sb, so), (db, do) = ((tables.gather(1, x // bs), x % bs) for x in (src, dst))
    st["k"][:, db, :, do] = st["k"][:, sb, :, so]
    st["v"][:, db, :, do] = st["v"][:, sb, :, so]
    return st["k"], st["v"]


# ---------------------------------------------------------------------------------- one pass
def _ops():
    """The framework's tensor-level entry points."""
    package = str(Path(__file__).resolve().parent.parent / "mini-inference_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from engine import paged_ops

    return paged_ops


def _own_pass(st):
    ops, case = _ops(), st["case"]
    if case["op"] == "attend":
        return {"out": ops.paged_tree(st["q"], st["k"], st["v"], st["tables"], st["cu_q"], st["ctx_start"], st["mask"],
                                      st["most"])}
    if case["op"] == "index":
        positions, slots, mask = ops.tree_index(st["parents"], st["cu_q"], st["ctx_start"], st["tables"], st["most"],
                                                case["block"])
        return {"positions": positions, "slots": slots, "mask": mask}
    if case["op"] == "verify":
        target, path, counts, following = ops.tree_verify(st["logits"], st["tokens"], st["parents"], st["cu_q"],
                                                          st["most"])
        return {"target": target, "path": path, "counts": counts, "next": following}
    ops.tree_commit(st["k"], st["v"], st["tables"], st["ctx_start"], st["path"], st["counts"])
    return {"k": st["k"], "v": st["v"]}


def run(state):
    if own:
        return _own_pass(state)
    op = state["case"]["op"]
    if op == "attend":
        return {"out": _plain_attend(state)}
    if op == "index":
        return dict(zip(("positions", "slots", "mask"), _plain_index(state)))
    if op == "verify":
        return dict(zip(("target", "path", "counts", "next"), _plain_verify(state)))
    return dict(zip(("k", "v"), _plain_commit(state)))


# ---------------------------------------------------------------------------------- costs
def work(case):
    ctx, nodes = _lengths(case)
    e = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    total, words = sum(nodes), -(-max(nodes) // 64)
    hq, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    table = sum(-(-(a + n) // case["block"]) * 4 for a, n in zip(ctx, nodes))
    if case["op"] == "attend":
        keys = sum(ctx) + total
        # A node of a tree sees about log2(n) nodes beside the cached ones, one of a chain half of them;
        # the products of masked pairs are not needed and not counted.
        seen = sum(n * a + n * (n + 1) / 2 if case["tree"] == "chain" else n * (a + 1 + math.log2(n))
                   for a, n in zip(ctx, nodes))
        return {"bytes": 2 * keys * hkv * d * e + 2 * total * hq * d * e + total * words * 8 + table + 12 * len(ctx),
                "flops": 4 * hq * d * seen}
    if case["op"] == "index":
        return {"bytes": total * (4 + 8 + 8 + 8 * words + 4 / case["block"]) + 12 * len(ctx), "flops": 0}
    if case["op"] == "verify":
        return {"bytes": total * (case["vocab"] * e + 8 + 8 + 4) + len(ctx) * (4 * max(nodes) + 16), "flops": 0}
    moved = sum(place != i for p in _paths(case) for place, i in enumerate(p))  # a row read and written, K and V
    return {"bytes": 4 * moved * case["layers"] * hkv * d * e + sum(4 * len(p) + 8 for p in _paths(case)), "flops": 0}


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    with torch.inference_mode():
        st = prepare(case, seed)
        return {"attend": _exact_attend, "index": _exact_index, "verify": _exact_verify,
                "commit": _exact_commit}[case["op"]](st)


def _node_sees(word_row, j):
    return (int(word_row[j // 64]) >> (j % 64)) & 1 == 1


def _exact_attend(st):
    case, bs, d = st["case"], st["case"]["block"], st["case"]["head_dim"]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    words, tables, at = st["mask"].cpu().numpy(), st["tables"].cpu(), 0
    for s, (a, n) in enumerate(zip(st["ctx"], st["nodes"])):
        blocks = tables[s, :-(-(a + n) // bs)].long().cuda()
        hidden = torch.ones(n, a + n, dtype=torch.bool)
        hidden[:, :a] = False
        for i in range(n):
            for j in range(n):
                if _node_sees(words[at + i], j):
                    hidden[i, a + j] = False
        hidden, empty = hidden.cuda(), hidden.all(1).cuda()
        for h in range(case["kv_heads"]):
            k, v = (st[x][blocks, h].reshape(-1, d)[:a + n].double() for x in ("k", "v"))
            for g in range(h * group, (h + 1) * group):
                score = torch.mm(st["q"][at:at + n, g].double(), k.t()).div_(math.sqrt(d))
                weight = torch.softmax(score.masked_fill_(hidden, -math.inf), dim=1)
                out[at:at + n, g] = torch.mm(weight.masked_fill_(empty[:, None], 0.0), v)
        at += n
    return {"out": out}


def _exact_index(st):
    bs, tables = st["case"]["block"], st["tables"].cpu().tolist()
    positions, slots, seen = [], [], []
    for s, (a, tree) in enumerate(zip(st["ctx"], st["trees"])):
        for i in range(len(tree)):
            up, chain = i, []
            while up >= 0:
                chain.append(up)
                up = tree[up]
            positions.append(a + len(chain) - 1)
            slots.append(tables[s][(a + i) // bs] * bs + (a + i) % bs)
            seen.append(chain)
    return {"positions": torch.tensor(positions), "slots": torch.tensor(slots),
            "mask": _bit_words(seen, -(-st["most"] // 64))}


def _exact_verify(st):
    target = []
    for row in st["logits"]:
        target.append(int((row == row.max()).nonzero()[0, 0]))
    tokens, at, paths, following = st["tokens"].cpu().tolist(), 0, [], []
    for tree in st["trees"]:
        path = [0]
        while True:
            want = target[at + path[-1]]
            on = [i for i, p in enumerate(tree) if p == path[-1] and tokens[at + i] == want]
            if not on:
                break
            path.append(on[0])
        paths.append(path)
        following.append(target[at + path[-1]])
        at += len(tree)
    padded = [p + [-1] * (st["most"] - len(p)) for p in paths]
    return {"target": torch.tensor(target), "path": torch.tensor(padded, dtype=torch.int32),
            "counts": torch.tensor([len(p) for p in paths], dtype=torch.int32), "next": torch.tensor(following)}


def _exact_commit(st):
    bs, tables, before = st["case"]["block"], st["tables"].cpu().tolist(), {"k": st["k"], "v": st["v"]}
    after = {x: pool.double() for x, pool in before.items()}
    for s, path in enumerate(_paths(st["case"])):
        for place, node in enumerate(path):
            (b, o), (to_b, to_o) = ((tables[s][(st["ctx"][s] + i) // bs], (st["ctx"][s] + i) % bs) for i in (node, place))
            for x in ("k", "v"):
                after[x][:, to_b, :, to_o] = before[x][:, b, :, o].double()
    return after
