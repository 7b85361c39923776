"""Several candidates for a sequence of the paged cache -- drafted trees and beams -- as cases to time.

A speculative step appends a tree of drafted tokens to a sequence, as its last n positions: node i is row
i of the sequence, and row i of `masks` (int64 words, bit j: node j) holds the node and its ancestors. A
row without bits is no node (trees padded to one size). A beam search keeps `beams` sequences for each
prompt. `run` makes one pass through an operator. Kinds:

  attention  paged_tree_attention: a node sees the positions before the tree (the last `window` of them,
             counted from its depth in the tree, where a window is set) and the nodes of its mask
  verify     tree_verify: the token that every node's largest logit names, and the greedy walk from node 0
             to the child that it names, as long as there is one: the node it ends at, and the token behind
  commit     paged_tree_commit: the accepted node's path becomes the sequence's positions behind the ones
             before the tree, in every layer, and the sequence ends there
  select     beam_select: the best `beams` of a group's candidates score + log softmax(logits), with the
             beams they come from
  reorder    paged_cache_reorder: every sequence becomes what its parent was: full pages shared, a
             partly filled last page copied for all but one of its children

Calls that change the table start from the same one in every pass: the pass copies it in first, as a
scheduler's upload does. K and V are bf16, or E4M3 codes with one f32 scale per layer and KV head. Head
layouts are those of the sliding layers (16 query heads, 8 KV heads of 256, a window of 1024), of the
full-attention layers (16 query heads, one KV head of 512), and generic ones; 262144 is the vocabulary.
"""
import math
import os
import random
import sys

import torch

DEV = "cuda"
own = False


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the drafted tree of one short conversation in a sliding layer: latency
        {"name": "tree_sliding_one", "kind": "attention", "heads": 16, "kv_heads": 8, "dim": 256, "fmt": "bf16", "slots": 64,
         "window": 1024, "seqs": 1, "nodes_lo": 8, "nodes_hi": 8, "kv_lo": 700, "kv_hi": 700, "mix": 1},
        # a batch of large trees in a full-attention layer, every sequence at its own length
        {"name": "tree_full", "kind": "attention", "heads": 16, "kv_heads": 1, "dim": 512, "fmt": "bf16", "slots": 512,
         "window": 0, "seqs": 12, "nodes_lo": 30, "nodes_hi": 63, "kv_lo": 900, "kv_hi": 16000, "mix": 2},
        # a batch of medium trees in a sliding layer
        {"name": "tree_sliding_batch", "kind": "attention", "heads": 16, "kv_heads": 8, "dim": 256, "fmt": "bf16", "slots": 128,
         "window": 1024, "seqs": 40, "nodes_lo": 9, "nodes_hi": 33, "kv_lo": 10, "kv_hi": 5000, "mix": 3},
        # small trees over a long E4M3 cache in small pages
        {"name": "tree_e4m3", "kind": "attention", "heads": 32, "kv_heads": 8, "dim": 128, "fmt": "e4m3", "slots": 16,
         "window": 0, "seqs": 32, "nodes_lo": 5, "nodes_hi": 16, "kv_lo": 100, "kv_hi": 9000, "mix": 4},
        # the verification of one tree
        {"name": "verify_one", "kind": "verify", "vocab": 262144, "seqs": 1, "nodes_lo": 8, "nodes_hi": 8, "mix": 5},
        # and of a batch's
        {"name": "verify_batch", "kind": "verify", "vocab": 262144, "seqs": 24, "nodes_lo": 5, "nodes_hi": 33, "mix": 6},
        # one sequence keeps a path of its tree, in every layer of a small pool
        {"name": "commit_one", "kind": "commit", "kv_heads": 8, "dim": 256, "fmt": "bf16", "slots": 64, "layers": 8,
         "seqs": 1, "nodes_lo": 16, "nodes_hi": 16, "kv_lo": 700, "kv_hi": 700, "mix": 7},
        # a batch does
        {"name": "commit_batch", "kind": "commit", "kv_heads": 8, "dim": 256, "fmt": "bf16", "slots": 64, "layers": 10,
         "seqs": 60, "nodes_lo": 20, "nodes_hi": 63, "kv_lo": 10, "kv_hi": 200, "mix": 8},
        # one prompt's beams
        {"name": "select_one", "kind": "select", "vocab": 262144, "groups": 1, "beams": 4, "done": 0, "mix": 9},
        # many prompts' beams, some of them finished
        {"name": "select_batch", "kind": "select", "vocab": 262144, "groups": 20, "beams": 8, "done": 9, "mix": 10},
        # one prompt's beams follow the selection, over an E4M3 cache
        {"name": "reorder_one", "kind": "reorder", "kv_heads": 1, "dim": 512, "fmt": "e4m3", "slots": 128, "layers": 2,
         "groups": 1, "beams": 4, "kv_lo": 500, "kv_hi": 500, "tail": 300, "mix": 11},
        # many prompts' beams do
        {"name": "reorder_batch", "kind": "reorder", "kv_heads": 8, "dim": 256, "fmt": "bf16", "slots": 64, "layers": 6,
         "groups": 12, "beams": 8, "kv_lo": 20, "kv_hi": 500, "tail": 150, "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _draw(rng, kind):
    mix = rng.randrange(1 << 20)
    nodes = _log_int(rng, 1, 200)
    trees = {"nodes_lo": max(1, nodes - rng.choice([0, nodes // 2, nodes])), "nodes_hi": nodes}
    kv_lo = _log_int(rng, 1, 500)
    cache = {"fmt": rng.choice(["bf16", "e4m3"]), "slots": rng.choice([1, 16, 24, 48, 64, 100, 512]), "kv_lo": kv_lo}
    if kind == "attention":
        kv_heads, group, dim = rng.choice([(8, 2, 256), (1, 16, 512), (8, 4, 128), (4, 1, 256), (2, 7, 128), (1, 8, 512), (12, 1, 64), (4, 8, 128)])
        return dict(cache, **trees, kind=kind, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, window=rng.choice([0, 0, 1024, _log_int(rng, 256, 5000)]),
                    seqs=_log_int(rng, 1, 60), kv_hi=kv_lo + _log_int(rng, 1, 16000), mix=mix)
    vocab = rng.choice([262144, 262144, 32000, 50000, _log_int(rng, 100, 150000)])
    if kind == "verify":
        return dict(trees, kind=kind, vocab=vocab, seqs=_log_int(rng, 1, 60), mix=mix)
    kv_heads, dim = rng.choice([(8, 256), (1, 512), (8, 128), (2, 64), (3, 128)])
    cache = dict(cache, kv_heads=kv_heads, dim=dim, layers=rng.randrange(1, 9), kv_hi=kv_lo + _log_int(rng, 1, 500))
    if kind == "commit":
        return dict(cache, **trees, kind=kind, seqs=_log_int(rng, 1, 80), mix=mix)
    groups, beams = _log_int(rng, 1, 24), rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 32])
    if kind == "select":
        return {"kind": kind, "vocab": vocab, "groups": groups, "beams": beams, "done": rng.randrange(0, groups * beams // 2 + 1), "mix": mix}
    return dict(cache, kind=kind, groups=groups, beams=beams, tail=_log_int(rng, 1, 400), mix=mix)


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "verify", "commit", "select", "select", "reorder"])
    tops = [work(c) for c in listed() if c["kind"] == kind]
    most_bytes, most_flops = max(w["bytes"] for w in tops), max(w["flops"] for w in tops)
    while True:  # until a case costs no more than the largest listed one
        c = _draw(rng, kind)
        w = work(c)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops and _held(c) <= 1 << 30 and _padded(c) <= 1 << 30:
            return c


def _pages(n, slots):
    return -(-n // slots)


# Trees. A node's parent lies a level above it; levels follow each other, so a parent has the lower number.

def _tree(r, n):
    """Parents of n nodes, the first of them the root (-1); now and then a chain."""
    parents, level, width = [-1], [0], 1 if r.random() < 0.15 else r.randint(2, 10)
    while len(parents) < n:
        here = sorted(r.choice(level) for _ in range(min(n - len(parents), width if width == 1 else max(2, width - r.randint(0, 2)))))
        level = list(range(len(parents), len(parents) + len(here)))
        parents += here
    return parents


def _path(parents, i):
    p = []
    while i >= 0:
        p.append(i)
        i = parents[i]
    return p[::-1]


def _accepted(r, parents):
    """A node whose path, moved to the front, lands on none of its own nodes but those that stay, so that passes repeat."""
    best = [0]
    for _ in range(8):
        p = _path(parents, r.randrange(len(parents)))
        while any(j != i and j < len(p) for i, j in enumerate(p)):
            p.pop()
        best = max(best, p, key=len)
    return best


def _trees(c):
    """Of each sequence: positions before the tree, the tree's parents, rows in all (some are no nodes)."""
    r = random.Random(c["mix"])
    before, trees, rows = [], [], []
    for _ in range(c["seqs"]):
        before.append(r.randint(c.get("kv_lo", 0), c.get("kv_hi", 0)))
        n = r.randint(c["nodes_lo"], c["nodes_hi"])
        trees.append(_tree(r, n))
        rows.append(n + (r.randint(0, 2) if c["kind"] == "attention" and r.random() < 0.3 else 0))
    return before, trees, rows


def _kept(c):
    """Of each sequence, the path it keeps: the root at least, of few sequences nothing."""
    _, trees, _ = _trees(c)
    r = random.Random(c["mix"] + 1)
    return [[] if len(trees) > 4 and r.random() < 0.05 else _accepted(r, t) for t in trees]


# Beams: the sequences of a group share the full pages of their prompt; behind it each has its own. Some groups stand still, and
# some have beams that ended early.

def _beams(c):
    """Of each sequence: positions of its prompt, of all; its parent."""
    r = random.Random(c["mix"])
    prompts, lens, parents = [], [], []
    for g in range(c["groups"]):
        prompt, n = r.randint(c["kv_lo"], c["kv_hi"]), r.randint(1, c["tail"])
        still, ragged = c["groups"] > 3 and r.random() < 0.1, r.random() < 0.2
        for b in range(c["beams"]):
            prompts.append(prompt)
            lens.append(prompt + (r.randint(1, n) if ragged else n))
            parents.append(g * c["beams"] + (b if still else min(r.randrange(c["beams"]), r.randrange(c["beams"]))))
    return prompts, lens, parents


def _beam_pages(c):
    """Pages in use: a prompt's full ones once a group, the others once a sequence."""
    prompts, lens, _ = _beams(c)
    return sum(_pages(n, c["slots"]) - p // c["slots"] for p, n in zip(prompts, lens)) + sum(p // c["slots"] for p in prompts[::c["beams"]])


def _copies(c):
    """(parent, child) of the partly filled pages that are copied: for every child of a parent but itself, or its first."""
    _, lens, parents = _beams(c)
    keeper = {}
    for s, p in enumerate(parents):
        if p not in keeper or s == p:
            keeper[p] = s
    return [(p, s) for s, p in enumerate(parents) if keeper[p] != s and lens[p] % c["slots"]]


def _slot_bytes(c):
    return c["kv_heads"] * c["dim"] * (2 if c["fmt"] == "bf16" else 1)


def _held(c):
    """Bytes of K and V pages, or of logits."""
    if c["kind"] in ("verify", "select"):
        rows = sum(_trees(c)[2]) if c["kind"] == "verify" else c["groups"] * c["beams"]
        return 2 * rows * c["vocab"]
    if c["kind"] == "reorder":
        n = _beam_pages(c) + len(_copies(c)) + 2
    else:
        before, _, rows = _trees(c)
        n = sum(_pages(b + m, c["slots"]) + 1 for b, m in zip(before, rows))
    return 2 * n * c["slots"] * _slot_bytes(c) * c.get("layers", 1)


def _padded(c):
    """Elements of the scores, or of K, with every sequence padded to the longest."""
    if c["kind"] != "attention":
        return 0
    before, _, rows = _trees(c)
    keys = max(b + n for b, n in zip(before, rows))
    return c["seqs"] * keys * max(c["heads"] * max(rows), c["kv_heads"] * c["dim"])


def work(case):
    c, kind = case, case["kind"]
    if kind == "verify":
        rows = sum(_trees(c)[2])
        return {"bytes": rows * (2.0 * c["vocab"] + 16) + 12.0 * c["seqs"], "flops": 0.0}
    if kind == "select":
        n = c["groups"] * c["beams"]
        return {"bytes": (n - c["done"]) * 2.0 * c["vocab"] + 24.0 * n, "flops": 2.0 * (n - c["done"]) * c["vocab"]}
    slot = _slot_bytes(c)
    if kind == "reorder":
        _, lens, parents = _beams(c)
        moved = sum(lens[p] % c["slots"] for p, _ in _copies(c))
        entries = sum(_pages(lens[p], c["slots"]) for s, p in enumerate(parents) if p != s)
        return {"bytes": 4.0 * c["layers"] * moved * slot + 8.0 * entries + 12.0 * len(lens), "flops": 0.0}
    before, trees, rows = _trees(c)
    if kind == "commit":
        moved = sum(sum(1 for i, j in enumerate(p) if i != j) for p in _kept(c))
        return {"bytes": 4.0 * c["layers"] * moved * slot + 12.0 * c["seqs"], "flops": 0.0}
    keys = pairs = 0
    for b, t in zip(before, trees):
        depths = [len(_path(t, i)) for i in range(len(t))]
        w = c["window"]
        pairs += sum(min(b + d, w or b + d) for d in depths)
        keys += min(b, w - 1 if w else b) + len(t)
    return {"bytes": 2.0 * keys * slot + sum(rows) * (4.0 * c["heads"] * c["dim"] + 8) + 4.0 * keys / c["slots"],
            "flops": 4.0 * pairs * c["heads"] * c["dim"]}


# ----------------------------------------------------------------------------------------- inputs

def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * std


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _signed(word):
    return word - (1 << 64) if word >> 63 else word


def _masks(trees, rows):
    words = -(-max(rows) // 64)
    masks = []
    for t, n in zip(trees, rows):
        seen = []
        for i, p in enumerate(t):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        masks += [[_signed(m >> 64 * w & (1 << 64) - 1) for w in range(words)] for m in seen + [0] * (n - len(t))]
    return torch.tensor(masks, dtype=torch.int64, device=DEV)


def _starts(rows):
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    return _i32(starts)


def _cache(s, c, g, rows_of_table, lens, pages):
    """The cache of a case: rows_of_table, the pages that each sequence names (numbers below `pages`, some of them free)."""
    S, layers, hk, d = len(lens), c.get("layers", 1), c["kv_heads"], c["dim"]
    columns = max(len(t) for t in rows_of_table)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    at = torch.tensor([t + [-1] * (columns - len(t)) for t in rows_of_table], device=DEV)
    table = torch.where(at >= 0, order[at.clamp_min(0)], torch.zeros_like(order[:1])).to(torch.int32)
    refs = torch.bincount(table[at >= 0].long(), minlength=pages).to(torch.int32)
    # the table, the lengths and the reference counts in one allocation, and the values they start from
    s["ints"] = torch.cat([table.reshape(-1), _i32(lens), refs])
    s["ints_at_start"] = s["ints"].clone()
    a, b = table.numel(), table.numel() + S
    s["table"], s["lens"], s["refs"] = s["ints"][:a].view(table.shape), s["ints"][a:b], s["ints"][b:]
    shape = (layers, pages, c["slots"], hk, d)
    if c["fmt"] == "bf16":
        s["k"], s["v"] = _normal(g, shape).to(torch.bfloat16), _normal(g, shape).to(torch.bfloat16)
        s["k_scale"] = s["v_scale"] = None
    else:                                                                  # the largest of the values at about 448
        s["k_scale"], s["v_scale"] = ((0.9 + 0.2 * torch.rand((layers, hk), generator=g, device=DEV)) * (6.0 / 448.0) for _ in range(2))
        s["k"], s["v"] = ((_normal(g, shape, 448.0 / 6.0)).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn) for _ in range(2))
    if own:
        s["cache"] = _ops().PagedCache(s["k"], s["v"], s["table"], s["lens"], s["refs"], s["k_scale"], s["v_scale"])


def _logits(g, rows, vocab):
    """Logits as a language model's: a wide bulk, and a few tokens that stand out; at most +-30."""
    x = _normal(g, (rows, vocab), 3.0)
    likely = torch.randint(0, vocab, (rows, min(vocab, 24)), generator=g, device=DEV)
    x.scatter_add_(1, likely, 8.0 + _normal(g, likely.shape, 3.0))
    return (30.0 * torch.tanh(x / 30.0)).to(torch.bfloat16)


def prepare(case, seed):
    c, kind = case, case["kind"]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": c, "kind": kind}
    if kind == "select":
        n = c["groups"] * c["beams"]
        s["logits"] = _logits(g, n, c["vocab"])
        # beams of a prompt lie a few units apart
        s["scores"] = -10.0 * torch.rand(n, generator=g, device=DEV) - 2.0
        s["finished"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        s["finished"][random.Random(c["mix"]).sample(range(n), c["done"])] = 1
        s["eos"] = 1
        s["out_scores"], s["out_finished"] = torch.empty_like(s["scores"]), torch.empty_like(s["finished"])
        s["parents"], s["tokens"] = torch.empty_like(s["finished"]), torch.empty_like(s["finished"])
        return s
    if kind == "reorder":
        prompts, lens, parents = _beams(c)
        rows_of_table, n = [], 0
        for i, (p, m) in enumerate(zip(prompts, lens)):
            full = p // c["slots"]
            if i % c["beams"] == 0:
                shared = list(range(n, n + full))
                n += full
            more = _pages(m, c["slots"]) - full
            rows_of_table.append(shared + list(range(n, n + more)))
            n += more
        _cache(s, c, g, rows_of_table, lens, n + len(_copies(c)) + 2)
        s["parents"] = _i32(parents)
        return s
    before, trees, rows = _trees(c)
    s["masks"], s["row_starts"], s["total"], s["longest"] = _masks(trees, rows), _starts(rows), sum(rows), max(rows)
    if kind == "verify":
        s["logits"] = _logits(g, s["total"], c["vocab"])
        s["draft"] = torch.randint(0, c["vocab"], (s["total"],), generator=g, device=DEV).to(torch.int32)
        # a good draft: most nodes' largest logits name one of their children
        r = random.Random(seed)
        first = 0
        row, col = [], []
        for t, n in zip(trees, rows):
            for i in range(len(t)):
                children = [j for j, p in enumerate(t) if p == i]
                if children and r.random() < 0.8:
                    row.append(first + i)
                    col.append(first + r.choice(children))
            first += n
        if row:
            s["logits"][torch.tensor(row, device=DEV), s["draft"][torch.tensor(col, device=DEV)].long()] = 30.0
        s["best"] = torch.empty_like(s["draft"])
        s["leaves"], s["next"] = (torch.empty(len(rows), dtype=torch.int32, device=DEV) for _ in range(2))
        return s
    lens = [b + n for b, n in zip(before, rows)]
    rows_of_table, n = [], 0
    for m in lens:
        rows_of_table.append(list(range(n, n + _pages(m, c["slots"]))))
        n += _pages(m, c["slots"])
    _cache(s, c, g, rows_of_table, lens, n + len(lens) // 4 + 1)           # a few pages stay free
    s["keys"] = max(lens)
    if kind == "commit":
        s["leaves"] = _i32([p[-1] if p else -1 for p in _kept(c)])
        return s
    # head norms leave q . k with a spread of about two
    d = c["dim"]
    s["scale"], s["window"] = (1.0 if d >= 256 else 1.0 / math.sqrt(d)), c["window"]
    s["q"] = _normal(g, (s["total"], c["heads"], d), 2.0 / math.sqrt(d) / s["scale"]).to(torch.bfloat16)
    s["out"] = torch.empty_like(s["q"])
    return s


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moa-workspace_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from moa_amd import ops
    return ops


# ------------------------------------------------------------------------------------- plain forms

def _nodes(s):
    """Each row's sequence and its number there; and the masks as truth values [rows, longest]."""
    row = torch.arange(s["total"], device=DEV)
    starts = s["row_starts"].long()
    seq = torch.searchsorted(starts, row, right=True) - 1
    j = torch.arange(s["longest"], device=DEV)
    sees = (s["masks"][:, j // 64] >> (j % 64)) & 1 == 1
    return seq, row - starts[seq], sees & (j[None, :] < (starts[1:] - starts[:-1])[seq][:, None])


def _attention(s):
    c, slots, hk = s["case"], s["case"]["slots"], s["case"]["kv_heads"]
    group, d, nq, nk = c["heads"] // hk, c["dim"], s["longest"], s["keys"]
    S = s["lens"].numel()
    key = torch.arange(nk, device=DEV)
    page = s["table"].long()[:, key // slots]                               # [S, keys]
    k, v = _bits(s["k"])[0][page, key % slots], _bits(s["v"])[0][page, key % slots]
    if s["k_scale"] is None:
        k, v = k.float(), v.float()
    else:
        k = k.view(torch.float8_e4m3fn).float() * s["k_scale"][0][:, None]
        v = v.view(torch.float8_e4m3fn).float() * s["v_scale"][0][:, None]
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()  # [S, heads, d, keys], [S, heads, keys, d]
    seq, i, nodes = _nodes(s)
    counts = (s["row_starts"][1:] - s["row_starts"][:-1]).long()
    base = (s["lens"].long() - counts)[seq][:, None]                        # [rows, 1]
    at = key[None, :] - base                                                # the key's node
    seen = torch.gather(nodes, 1, at.clamp(0, nq - 1)) & (at >= 0) & (at < nq)
    depth = nodes.sum(1, keepdim=True)
    seen |= (at < 0) & (depth > 0) & (at > depth - 1 - (s["window"] or 1 << 40))
    sees = torch.zeros((S, nq, nk), dtype=torch.bool, device=DEV)
    sees[seq, i] = seen
    q = torch.zeros((S, nq, c["heads"], d), device=DEV)
    q[seq, i] = s["q"].float()
    q = q.view(S, nq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(S, hk, group * nq, d)
    x = (torch.matmul(q, k) * s["scale"]).view(S, hk, group, nq, nk)
    x = x.masked_fill(~sees[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-3e38))
    x = x / x.sum(-1, keepdim=True).clamp_min(1e-38)
    o = torch.matmul(x.view(S, hk, group * nq, nk), v).view(S, hk, group, nq, d)
    return o.permute(0, 3, 1, 2, 4).reshape(S, nq, c["heads"], d)[seq, i].to(torch.bfloat16)


def _bits(pages):
    return pages.view(torch.uint8) if pages.dtype == torch.float8_e4m3fn else pages


def _verify(s):
    x = s["logits"].float()
    v = torch.arange(x.shape[1], device=DEV)
    best = torch.where(x == x.amax(1, keepdim=True), v, x.shape[1]).amin(1)  # [rows], ties to the lowest token
    seq, i, sees = _nodes(s)
    nq, S = s["longest"], s["leaves"].numel()
    nodes = torch.zeros((S, nq, nq), dtype=torch.bool, device=DEV)
    nodes[seq, i] = sees
    token = torch.full((S, nq), -1, dtype=torch.long, device=DEV)
    token[seq, i] = s["draft"].long()
    names = torch.zeros((S, nq), dtype=torch.long, device=DEV)
    names[seq, i] = best
    eye = torch.eye(nq, dtype=torch.bool, device=DEV)[None]
    itself, others = (nodes & eye).any(2), nodes & ~eye
    cur = torch.zeros(S, dtype=torch.long, device=DEV)
    all_s = torch.arange(S, device=DEV)
    for _ in range(nq):
        child = itself & (others == nodes[all_s, cur][:, None]).all(2) & (token == names[all_s, cur][:, None])
        first = torch.where(child, torch.arange(nq, device=DEV), nq).amin(1)
        cur = torch.where(first < nq, first, cur)
    s["best"].copy_(best)
    s["leaves"].copy_(cur)
    s["next"].copy_(names[all_s, cur])


def _commit(s):
    table, lens, refs, slots = s["table"], s["lens"], s["refs"], s["case"]["slots"]
    counts = (s["row_starts"][1:] - s["row_starts"][:-1]).long()
    base = lens.long() - counts
    _, _, sees = _nodes(s)
    kept = sees[(s["row_starts"][:-1].long() + s["leaves"].long()).clamp_min(0)] & (s["leaves"] >= 0)[:, None]
    rank = kept.long().cumsum(1) - 1
    seq, node = torch.nonzero(kept, as_tuple=True)
    src, dst = base[seq] + node, base[seq] + rank[seq, node]
    t = table.long()
    for pages in (_bits(s["k"]), _bits(s["v"])):
        pages[:, t[seq, dst // slots], dst % slots] = pages[:, t[seq, src // slots], src % slots]
    new = base + kept.sum(1)
    col = torch.arange(table.shape[1], device=DEV)[None, :]
    gone = (col >= ((new + slots - 1) // slots)[:, None]) & (col < ((lens.long() + slots - 1) // slots)[:, None])
    refs.index_add_(0, table[gone].long(), -torch.ones_like(table[gone]))
    lens.copy_(new)


def _select(s):
    beams, vocab = s["case"]["beams"], s["case"]["vocab"]
    x = s["logits"].double()                                               # totals that lie close are told apart
    m = x.amax(1, keepdim=True)
    total = s["scores"].double()[:, None] + (x - m - torch.log(torch.exp(x - m).sum(1, keepdim=True)))
    done = s["finished"] != 0
    total[done] = -math.inf
    total[done, s["eos"]] = s["scores"][done].double()
    total = torch.where(total.isnan(), -math.inf, total).view(-1, beams * vocab)
    order = torch.argsort(total, dim=1, descending=True, stable=True)[:, :beams]
    score = torch.gather(total, 1, order).reshape(-1)
    group = torch.arange(total.shape[0], device=DEV)[:, None] * beams
    parent, token = (group + order // vocab).reshape(-1), (order % vocab).reshape(-1)
    dead = score == -math.inf
    parent = torch.where(dead, torch.arange(score.numel(), device=DEV), parent)
    token = torch.where(dead, s["eos"], token)
    s["out_scores"].copy_(score)
    s["parents"].copy_(parent)
    s["tokens"].copy_(token)
    s["out_finished"].copy_(done[parent] | (token == s["eos"]))


def _reorder(s):
    table, lens, refs, slots = s["table"], s["lens"], s["refs"], s["case"]["slots"]
    p, S = s["parents"].long(), s["parents"].numel()
    me = torch.arange(S, device=DEV)
    chosen = torch.zeros(S, dtype=torch.bool, device=DEV)
    chosen[p] = True
    keeper = torch.where(p == me, me - S, me)                              # itself before the others
    keeper = torch.full((S,), S, device=DEV).scatter_reduce_(0, p, keeper, "amin")
    keeper = torch.where(keeper < 0, keeper + S, keeper)
    full, part = lens.long() // slots, lens.long() % slots
    copies = torch.nonzero((keeper[p] != me) & (part[p] > 0))[:, 0]
    last = table[me, full.clamp_max(table.shape[1] - 1)].long()
    spare = (~chosen) & (part > 0) & (refs[last] == 1)
    pages = torch.cat([last[spare], torch.nonzero(refs == 0)[:, 0]])[:copies.numel()]
    col = torch.arange(table.shape[1], device=DEV)[None, :]
    new = torch.where(col < ((lens[p] + slots - 1) // slots)[:, None], table[p], table)
    new[copies, full[p[copies]]] = pages.to(torch.int32)
    old_lens, new_lens = lens.clone(), lens[p]
    for t, n, sign in ((table, old_lens, -1), (new, new_lens, 1)):
        e = t[col < ((n + slots - 1) // slots)[:, None]].long()
        refs.index_add_(0, e, torch.full_like(e, sign, dtype=torch.int32))
    src = last[p[copies]]
    used = torch.arange(slots, device=DEV)[None, :] < part[p[copies]][:, None]
    which, slot = torch.nonzero(used, as_tuple=True)
    for t in (_bits(s["k"]), _bits(s["v"])):
        t[:, pages[which], slot] = t[:, src[which], slot]
    table.copy_(new)
    lens.copy_(new_lens)


# ------------------------------------------------------------------------------------------- a pass

def run(state):
    s, kind = state, state["kind"]
    if kind == "attention":
        if not own:
            return {"out": _attention(s)}
        _ops().paged_tree_attention(s["q"], s["cache"], s["row_starts"], s["masks"], s["out"], window=s["window"], scale=s["scale"],
                                    max_rows=s["longest"])
        return {"out": s["out"]}
    if kind == "verify":
        if own:
            _ops().tree_verify(s["logits"], s["draft"], s["row_starts"], s["masks"], s["best"], s["leaves"], s["next"])
        else:
            _verify(s)
        return {"best": s["best"], "leaves": s["leaves"], "next": s["next"]}
    if kind == "select":
        if own:
            _ops().beam_select(s["logits"], s["scores"], s["finished"], s["out_scores"], s["out_finished"], s["parents"], s["tokens"],
                               beams=s["case"]["beams"], eos=s["eos"])
        else:
            _select(s)
        return {"scores": s["out_scores"], "finished": s["out_finished"], "parents": s["parents"], "tokens": s["tokens"]}
    s["ints"].copy_(s["ints_at_start"])
    if kind == "commit":
        if own:
            _ops().paged_tree_commit(s["cache"], s["row_starts"], s["masks"], s["leaves"])
        else:
            _commit(s)
    elif own:
        _ops().paged_cache_reorder(s["cache"], s["parents"], beams=s["case"]["beams"])
    else:
        _reorder(s)
    return {"k": s["k"], "v": s["v"], "table": s["table"], "lens": s["lens"], "refs": s["refs"]}


# --------------------------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    """Attention node by node's sequence and head by head in float64, beams' candidates group by group. A verification compares,
    and commits and reorders move values: nothing is computed."""
    if case["kind"] == "select":
        return _exact_select(case, seed)
    if case["kind"] != "attention" or work(case)["flops"] > 3e12:
        return None
    c = case
    s = prepare(c, seed)
    before, trees, rows = _trees(c)
    hk, group = c["kv_heads"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    ones = torch.ones(hk, dtype=torch.float64, device=DEV)
    ks, vs = (ones, ones) if s["k_scale"] is None else (s["k_scale"][0].double(), s["v_scale"][0].double())
    first = 0
    for i, (b, t, n) in enumerate(zip(before, trees, rows)):
        p = torch.arange(0, b + len(t), device=DEV)
        page, slot = s["table"][i].long()[torch.div(p, c["slots"], rounding_mode="floor")], torch.remainder(p, c["slots"])
        paths = [_path(t, j) for j in range(len(t))]
        hidden = torch.ones((len(t), b + len(t)), dtype=torch.bool)
        for j, path in enumerate(paths):
            hidden[j, [b + a for a in path]] = False
            hidden[j, max(0, b + len(path) - c["window"]) if c["window"] else 0:b] = False
        hidden = hidden.to(DEV)
        for h in range(hk):
            kh = s["k"][0, :, :, h].float()[page, slot].double() * ks[h]
            vh = s["v"][0, :, :, h].float()[page, slot].double() * vs[h]
            for j in range(h * group, (h + 1) * group):
                w = s["q"][first:first + len(t), j].double() @ kh.T * s["scale"]
                w[hidden] = -math.inf
                out[first:first + len(t), j] = torch.softmax(w, dim=1) @ vh
        first += n
    return {"out": out}


def _exact_select(c, seed):
    s = prepare(c, seed)
    beams, n = c["beams"], c["groups"] * c["beams"]
    logs = torch.log_softmax(s["logits"].double(), dim=1)
    most = torch.topk(logs, min(c["vocab"], beams + 1), dim=1).values[:, -1].tolist()
    scores, done = s["scores"].double().tolist(), s["finished"].tolist()
    got = {"scores": [], "finished": [], "parents": [], "tokens": []}
    for g in range(c["groups"]):
        found = []
        for r in range(g * beams, (g + 1) * beams):
            if done[r]:
                found.append((-scores[r], r, s["eos"]))
                continue
            at = torch.nonzero(logs[r] >= most[r])[:, 0]
            found += [(-(scores[r] + x), r, v) for x, v in zip(logs[r][at].tolist(), at.tolist())]
        for total, r, v in sorted(found)[:beams]:
            got["scores"].append(-total)
            got["parents"].append(r)
            got["tokens"].append(v)
            got["finished"].append(1 if done[r] or v == s["eos"] else 0)
    assert len(got["scores"]) == n
    return {"scores": torch.tensor(got["scores"], dtype=torch.float64, device=DEV),
            **{k: torch.tensor(got[k], dtype=torch.int32, device=DEV) for k in ("finished", "parents", "tokens")}}
