"""Drafted trees and beams in plain form for the tests: trees and masks as Python integers, state changes on paged_model.State, values
in float64."""
from __future__ import annotations

import math
import random

import torch

from paged_model import pages_of


def tree(rng, n, chain=False):
    """Masks (integers) of a random tree of n nodes: a node's parent has a lower number."""
    masks = [1][:n]
    for i in range(1, n):
        p = i - 1 if chain else rng.randrange(max(0, i - 9), i)
        masks.append(masks[p] | 1 << i)
    return masks


def words_of(n):
    return max(1, -(-n // 64))


def mask_tensor(masks, words, device):
    """int64 [rows, words] of the rows' integers."""
    def word(m, w):
        x = m >> 64 * w & (1 << 64) - 1
        return x - (1 << 64) if x >> 63 else x

    return torch.tensor([[word(m, w) for w in range(words)] for m in masks], dtype=torch.int64, device=device).reshape(len(masks), words)


def attention(q, k, v, table, lens, starts, masks, slots, window, scale, k_scale=None, v_scale=None):
    """Per row in float64: (out, a, d) as paged_model.attention."""
    R, H, D = q.shape
    hk = k.shape[2]
    g = H // hk
    out = torch.full((R, H, D), float("nan"), dtype=torch.float64, device=q.device)
    a, d = out.clone(), torch.zeros((R, H), dtype=torch.float64, device=q.device)
    ks = torch.ones(hk, dtype=torch.float64, device=q.device) if k_scale is None else k_scale.double().reshape(hk)
    vs = torch.ones(hk, dtype=torch.float64, device=q.device) if v_scale is None else v_scale.double().reshape(hk)
    for s, n in enumerate(lens):
        m0, m1 = starts[s], starts[s + 1]
        if m0 == m1:
            continue
        base = n - (m1 - m0)
        t = torch.arange(n, device=q.device)
        page = torch.tensor(table[s], device=q.device)[t // slots]
        kk = (k[page, t % slots].double() * ks[:, None]).permute(1, 2, 0).contiguous()
        vv = (v[page, t % slots].double() * vs[:, None]).permute(1, 0, 2).contiguous()
        for m in range(m0, m1):
            nodes = [j for j in range(m1 - m0) if masks[m] >> j & 1]
            if not nodes:
                out[m], a[m] = 0.0, 0.0
                continue
            p = base + len(nodes) - 1
            sees = list(range(max(0, p - window + 1) if window else 0, base)) + [base + j for j in nodes]
            sees = torch.tensor(sees, device=q.device)
            qh, kr, vr = q[m].double().view(hk, g, D), kk[:, :, sees].contiguous(), vv[:, sees].contiguous()
            w = torch.softmax(torch.matmul(qh, kr) * scale, dim=-1)
            out[m], a[m] = torch.matmul(w, vr).reshape(H, D), torch.matmul(w, vr.abs()).reshape(H, D)
            d[m] = (torch.matmul(qh.abs(), kr.abs()) * abs(scale)).amax(-1).reshape(H)
    return out, a, d


def verify(logits, tokens, starts, masks):
    """(best, leaves, next) of float logits [rows, vocab] (a tensor): NaN below everything, ties to the lowest token."""
    x = torch.where(logits.isnan(), -math.inf, logits.double())
    rank = torch.where(logits.isnan(), -1, 0)
    best = []
    for r in range(x.shape[0]):
        if bool((rank[r] == 0).any()):
            ok = (x[r] == x[r].max()) & (rank[r] == 0)
            best.append(int(torch.nonzero(ok)[0]))
        else:
            best.append(0)
    leaves, nexts = [], []
    for s in range(len(starts) - 1):
        m0, n = starts[s], starts[s + 1] - starts[s]
        low = (1 << max(n, 0)) - 1
        if n == 0 or not masks[m0] & 1:
            leaves.append(-1)
            nexts.append(-1)
            continue
        cur = 0
        while True:
            sees = masks[m0 + cur] & low
            child = [c for c in range(n) if tokens[m0 + c] == best[m0 + cur] and masks[m0 + c] >> c & 1 and not sees >> c & 1
                     and masks[m0 + c] & low & ~(1 << c) == sees]
            if not child:
                break
            cur = child[0]
        leaves.append(cur)
        nexts.append(best[m0 + cur])
    return best, leaves, nexts


def commit(st, starts, masks, leaves):
    """Moves ((page, slot), (page, slot)) of a commit on a paged_model.State, and the sequences that stay as they were."""
    moves, left = [], []
    for s in range(len(st.lens)):
        n = starts[s + 1] - starts[s]
        if n == 0:
            continue
        base = st.lens[s] - n
        pages = [st.table[s][(base + i) // st.slots] for i in range(n)] if base >= 0 else [-1]
        if not -1 <= leaves[s] < n or any(not 0 <= p < len(st.refs) or st.refs[p] != 1 for p in pages):
            left.append(s)
            continue
        kept = [j for j in range(n) if leaves[s] >= 0 and masks[starts[s] + leaves[s]] >> j & 1]
        place = lambda t: (st.table[s][t // st.slots], t % st.slots)
        moves += [(place(base + j), place(base + i)) for i, j in enumerate(kept) if i != j]
        for i in range(pages_of(base + len(kept), st.slots), pages_of(st.lens[s], st.slots)):
            st.refs[st.table[s][i]] = 0
        st.lens[s] = base + len(kept)
    return moves, left


def reorder(st, parents, beams):
    """Page copies (source, target, slots) of a reorder on a paged_model.State; None where it is refused."""
    n, slots = len(parents), st.slots
    if any(not s // beams * beams <= p < s // beams * beams + beams for s, p in enumerate(parents)):
        return None
    keeper = {}
    for s, p in enumerate(parents):
        if p not in keeper or s == p:
            keeper[p] = s
    copies = [s for s, p in enumerate(parents) if keeper[p] != s and st.lens[p] % slots]
    last = lambda s: st.table[s][st.lens[s] // slots]
    targets = [last(s) for s in range(n) if s not in keeper and st.lens[s] % slots and st.refs[last(s)] == 1]
    targets += [p for p, r in enumerate(st.refs) if r == 0]
    if len(targets) < len(copies):
        return None
    moves = [(last(parents[s]), t, st.lens[parents[s]] % slots) for s, t in zip(copies, targets)]
    old, lens = [list(r) for r in st.table], list(st.lens)
    for s in range(n):
        for i in range(pages_of(lens[s], slots)):
            st.refs[old[s][i]] -= 1
        p = parents[s]
        st.table[s][:pages_of(lens[p], slots)] = old[p][:pages_of(lens[p], slots)]
        st.lens[s] = lens[p]
    for s, (_, t, _) in zip(copies, moves):
        st.table[s][st.lens[s] // slots] = t
    for s in range(n):
        for i in range(pages_of(st.lens[s], slots)):
            st.refs[st.table[s][i]] += 1
    return moves


def select(logits, scores, finished, beams, eos):
    """(scores, finished, parents, tokens) of logits [rows, vocab], totals in float64."""
    x = logits.double()
    out = ([], [], [], [])
    for g in range(0, len(scores), beams):
        found = []
        for r in range(g, g + beams):
            if finished[r]:
                if eos >= 0:
                    found.append((scores[r], r, eos))
                continue
            m = x[r].max()
            t = scores[r] + (x[r] - (m + torch.log(torch.exp(x[r] - m).sum())))
            t = torch.where(t.isnan(), -math.inf, t)
            order = torch.argsort(t, descending=True, stable=True)[:beams].tolist()
            found += [(float(t[v]), r, v) for v in order]
        found = sorted([f for f in found if f[0] > -math.inf], key=lambda f: (-f[0], f[1], f[2]))[:beams]
        for i in range(beams):
            total, p, v = found[i] if i < len(found) else (-math.inf, g + i, max(eos, 0))
            out[0].append(total)
            out[1].append(1 if i >= len(found) or finished[p] or v == eos else 0)
            out[2].append(p)
            out[3].append(v)
    return out


def rng(seed):
    return random.Random(seed)
