"""The paged cache in plain form for the tests: integer state as Python lists, values in float64."""
from __future__ import annotations

import torch


def pages_of(n, slots):
    return -(-n // slots)


class State:
    """Table, lengths and reference counts, changed as moa_paged.h says; a refused call returns False and changes
    nothing. `moves` collects the (source, target) page copies of the last call."""

    def __init__(self, table, lens, refs, slots):
        self.table, self.lens, self.refs, self.slots = [list(r) for r in table], list(lens), list(refs), slots
        self.moves = []

    def _lowest_free(self, n):
        free = [p for p, r in enumerate(self.refs) if r == 0][:n]
        return free if len(free) == n else None

    def reserve(self, new):
        cap = len(self.table[0]) * self.slots
        if any(n < 0 or length + n > cap for n, length in zip(new, self.lens)):
            return False
        need = [pages_of(length + n, self.slots) - pages_of(length, self.slots) for n, length in zip(new, self.lens)]
        free = self._lowest_free(sum(need))
        if free is None:
            return False
        for s, n in enumerate(need):
            at = pages_of(self.lens[s], self.slots)
            for i in range(n):
                self.table[s][at + i] = free[0]
                self.refs[free.pop(0)] = 1
            self.lens[s] += new[s]
        return True

    def fork(self, parents, children):
        S, self.moves = len(self.lens), []
        if any(not 0 <= s < S for s in parents + children) or len(set(children)) < len(children):
            return False
        if any(self.lens[c] for c in children) or set(parents) & set(children):
            return False
        free = self._lowest_free(sum(1 for p in parents if self.lens[p] % self.slots))
        if free is None:
            return False
        for p, c in zip(parents, children):
            full = self.lens[p] // self.slots
            for i in range(full):
                self.table[c][i] = self.table[p][i]
                self.refs[self.table[p][i]] += 1
            if self.lens[p] % self.slots:
                self.moves.append((self.table[p][full], free[0]))
                self.table[c][full] = free[0]
                self.refs[free.pop(0)] = 1
            self.lens[c] = self.lens[p]
        return True

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.lens):
                for i in range(pages_of(self.lens[s], self.slots)):
                    self.refs[self.table[s][i]] -= 1
                self.lens[s] = 0

    def compact(self):
        n = sum(1 for r in self.refs if r > 0)
        to = [p for p in range(n) if self.refs[p] == 0]
        src = [p for p in range(n, len(self.refs)) if self.refs[p] > 0]
        place = dict(zip(src, to))
        for s, length in enumerate(self.lens):
            for i in range(pages_of(length, self.slots)):
                self.table[s][i] = place.get(self.table[s][i], self.table[s][i])
        for a, b in place.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.moves = list(place.items())


def positions(row_starts, lens):
    """(row, sequence, position) of every row that belongs to a sequence."""
    return [(m, s, lens[s] - (row_starts[s + 1] - m)) for s in range(len(lens)) for m in range(row_starts[s], row_starts[s + 1])]


def attention(q, k, v, table, lens, row_starts, slots, window, scale, k_scale=None, v_scale=None):
    """Per row in float64 on the tensors' device: (out, a, d) [rows, heads, dim], [rows, heads, dim], [rows, heads].
    a: the attention of |v|; d: the largest scale * sum_i |q_i k_i| among the visible positions, what the rounding of a
    score is relative to. k, v [pages, slots, kv_heads, dim] values; rows of no sequence stay NaN."""
    R, H, D = q.shape
    hk = k.shape[2]
    g = H // hk
    out = torch.full((R, H, D), float("nan"), dtype=torch.float64, device=q.device)
    a, d = out.clone(), torch.zeros((R, H), dtype=torch.float64, device=q.device)
    ks = torch.ones(hk, dtype=torch.float64, device=q.device) if k_scale is None else k_scale.double().reshape(hk)
    vs = torch.ones(hk, dtype=torch.float64, device=q.device) if v_scale is None else v_scale.double().reshape(hk)
    for s, n in enumerate(lens):
        m0, m1 = row_starts[s], row_starts[s + 1]
        if m0 == m1:
            continue
        first = max(0, n - (m1 - m0) + 1 - window) if window else 0
        t = torch.arange(first, max(n, first), device=q.device)
        page = torch.tensor(table[s], device=q.device)[t // slots] if n else t
        kk, vv = k[page, t % slots].double() * ks[:, None], v[page, t % slots].double() * vs[:, None]  # [keys, hk, D]
        for m in range(m0, m1):
            p = n - (m1 - m)
            lo = max(first, p - window + 1) if window else first
            if p < lo:
                out[m], a[m] = 0.0, 0.0
                continue
            kr, vr = kk[lo - first:p + 1 - first], vv[lo - first:p + 1 - first]
            qh = q[m].double().view(hk, g, D)
            kt, vt = kr.permute(1, 2, 0).contiguous(), vr.permute(1, 0, 2).contiguous()
            w = torch.softmax(torch.matmul(qh, kt) * scale, dim=-1)
            out[m], a[m] = torch.matmul(w, vt).reshape(H, D), torch.matmul(w, vt.abs()).reshape(H, D)
            d[m] = (torch.matmul(qh.abs(), kt.abs()) * abs(scale)).amax(-1).reshape(H)
    return out, a, d
