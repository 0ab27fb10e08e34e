"""Plain implementations of the paged-cache operators (test infrastructure).

Floating point in 64 bits, one row at a time; page bookkeeping as Python lists, one sequence at a
time.  Nothing here shares code with the operators.
"""

from __future__ import annotations

import math

import torch


def attention(q, k_pages, v_pages, table, kv_lens, query_start, mask=None, scale=None, causal=True):
    """``(output, sum_j p_j |v_j|)`` in 64 bits, ``[N,Hq,D]`` each; rows behind the last sequence zero."""
    q, k_pages, v_pages = (t.detach().cpu().double() for t in (q, k_pages, v_pages))
    table, kv_lens, query_start = table.tolist(), kv_lens.tolist(), query_start.tolist()
    N, Hq, D = q.shape
    page, Hk = k_pages.shape[1], k_pages.shape[2]
    rep = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    on = torch.ones(N, Hq, dtype=torch.bool)
    if mask is not None:
        on = (mask.cpu() != 0).repeat_interleave(Hq // mask.shape[1], dim=1)
    for s, L in enumerate(kv_lens):
        a, b = query_start[s], query_start[s + 1]
        if L == 0 or a == b:
            continue
        ids = table[s][:-(-L // page)]
        k = k_pages[ids].reshape(-1, Hk, D)[:L].repeat_interleave(rep, dim=1)
        v = v_pages[ids].reshape(-1, Hk, D)[:L].repeat_interleave(rep, dim=1)
        for t in range(a, b):
            n = min(L, L - (b - a) + (t - a) + 1) if causal else L
            if n <= 0:
                continue
            z = torch.einsum("hd,khd->hk", q[t], k[:n]) * scale
            p = torch.softmax(z, dim=1)
            out[t] = torch.einsum("hk,khd->hd", p, v[:n]) * on[t][:, None]
            size[t] = torch.einsum("hk,khd->hd", p, v[:n].abs()) * on[t][:, None]
    return out, size


def rotate(x, positions, inv_freq, axis_of_pair, interleaved=False, scale=1.0):
    """``x [N,heads,D]`` turned, and ``|a| + |b|`` of the pair of every channel, in 64 bits."""
    x = x.detach().cpu().double()
    pos, f = positions.cpu().double(), inv_freq.cpu().double()
    if pos.dim() == 1:
        pos = pos[None]
    out, size = x.clone(), x.abs().clone()
    half = len(f)
    for i in range(half):
        angle = pos[axis_of_pair[i]] * f[i]
        c, s = (torch.cos(angle) * scale)[:, None], (torch.sin(angle) * scale)[:, None]
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
        a, b = x[..., ia], x[..., ib]
        out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
        size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * abs(scale)
    return out, size


class Pages:
    """The state of a cache as Python integers, and the operators on it."""

    def __init__(self, table, lens, refs, page):
        self.table, self.lens = [list(r) for r in table], list(lens)
        self.refs, self.page = list(refs), page

    def held(self, s):
        return math.ceil(self.lens[s] / self.page)

    def extend(self, add):
        """``(granted, [(src page, dst page, rows)])``."""
        S, W, page = len(self.lens), len(self.table[0]), self.page
        free = [p for p, r in enumerate(self.refs) if r == 0]
        fits = [a >= 0 and math.ceil((n + a) / page) <= W for n, a in zip(self.lens, add)]
        tail = [self.table[s][self.held(s) - 1] if fits[s] and add[s] > 0 and self.lens[s] % page else -1
                for s in range(S)]
        tail = [t if t >= 0 and self.refs[t] > 1 else -1 for t in tail]
        copies, keeps = [False] * S, [None] * S
        for s in range(S):
            if tail[s] < 0:
                continue
            writers = [j for j in range(S) if tail[j] == tail[s]]
            if len(writers) == self.refs[tail[s]] and writers[0] == s:
                keeps[s] = writers[-1]
            else:
                copies[s] = True
        need = [(math.ceil((self.lens[s] + add[s]) / page) - self.held(s) if fits[s] else 0) + copies[s]
                for s in range(S)]
        upto, total = [], 0
        for n in need:
            total += n
            upto.append(total)
        granted = [fits[s] and (need[s] == 0 or upto[s] <= len(free))
                   and (keeps[s] is None or upto[keeps[s]] <= len(free)) for s in range(S)]
        moves = []
        for s in range(S):
            if not granted[s]:
                continue
            mine = free[upto[s] - need[s]:upto[s]]
            held = self.held(s)
            if copies[s]:
                moves.append((tail[s], mine[0], self.lens[s] % page))
                self.refs[tail[s]] -= 1
                self.table[s][held - 1] = mine[0]
                self.refs[mine[0]] = 1
                mine = mine[1:]
            for j, p in enumerate(mine):
                self.table[s][held + j] = p
                self.refs[p] = 1
            self.lens[s] += add[s]
        return granted, moves

    def fork(self, parents, children):
        before, done = list(self.lens), []
        for i, (p, c) in enumerate(zip(parents, children)):
            ok = 0 <= p < len(before) and 0 <= c < len(before) and c not in children[:i] and before[c] == 0
            done.append(ok)
            if ok:
                for j in range(math.ceil(before[p] / self.page)):
                    self.table[c][j] = self.table[p][j]
                    self.refs[self.table[p][j]] += 1
                self.lens[c] = before[p]
        return done

    def trim(self, rows, keep):
        for i, (s, to) in enumerate(zip(rows, keep)):
            if s in rows[:i] or not 0 <= s < len(self.lens) or to < 0 or to >= self.lens[s]:
                continue
            for j in range(math.ceil(to / self.page), self.held(s)):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lens[s] = to

    def compact(self):
        """``(live, [(src page, dst page)])``."""
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(len(self.lens)):
            for j in range(self.held(s)):
                self.table[s][j] = to.get(self.table[s][j], self.table[s][j])
        return live, list(to.items())
