"""Oracle of the paged 8-bit cache and of attention over packed sequences: plain torch on the CPU.

Codes and scales in float32 as the format defines them (each operation rounded), attention in float64.
"""
from __future__ import annotations

import torch

TOP = {"int8": 127.0, "e4m3": 448.0}


def quantise(block: torch.Tensor, code: str):
    """One head's block (page, d) -> (codes as float32, scale): a = max(|x|, 2^-100), scale =
    a * (1 / top), code = rne(x * ((1 / a) * top)), each operation rounded; a block with an infinity or a NaN: zeros, scale NaN."""
    x = block.float()
    if not torch.isfinite(x).all():
        return torch.zeros_like(x), torch.tensor(float("nan"))
    a = x.abs().max().clamp_min(2.0 ** -100)
    top = torch.tensor(TOP[code])
    y = x * ((torch.ones(()) / a) * top)
    c = torch.round(y) if code == "int8" else y.to(torch.float8_e4m3fn).float()
    return c, a * (torch.ones(()) / top)


def cached(x: torch.Tensor, page: int, code: str) -> torch.Tensor:
    """Tokens (n, H, d) as the cache holds them, float64: full blocks code * scale, the rest as it came."""
    y = x.double().clone()
    for j in range(x.shape[0] // page):
        for h in range(x.shape[1]):
            c, s = quantise(x[j * page:(j + 1) * page, h], code)
            y[j * page:(j + 1) * page, h] = c.double() * s.double()
    return y


def attend(q, k, v, scaling, causal=True):
    """q (t, Hq, d) over k, v (n, Hkv, d), the last query at the last key.  Returns (out, mass, score): the
    outputs, sum_j p_j |v_j| and the largest scaling * sum_c |q_c k_c| of the visible keys, float64."""
    (t, Hq, d), (n, Hkv, _) = q.shape, k.shape
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros((t, Hq, d), dtype=torch.float64)
    mass, score = torch.zeros_like(out), torch.zeros((t, Hq, 1), dtype=torch.float64)
    for i in range(t):
        m = min(n, max(0, i + 1 + n - t)) if causal else n
        for h in range(Hq):
            if m == 0:
                continue
            kk, vv = k[:m, h // (Hq // Hkv)], v[:m, h // (Hq // Hkv)]
            p = torch.softmax((kk @ q[i, h]) * scaling, 0)
            out[i, h], mass[i, h] = p @ vv, p @ vv.abs()
            score[i, h] = (kk.abs() @ q[i, h].abs()).max() * abs(scaling)
    return out, mass, score


class Accounts:
    """The page accounts: who holds which page, the lowest free page first."""

    def __init__(self, slots, pages, page):
        self.page, self.refs = page, [0] * pages
        self.lens, self.table = [0] * slots, [[] for _ in range(slots)]

    def extend(self, slots, counts):
        for s, c in zip(slots, counts):
            self.lens[s] += c
            while len(self.table[s]) < self.lens[s] // self.page:
                i = self.refs.index(0)
                self.refs[i] = 1
                self.table[s].append(i)

    def fork(self, src, dst):
        for a, b in zip(src, dst):
            self.lens[b], self.table[b] = self.lens[a], list(self.table[a])
            for p in self.table[b]:
                self.refs[p] += 1

    def free(self, slots):
        for s in slots:
            for p in self.table[s]:
                self.refs[p] -= 1
            self.lens[s], self.table[s] = 0, []

    def move(self, end, pages):
        """Pages >= end to the lowest free places, in order; then ``pages`` pages."""
        live = [p for p, r in enumerate(self.refs) if r]
        holes = [p for p in range(min(end, len(self.refs))) if not self.refs[p]]
        to = {p: p for p in live}
        for p, hole in zip([p for p in live if p >= end], holes):
            to[p] = hole
        refs = [0] * pages
        for p in live:
            refs[to[p]] = self.refs[p]
        self.refs, self.table = refs, [[to[p] for p in t] for t in self.table]
