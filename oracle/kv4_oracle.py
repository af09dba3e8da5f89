"""Plain restatement of the paged 4-bit KV cache and of token scoring, in 64 bits on the CPU.

``quantise`` / ``value`` are the number format, ``Pages`` the page management with Python lists, ``attend`` the attention
over a row's dequantised keys and values, ``score`` the log probabilities, entropy and alternatives of logits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE = 64
OVERFLOW = 2.0 ** 122


def quantise(x: torch.Tensor):
    """Integers -7..7 [..., hd] and scales [..., hd / 32] in float64."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)                       # NaN where the group has one
    bad = ~(top < OVERFLOW)
    t = np.where(bad.numpy(), 0.0, top.numpy()) / 7.0
    mant, exp = np.frexp(t.astype(np.float32).astype(np.float64))
    # 4 significant bits; below the smallest normal float32 the spacing stays that of the smallest normal's
    low = np.maximum(0, -125 - exp)
    s = np.ldexp(np.rint(np.ldexp(mant, 4 - low)), exp + low - 4)
    s = torch.from_numpy(np.where(bad.numpy(), 0.0, s))
    n = torch.where(s[..., None] > 0, g.nan_to_num(0, 0, 0) / torch.where(s > 0, s, 1.0)[..., None], 0.0)
    n = torch.from_numpy(np.rint(n.numpy())).clamp(-7, 7)
    return n.flatten(-2), torch.where(bad, float("nan"), s)


def value(n: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    return (n.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def dequantised(x: torch.Tensor) -> torch.Tensor:
    return value(*quantise(x))


class Pages:
    """Tables, lengths and holders of a cache; ``content[page]`` is a dict slot -> whatever was written there."""

    def __init__(self, rows: int, row_pages: int, pages: int):
        self.table = [[] for _ in range(rows)]
        self.row_pages, self.n = row_pages, pages
        self.lengths, self.counts = [0] * rows, [0] * rows
        self.content = [dict() for _ in range(pages)]
        self.error = False

    def refs(self):
        r = [0] * self.n
        for t in self.table:
            for p in t:
                r[p] += 1
        return r

    def extend(self, counts):
        R = len(self.table)
        refs = self.refs()
        if any(c < 0 or l + c > self.row_pages * PAGE for c, l in zip(counts, self.lengths)):
            return self._refuse()
        copy = []
        left = list(refs)
        for r in range(R):
            part = self.table[r][-1] if counts[r] > 0 and self.lengths[r] % PAGE else None
            copy.append(part is not None and left[part] > 1)
            if copy[r]:
                left[part] -= 1
        fresh = [-(-(l + c) // PAGE) - -(-l // PAGE) if c > 0 else 0 for l, c in zip(self.lengths, counts)]
        free = [p for p in range(self.n) if refs[p] == 0]
        if sum(fresh) + sum(copy) > len(free):
            return self._refuse()
        for r in range(R):
            if copy[r]:
                p = free.pop(0)
                self.content[p] = dict(self.content[self.table[r][-1]])
                self.table[r][-1] = p
            for _ in range(fresh[r]):
                self.table[r].append(free.pop(0))
            self.lengths[r] += counts[r]
        self.counts = list(counts)

    def _refuse(self):
        self.counts = [0] * len(self.table)
        self.error = True

    def write(self, r, pos, what):
        self.content[self.table[r][pos // PAGE]][pos % PAGE] = what

    def row(self, r):
        return [self.content[self.table[r][p // PAGE]].get(p % PAGE) for p in range(self.lengths[r])]

    def fork(self, parents):
        table = [list(t) for t in self.table]
        lengths = list(self.lengths)
        for r, p in enumerate(parents):
            if p >= len(parents):
                self.error = True
                continue
            self.table[r] = [] if p < 0 else list(table[p])
            self.lengths[r] = 0 if p < 0 else lengths[p]
        self.counts = [0] * len(parents)

    def rollback(self, n):
        for r, k in enumerate(n):
            if k < 0 or k > self.lengths[r]:
                self.error = True
                continue
            self.lengths[r] -= k
            del self.table[r][-(-self.lengths[r] // PAGE):]
        self.counts = [0] * len(self.table)

    def free(self, rows):
        for r in rows:
            self.table[r], self.lengths[r], self.counts[r] = [], 0, 0

    def compact(self):
        refs = self.refs()
        used = sum(x > 0 for x in refs)
        to = dict(zip([p for p in range(used, self.n) if refs[p]], [p for p in range(used) if not refs[p]]))
        for a, b in to.items():
            self.content[b] = self.content[a]
            self.content[a] = dict()
        self.table = [[to.get(p, p) for p in t] for t in self.table]
        return used


def attend(q, k, v, length: int, count: int, scale: float, window: int = 0) -> torch.Tensor:
    """q [S, Hq, hd], k / v [length, Hkv, hd] float64 -> [S, Hq, hd]; zeros behind ``count`` queries."""
    S, Hq, hd = q.shape
    out = torch.zeros(S, Hq, hd, dtype=torch.float64)
    G = Hq // k.shape[1]
    for i in range(count):
        pos = length - count + i
        lo = max(0, pos - window + 1) if window else 0
        for h in range(Hq):
            s = scale * (k[lo:pos + 1, h // G] @ q[i, h].double())
            out[i, h] = torch.softmax(s, 0) @ v[lo:pos + 1, h // G]
    return out


def score(x: torch.Tensor, token: int, top_n: int):
    """(log p, entropy, [(id, log p)]) of one logits row, in Python's 64-bit floats."""
    x = [float(t) for t in x.double()]
    m = max(x)
    if any(t != t for t in x) or not math.isfinite(m):
        nan = float("nan")
        return nan, nan, None
    lse = m + math.log(math.fsum(math.exp(t - m) for t in x))
    ent = -math.fsum(math.exp(t - lse) * (t - lse) for t in x if t > -math.inf)
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))[:top_n]
    lp = 0.0 if token < 0 else x[token] - lse if token < len(x) else float("nan")
    return lp, ent, [(i, x[i] - lse) for i in order]
