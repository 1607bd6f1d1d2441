"""Page tables kept by plain lists, drafted trees, and attention over a request's keys in
64 bits with its error bounds."""

from __future__ import annotations

import math

import torch


class Book:
    """The tables of ``gki.PageTable``: pages from a queue, in the order of requests and
    positions; dead ones return to its end in the same order before any are taken."""

    def __init__(self, requests, pages, page, sink, window, max_pages=None):
        self.page, self.sink, self.window = page, sink, window
        self.max_pages = pages if max_pages is None else max_pages
        self.queue, self.table = list(range(pages)), [{} for _ in range(requests)]
        self.length, self.taken = [0] * requests, [0] * requests

    def refusal(self, counts, rows, max_count):
        """Bits of why a step does not fit."""
        bad = any(c < 0 or c > max_count or n + c > self.max_pages * self.page for c, n in zip(counts, self.length))
        if bad:
            return 4
        why = 2 if sum(counts) > rows else 0
        dead = sum(len(self._dead(r)) for r, c in enumerate(counts) if c)
        new = sum(max(0, -(-(n + c) // self.page) - t) for c, n, t in zip(counts, self.length, self.taken) if c > 0)
        return why | (1 if new > len(self.queue) + dead else 0)

    def _dead(self, r):
        """Pages without sinks that the next token (at position length) and later ones do not
        see, the one it goes to left out."""
        n = self.length[r]
        return [i for i in sorted(self.table[r]) if i * self.page >= self.sink and (i + 1) * self.page <= n
                and i * self.page + self.page - 1 <= n - self.window]

    def extend(self, counts):
        for r, c in enumerate(counts):
            for i in self._dead(r) if c else ():
                self.queue.append(self.table[r].pop(i))
        base = list(self.length)
        for r, c in enumerate(counts):
            for i in range(self.taken[r], -(-(self.length[r] + c) // self.page) if c else 0):
                self.table[r][i] = self.queue.pop(0)
                self.taken[r] = i + 1
            self.length[r] += c
        return base

    def release(self, done):
        for r, d in enumerate(done):
            if d:
                self.queue += [self.table[r][i] for i in sorted(self.table[r])]
                self.table[r], self.length[r], self.taken[r] = {}, 0, 0

    def slot(self, r, x):
        return self.table[r][x // self.page] * self.page + x % self.page


def chains(parents):
    """Each node's ancestors and itself, the root first; a parent that is no earlier node counts as none."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def seen(base, n, sink, window, parents=None):
    """bool [n, base + n]: which stored keys each of a request's new rows sees."""
    out = torch.zeros(n, base + n, dtype=torch.bool)
    x = torch.arange(base + n)
    if parents is None:
        p = base + torch.arange(n)[:, None]
        return (x <= p) & ((x < sink) | (x > p - window))
    for i, chain in enumerate(chains(parents)):
        p = base + len(chain) - 1
        out[i, :base] = (x[:base] < sink) | (x[:base] > p - window)
        for depth, j in enumerate(chain):
            out[i, base + j] = base + depth < sink or base + depth > p - window
    return out


def attend(q, k, v, visible, scale, dtype):
    """One request: q [n, H, D], k / v [m, H_kv, D], visible [n, m]. O, LSE, the bound of each
    output and its mean square error (roundings of half a unit: of P, of a row sum over rounded
    P, of O; an fp16 number below 2^-14 is off by up to 2^-25), the bound of the LSE."""
    n, H, D = q.shape
    group = H // k.shape[1]
    half = torch.finfo(dtype).eps / 2
    u = 2.0**-25 if dtype == torch.float16 else 0.0
    q, k, v = q.double(), k.double().repeat_interleave(group, 1), v.double().repeat_interleave(group, 1)
    q, k, v = q.transpose(0, 1), k.permute(1, 2, 0).contiguous(), v.transpose(0, 1).contiguous()
    s = (q @ k) * scale
    s = torch.where(visible, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top.isinf(), torch.zeros_like(top), top))
    l = e.sum(-1, keepdim=True)
    P = e / torch.where(l == 0, torch.ones_like(l), l)
    o = P @ v
    lse = torch.where(l == 0, torch.zeros_like(l), torch.where(l == 0, torch.zeros_like(top), top) + torch.log(l.clamp(min=1e-300)))
    size = torch.where(visible, (q.abs() @ k.abs()) * abs(scale), torch.zeros_like(s)).amax(-1, keepdim=True)
    # fp32: scores of D <= 128 terms off by 136 units of 2^-24 of their size, sums by 2^-24 a term
    f32 = 2 * 136 * 2.0**-24 * size + (k.shape[2] + 300) * 2.0**-24
    pv, keys = P @ v.abs(), visible.sum(-1)[:, None]
    small = u * (visible.double() @ v.abs() + keys * pv)
    bound = half * o.abs() + (2 * half + f32) * 1.02 * pv + small + u
    mean = half**2 * (P**2 @ v**2 + 2 * o**2) + (f32 * pv) ** 2 + u**2 * (visible.double() @ v**2 + keys * o**2 + 1)
    lse_bound = 1.01 * half + f32 + 2.0**-23 * lse.abs() + u * keys
    out = [t.transpose(0, 1) for t in (o, bound, mean)]
    return out[0], lse[..., 0].T, out[1], out[2], lse_bound[..., 0].T
