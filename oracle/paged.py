"""The paged KV cache in 64 bits, from its definition.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). Rows are laid out one position
at a time from the page table, in Python.
"""
from __future__ import annotations

import math

import torch


def cell(table, pages, page, row, position):
    """``(page, place)`` of a position, or None where it has no page."""
    if not 0 <= row < table.shape[0] or not 0 <= position < table.shape[1] * page:
        return None
    at = int(table[row, position // page])
    return (at, position % page) if 0 <= at < pages else None


def row(pool, table, b, n):
    """Positions ``0 .. n-1`` of row ``b`` of ``pool [P, H, page, D]``: ``[H, n, D]`` in 64 bits, and which of
    them have a page."""
    pages, heads, page, dim = pool.shape
    n = max(0, min(n, table.shape[1] * page))
    out, there = torch.zeros(heads, n, dim, dtype=torch.float64), torch.zeros(n, dtype=torch.bool)
    for first in range(0, n, page):
        c, last = cell(table, pages, page, b, first), min(n, first + page)
        if c:
            out[:, first:last] = pool[c[0], :, :last - first].double()
            there[first:last] = True
    return out, there


def attention(q, pk, pv, table, used, scale, limit=None):
    """``q [B, Hq, D]`` over the rows of ``pk, pv``: the result, and per row the probabilities ``[Hkv, G, n]``
    (0 without a page); a row with nothing gives zeros."""
    b, hq, d = q.shape
    hkv = pk.shape[1]
    out, probabilities = torch.zeros(b, hq, d, dtype=torch.float64), []
    for i in range(b):
        n = int(used[i]) if limit is None else min(int(used[i]), limit)
        k, there = row(pk, table, i, n)
        v, _ = row(pv, table, i, n)
        p = torch.zeros(hkv, hq // hkv, k.shape[1], dtype=torch.float64)
        if bool(there.any()):
            s = (q[i].double().view(hkv, hq // hkv, d) @ k.transpose(1, 2) * scale)[:, :, there]
            p[:, :, there] = torch.softmax(s, -1)
            out[i] = (p @ v).reshape(hq, d)
        probabilities.append(p)
    return out, probabilities


def angles(positions, rotary, theta):
    """cos, sin ``[T, rotary / 2]`` in 64 bits."""
    inv = torch.tensor([theta ** (-2 * i / rotary) for i in range(rotary // 2)], dtype=torch.float64)
    a = positions.double()[:, None] * inv
    return a.cos(), a.sin()


def rotate(x, cos, sin, neox, rounded=False):
    """``x [T, heads, D]`` turned by ``cos, sin [T, R / 2]`` in 64 bits; ``rounded``: each product and sum to bf16,
    as a bf16 table has it."""
    def held(t):
        # a product of two bf16 values is exact in fp32, and so is what it rounds from
        return t.to(torch.bfloat16).double() if rounded else t
    o, r = x.double().clone(), 2 * cos.shape[-1]
    for i in range(r // 2):
        a, b = (i, i + r // 2) if neox else (2 * i, 2 * i + 1)
        x1, x2, c, s = x[..., a].double(), x[..., b].double(), cos[:, None, i], sin[:, None, i]
        o[..., a] = held(held(x1 * c) - held(x2 * s))
        o[..., b] = held(held(x2 * c) + held(x1 * s))
    return o


def keep(weights, n, count, recent):
    """The positions that stay of one row's ``n``: sorted by weight, the first of equal ones, one at a time."""
    if n <= count:
        return list(range(n))
    free = n - recent

    def rank(j):
        w = float(weights[j])
        return (0, 0.0, j) if math.isnan(w) else (1, -w, j)
    return sorted(sorted(range(free), key=rank)[:count - recent] + list(range(free, n)))
