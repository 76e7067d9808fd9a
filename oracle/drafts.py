"""Verification of drafted tokens with exact fractions, token by token."""
from __future__ import annotations

import math
from fractions import Fraction

import torch


def _part(x: float) -> Fraction:
    return Fraction(x) if x > 0 and math.isfinite(x) else Fraction(0)


def _pick(rest, r: float) -> int:
    """The first index at which the running sum passes r times the total; -1 for nothing."""
    total = sum(rest, Fraction(0))
    if total == 0:
        return -1
    edge = (Fraction(min(r, 1.0)) if r > 0 else Fraction(0)) * total
    run, last = Fraction(0), -1
    for i, x in enumerate(rest):
        if x > 0:
            run, last = run + x, i
            if run > edge:
                return i
    return last


def verify(target, draft, tokens, accept, sample, counts=None):
    b, k = tokens.shape
    vocab = target.shape[2]
    out, taken = torch.full((b, k + 1), -1, dtype=torch.int64), torch.zeros(b, dtype=torch.int32)
    for i in range(b):
        count = k if counts is None else max(0, min(k, int(counts[i])))
        n, rest = 0, None
        while n < count:
            x = int(tokens[i, n])
            inside = 0 <= x < vocab
            p = float(target[i, n, x]) if inside else 0.0
            q = (1.0 if draft is None else float(draft[i, n, x])) if inside else 0.0
            u = float(accept[i, n])
            if inside and all(map(math.isfinite, (u, p, q))) and Fraction(u) * Fraction(q) < Fraction(p):
                out[i, n] = x
                n += 1
                continue
            row = [float(y) for y in target[i, n]]
            if draft is None:
                rest = [Fraction(0) if j == x else _part(y) for j, y in enumerate(row)]
            else:
                other = [float(y) for y in draft[i, n]]
                rest = [max(Fraction(y) - Fraction(z), Fraction(0)) if _part(y) and math.isfinite(z) else Fraction(0)
                        for y, z in zip(row, other)]
            if sum(rest, Fraction(0)) == 0:
                rest = [_part(y) for y in row]
            break
        if rest is None:
            rest = [_part(float(y)) for y in target[i, n]]
        out[i, n] = _pick(rest, float(sample[i]))
        taken[i] = n
    return out, taken
