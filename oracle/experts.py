"""Expert routing, dispatch and combine in 64 bits, token by token."""
from __future__ import annotations

import math

import torch


def _before(a, i, b, j):
    """Score a of index i stands before score b of index j: NaN first, then the
    higher, then the lower index (+0 and -0 equal)."""
    an, bn = math.isnan(a), math.isnan(b)
    if an or bn:
        return (an and not bn) or (an and bn and i < j)
    return a > b or (a == b and i < j)


class _Ranked:
    def __init__(self, score, index):
        self.score, self.index = score, index

    def __lt__(self, other):
        return _before(self.score, self.index, other.score, other.index)


def best(scores, k):
    """Indices of the k best of a list of floats, best first."""
    return [r.index for r in sorted(_Ranked(float(s), i) for i, s in enumerate(scores))[:k]]


def scores64(logits, kind):
    x = logits.double()
    if kind == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    e = torch.exp(x - x.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def route(logits, top_k, bias=None, scores="softmax", groups=1, top_groups=1, renormalize=True, scale=1.0):
    """(weights float64, experts int32) of logits [T, E] on the CPU."""
    t, e = logits.shape
    s = scores64(logits, scores)
    choice = logits.double() if bias is None else s + bias.double()
    size = e // groups
    weights = torch.empty((t, top_k), dtype=torch.float64)
    experts = torch.empty((t, top_k), dtype=torch.int32)
    for i in range(t):
        row = choice[i].tolist()
        allowed = list(range(e))
        if top_groups < groups:
            group_scores = []
            for g in range(groups):
                part = row[g * size:(g + 1) * size]
                pick = best(part, 1 if bias is None else min(2, size))
                group_scores.append(part[pick[0]] if len(pick) == 1 else part[pick[0]] + part[pick[1]])
            kept = sorted(best(group_scores, top_groups))
            allowed = [g * size + j for g in kept for j in range(size)]
        chosen = [allowed[j] for j in best([row[a] for a in allowed], top_k)]
        experts[i] = torch.tensor(chosen, dtype=torch.int32)
        w = s[i, chosen]
        weights[i] = (w / w.sum() if renormalize else w) * scale
    return weights, experts


def dispatch(x, experts, num_experts):
    """(tokens of the filled rows, offsets, slots) by walking the assignments."""
    t, k = experts.shape
    slots = torch.full((t, k), -1, dtype=torch.int32)
    tokens, offsets = [], [0]
    for e in range(num_experts):
        for i in range(t):
            for j in range(k):
                if int(experts[i, j]) == e:
                    slots[i, j] = len(tokens)
                    tokens.append(i)
        offsets.append(len(tokens))
    return torch.tensor(tokens, dtype=torch.int64), torch.tensor(offsets, dtype=torch.int32), slots


def combine(y, weights, slots):
    """(float64 sums, sum of |weight * element|) of each output."""
    rows = y.double()[slots.clamp(min=0).long()]
    valid = ((slots >= 0) & (slots < y.shape[0])).unsqueeze(-1)
    terms = torch.where(valid, rows * weights.double().unsqueeze(-1), torch.zeros((), dtype=torch.float64))
    return terms.sum(1), terms.abs().sum(1)
