"""Token log probabilities, entropies and alternatives in 64 bits."""
from __future__ import annotations

import torch

from oracle.experts import best


def token_logprobs(logits, tokens, top):
    """(logprobs, entropy, top_logprobs, top_ids) of logits [R, V], floats in
    float64: log p = x - m - log sum exp(x - m), entropy = -sum p log p (0 log 0 = 0)."""
    x = logits.double()
    m = x.amax(1, keepdim=True)
    # (x - m) first: next to a maximum of 1e38, log(sum) is lost even in 64 bits
    logp = (x - m) - torch.log(torch.exp(x - m).sum(1, keepdim=True))
    p = torch.exp(logp)
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(1)
    r, v = x.shape
    inside = (tokens >= 0) & (tokens < v)
    lp = torch.where(inside, logp.gather(1, tokens.clamp(0, v - 1)[:, None])[:, 0], torch.full((r,), float("nan")).double())
    ids = torch.empty((r, top), dtype=torch.int64)
    for i in range(r):
        ids[i] = torch.tensor(best(x[i].tolist(), top), dtype=torch.int64)
    return lp, entropy, logp.gather(1, ids), ids
