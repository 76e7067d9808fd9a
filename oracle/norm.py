"""Group norm in 64 bits, from the definition, one group at a time."""
from __future__ import annotations

import torch


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, silu=False):
    """float64 result of channels-last x [N, ..., C], and the pieces that the
    tests' error bounds need: {"y", "mean", "scale", "before"} with one mean and
    one 1 / sqrt(var + eps) * |weight| per element, and y before the SiLU."""
    n, c = x.shape[0], x.shape[-1]
    per = c // groups
    v = x.double().reshape(n, -1, c)
    mean, inv = torch.empty_like(v), torch.empty_like(v)
    for i in range(n):
        for g in range(groups):
            part = v[i, :, g * per:(g + 1) * per]
            mu = part.sum() / part.numel()
            mean[i, :, g * per:(g + 1) * per] = mu
            inv[i, :, g * per:(g + 1) * per] = 1.0 / torch.sqrt(((part - mu) ** 2).sum() / part.numel() + eps)
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    before = (v - mean) * inv * w + b
    y = before / (1.0 + torch.exp(-before)) if silu else before
    shape = x.shape
    return {"y": y.view(shape), "mean": mean.view(shape), "scale": (inv * w.abs()).view(shape),
            "before": before.view(shape)}


def blocked(t, channels):
    """NC1HWC0 -> channels-last [N, H, W, channels]."""
    n, c1, h, w, _ = t.shape
    return t.permute(0, 2, 3, 1, 4).reshape(n, h, w, c1 * 16)[..., :channels]
