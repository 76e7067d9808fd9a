"""Rotary positions with several axes in 64 bits, pair by pair."""
from __future__ import annotations

import torch


def rotary_axes(x, positions, freqs, axes, interleaved=False, inverse=False):
    """(float64 result, |a| + |b| of each element's pair) of x [B, T, H, D]."""
    out, size = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    pairs = freqs.numel()
    for i in range(pairs):
        first, second = (2 * i, 2 * i + 1) if interleaved else (i, pairs + i)
        a, b = x[..., first].double(), x[..., second].double()
        axis = int(axes[i])
        if not 0 <= axis < positions.shape[0]:
            continue
        angle = (positions[axis].double() * float(freqs[i]))[..., None]
        cos, sin = torch.cos(angle), torch.sin(angle) * (-1.0 if inverse else 1.0)
        out[..., first] = a * cos - b * sin
        out[..., second] = b * cos + a * sin
        size[..., first] = size[..., second] = a.abs() + b.abs()
    return out, size
