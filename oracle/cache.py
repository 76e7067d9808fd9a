"""The 8-bit cache in exact arithmetic, sequence by sequence and page by page."""
from __future__ import annotations

import math

import torch

from oracle import attend as at

TOP = 448.0
LEAST = -110


def decode(codes):
    """float64 values of e4m3 codes in bytes (sign, 4 bits of exponent with bias 7, 3 of fraction; 0x7F is NaN)."""
    c = codes.long()
    exponent, fraction = (c >> 3) & 15, (c & 7).double()
    value = torch.where(exponent == 0, fraction * 2.0 ** -9, (1 + fraction / 8) * torch.exp2((exponent - 7).double()))
    value = torch.where((c & 0x7F) == 0x7F, torch.full_like(value, math.nan), value)
    return torch.where(c >= 128, -value, value)


def encode(x):
    """Codes of the nearest e4m3 values, ties to even; what is larger becomes the largest, NaN 0x7F."""
    a = x.abs().clamp(max=TOP)
    finite = torch.where(torch.isnan(a), torch.zeros_like(a), a)
    exponent = (torch.frexp(finite)[1] - 1).clamp(min=-6)
    steps = torch.round(finite * torch.exp2((3 - exponent).double()))  # torch.round is to even
    up = steps == 16
    exponent, steps = torch.where(up, exponent + 1, exponent).long(), torch.where(up, torch.full_like(steps, 8), steps).long()
    code = torch.where(steps < 8, steps, ((exponent + 7) << 3) + (steps - 8))
    code = torch.where(torch.isnan(x), torch.full_like(code, 0x7F), code)
    return (code + torch.where(torch.signbit(x), 128, 0)).to(torch.uint8)


def scale_for(amax: float) -> float:
    """2^e, the least with amax <= 448 * 2^e and e >= -110."""
    fraction, exponent = math.frexp(amax)  # amax = fraction * 2^exponent, 448 = 0.875 * 2^9
    return 2.0 ** max(LEAST, exponent - 9 + (fraction > 0.875))


def write(k, v, k_cache, v_cache, k_scales, v_scales, table, lengths, counts=None):
    """Writes in place (codes uint8, scales float32), on the CPU."""
    b, t, heads, _ = k.shape
    pages, _, page, _ = k_cache.shape
    for i in range(b):
        n = t if counts is None else max(0, min(t, int(counts[i])))
        begin = max(int(lengths[i]), 0) - n
        for slot in range(table.shape[1]):
            low, high = max(begin, slot * page), min(begin + n, (slot + 1) * page)
            id_ = int(table[i, slot])
            if low >= high or not 0 <= id_ < pages:
                continue
            off, count = low - slot * page, high - low
            for x, codes, scales in ((k, k_cache, k_scales), (v, v_cache, v_scales)):
                for h in range(heads):
                    new = x[i, low - begin:high - begin, h].double()
                    fine = new[torch.isfinite(new)].abs()
                    amax = float(fine.max()) if fine.numel() else 0.0
                    was = float(scales[id_, h])
                    keeps = off > 0 and 0.0 < was < math.inf
                    s = scale_for(amax) if amax > 0 else was if keeps else 1.0
                    if keeps and was >= s:
                        s = was
                    if off and s != was:
                        codes[id_, h, :off] = encode(decode(codes[id_, h, :off]) * was / s)
                    codes[id_, h, off:off + count] = encode(new / s)
                    scales[id_, h] = s


def attention(q, k_cache, v_cache, k_scales, v_scales, table, lengths, counts=None, scale=None):
    """attend()'s three over each sequence's cached tokens; rows from counts on are 0."""
    b, t, h, d = q.shape
    pages, heads, page, _ = k_cache.shape
    every = []
    for i in range(b):
        n = t if counts is None else max(0, min(t, int(counts[i])))
        length = max(0, min(int(lengths[i]), table.shape[1] * page))
        before = max(int(lengths[i]), 0) - n
        ids = [int(x) for x in table[i, :-(-length // page)]]
        there = torch.tensor([0 <= x < pages for x in ids], dtype=torch.bool).repeat_interleave(page)[:length]
        ids = [x if 0 <= x < pages else 0 for x in ids]

        def gathered(codes, scales):
            if not length:
                return torch.zeros((0, heads, d), dtype=torch.float64)
            x = torch.stack([decode(codes[j]) * scales[j].double()[:, None, None] for j in ids])
            return x.permute(0, 2, 1, 3).reshape(-1, heads, d)[:length]

        seen = there[None] & (torch.arange(length)[None] <= before + torch.arange(t)[:, None])
        seen = seen & (torch.arange(t) < n)[:, None]
        every.append(at.attend(q[i], gathered(k_cache, k_scales), gathered(v_cache, v_scales), seen, d ** -0.5 if scale is None else scale))
    return tuple(torch.stack(x) for x in zip(*every))
