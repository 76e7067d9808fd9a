"""Attention of rows to the keys that each sees, in 64 bits."""
from __future__ import annotations

import torch


def attend(q, k, v, seen, scale):
    """Of q [T, H, D], k and v [S, Hk, D] and seen [T, S]: the result [T, H, D], the
    sums of p |v| with the same weights, and the largest scale * sum |q k| of what a
    row sees [T, H].  What is not seen takes no part; rows that see nothing are 0."""
    t, h, d = q.shape
    group = h // k.shape[1]
    out, size, reach = torch.zeros((t, h, d), dtype=torch.float64), torch.zeros((t, h, d), dtype=torch.float64), torch.zeros((t, h), dtype=torch.float64)
    q, k, v = q.double(), k.double(), v.double()
    apart = not (torch.isfinite(k).all() and torch.isfinite(v).all())
    for j in range(h):
        kj, vj = k[:, j // group], v[:, j // group]
        for rows in ([slice(i, i + 1) for i in range(t)] if apart else [slice(0, t)]):
            see = seen[rows]
            cols = see[0] if apart else torch.ones(k.shape[0], dtype=torch.bool)
            if not see.any():
                continue
            kk, vv, see = kj[cols], vj[cols], see[:, cols]
            s = (q[rows, j] @ kk.t() * scale).masked_fill(~see, -torch.inf)
            reach[rows, j] = (q[rows, j].abs() @ kk.abs().t() * scale).masked_fill(~see, 0).amax(1)
            m = s.amax(1, keepdim=True)
            e = torch.exp(s - torch.where(m == -torch.inf, torch.zeros_like(m), m))
            total = e.sum(1, keepdim=True)
            p = torch.where(total == 0, torch.zeros_like(e), e / total)
            out[rows, j], size[rows, j] = p @ vv, p @ vv.abs()
    return out, size, reach


def cross_attention(q, k, v, lengths=None, mask=None, scale=None):
    b, t, _, d = q.shape
    s = k.shape[1]
    parts = []
    for i in range(b):
        seen = torch.ones(s, dtype=torch.bool) if mask is None else mask[i].bool()
        if lengths is not None:
            seen = seen & (torch.arange(s) < int(lengths[i]))
        parts.append(attend(q[i], k[i], v[i], seen[None].expand(t, s), d ** -0.5 if scale is None else scale))
    return tuple(torch.stack(x) for x in zip(*parts))


def allowed(q, result, keys, extra=0.0):
    """How far the kernels' outputs may be from `result` of attend(), with u = 2^-24
    and h = eps / 2 of the type:
      a score is off by D u of scale sum |q k| (products exact, sums in 32 bits),
        and by 2 u of itself times its constants;
      its exponent (in bits, log2(e) of that) by 4 u more of the score and the
        maximum; the exponential by 2 u, and by 2 u for each of up to 32 rescalings;
      a weight is rounded once to the type (h), or, subnormal as a half, by 2^-33 of
        the largest (they are scaled by 2^8); the total keeps the unrounded ones;
        one below 2^-126 of the largest, the least normal of 32 bits, is lost
        (`extra`: the largest value that a weight may come with);
      the sums over the keys by `keys` u at most, in the total and in the mix;
      the result is rounded once (h, or half a subnormal)."""
    out, size, reach = result
    u, h = 2.0 ** -24, torch.finfo(q.dtype).eps / 2
    eps = (q.shape[-1] + 12) * u * reach[..., None] * 1.01 + 80 * u
    tiny = keys * (2.0 ** -33 if q.dtype == torch.float16 else 2.0 ** -126)
    return 1.01 * ((h + 2 * eps + 2 * keys * u) * size + h * out.abs()) + tiny * extra + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
