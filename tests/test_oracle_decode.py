"""The 64-bit definitions of the rotary positions, the cache and the drafts
against other ways to the same values."""
import math

import torch

from oracle import attend, cache, drafts, rotary
from tests.helpers import gen


def test_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.int64).to(torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double()
    got = cache.decode(codes)
    assert torch.equal(got.nan_to_num(999.0), want.nan_to_num(999.0))
    x = torch.cat([torch.randn(20000, generator=gen(1)) * 30, torch.rand(20000, generator=gen(2)) * 0.02,
                   torch.arange(-4500, 4500) * 0.1, torch.tensor([0.0, -0.0, 448.0, -448.0, 2.0 ** -10, 3 * 2.0 ** -10])]).clamp(-448, 448)
    assert torch.equal(cache.encode(x.double()), x.to(torch.float8_e4m3fn).view(torch.uint8))
    assert cache.encode(torch.tensor([math.inf, -1e9, math.nan]).double()).tolist() == [0x7E, 0xFE, 0x7F]
    kept = codes[(codes & 0x7F) != 0x7F]
    assert torch.equal(cache.encode(cache.decode(kept)), kept)


def test_scales():
    for amax in (448.0, 448.0001, 449.0, 224.0, 1.0, 1e-30, 3.3e38, 1e-38):
        s = cache.scale_for(amax)
        assert amax <= 448 * s and (amax > 224 * s or s == 2.0 ** -110)


def test_attend_is_softmax():
    q, k, v = (torch.randn(s, generator=gen(i)).double() for i, s in enumerate(((3, 4, 8), (9, 2, 8), (9, 2, 8))))
    seen = torch.rand((3, 9), generator=gen(5)) < 0.6
    seen[1] = False
    out, size, _ = attend.attend(q, k, v, seen, 0.3)
    for t in range(3):
        for h in range(4):
            kk, vv = k[seen[t], h // 2], v[seen[t], h // 2]
            want = torch.softmax(0.3 * kk @ q[t, h], 0) @ vv if seen[t].any() else torch.zeros(8).double()
            torch.testing.assert_close(out[t, h], want)
    assert (size >= out.abs() - 1e-12).all()


def test_rotary_keeps_lengths_and_turns_back():
    x = torch.randn((2, 3, 2, 10), generator=gen(1)).double()
    positions = torch.randint(0, 1000, (2, 2, 3), generator=gen(2))
    freqs, axes = torch.tensor([1.0, 0.5, 0.01, 0.3]), torch.tensor([0, 1, 0, 1], dtype=torch.int32)
    for inter in (False, True):
        y, _ = rotary.rotary_axes(x, positions, freqs, axes, inter)
        torch.testing.assert_close(y.norm(dim=-1), x.norm(dim=-1))
        assert torch.equal(y[..., 8:], x[..., 8:])
        back, _ = rotary.rotary_axes(y, positions, freqs, axes, inter, True)
        torch.testing.assert_close(back, x)


def test_drafts_follow_the_target():
    """Over random numbers, the first token has the target's distribution."""
    p, q = torch.tensor([0.5, 0.2, 0.3]), torch.tensor([0.1, 0.6, 0.3])
    counts = torch.zeros(3)
    steps = 60
    for x in range(3):  # the draft's token, weighed by its probability
        for i in range(steps):
            for j in range(steps):
                u, r = (i + 0.5) / steps, (j + 0.5) / steps
                out, _ = drafts.verify(torch.stack([p, p])[None], q[None, None], torch.tensor([[x]]), torch.tensor([[u]]), torch.tensor([r]))
                counts[out[0, 0]] += float(q[x]) / steps ** 2
    assert (counts - p).abs().max() < 0.02
