"""Rotary positions and verification of drafts where a pair has no axis, a draft's
probability is none, or a sum's rounding decides."""
import math
from fractions import Fraction
from itertools import accumulate

import pytest
import torch

from oracle import drafts
from tests.helpers import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,pairs", [(16, 8), (48, 23), (80, 32)])
def test_pairs_of_no_axis_keep_their_bits(gpu, dtype, interleaved, d, pairs):
    """Beside infinities, NaN and negative zeros too, in place or not, turned back or not."""
    from thintnpu_amd import capi
    g = gen(d)
    q = torch.randn((2, 5, 3, d), generator=g)
    odd = torch.tensor([math.nan, math.inf, -math.inf, -0.0, 0.0, 1.0])
    q = torch.where(torch.rand(q.shape, generator=g) < 0.5, odd[torch.randint(0, 6, q.shape, generator=g)], q).to(dtype)
    axes = torch.randint(0, 2, (pairs,), generator=g, dtype=torch.int32)
    outside = torch.rand(pairs, generator=g) < 0.5
    axes[outside] = torch.tensor([-1, 2, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)[torch.randint(0, 4, (int(outside.sum()),), generator=g)]
    positions = torch.randint(-99, 99, (2, 2, 5), generator=g, dtype=torch.int32)
    tables = [x.to(gpu) for x in (positions, torch.rand(pairs, generator=g), axes)]
    i = torch.arange(pairs)[outside]
    dims = torch.cat([2 * i, 2 * i + 1] if interleaved else [i, pairs + i])
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    for inverse in (False, True):
        x = q.to(gpu)
        for out in (None, x):
            got = capi.rotary_axes(x, *tables, interleaved=interleaved, inverse=inverse, out=out).cpu()[..., dims]
            want = q[..., dims]
            nan = torch.isnan(want)
            assert torch.equal(torch.isnan(got), nan) and torch.equal(got.view(bits)[~nan], want.view(bits)[~nan])


def verify(gpu, target, draft, tokens, accept, sample):
    from thintnpu_amd import capi
    got = capi.verify_drafts(*(x.to(gpu) for x in (target, draft, tokens, accept, sample)))
    return got[0].cpu(), got[1].cpu()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [40, 6000])
def test_draft_probabilities_that_are_none(gpu, dtype, v):
    """A draft whose own probability is not finite falls, whatever the target's and the random number."""
    rows = [(q, p, u) for q in (-math.inf, math.inf, math.nan) for p in (0.0, 0.25, 1.0) for u in (0.0, 0.5, 0.99)]
    n = len(rows)
    target = torch.softmax(torch.randn((n, 3, v), generator=gen(v)), 2)
    draft = torch.softmax(torch.randn((n, 2, v), generator=gen(v + 1)), 2)
    tokens = torch.randint(0, v, (n, 2), generator=gen(3))
    accept = torch.zeros((n, 2))
    for i, (q, p, u) in enumerate(rows):
        at = i % 2
        target[i, at, tokens[i, at]], draft[i, at, tokens[i, at]], accept[i, at] = p, q, u
    target, draft = target.to(dtype), draft.to(dtype)
    sample = torch.rand((n,), generator=gen(4))
    out, taken = verify(gpu, target, draft, tokens, accept, sample)
    want = drafts.verify(target, draft, tokens, accept, sample)
    assert torch.equal(taken, torch.arange(n, dtype=torch.int32) % 2)
    assert torch.equal(taken, want[1]) and torch.equal(out, want[0])


# Roundings of 64 bits between a sum that is compared with the border and its exact
# value, each 2^-53 of the total at most.  The sum ahead of the tile: tiles' own 17 (an
# element's difference, 7 along a thread's, 6 over the lanes, 3 over the wavefronts), 6
# and one for each 64 tiles, 2 to take the tile apart.  Within it 28: 14 to a lane, 3 over
# the wavefronts, 3 to join them, 8 along a thread's.  The border: a total's 17, 6 and one for
# each 64 tiles, and the product.
def roundings(vocab):
    rounds = -(-vocab // (64 * 2048))
    return (17 + 6 + rounds + 2) + 28 + (17 + 6 + rounds + 1)


@pytest.mark.parametrize("v", [1500, 6000, 50001, 140000])
@pytest.mark.parametrize("least", [-60, -20])
def test_borders_by_rounding(gpu, v, least):
    """Rows of many exponents whose sum up to the middle is a half of the total but for
    2^-50 of it: the token is the exact one, or the random number lies within the
    roundings of the border between the two."""
    half = (v - 2) // 2
    n = 24 if v < 10000 else 6
    g = gen(v)
    first = torch.exp2(torch.rand((n, half), generator=g) * least)
    rest = first.gather(1, torch.rand((n, half), generator=g).argsort(1))
    target = torch.zeros((n, v))
    target[:, 1:1 + half], target[:, 1 + half:1 + 2 * half] = first, rest
    # a token at either end moves the border past a half, or short of it, or there is none
    extra = torch.exp2(torch.floor(torch.log2(first.double().sum(1))) - torch.randint(44, 53, (n,), generator=g)).float()
    for i in range(n):
        if i % 3 < 2:
            target[i, (0, 1 + 2 * half)[i % 3]] = extra[i]
    sample = torch.full((n,), 0.5)
    out, taken = verify(gpu, target[:, None], torch.zeros((n, 0, v)), torch.zeros((n, 0), dtype=torch.int64), torch.zeros((n, 0)), sample)
    assert not taken.any()
    for i in range(n):
        row = [int(x * 2.0 ** 120) for x in target[i].tolist()]  # exact
        prefix = list(accumulate(row))
        whole = prefix[-1]
        edge = Fraction(whole, 2)
        want = next(j for j, y in enumerate(prefix) if y > edge)
        got = int(out[i, 0])
        allowed = roundings(v) * Fraction(1, 2 ** 53) * whole
        # the token's own stretch of the distribution, widened by the roundings
        assert row[got] > 0 and prefix[got] + allowed > edge >= prefix[got] - row[got] - allowed, (i, got, want)
