"""Rotary positions and verification of drafts where a pair has no axis or a draft's
probability is none."""
import math

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
