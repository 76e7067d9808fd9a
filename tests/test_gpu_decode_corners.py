"""Rotary positions where a pair has no axis."""
import math

import pytest
import torch

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
