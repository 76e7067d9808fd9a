"""thin_cache_attention where values and scales of some rows' tokens are not others':
against the 64-bit definition, within oracle.attend.allowed() of what each row sees."""
import math

import pytest
import torch

from tests.helpers import gen
from tests.test_gpu_cache import HALVES, Cache, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("d", [96, 128, 208, 256])
def test_nan_values_among_the_first_keys(gpu, dtype, d):
    """Many rows that begin with the sequence: NaN values of the first 32 keys, in
    dims of every wavefront's, reach the rows from their key on and no earlier one."""
    c = Cache(gpu, 3, 3, 16, 2, d, d)
    keys = (0, 5, 16, 31)
    for i in range(3):
        for n, j in enumerate(keys):
            c.host[1][c.table[i, j // 16].long(), n % 2, j % 16, (n + i) * (d // 8) + d // 4::d // 2] = 0x7F
    c.dev = [x.to(gpu) for x in c.host]
    q = queries(3, 40, 4, d, HALVES[dtype], 1)
    got = c.attend(q, torch.tensor([40, 41, 48], dtype=torch.int32))
    nan = torch.isnan(got.cpu())
    assert nan[0, 0, :2].any() and not nan[0, :5, 2:].any() and nan[0, 5:, 2:].any(2).all()
    c.attend(q, torch.tensor([40, 40, 40], dtype=torch.int32), torch.tensor([40, 33, 39], dtype=torch.int32))


def seen_top(c, lengths, counts, t, table=None):
    """[B, T, H]: the largest of the values' scales among the pages that each row sees."""
    table = c.table if table is None else table
    pages, heads, page, _ = c.shape
    top = torch.zeros((table.shape[0], t, heads), dtype=torch.float64)
    for b in range(table.shape[0]):
        n = t if counts is None else int(counts[b])
        for i in range(n):
            keys = max(0, min(int(lengths[b]) - n + i + 1, table.shape[1] * page))
            ids = table[b, :-(-keys // page)].long()
            if keys:
                top[b, i] = c.host[3][ids].double().amax(0)
    return top


def check(c, q, lengths, counts=None, scale=None):
    """attend() with an allowance by what a row sees alone."""
    from oracle import attend
    from oracle import cache as oracle
    from thintnpu_amd import capi
    c.dev = [x.to(c.gpu) for x in c.host]
    got = capi.cache_attention(q.to(c.gpu), *c.dev, c.table.to(c.gpu), lengths.to(c.gpu),
                               None if counts is None else counts.to(c.gpu), scale).cpu().double()
    ref = oracle.attention(q, *c.host, c.table, lengths, counts, scale)
    group = q.shape[2] // c.shape[1]
    top = seen_top(c, lengths, counts, q.shape[1]).repeat_interleave(group, 2)[..., None] * 448
    allowed = attend.allowed(q, ref, c.table.shape[1] * c.shape[2], top)
    assert torch.isfinite(got).all()
    far = (got - ref[0]).abs() / allowed
    assert far.max() <= 1, (float(far.max()), (far > 1).nonzero()[:4].tolist())


@pytest.mark.parametrize("t,h", [(2, 4), (5, 8), (6, 10), (16, 4), (40, 4), (130, 2)])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("up,zeros", [(26, False), (60, True), (120, True)])
def test_scales_of_later_tokens(gpu, t, h, dtype, up, zeros):
    """A page that begins with one of the call's own tokens and whose values have a
    far larger scale: the rows before it lose nothing, those behind it see it."""
    c = Cache(gpu, 3, 26, 16, 2, 64, t + h)
    c.host[0] = torch.randint(0x20, 0x34, c.shape, generator=c.g).to(torch.uint8)  # 2^-3 to 0.7: no row sees one key alone
    c.host[2][:] = 0.25
    c.host[3][:] = 2.0 ** -16
    lengths = torch.tensor([max(t, 17 + (t - 1) // 2), 364, 16 * 16 + t], dtype=torch.int32)
    for b in range(3):
        last = int(lengths[b]) - 1
        for at, scale in (((last, 2.0 ** up),), ((last - t // 2, 2.0 ** (up / 2)), (last, 2.0 ** up * 1.7)), ((last, 2.0 ** up),))[b]:
            page = c.table[b, at // 16].long()
            c.host[3][page] = 2.0 ** -16 * scale
            if zeros:  # (else what the type holds is passed)
                c.host[1][page] = 0
    q = queries(3, t, h, 64, HALVES[dtype], 3)
    check(c, q, lengths)
    check(c, q, lengths, torch.tensor([t, t - 1, max(1, t // 2)], dtype=torch.int32))


@pytest.mark.parametrize("t,n", [(4, 81), (40, 97)])
def test_scales_of_later_tokens_as_written(gpu, t, n):
    """The same through the write: a last token of huge values, which begins a page,
    changes no bit of the rows before it."""
    from thintnpu_amd import capi
    results = []
    for huge in (1.0, 2.0 ** 40):
        c = Cache(gpu, 1, 8, 16, 2, 64, 5, filled=False)
        k, v = (torch.randn((1, n, 2, 64), generator=gen(i)) * 1e-3 for i in (1, 2))
        v[:, -1] *= huge
        c.write(k[:, :n - t], v[:, :n - t], torch.tensor([n - t], dtype=torch.int32))
        c.write(k[:, n - t:], v[:, n - t:], torch.tensor([n], dtype=torch.int32))
        q = queries(1, t, 4, 64, torch.float16, 6)
        got = capi.cache_attention(q.to(gpu), *c.dev, c.table.to(gpu), torch.tensor([n], dtype=torch.int32, device=gpu))
        assert got[0, :-1].abs().amax(2).min() > 0
        results.append(got[0, :-1])
    assert torch.equal(*results)


@pytest.mark.parametrize("t", [1, 6, 40])
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("high,low", [(0, -40), (0, -66), (10, -110), (10, -117), (10, -120), (119, -110)])
def test_weights_of_tiny_scales_count(gpu, t, dtype, high, low):
    """Values' scales 2^40 to 2^229 apart: keys of the small ones have next to no part
    in the mix and their whole part in the total."""
    if dtype == "fp16" and high > 10:
        high, low = 10, -126  # (2^119 is past a half)
    c = Cache(gpu, 2, 24, 16, 2, 64, high - low)
    c.host[0][:] = 0
    c.host[0][..., 0] = 0x58  # 16: what the scores come from
    c.host[1] = torch.randint(0x28, 0x44, c.shape, generator=c.g).to(torch.uint8)
    c.host[2][:] = 1.0
    c.host[3][:] = 2.0 ** low
    for b in range(2):
        first = c.table[b, 3 + 5 * b].long()
        c.host[3][first] = 2.0 ** high
        c.host[0][first, ..., 0] = 0x5C  # 24
    q = torch.zeros((2, t, 4, 64))
    q[..., 0] = torch.rand((2, t, 4), generator=c.g) + 0.5  # scores 4 to 12 apart: shares of 2^-6 to 2^-18 each
    check(c, q.to(HALVES[dtype]), torch.tensor([384, 350], dtype=torch.int32), None, 1.0)


@pytest.mark.parametrize("t", [1, 6, 40])
@pytest.mark.parametrize("mixed", [False, True])
def test_subnormal_scales(gpu, t, mixed):
    """Values whose scales are below the least normal number, all of them or but for a page."""
    c = Cache(gpu, 2, 8, 16, 2, 64, t)
    c.host[0] = torch.randint(0x20, 0x34, c.shape, generator=c.g).to(torch.uint8)
    c.host[1] = torch.randint(0x70, 0x7F, c.shape, generator=c.g).to(torch.uint8)  # 128 to 448
    c.host[2][:] = 0.25
    c.host[3][:] = 1.25 * 2.0 ** -128
    if mixed:
        c.host[3][c.table[:, 2].long()] = 2.0 ** -124
    check(c, queries(2, t, 4, 64, torch.bfloat16, 3), torch.tensor([128, 100], dtype=torch.int32))


@pytest.mark.parametrize("below", [3e-5, 1e-5])
@pytest.mark.parametrize("t", [1, 40])
def test_weights_fit_a_half(gpu, t, below):
    """Scales just below twice a power of two, and a score next to 7 bits above the
    first: its weight, scaled, is still a half."""
    c = Cache(gpu, 1, 8, 16, 1, 64, 1)
    c.host[0][:] = 0xF8  # -256: 28 bits below
    c.host[0][c.table[0, :4].long()] = 0  # scores of 0 in the first 64 keys
    c.host[0][c.table[0, 5].long(), 0, 3] = 0x68  # one of 64
    c.host[1] = torch.randint(0x28, 0x44, c.shape, generator=c.g).to(torch.uint8)
    c.host[2][:] = 1.0
    c.host[3][:] = 2 - 2.0 ** -16
    q = torch.zeros((1, t, 4, 64), dtype=torch.float16)
    q[..., 0] = 1.0
    check(c, q, torch.tensor([128], dtype=torch.int32), None, 7 * (1 - below) * math.log(2) / 64)


@pytest.mark.parametrize("t", [1, 6, 40])
@pytest.mark.parametrize("which", [2, 3])
def test_scales_of_nan_reach_their_rows(gpu, t, which):
    """A page with a scale of NaN, part of which the first rows see: all rows that
    see a token of it are NaN, those before it are not."""
    from thintnpu_amd import capi
    c = Cache(gpu, 1, 8, 16, 2, 64, t)
    c.host[which][c.table[0, 4].long(), 1] = math.nan
    c.dev = [x.to(gpu) for x in c.host]
    for length in (66, 70, 64 + t, 63 + t, 100):
        length = max(length, t)
        q = queries(1, t, 4, 64, torch.float16, length)
        got = capi.cache_attention(q.to(gpu), *c.dev, c.table.to(gpu), torch.tensor([length], dtype=torch.int32, device=gpu))
        sees = torch.arange(length - t, length) >= 64
        nan = torch.isnan(got[0].cpu())
        assert not nan[:, :2].any() and torch.equal(nan[:, 2:].all(2), sees[:, None].expand(t, 2))
        assert torch.equal(nan[:, 2:].any(2), sees[:, None].expand(t, 2))


@pytest.mark.parametrize("d,page", [(32, 16), (64, 48), (128, 16), (144, 32), (256, 32)])
def test_codes_at_odd_addresses_many_rows(gpu, d, page):
    """Pages, heads and tokens at odd byte distances, read by the kernel for many rows."""
    from thintnpu_amd import capi
    from tests.test_gpu_cache import close
    from oracle import cache as oracle
    c = Cache(gpu, 2, 7, page, 2, d, d)
    lengths = torch.tensor([7 * page - 3, 81], dtype=torch.int32)
    for shift in (1, 3, 8):
        views = []
        for x in c.host[:2]:
            p, h, n, _ = c.shape
            base = torch.full((p, n, h, d + 5), 0x7F, dtype=torch.uint8, device=gpu)  # tokens before heads
            view = torch.full((base.numel() + 64,), 0x7F, dtype=torch.uint8, device=gpu)[shift:shift + base.numel()].view_as(base)
            view[..., 3:3 + d] = x.permute(0, 2, 1, 3).to(gpu)
            views.append(view[..., 3:3 + d].permute(0, 2, 1, 3))
        for t, h in ((33, 2), (50, 6)):
            q = queries(2, t, h, d, torch.bfloat16, t)
            got = capi.cache_attention(q.to(gpu), *views, *c.dev[2:], c.table.to(gpu), lengths.to(gpu))
            close(got, oracle.attention(q, *c.host, c.table, lengths), q, 7 * page, c.host)
