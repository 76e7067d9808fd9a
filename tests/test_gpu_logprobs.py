"""thin_token_logprobs against the 64-bit definition.

Ids are equal.  With u = 2^-24: a lane adds 64 terms one after another and the
joins add about 20 levels, each term 2^y carries 2 u of exp2 and ln 2 |y| u of
its rounded exponent, and sum p |y| <= log2(V) + 2 <= 25 bits for every V here;
log2 is off by 2 u of at most 23.  So
  log s is off by (64 + 20 + 2 + 25 + 46) u <= 160 u,
a log probability by that and 4 u of its own size; the entropy's u / s has terms
of 25 u more, on sums whose size is the entropy itself and one bit."""
import math

import pytest
import torch

from oracle import logprobs as oracle
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
U = 2.0 ** -24


def close(got, ref, allowed):
    got = got.cpu().double()
    ref = torch.where(ref < -torch.finfo(torch.float32).max, torch.full_like(ref, -math.inf), ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got == -math.inf, ref == -math.inf)
    fine = torch.isfinite(ref)
    assert ((got - ref).abs() <= allowed)[fine].all(), float(((got - ref).abs() / allowed)[fine].max())


def check(gpu, logits, tokens, top, view=None):
    from thintnpu_amd import capi
    got = capi.token_logprobs(logits.to(gpu) if view is None else view, tokens.to(gpu), top)
    ref = oracle.token_logprobs(logits, tokens, top)
    assert torch.equal(got[3].cpu(), ref[3])
    close(got[0], ref[0], (160 + 4 * ref[0].abs()) * U)
    close(got[1], ref[1], 200 * (2 + ref[1].abs()) * U)
    close(got[2], ref[2], (160 + 4 * ref[2].abs()) * U)
    return got


def rows(r, v, dtype, seed):
    g = gen(seed)
    x = torch.randn((r, v), generator=g) * 2
    x[torch.arange(r), torch.randint(0, v, (r,), generator=g)] = 9.0
    return x.to(dtype), torch.randint(0, v, (r,), generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1, 2, 15, 16, 17, 32, 33, 64, 80, 128, 129, 256, 500, 512, 513, 1000, 1024, 1025, 1100, 4095,
                               4096, 4097, 8192, 9001, 50001])
def test_every_width(gpu, v, dtype):
    x, tokens = rows(5, v, TYPES[dtype], v)
    for top in sorted({0, 1, min(5, v), min(20, v), min(32, v)}):
        check(gpu, x, tokens, top)


@pytest.mark.parametrize("r", [1, 3, 64, 257])
def test_row_counts(gpu, r):
    for v in (80, 1000, 5000):
        x, tokens = rows(r, v, torch.bfloat16, r + v)
        check(gpu, x, tokens, 3)


@pytest.mark.parametrize("v", [4090, 4097, 20000, 140001])
def test_many_rows(gpu, v):
    """Rows enough that a wavefront ends each: a few kinds of them, all over."""
    from thintnpu_amd import capi
    kinds = (torch.randn((7, v), generator=gen(v)) * 2).half()
    kinds[1] = -math.inf
    kinds[1, v // 2: v // 2 + 9] = 1.0
    kinds[2] = 0.5
    kinds[3] = torch.randint(0, 3, (v,), generator=gen(v + 1)).half()
    kinds[4, 7] = kinds[4, v - 2] = math.nan
    kinds[5, 9] = math.inf
    kinds[6] = -math.inf
    which = torch.randint(0, 7, (900,), generator=gen(v + 2))
    tokens = torch.randint(0, v, (7,), generator=gen(v + 3))
    for top in (0, 1, 5, 32):
        few = check(gpu, kinds, tokens, top)
        many = capi.token_logprobs(kinds.to(gpu)[which.to(gpu)], tokens[which].to(gpu), top)
        for a, b in zip(many, few):
            torch.testing.assert_close(a, b[which.to(gpu)], rtol=0, atol=0 if a.dtype == torch.int64 else 64 * U, equal_nan=True)


def test_wide_row(gpu):
    x, tokens = rows(2, 200003, torch.float32, 1)
    check(gpu, x, tokens, 32)
    x, tokens = rows(1, 1 << 20, torch.float16, 2)  # more tiles than lanes
    check(gpu, x, tokens, 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [96, 700, 5003, 12000])
def test_ties(gpu, v, dtype):
    """Equal logits all over, in runs, and a few masked-in tokens among -inf:
    the lower ids come first."""
    x = torch.zeros((8, v))
    x[1] = torch.randint(0, 3, (v,), generator=gen(v)).float()
    x[2] = -math.inf
    x[2, v // 2:v // 2 + 7] = 1.5
    x[3] = -math.inf
    x[3, v - 1] = 0.0
    x[4] = torch.arange(v) // 70
    x[5] = -(torch.arange(v) // 70).float()
    x[6, ::3] = -0.0
    x[7, v // 3:] = 4.0
    tokens = torch.tensor([0, 5, v // 2, 1, v - 1, 0, 3, v - 2])
    for top in (1, 6, 32):
        check(gpu, x.to(TYPES[dtype]), tokens, top)


@pytest.mark.parametrize("v", [40, 900, 3000, 9000])
def test_special_values(gpu, v):
    x = torch.randn((9, v), generator=gen(v))
    nan, inf = math.nan, math.inf
    x[0, 17] = nan
    x[1, 20] = inf
    x[2] = -inf
    x[3, 5] = -inf
    x[4, v - 1] = nan
    x[4, 2] = nan
    x[5, 8] = x[5, v - 3] = inf
    x[6] = nan
    x[7, 3:] = -inf
    x[8] = x[8].clamp(-1, 1) * 1e-30
    tokens = torch.tensor([17, 20, 0, 5, 1, 0, 0, 9, 4])
    for dtype in TYPES.values():
        check(gpu, x.to(dtype), tokens, 12)


@pytest.mark.parametrize("v", [300, 7000])
def test_lowest_values_of_the_type(gpu, v):
    """Masks of the type's lowest value, and a row of nothing else."""
    for dtype in TYPES.values():
        low = torch.finfo(dtype).min
        x = torch.randn((3, v), generator=gen(v)).to(dtype)
        x[0, 10:] = low
        x[1] = low
        x[2, ::2] = torch.finfo(dtype).max / 2
        check(gpu, x, torch.tensor([3, 4, 2]), 14)


def test_tokens_outside(gpu):
    for v in (50, 6000):
        x, _ = rows(5, v, torch.float16, v)
        tokens = torch.tensor([-100, v, 0, -1, 2 ** 40])
        check(gpu, x, tokens, 4)


@pytest.mark.parametrize("v", [61, 5001])
def test_views(gpu, v):
    from thintnpu_amd import capi
    base = (torch.randn((12, 2, v + 9), generator=gen(3)) * 2).to(torch.bfloat16)
    dev = base.to(gpu)
    tokens = torch.arange(12)
    check(gpu, base[:, 1, 5:5 + v], tokens, 7, view=dev[:, 1, 5:5 + v])
    ref = capi.token_logprobs(dev[:, 0, :v], tokens.to(gpu), 4)
    big = torch.zeros((12, 4), device=gpu), torch.zeros((12, 3), device=gpu), torch.zeros((4, 12), device=gpu), torch.zeros((12, 9), dtype=torch.int64, device=gpu)
    out = big[0][:, 1], big[1][:, 2], big[2].t(), big[3][:, 1:5]
    every = torch.arange(24, device=gpu)[::2] // 2
    capi.token_logprobs(dev[:, 0, :v], every, 4, out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, ref))
    assert not big[3][:, 0].any() and not big[3][:, 5:].any() and not big[0][:, 0].any()


def test_no_rows(gpu):
    from thintnpu_amd import capi
    out = capi.token_logprobs(torch.empty((0, 50), device=gpu), torch.empty(0, dtype=torch.int64, device=gpu), 3)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0, 3), (0, 3)]


def test_rows_beyond_32_bits(gpu):
    far = 2 ** 32 + 8
    base = torch.empty(far + 8192, dtype=torch.float16, device=gpu)
    for v in (200, 6000):
        x, tokens = rows(2, v, torch.float16, v)
        view = base.as_strided((2, v), (far, 1))
        view.copy_(x)
        check(gpu, x, tokens, 5, view=view)


@pytest.mark.parametrize("v", [100, 9000])
def test_same_bits_and_captured(gpu, v):
    from thintnpu_amd import capi
    x, tokens = (t.to(gpu) for t in rows(40, v, torch.bfloat16, 5))
    ref = capi.token_logprobs(x, tokens, 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = capi.token_logprobs(x, tokens, 6, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    xs, outs, graphs = [x.clone(), x.clone()], [], []
    for v_ in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(capi.token_logprobs(v_, tokens, 6))
        graphs.append(graph)
    for step in range(3):
        for i, v_ in enumerate(xs):
            v_.copy_(x * (0.5 + step + i))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for v_, out in zip(xs, outs):
            assert all(torch.equal(a, b) for a, b in zip(out, capi.token_logprobs(v_, tokens, 6)))


def _steps_lost(low, high, count, seed):
    """fp32 numbers m whose m log2(e) is off by low to high in its 32-bit rounding."""
    m = torch.rand(1 << 20, generator=gen(seed)).add(1.0).mul(2.0 ** 30).float()
    product = m.double() * float(torch.tensor(1.4426950408889634, dtype=torch.float32))
    off = product - (m * 1.4426950408889634).double()
    return m[(off > low) & (off < high)][:count].tolist()


@pytest.mark.parametrize("v", [40, 900, 3000, 9000])
def test_large_maxima(gpu, v):
    """Maxima far from zero, where m log2(e) loses more than the exponent's range."""
    lost = _steps_lost(-128, -126, 3, 1) + _steps_lost(126, 128, 3, 2) + _steps_lost(60, 64, 2, 3)
    assert len(lost) == 8 and min(lost) > 1e9
    peaks = [1601153152.0, *lost, *(1.3 * 2.0 ** e for e in range(8, 126, 6))]
    peaks += [-p for p in peaks if p < 1e28]
    x = torch.empty((len(peaks), v))
    for i, m in enumerate(peaks):
        x[i] = m - abs(m) * torch.rand(v, generator=gen(i))
        x[i, i % v], x[i, (7 * i + 5) % v], x[i, v - 1 - i % 3] = m, m, m
        x[i, 9] = m * (1 - 2.0 ** -22 if m > 0 else 1 + 2.0 ** -22)
    tokens = torch.tensor([(i % v, 9, 11)[i % 3] for i in range(len(peaks))])
    for dtype in (torch.float32, torch.bfloat16):
        check(gpu, x.to(dtype), tokens, 9)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("v", [700, 1100, 5000, 9001])
def test_low_masks(gpu, v, dtype):
    """Masked logits of any finite size: no run that the row ends in stands above another."""
    edge = 2.3586574e38  # about the largest whose product with log2(e) is finite
    base = torch.zeros((12, v + 8), dtype=TYPES[dtype])
    for i, low in enumerate((-1e28, -9e29, -1e30, -1.01e30, -1e31, -1e35, -2e38, -edge * 0.999, -edge, -edge * 1.001, -3e38, -3.38e38)):
        base[i] = low
    tokens = torch.arange(12)
    dev = base.to(gpu)
    for skew in (0, 3):
        x, view = base[:, skew:skew + v], dev[:, skew:skew + v]
        x[:, 100] = view[:, 100] = 0.5
        x[:, v - 600] = view[:, v - 600] = -0.25
        for top in (3, 32):
            check(gpu, x, tokens, top, view=view)
        x[:, v // 2] = view[:, v // 2] = -math.inf
        check(gpu, x, tokens, 5, view=view)
