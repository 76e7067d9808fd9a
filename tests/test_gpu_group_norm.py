"""thin_group_norm against the 64-bit definition: layouts, types, group sizes
that divide a vector, fill it or straddle it, strided and unaligned views, one
row to many, and the special values.

Bound of an element, from the kernel's arithmetic (u = 2^-24, half a step of
fp32).  A thread adds at most `serial` terms one after another before the
pairwise joins (about 20 levels): sums are off by (serial + 20) u of their
absolute value, the variance by twice that relatively, its inverse root by half
of it, and the mean by (serial + 20) u times the mean absolute deviation from
the shift.  x - mean, the product and the sum add 3 u of their operands:
  before <= scale * dev * 3 (serial + 20) u + 4 u (scale (|x| + |mean|) + |bias|)
with dev = |x - mean| + sigma.  SiLU has a slope below 1.1 and an own relative
error below (8 + 2 |y|) u (exp2 of a rounded argument, one add, rcp, one
product).  The output's rounding adds half a step of its type."""
import math

import pytest
import torch

from oracle import norm
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
U = 2.0 ** -24
SERIAL = 512  # no test gives a thread more terms of a sum in a row


def bound(x, ref, bias, dtype, silu):
    v = x.double()
    scale = ref["scale"]
    inverse = scale.clamp(min=1e-300)
    dev = (v - ref["mean"]).abs() + (v - ref["mean"]).pow(2).mean().sqrt()
    b = torch.zeros(x.shape[-1]) if bias is None else bias.abs()
    before = inverse * dev * 3 * (SERIAL + 20) * U + 4 * U * (inverse * (v.abs() + ref["mean"].abs()) + b.double())
    out = before
    if silu:
        out = 1.1 * before + ref["y"].abs() * (8 + 2 * ref["before"].abs()) * U
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return out + torch.finfo(dtype).eps / 2 * (ref["y"].abs() + out) + tiny


def inputs(shape, dtype, seed, params):
    g = gen(seed)
    c = shape[-1]
    x = (torch.randn(shape, generator=g) * (torch.rand(c, generator=g) + 0.5) + torch.randn(c, generator=g)).to(dtype)
    w = b = None
    if params:
        kind = dtype if params == "same" else torch.float32
        w, b = torch.randn(c, generator=g).to(kind), (torch.randn(c, generator=g) * 0.3).to(kind)
    return x, w, b


def put(t, dev):
    return None if t is None else t.to(dev)


def check(got, x, groups, w, b, eps, silu):
    ref = norm.group_norm(x, groups, w, b, eps, silu)
    err = (got.cpu().double() - ref["y"]).abs()
    allowed = bound(x, ref, b, x.dtype, silu)
    worst = (err / allowed).max()
    assert worst <= 1, float(worst)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [
    ((2, 9, 7, 64), 32), ((1, 33, 21, 128), 32), ((3, 5, 96), 4), ((2, 1, 1, 48), 48), ((1, 40, 40, 27), 27),
    ((2, 11, 13, 27), 9), ((2, 6, 5, 27), 3), ((1, 17, 30), 1), ((4, 24), 3), ((1, 1, 1), 1), ((1, 300, 72), 24),
    ((2, 10, 10, 1040), 5), ((1, 7, 9, 2047), 1), ((1, 3, 5, 2403), 3), ((2, 50, 8), 2), ((1, 25, 25, 648), 24),
    ((1, 100, 100, 16), 4), ((40, 4, 4, 32), 8)])
def test_channels_last(gpu, shape, groups, dtype):
    from thintnpu_amd import capi
    for i, (params, silu) in enumerate((("same", True), ("fp32", False), (None, True))):
        x, w, b = inputs(shape, TYPES[dtype], 100 + i, params)
        got = capi.group_norm(x.to(gpu), groups, put(w, gpu), put(b, gpu), eps=1e-5, silu=silu)
        check(got, x, groups, w, b, 1e-5, silu)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c,h,w,groups", [
    (1, 128, 20, 20, 32), (2, 64, 9, 7, 32), (1, 48, 5, 5, 2), (2, 27, 6, 7, 3), (1, 27, 40, 33, 27), (1, 20, 3, 3, 1),
    (1, 100, 8, 8, 4), (2, 16, 1, 1, 16), (1, 1, 2, 3, 1), (1, 200, 4, 6, 5), (1, 512, 6, 6, 1), (1, 1001, 3, 4, 7),
    (1, 256, 20, 20, 16), (3, 130, 4, 4, 2)])
def test_blocked(gpu, n, c, h, w, groups, dtype):
    from thintnpu_amd import capi
    x, wt, b = inputs((n, h, w, c), TYPES[dtype], 7, "same")
    c1 = (c + 15) // 16
    full = torch.full((n, h, w, c1 * 16), float("nan"), dtype=x.dtype)  # what the padding holds must not matter
    full[..., :c] = x
    blocked = full.view(n, h, w, c1, 16).permute(0, 3, 1, 2, 4).contiguous()
    for silu in (True, False):
        got = capi.group_norm_nc1hwc0(blocked.to(gpu), groups, wt.to(gpu), b.to(gpu), silu=silu, channels=c).cpu()
        check(norm.blocked(got, c), x, groups, wt, b, 1e-5, silu)
        rest = norm.blocked(got, c1 * 16)[..., c:]
        assert torch.equal(rest, torch.zeros_like(rest))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,groups", [
    ((17, 12, 12, 64), 8),     # one launch, samples dealt to the XCDs with some left over
    ((2, 70, 70, 32), 4), ((9, 50, 60, 64), 16),  # 4, 8 and 16 vectors a thread
    ((2, 110, 100, 128), 32),  # two launches, streaming stores
    ((1, 160, 150, 72), 9), ((1, 90, 120, 328), 41), ((1, 64, 65, 520), 65)])
def test_larger(gpu, shape, groups, dtype):
    from thintnpu_amd import capi
    x, w, b = inputs(shape, TYPES[dtype], 31, "same")
    check(capi.group_norm(x.to(gpu), groups, w.to(gpu), b.to(gpu), silu=True), x, groups, w, b, 1e-5, True)
    n, h, w_, c = shape
    if c % 16 == 0:
        blocked = x.view(n, h, w_, c // 16, 16).permute(0, 3, 1, 2, 4).contiguous()
        got = capi.group_norm_nc1hwc0(blocked.to(gpu), groups, w.to(gpu), b.to(gpu), silu=True)
        check(norm.blocked(got.cpu(), c), x, groups, w, b, 1e-5, True)


def test_whole_blocks_need_no_channel_count(gpu):
    from thintnpu_amd import capi
    x = torch.randn((1, 2, 3, 4, 16), generator=gen(1)).half()
    got = capi.group_norm_nc1hwc0(x.to(gpu), 8).cpu()
    check(norm.blocked(got, 32), norm.blocked(x, 32), 8, None, None, 1e-5, False)


@pytest.mark.parametrize("dtype", TYPES)
def test_views(gpu, dtype):
    """A channel range, a crop, an unaligned start, a stepped batch, an output view."""
    from thintnpu_amd import capi
    base = (torch.randn((4, 12, 14, 90), generator=gen(5)) + 0.5).to(TYPES[dtype])
    dev = base.to(gpu)
    for cut in ((slice(None), slice(None), slice(None), slice(45, 90)), (slice(0, 4, 2), slice(2, 9), slice(3, 11), slice(1, 61)),
                (slice(1, 2), slice(0, 12, 3), slice(None), slice(0, 30))):
        x, v = base[cut], dev[cut]
        room = torch.zeros((*x.shape[:-1], x.shape[-1] + 7), dtype=x.dtype, device=gpu)
        out = room[..., 3:3 + x.shape[-1]]
        capi.group_norm(v, 15, silu=True, out=out)
        check(out, x, 15, None, None, 1e-5, True)
        assert not room[..., :3].any() and not room[..., 3 + x.shape[-1]:].any()
    # the half of a blocked tensor, and a blocked output inside another
    x = (torch.randn((2, 8, 6, 5, 16), generator=gen(6))).to(TYPES[dtype])
    got = capi.group_norm_nc1hwc0(x.to(gpu)[:, 4:], 16, silu=True)
    check(norm.blocked(got.cpu(), 64), norm.blocked(x[:, 4:], 64), 16, None, None, 1e-5, True)


@pytest.mark.parametrize("h", [8, 150])
def test_between_channel_ranges(gpu, h):
    """From one channel range of a tensor to another, and between blocks of one."""
    from thintnpu_amd import capi
    base = torch.randn((2, h, h, 160), generator=gen(h)).half()
    dev = base.to(gpu)
    capi.group_norm(dev[..., :64], 8, silu=True, out=dev[..., 96:])
    check(dev[..., 96:], base[..., :64], 8, None, None, 1e-5, True)
    assert torch.equal(dev[..., :96].cpu(), base[..., :96])
    base = torch.randn((2, 8, h, h, 16), generator=gen(h + 1)).half()
    dev = base.to(gpu)
    capi.group_norm_nc1hwc0(dev[:, 4:], 8, silu=True, out=dev[:, :4])
    check(norm.blocked(dev[:, :4].cpu(), 64), norm.blocked(base[:, 4:], 64), 8, None, None, 1e-5, True)
    assert torch.equal(dev[:, 4:].cpu(), base[:, 4:])


@pytest.mark.parametrize("shape,groups", [((2, 8, 8, 64), 8), ((1, 150, 150, 64), 16)])
def test_in_place(gpu, shape, groups):
    from thintnpu_amd import capi
    x, w, b = inputs(shape, torch.float16, 9, "same")
    dev = x.to(gpu)
    ref = capi.group_norm(dev, groups, w.to(gpu), b.to(gpu), silu=True)
    assert capi.group_norm(dev, groups, w.to(gpu), b.to(gpu), silu=True, out=dev) is dev
    assert torch.equal(dev, ref)


@pytest.mark.parametrize("dtype", TYPES)
def test_mean_far_from_zero(gpu, dtype):
    """Values a thousand deviations from zero: squares formed before the mean is
    taken off would leave nothing of the variance in 32 bits."""
    from thintnpu_amd import capi
    x = (torch.randn((1, 64, 64, 32), generator=gen(2)) * 4 + 1000).to(TYPES[dtype])
    got = capi.group_norm(x.to(gpu), 4)
    check(got, x, 4, None, None, 1e-5, False)


def test_special_values(gpu):
    from thintnpu_amd import capi
    x = torch.randn((2, 4, 4, 32), generator=gen(3)).half()
    x[0, 1, 1, 3] = math.nan
    x[0, 2, 2, 9] = math.inf
    x[1, 0, 0, 20] = -math.inf
    x[1, :, :, 0:8] = 2.5  # no spread: zero, whatever eps
    got = capi.group_norm(x.to(gpu), 4, silu=False).cpu()
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, :, :, 0:8] = bad[0, :, :, 8:16] = bad[1, :, :, 16:24] = True
    assert torch.equal(torch.isnan(got), bad)
    assert not got[1, :, :, 0:8].any()
    assert torch.isnan(capi.group_norm(x[1:, :, :, :8].to(gpu), 1, eps=0.0).cpu()).all()  # 0 / 0


def test_large_eps_and_empty(gpu):
    from thintnpu_amd import capi
    x, w, b = inputs((2, 6, 6, 16), torch.float32, 4, "same")
    got = capi.group_norm(x.to(gpu), 4, w.to(gpu), b.to(gpu), eps=3.0)
    check(got, x, 4, w, b, 3.0, False)
    for shape in ((0, 4, 16), (2, 0, 16)):
        assert capi.group_norm(torch.empty(shape, dtype=torch.float16, device=gpu), 4).shape == shape


def test_offsets_beyond_32_bits(gpu):
    """Samples and rows whose element offsets pass 2^32."""
    from thintnpu_amd import capi
    far = 2 ** 32 + 24
    base = torch.empty(far + 2 ** 20, dtype=torch.float16, device=gpu)
    x, w, b = inputs((2, 6, 5, 24), torch.float16, 12, "same")
    v = base.as_strided((2, 6, 5, 24), (far, 5 * 24, 24, 1))
    v.copy_(x)
    check(capi.group_norm(v, 3, w.to(gpu), b.to(gpu)), x, 3, w, b, 1e-5, False)
    v = base.as_strided((1, 2, 15, 24), (far, far, 24, 1))
    v.copy_(x[0].view(1, 2, 15, 24))
    check(capi.group_norm(v, 3, w.to(gpu), b.to(gpu), out=v), x[:1].view(1, 2, 15, 24), 3, w, b, 1e-5, False)


@pytest.mark.parametrize("shape", [(2, 8, 8, 64), (1, 160, 160, 64)])
def test_same_bits_and_captured(gpu, shape):
    """Two calls, a call on another stream and replays of two graphs captured
    one after the other (each with its own workspace) give the same bits."""
    from thintnpu_amd import capi
    x, w, b = (put(t, gpu) for t in inputs(shape, torch.float16, 21, "same"))
    ref = capi.group_norm(x, 8, w, b, silu=True)
    assert torch.equal(capi.group_norm(x, 8, w, b, silu=True), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = capi.group_norm(x, 8, w, b, silu=True, stream=side)
    side.synchronize()
    assert torch.equal(got, ref)
    graphs, outs, xs = [], [], [x.clone(), x.clone()]
    for v in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(capi.group_norm(v, 8, w, b, silu=True))
        graphs.append(graph)
    for step in range(3):
        for v in xs:
            v.copy_(x * (step + 1))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        expect = capi.group_norm(x * (step + 1), 8, w, b, silu=True)
        assert all(torch.equal(o, expect) for o in outs)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("c,groups,h", [(130, 2, 9), (130, 2, 40), (1001, 7, 5), (268, 4, 11), (1044, 4, 4)])
def test_groups_that_begin_inside_a_vector(gpu, c, groups, h, dtype):
    """A blocked group that begins between two whole vectors: the channels before
    it are another group's, whose NaN, infinities and far values are not its own."""
    from thintnpu_amd import capi
    base, w, b = inputs((2, h, 7, c), TYPES[dtype], c + h, "same")
    per = c // groups
    for value in (math.nan, math.inf, -math.inf, 1000.0, -1e4, 6e4):
        for odd in (0, 1):
            x = base.clone().view(2, h, 7, groups, per)
            x[:, :, :, odd::2] = value if not math.isfinite(value) else (x[:, :, :, odd::2].float() + value).to(x.dtype)
            x = x.view(2, h, 7, c)
            full = torch.zeros((2, h, 7, (c + 15) // 16 * 16), dtype=x.dtype)
            full[..., :c] = x
            blocked = full.view(2, h, 7, -1, 16).permute(0, 3, 1, 2, 4).contiguous()
            got = norm.blocked(capi.group_norm_nc1hwc0(blocked.to(gpu), groups, w.to(gpu), b.to(gpu), channels=c).cpu(), c)
            for i in range(groups):
                own = slice(i * per, (i + 1) * per)
                if math.isfinite(value) or i % 2 != odd:
                    check(got[..., own], x[..., own], 1, w[own], b[own], 1e-5, False)
                else:
                    assert torch.isnan(got[..., own]).all()
