"""Expert routing, dispatch and combine against the 64-bit definitions.

Experts and slots are whole numbers and equal.  A weight is s / sum * scale in
fp32: expf is off by 2 u relatively (u = 2^-24, half a step; one unit in the
last place is 2 u) plus its argument's rounding, |argument| u; 1 / (1 + e), the
quotient, the product and the sum of k terms add (k + 8) u:
  |error| <= |w| (2 * max|argument| + 2 k + 24) u, twice over for s and the sum.
combine adds k products one after another: k u of sum |w y|, and half a step of
its type."""
import math
import random

import pytest
import torch

from oracle import experts as ex
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
U = 2.0 ** -24


def check_route(gpu, logits, k, bias=None, view=None, **options):
    from thintnpu_amd import capi
    dev = logits.to(gpu) if view is None else view
    w, e = capi.expert_route(dev, k, bias=None if bias is None else bias.to(gpu), **options)
    rw, re = ex.route(logits, k, bias, **options)
    assert torch.equal(e.cpu(), re)
    got, finite = w.cpu().double(), torch.isfinite(rw)
    assert torch.equal(torch.isnan(got), torch.isnan(rw))
    span = logits.double()[torch.isfinite(logits)].abs().max().item() * 2 if logits.numel() else 0.0
    allowed = rw.abs() * (2 * span + 2 * k + 24) * 2 * U + 1e-37
    assert ((got - rw).abs() <= allowed)[finite].all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("e", [1, 3, 4, 16, 17, 32, 60, 64, 65, 128, 200, 256, 300, 512, 513, 1000, 1024])
def test_every_width(gpu, e, dtype):
    g = gen(e)
    logits = (torch.randn((13, e), generator=g) * 2).to(TYPES[dtype])
    for k in sorted({1, min(e, 6), min(e, 32)}):
        check_route(gpu, logits, k)
        check_route(gpu, logits, k, bias=torch.randn(e, generator=g) * 0.1, scores="sigmoid", scale=2.5)
        check_route(gpu, logits, k, bias=torch.randn(e, generator=g) * 0.01, scores="softmax", renormalize=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("e,groups,top,k", [(256, 8, 4, 8), (256, 8, 1, 32), (64, 8, 3, 6), (60, 4, 2, 5), (60, 30, 7, 9),
                                            (16, 16, 5, 5), (1024, 64, 9, 17), (640, 64, 1, 10), (12, 2, 1, 6), (256, 4, 4, 8)])
def test_groups(gpu, e, groups, top, k, dtype):
    g = gen(e * groups)
    logits = (torch.randn((9, e), generator=g) * 2).to(TYPES[dtype])
    bias = torch.randn(e, generator=g) * 0.1
    for scores in ("softmax", "sigmoid"):
        check_route(gpu, logits, k, scores=scores, groups=groups, top_groups=top)
        check_route(gpu, logits, k, bias=bias, scores=scores, groups=groups, top_groups=top, renormalize=False, scale=0.5)


@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 300])
def test_token_counts_and_views(gpu, t):
    base = torch.randn((t, 2, 100), generator=gen(t)).half()
    dev = base.to(gpu)
    check_route(gpu, base[:, 1, 3:97], 4, view=dev[:, 1, 3:97])
    bias = torch.randn((94, 2), generator=gen(t + 1))[:, 1]
    check_route(gpu, base[:, 0, 3:97], 4, bias=bias, view=dev[:, 0, 3:97], scores="sigmoid")
    from thintnpu_amd import capi
    room = torch.zeros((t, 12), device=gpu), torch.zeros((4, t), dtype=torch.int32, device=gpu)
    out = room[0][:, 2:10:2], room[1].t()
    capi.expert_route(dev[:, 0], 4, out=out)
    w, e = capi.expert_route(dev[:, 0], 4)
    assert torch.equal(out[0], w) and torch.equal(out[1], e)
    assert not room[0][:, 1::2].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("e", [3, 16, 30, 60, 128, 250, 256, 512, 700])
def test_many_tokens(gpu, e, dtype):
    """More tokens than get a wavefront each: rows of a few kinds, all over."""
    from thintnpu_amd import capi
    g = gen(e)
    kinds = (torch.randn((11, e), generator=g) * 2).to(TYPES[dtype])
    kinds[3] = 0
    kinds[4, e // 2:] = -math.inf
    kinds[5, 0] = math.nan
    which = torch.randint(0, 11, (1500,), generator=g)
    bias = torch.randn(e, generator=g) * 0.1
    k, groups, top = min(e, 9), 5 if e % 5 == 0 else 4 if e % 4 == 0 else 1, 2
    for options in ({}, {"bias": bias, "scores": "sigmoid"}, {"bias": bias, "renormalize": False},
                    {"groups": groups, "top_groups": min(top, groups)},
                    {"bias": bias, "scores": "sigmoid", "groups": groups, "top_groups": min(top, groups), "scale": 2.5}):
        if options.get("groups", 1) > 1 and k > e // groups * 2:
            continue
        rw, re = ex.route(kinds, k, **options)
        moved = {**options, "bias": bias.to(gpu)} if "bias" in options else options
        w, experts = capi.expert_route(kinds[which].to(gpu), k, **moved)
        assert torch.equal(experts.cpu(), re[which])
        few = capi.expert_route(kinds.to(gpu), k, **moved)[0].cpu()
        # the two differ in the order of a sum of positive terms: 16 in a lane at most and 6 joins, so 22 u on
        # either side, and 2 u each for the quotient and the product
        torch.testing.assert_close(w.cpu(), few[which], rtol=48 * U, atol=0, equal_nan=True)
        torch.testing.assert_close(few.double(), rw, rtol=(2 * 20 + 2 * k + 24) * 2 * U, atol=1e-37, equal_nan=True)


def test_ties_go_to_the_lower_index(gpu):
    logits = torch.zeros((5, 96))
    logits[1, 50:] = 1
    logits[2, ::2] = -0.0
    logits[3] = torch.tensor([1.0, 2.0] * 48)
    logits[4] = -math.inf
    logits[4, 40:44] = 3.0
    for dtype in TYPES.values():
        check_route(gpu, logits.to(dtype), 7)
        check_route(gpu, logits.to(dtype), 7, groups=12, top_groups=2)
        check_route(gpu, logits.to(dtype), 7, scores="sigmoid")
        check_route(gpu, logits.to(dtype), 7, bias=torch.full((96,), 0.25), scores="sigmoid")


def test_borders_that_32_bits_cannot_tell(gpu):
    """s + bias within 2^-30 of each other, in either order: 1/2 + b against
    sigmoid(x) with the bias that lifts it just above or below."""
    e = 64
    x = torch.linspace(-2, 2, e, dtype=torch.float32).repeat(8, 1)
    s = 1.0 / (1.0 + torch.exp(-x[0].double()))
    rng = random.Random(5)
    bias = (0.9 - s).float()  # every choice score is about 0.9, off by the bias's rounding alone
    order = list(range(e))
    rng.shuffle(order)
    x, bias = x[:, order].contiguous(), bias[order].contiguous()
    choice = ex.scores64(x, "sigmoid")[0] + bias.double()
    gaps = choice.sort().values.diff()
    assert gaps.max() < 2.0 ** -22  # 32 bits see ties all over
    check_route(gpu, x, 8, bias=bias, scores="sigmoid")
    check_route(gpu, x, 5, bias=bias, scores="sigmoid", groups=8, top_groups=3)
    check_route(gpu, x, 32, bias=bias, scores="sigmoid", groups=4, top_groups=3)


@pytest.mark.parametrize("e,groups,top,k", [(60, 5, 2, 8), (120, 8, 3, 6), (250, 5, 2, 9), (500, 20, 7, 8), (1000, 8, 3, 8)])
def test_close_choices_in_groups_of_any_size(gpu, e, groups, top, k):
    """Every other row's choice scores are equal but for the bias's rounding, so
    that waves choose again in 64 bits while others rank groups whose sizes are
    not powers of two; few tokens and many."""
    from thintnpu_amd import capi
    g = gen(e)
    x = torch.randn((12, e), generator=g)
    s = 1.0 / (1.0 + torch.exp(-x[0].double()))
    bias = (0.9 - s).float()
    x[::2] = x[0]
    x[4] = x[0].flip(0)
    options = {"scores": "sigmoid", "groups": groups, "top_groups": top}
    want = ex.route(x, k, bias, **options)[1]
    for tokens in (333, 2100):
        which = torch.randint(0, 12, (tokens,), generator=g)
        got = capi.expert_route(x[which].to(gpu), k, bias=bias.to(gpu), **options)[1]
        assert torch.equal(got.cpu(), want[which])


def test_route_special_values(gpu):
    nan, inf = math.nan, math.inf
    logits = torch.randn((6, 40), generator=gen(8))
    logits[0, 7] = nan
    logits[1, 3] = inf
    logits[2] = -inf
    logits[3, 5:] = -inf
    logits[4, 2] = -inf
    logits[5, 30] = nan
    logits[5, 11] = nan
    for dtype in TYPES.values():
        for scores in ("softmax", "sigmoid"):
            check_route(gpu, logits.to(dtype), 6, scores=scores)
            check_route(gpu, logits.to(dtype), 6, bias=torch.randn(40, generator=gen(9)) * 0.1, scores=scores)
            check_route(gpu, logits.to(dtype), 6, scores=scores, groups=5, top_groups=2)


def test_route_captured_and_repeated(gpu):
    from thintnpu_amd import capi
    logits = torch.randn((50, 256), generator=gen(1)).to(gpu)
    bias = (torch.randn(256, generator=gen(2)) * 0.1).to(gpu)
    call = lambda: capi.expert_route(logits, 8, bias=bias, scores="sigmoid", groups=8, top_groups=4)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, e = call()
    for step in range(3):
        logits.copy_(torch.randn((50, 256), generator=gen(10 + step)))
        graph.replay()
        torch.cuda.synchronize()
        rw, re = call()
        assert torch.equal(w, rw) and torch.equal(e, re)


# ---------------------------------------------------------------- rows
def check_dispatch(gpu, x, experts, count, xv=None, ev=None):
    from thintnpu_amd import capi
    t, k = experts.shape
    rows = torch.full((t * k, x.shape[1]), 7.0, dtype=x.dtype, device=gpu)
    offsets = torch.full((count + 1,), -5, dtype=torch.int32, device=gpu)
    slots = torch.full((t, k), -5, dtype=torch.int32, device=gpu)
    capi.expert_dispatch(x.to(gpu) if xv is None else xv, experts.to(gpu) if ev is None else ev, count,
                         out=(rows, offsets, slots))
    tokens, ro, rs = ex.dispatch(x, experts, count)
    assert torch.equal(offsets.cpu(), ro) and torch.equal(slots.cpu(), rs)
    got = rows.cpu()
    assert torch.equal(got[:len(tokens)].view(torch.uint8), x[tokens].contiguous().view(torch.uint8))
    assert (got[len(tokens):] == 7.0).all()  # rows of no assignment stay
    return rows, offsets, slots


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,k,e,width", [(1, 1, 1, 1), (1, 8, 16, 64), (3, 2, 5, 7), (48, 8, 256, 520), (33, 3, 1024, 2049),
                                         (100, 1, 7, 16), (5, 32, 40, 3), (512, 8, 64, 40), (513, 8, 64, 33),
                                         (700, 6, 1000, 9), (1500, 4, 3, 300), (4097, 1, 600, 24), (1200, 4, 1024, 8)])
def test_dispatch(gpu, t, k, e, width, dtype):
    g = gen(t * k)
    x = torch.randn((t, width), generator=g).to(TYPES[dtype])
    experts = torch.randint(0, e, (t, k), generator=g).int()  # the same expert twice in a token included
    check_dispatch(gpu, x, experts, e)


@pytest.mark.parametrize("t,k", [(20, 4), (2000, 4)])
def test_dispatch_without_expert(gpu, t, k):
    """Ids outside the experts: slot -1, the rows behind the last stay."""
    g = gen(t)
    x = torch.randn((t, 24), generator=g).half()
    experts = torch.randint(-3, 12, (t, k), generator=g).int()
    experts[1] = -1
    experts[2, 0], experts[2, 1] = 2 ** 31 - 1, -2 ** 31
    check_dispatch(gpu, x, experts, 9)
    check_dispatch(gpu, x, torch.full((t, k), -1, dtype=torch.int32), 9)
    check_dispatch(gpu, x, torch.full((t, k), 8, dtype=torch.int32), 9)


@pytest.mark.parametrize("t", [30, 3000])
def test_dispatch_views_and_bits(gpu, t):
    g = gen(t)
    bits = torch.randint(-32768, 32768, (t, 2, 37), dtype=torch.int16, generator=g).view(torch.float16)
    ids = torch.randint(0, 6, (3, t), generator=g).int()
    dev, idev = bits.to(gpu), ids.to(gpu)
    check_dispatch(gpu, bits[:, 1, 2:35], ids.t(), 6, dev[:, 1, 2:35], idev.t())


def test_dispatch_nothing(gpu):
    for t, width in ((0, 16), (4, 0), (3000, 0)):
        x, experts = torch.empty((t, width)).half(), torch.zeros((t, 2), dtype=torch.int32)
        check_dispatch(gpu, x, experts, 3)


@pytest.mark.parametrize("t", [6, 5000])
def test_dispatch_captured_twice(gpu, t):
    """Two captured graphs with workspaces of their own, replayed in turn."""
    from thintnpu_amd import capi
    x = torch.randn((t, 40), generator=gen(3)).half().to(gpu)
    ids = [torch.randint(0, 9, (t, 3), generator=gen(s)).int().to(gpu) for s in (1, 2)]
    capi.expert_dispatch(x, ids[0], 9)
    graphs, outs = [], []
    for e in ids:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(capi.expert_dispatch(x, e, 9))
        graphs.append(graph)
    for step in range(3):
        for i, e in enumerate(ids):
            e.copy_(torch.randint(-1, 9, (t, 3), generator=gen(20 + 2 * step + i)).int())
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for e, got in zip(ids, outs):
            ref = capi.expert_dispatch(x, e, 9)
            n = int(ref[1][-1])
            assert torch.equal(got[0][:n], ref[0][:n]) and torch.equal(got[1], ref[1]) and torch.equal(got[2], ref[2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,k,width", [(1, 1, 1), (1, 8, 64), (5, 2, 7), (48, 8, 520), (33, 3, 2049), (300, 9, 16), (7, 32, 3),
                                       (64, 5, 8), (3, 4, 8200)])
def test_combine(gpu, t, k, width, dtype):
    from thintnpu_amd import capi
    g = gen(t * k + width)
    rows = t * k + 3
    y = torch.randn((rows, width), generator=g).to(TYPES[dtype])
    w = torch.randn((t, k), generator=g)
    slots = torch.randint(-2, rows + 2, (t, k), generator=g).int()  # outside on both sides, and repeated
    got = capi.expert_combine(y.to(gpu), w.to(gpu), slots.to(gpu)).cpu()
    ref, size = ex.combine(y, w, torch.where(slots < rows, slots, torch.full_like(slots, -1)))
    f = torch.finfo(TYPES[dtype])
    allowed = size * k * U + f.eps / 2 * (ref.abs() + size * k * U) + f.tiny * f.eps
    assert ((got.double() - ref).abs() <= allowed).all()


def test_combine_views_and_special_values(gpu):
    from thintnpu_amd import capi
    g = gen(4)
    y = torch.randn((10, 3, 21), generator=g).half()
    y[4, 1, 5] = math.nan
    y[5, 1, 6] = math.inf
    w, slots = torch.rand((2, 6, 4), generator=g), torch.randint(0, 4, (4, 6), generator=g).int()
    slots[0, 2], slots[1, 3] = 4, 5
    room = torch.zeros((6, 40), dtype=torch.float16, device=gpu)
    out = room[:, 1:20]
    capi.expert_combine(y.to(gpu)[:, 1, 1:20], w.to(gpu)[1], slots.to(gpu).t(), out=out)
    ref, size = ex.combine(y[:, 1, 1:20], w[1], slots.t().contiguous())
    got = out.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    fine = torch.isfinite(ref)
    assert ((got - ref).abs() <= size * 4 * U + 2.0 ** -11 * ref.abs() * 1.01 + 2.0 ** -24)[fine].all()
    assert not room[:, 0].any() and not room[:, 20:].any()
    assert capi.expert_combine(y.to(gpu)[:, 1], w.to(gpu)[1][:0], slots.to(gpu).t()[:0]).shape == (0, 21)
    none = capi.expert_combine(y.to(gpu)[:, 1], w.to(gpu)[1][:, :0], slots.to(gpu).t()[:, :0])
    assert none.shape == (6, 21) and not none.any()


def test_rows_beyond_32_bits(gpu):
    """Row strides that take the offsets of x, rows, y and out past 2^32 elements."""
    from thintnpu_amd import capi
    far = 2 ** 31 + 40
    base = torch.empty(2 * far + 4096, dtype=torch.float16, device=gpu)
    x = torch.randn((3, 24), generator=gen(1)).half()
    v = base.as_strided((3, 24), (far, 1))
    v.copy_(x)
    experts = torch.tensor([[1], [0], [1]], dtype=torch.int32)
    check_dispatch(gpu, x, experts, 2, xv=v)
    room = torch.empty_like(base)
    rows = room.as_strided((3, 24), (far, 1))
    _, _, slots = capi.expert_dispatch(x.to(gpu), experts.to(gpu), 2, out=(
        rows, torch.empty(3, dtype=torch.int32, device=gpu), torch.empty((3, 1), dtype=torch.int32, device=gpu)))
    assert torch.equal(rows.cpu(), x[[1, 0, 2]])
    one = torch.ones((3, 1), device=gpu)
    back = capi.expert_combine(rows, one, slots, out=v)
    assert torch.equal(back.cpu(), x)


# ---------------------------------------------------------------- choices and weights that 32 bits lose
def check_routes(gpu, kinds, k, bias=None, **options):
    """check_route() of the rows, and of so many of them that 16 lanes take a token."""
    from thintnpu_amd import capi
    check_route(gpu, kinds, k, bias=bias, **options)
    which = torch.randint(0, kinds.shape[0], (1100,), generator=gen(k))
    moved = None if bias is None else bias.to(gpu)
    w, e = capi.expert_route(kinds[which].to(gpu), k, bias=moved, **options)
    few = capi.expert_route(kinds.to(gpu), k, bias=moved, **options)
    assert torch.equal(e.cpu(), few[1].cpu()[which])
    # as in test_many_tokens: the order of one sum of positive terms
    torch.testing.assert_close(w.cpu(), few[0].cpu()[which], rtol=48 * U, atol=1e-37, equal_nan=True)


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
@pytest.mark.parametrize("e,groups", [(4, 2), (16, 8), (24, 4), (32, 4), (256, 8), (240, 8), (1024, 4)])
@pytest.mark.parametrize("size", [1.0, 30.0, 137.0, 5000.0])
def test_group_borders_of_large_biases(gpu, e, groups, size, scores):
    """A group's two highest choice scores are near +h and -h, h another number
    for each group: their sums are alike, and off by the rounding of h in 32 bits."""
    per = e // groups
    g = gen(e + int(size))
    x = torch.randn((60, e), generator=g)
    s = ex.scores64(x[:1], scores)[0].view(groups, per)
    h = size * (1 + torch.arange(groups).double() / 7)
    bias = torch.full((groups, per), -4.0 * size, dtype=torch.float64)
    bias[:, 0], bias[:, 1] = h - s[:, 0], -h - s[:, 1]
    bias = bias.float()
    choice = s + bias.double()
    sums = choice.sort(1).values[:, -2:].sum(1)
    gaps = sums.sort().values.diff()
    assert gaps.max() < size * 2.0 ** -21 and gaps.min() > 1e-12  # within 32-bit rounding, and 64 bits tell them apart
    # rows whose first group's sum stands a little above or below another's: by the first logit alone
    for i in range(1, 60):
        x[i] = x[0]
        x[i, 0] += (i - 30) * size * 2.0 ** -22
    for top in sorted({1, groups // 2}):
        for k in (1, top * min(per, 2)):
            check_routes(gpu, x, k, bias=bias.view(-1), scores=scores, groups=groups, top_groups=top)


def test_group_borders_past_the_range(gpu):
    """Sums of two finite choice scores that 32 bits do not hold, and masks of
    -inf and of the lowest value."""
    low = torch.finfo(torch.float32).min
    x = torch.randn((9, 4), generator=gen(1))
    for bias in ([-3.4e38, -3e38, -3.4e38, -1e38], [3.4e38, 1e38, 3.4e38, 3e38], [low, low, low, 0.0], [low, low, low, low],
                 [low, 0.1, low, 0.2], [-math.inf, 0.0, 0.1, 0.2], [-math.inf, -math.inf, 0.1, 0.2],
                 [-math.inf, 1.0, -math.inf, 2.0], [math.inf, -1.0, math.inf, -2.0]):
        for scores in ("softmax", "sigmoid"):
            for k in (1, 2):
                check_route(gpu, x, k, bias=torch.tensor(bias), scores=scores, groups=2, top_groups=1, renormalize=False)


@pytest.mark.parametrize("e", [256, 300, 512, 1024])
def test_softmax_sums_that_32_bits_lose(gpu, e):
    """Terms that are each less than half a step of the sum that they join: the
    total, and with it the first score, is off by their sum."""
    x = torch.full((4, e), -200.0)
    small = list(range(1, 16)) + [16, 32, 64, 128] + ([256] if e > 300 else []) + ([512] if e > 512 else [])
    x[:, 0] = 0.0
    x[:, small] = -16.66
    x[1] = x[1].roll(3)
    lost = len(small) * math.exp(-16.66)
    for share in (0.5, 0.9, 0.97, 1.03):
        bias = torch.full((e,), -5.0)
        bias[0] = -1.0
        bias[3] = -1.0
        bias[200] = -lost * share
        for k in (1, 2):
            check_routes(gpu, x, k, bias=bias)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("e", [3, 16, 60, 256, 700])
def test_sigmoid_weights_of_very_negative_logits(gpu, e, dtype):
    """Sigmoids below the smallest fp32 number, whose quotients are not."""
    g = gen(e)
    x = (-85 - 215 * torch.rand((12, e), generator=g)).to(TYPES[dtype])
    x[1] = (-60 - 60 * torch.rand(e, generator=g)).to(x.dtype)
    x[2] = -100
    x[3] = torch.linspace(-95, -1, e).to(x.dtype)
    x[4, 1:] = -math.inf
    x[5] = (torch.randn(e, generator=g) - 1.5).to(x.dtype)
    x[6, 0] = 3.0
    for k in sorted({1, min(e, 8)}):
        check_routes(gpu, x, k, scores="sigmoid", scale=2.5)
        check_routes(gpu, x, k, bias=torch.rand(e, generator=gen(k)) + 0.5, scores="sigmoid")
