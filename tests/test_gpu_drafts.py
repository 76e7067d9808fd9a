"""thin_verify_drafts against exact fractions: the tokens and their number are equal."""
import math

import pytest
import torch

from oracle import drafts as oracle
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def inputs(b, k, v, dtype, seed, near=0.5):
    g = gen(seed)
    logits = torch.randn((b, k + 1, v), generator=g) * 2
    target = torch.softmax(logits, 2)
    draft = torch.softmax(logits[:, :k] + near * torch.randn((b, k, v), generator=g), 2)
    tokens = torch.multinomial(draft.reshape(-1, v), 1, generator=g).view(b, k) if k else torch.zeros((b, 0), dtype=torch.int64)
    return target.to(dtype), draft.to(dtype), tokens, torch.rand((b, k), generator=g), torch.rand((b,), generator=g)


def check(gpu, target, draft, tokens, accept, sample, counts=None):
    from thintnpu_amd import capi
    got = capi.verify_drafts(*(None if x is None else x.to(gpu) for x in (target, draft, tokens, accept, sample)),
                             counts=None if counts is None else counts.to(gpu))
    ref = oracle.verify(target, draft, tokens, accept, sample, counts)
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.int32
    assert torch.equal(got[1].cpu(), ref[1])
    assert torch.equal(got[0].cpu(), ref[0])
    return ref


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1, 2, 7, 8, 9, 100, 2047, 2048, 2049, 5001])
def test_vocabularies(gpu, dtype, v):
    for near in (0.3, 2.0):
        t, d, x, u, r = inputs(6, 3, v, TYPES[dtype], v, near)
        check(gpu, t, d, x, u, r)
        check(gpu, t, None, x, u, r)


@pytest.mark.parametrize("k", [0, 1, 2, 31, 32, 33, 63, 64])
def test_draft_counts(gpu, k):
    t, d, x, u, r = inputs(5, k, 300, torch.float32, k, 0.1)
    u = u * 0.5
    ref = check(gpu, t, d, x, u, r)
    assert k < 2 or ref[1].max() > 0
    check(gpu, t, d, x, u * 0, r)  # everything stays
    check(gpu, t, None, x, u * 0, r)
    check(gpu, t, d, x, u, r, torch.tensor([k, 0, k // 2, -5, 2 ** 31 - 1], dtype=torch.int32))


@pytest.mark.parametrize("b,v", [(1, 70001), (40, 9000), (300, 20000)])
def test_tiles(gpu, b, v):
    t, d, x, u, r = inputs(min(b, 6), 2, v, torch.float32, b, 1.0)
    ref = check(gpu, t, d, x, u, r)
    if b > 6:
        from thintnpu_amd import capi
        which = torch.randint(0, 6, (b,), generator=gen(b))
        got = capi.verify_drafts(*(a[which].to(gpu) for a in (t, d, x, u, r)))
        assert torch.equal(got[0].cpu(), ref[0][which]) and torch.equal(got[1].cpu(), ref[1][which])


def test_every_border(gpu):
    """Probabilities that binary fractions hold, random numbers at and next to every border."""
    v = 64
    target = torch.full((1, 2, v), 2.0 ** -6)
    draft = torch.full((1, 1, v), 2.0 ** -6)
    draft[0, 0, ::2], draft[0, 0, 1::2] = 2.0 ** -5, 0.0
    r = torch.cat([torch.arange(65) / 64, (torch.arange(64) / 64 + 2.0 ** -8), (torch.arange(1, 65) / 64 - 2.0 ** -20)])
    n = r.numel()
    for x, u in ((0, 0.5), (0, 0.5 - 2.0 ** -24), (1, 0.0), (1, 0.9), (0, 0.75)):
        check(gpu, target.repeat(n, 1, 1), draft.repeat(n, 1, 1), torch.full((n, 1), x), torch.full((n, 1), u), r)
        check(gpu, target.repeat(n, 1, 1), None, torch.full((n, 1), x), torch.full((n, 1), u / 64), r)


@pytest.mark.parametrize("v", [40, 6000])
def test_special_values(gpu, v):
    t, d, x, u, r = inputs(12, 2, v, torch.float32, v, 1.0)
    nan, inf = math.nan, math.inf
    t[0, :, 5], t[1, :, 7], t[2, :, 3] = nan, inf, -0.5
    d[3, :, 4], d[4, :, 9], d[5, :, 2] = nan, inf, -1.0
    t[6] = d[6].repeat_interleave(torch.tensor([1, 2]), 0) * 0.5  # nothing is left: the target's own row
    u[6] = 0.9
    t[7] = 0.0
    t[8] = nan
    t[9, :, 1:], t[9, :, 0] = 0.0, 1.0
    u[10], r[10] = nan, nan
    r[11] = 1.0
    for i in range(12):
        x[i, 0] = (5, 7, 3, 4, 9, 2, 0, 1, 2, 0, 3, 4)[i]
    check(gpu, t, d, x, u, r)
    check(gpu, t, None, x, u, r)
    check(gpu, t, d, x, u * 0 + 2.0, r * 0 - 1.0)
    check(gpu, t, d, x, u * 0 + 2.0, r * 0 + 7.0)


def test_tokens_outside(gpu):
    for v in (50, 4100):
        t, d, x, u, r = inputs(5, 2, v, torch.float16, v)
        x[:, 0] = torch.tensor([-1, v, 2 ** 40, -2 ** 62, v - 1])
        u *= 0
        check(gpu, t, d, x, u, r)
        check(gpu, t, None, x, u, r)


def test_distribution(gpu):
    """Drafts from q, accepted or replaced, are distributed as p: within five
    standard deviations over 2^17 of them."""
    from thintnpu_amd import capi
    n, v = 1 << 17, 12
    g = gen(3)
    p, q = torch.softmax(torch.randn(v, generator=g), 0), torch.softmax(torch.randn(v, generator=g), 0)
    tokens = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
    out, taken = capi.verify_drafts(p.expand(n, 2, v).to(gpu), q.expand(n, 1, v).to(gpu), tokens.to(gpu),
                                    torch.rand((n, 1), generator=g).to(gpu), torch.rand((n,), generator=g).to(gpu))
    share = torch.bincount(out[:, 0].cpu(), minlength=v).double() / n
    assert ((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()
    assert abs(float(taken.float().mean()) - float(torch.minimum(p, q).sum())) < 5 * 0.5 / n ** 0.5


@pytest.mark.parametrize("v", [61, 5003])
def test_views(gpu, v):
    from thintnpu_amd import capi
    t, d, x, u, r = inputs(7, 3, v, torch.bfloat16, v, 1.0)
    bt, bd = torch.zeros((4, 7, v + 5), dtype=t.dtype), torch.zeros((3, 7, v + 3), dtype=t.dtype)
    bt[..., 3:3 + v], bd[..., 1:1 + v] = t.transpose(0, 1), d.transpose(0, 1)
    args = (bt.to(gpu)[..., 3:3 + v].transpose(0, 1), bd.to(gpu)[..., 1:1 + v].transpose(0, 1),
            x.t().contiguous().to(gpu).t(), torch.stack([u, u + 1], 2).to(gpu)[..., 0], torch.stack([r, r], 1).to(gpu)[:, 1])
    big, few = torch.full((4, 9), 55, device=gpu), torch.full((7, 2), 55, dtype=torch.int32, device=gpu)
    out = big.t()[1:8], few[:, 1]
    got = capi.verify_drafts(*args, out=out)
    ref = oracle.verify(t, d, x, u, r)
    assert got[0] is out[0] and torch.equal(out[0].cpu(), ref[0]) and torch.equal(out[1].cpu(), ref[1])
    assert (big.t()[[0, 8]] == 55).all() and (few[:, 0] == 55).all()
    # one target for every sequence
    a = capi.verify_drafts(args[0][:1].expand(7, 4, v), *args[1:])
    b = capi.verify_drafts(args[0][:1].repeat(7, 1, 1), *args[1:])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_sequences(gpu):
    from thintnpu_amd import capi
    out, taken = capi.verify_drafts(torch.empty((0, 3, 9), device=gpu), torch.empty((0, 2, 9), device=gpu), torch.empty((0, 2), dtype=torch.int64, device=gpu),
                                    torch.empty((0, 2), device=gpu), torch.empty(0, device=gpu))
    assert out.shape == (0, 3) and taken.shape == (0,)


def test_beyond_32_bits(gpu):
    far = 2 ** 32 + 8
    base = torch.empty(far + 30000, dtype=torch.float16, device=gpu)
    t, d, x, u, r = inputs(1, 1, 5000, torch.float16, 2, 1.0)
    view = base.as_strided((1, 2, 5000), (0, far, 1))
    view.copy_(t)
    from thintnpu_amd import capi
    for stay in (0.0, 2.0):
        got = capi.verify_drafts(view, d.to(gpu), x.to(gpu), u.to(gpu) * 0 + stay, r.to(gpu))
        ref = oracle.verify(t, d, x, u * 0 + stay, r)
        assert torch.equal(got[0].cpu(), ref[0])


@pytest.mark.parametrize("v", [500, 50000])
def test_same_bits_streams_and_graphs(gpu, v):
    from thintnpu_amd import capi
    t, d, x, u, r = (a.to(gpu) for a in inputs(8, 4, v, torch.float32, v, 0.3))
    ref = capi.verify_drafts(t, d, x, u, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = capi.verify_drafts(t, d, x, u, r, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    us, outs, graphs = [u.clone(), u.clone()], [], []
    for a in us:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(capi.verify_drafts(t, d, x, a, r))
        graphs.append(graph)
    for step in range(3):
        r.mul_(0.9)
        for i, a in enumerate(us):
            a.copy_(u * (0.3 * step + 0.2 * i))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, out in zip(us, outs):
            assert all(torch.equal(y, z) for y, z in zip(out, capi.verify_drafts(t, d, x, a, r)))


@pytest.mark.parametrize("b", [700, 1100])
def test_several_tiles_a_workgroup(gpu, b):
    """Five tiles of a row, two or four of them to a workgroup."""
    from thintnpu_amd import capi
    t, d, x, u, r = inputs(4, 2, 9000, torch.float16, b, 1.0)
    ref = oracle.verify(t, d, x, u, r)
    many = [a.repeat(b // 4, *[1] * (a.dim() - 1)).to(gpu) for a in (t, d, x, u, r)]
    got = capi.verify_drafts(*many)
    assert torch.equal(got[0].cpu(), ref[0].repeat(b // 4, 1)) and torch.equal(got[1].cpu(), ref[1].repeat(b // 4))
