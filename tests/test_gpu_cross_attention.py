"""thin_cross_attention against the 64-bit definition, within oracle.attend.allowed()."""
import math

import pytest
import torch

from oracle import attend as oracle
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def inputs(b, t, s, h, hk, d, dtype, seed, std=1.0):
    g = gen(seed)
    q = (torch.randn((b, t, h, d), generator=g) * std).to(dtype)
    k, v = ((torch.randn((b, s, hk, d), generator=g)).to(dtype) for _ in range(2))
    return q, k, v


def close(got, ref, dtype, q, keys, vmax=8.0):
    got, out = got.cpu().double(), ref[0]
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    allowed = oracle.allowed(q, ref, keys, vmax)
    far = ((got - out).abs() / allowed)[~torch.isnan(out)]
    assert far.numel() == 0 or far.max() <= 1, float(far.max())


def check(gpu, q, k, v, lengths=None, mask=None, scale=None, views=None):
    from thintnpu_amd import capi
    dev = [x if x is None else x.to(gpu) for x in (q, k, v, lengths, mask)] if views is None else views
    got = capi.cross_attention(dev[0], dev[1], dev[2], dev[3], dev[4], scale)
    ref = oracle.cross_attention(q, k, v, lengths, mask, scale)
    close(got, ref, q.dtype, q, k.shape[1], float(v[torch.isfinite(v)].abs().max()) if v.numel() else 1.0)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 128, 136, 160, 192, 200, 256])
def test_head_dims(gpu, dtype, d):
    for t in (1, 20, 37):
        check(gpu, *inputs(2, t, 150, 4, 2, d, TYPES[dtype], d + t))


@pytest.mark.parametrize("s", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
def test_state_counts(gpu, s):
    for t, h, hk in ((1, 8, 1), (3, 6, 1), (70, 2, 2)):  # 8, 18 and 70 rows of a head
        check(gpu, *inputs(2, t, s, h, hk, 64, torch.bfloat16, s + t))


@pytest.mark.parametrize("t,h,hk", [(1, 1, 1), (15, 1, 1), (16, 1, 1), (17, 1, 1), (32, 1, 1), (33, 1, 1), (4, 8, 1), (5, 28, 4), (127, 1, 1), (128, 1, 1),
                                    (129, 2, 1), (300, 3, 3), (1, 40, 1), (43, 6, 2), (1, 129, 1)])
def test_row_counts(gpu, t, h, hk):
    check(gpu, *inputs(2, t, 200, h, hk, 32, torch.float16, t + h))


@pytest.mark.parametrize("b,t,s,h,hk", [(1, 1, 9000, 1, 1), (1, 6, 20011, 20, 4), (3, 100, 5001, 2, 2), (1, 300, 8400, 2, 1), (2, 1, 700, 4, 4)])
def test_keys_split(gpu, b, t, s, h, hk):
    """Few rows of many states: their states are split and joined."""
    from thintnpu_amd import capi
    q, k, v = inputs(b, t, s, h, hk, 64, torch.float16, s)
    need = capi.lib().thin_cross_attention_workspace(capi._packed(q), capi._packed(k))
    assert need > 0
    g = gen(s)
    lengths = torch.randint(0, s + 1, (b,), generator=g, dtype=torch.int32)
    lengths[0] = s
    for n, m in ((None, None), (lengths, None), (None, torch.rand((b, s), generator=g) < 0.5), (lengths, torch.rand((b, s), generator=g) < 0.02)):
        check(gpu, q, k, v, n, m)


@pytest.mark.parametrize("t", [1, 20, 60])
def test_lengths(gpu, t):
    q, k, v = inputs(9, t, 130, 2, 1, 32, torch.bfloat16, t)
    lengths = torch.tensor([0, 1, 64, 65, 129, 130, 131, -3, 2 ** 31 - 1], dtype=torch.int32)
    got = check(gpu, q, k, v, lengths)
    assert not got[0].any() and not got[7].any()


@pytest.mark.parametrize("t", [1, 20, 60])
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_places_may_hold_anything(gpu, t, dtype):
    """NaN, infinities and the largest values where the mask or the length hides them."""
    for s in (70, 600):
        q, k, v = inputs(4, t, s, 4, 2, 64, TYPES[dtype], s)
        g = gen(s + t)
        mask = torch.rand((4, s), generator=g) < 0.4
        mask[1] = False
        mask[2] = True
        mask[3, :s - 3] = False
        lengths = torch.tensor([s - 9, s, s // 2, s], dtype=torch.int32)
        hidden = ~mask | (torch.arange(s) >= lengths[:, None])
        for bad in (math.nan, math.inf, -math.inf, torch.finfo(TYPES[dtype]).max, torch.finfo(TYPES[dtype]).min):
            k2, v2 = k.clone(), v.clone()
            k2[hidden], v2[hidden] = bad, bad
            got = check(gpu, q, k2, v2, lengths, mask)
            assert torch.isfinite(got).all() and not got[1].any()


@pytest.mark.parametrize("t", [1, 40])
def test_special_values_seen(gpu, t):
    """NaN and infinities that are seen come out as the softmax gives them."""
    q, k, v = inputs(3, t, 100, 2, 2, 32, torch.float16, 5)
    v[0, 3, 0, 7] = math.nan
    k[1, 9, 1, 2] = math.nan
    q[2, 0, 1, 4] = math.nan
    from thintnpu_amd import capi
    got = capi.cross_attention(q.to(gpu), k.to(gpu), v.to(gpu)).cpu()
    bad = torch.isnan(got)
    assert bad[0, :, 0, 7].all() and int(bad[0].sum()) == t
    assert bad[1, :, 1].all() and not bad[1, :, 0].any()
    assert bad[2, 0, 1].all() and int(bad[2].sum()) == 32
    v[0, 3, 0, 7] = math.inf
    out = capi.cross_attention(q[:1].to(gpu), k[:1].to(gpu), v[:1].to(gpu)).cpu()
    assert (out[0, :, 0, 7] == math.inf).all() and int(torch.isfinite(out[0]).sum()) == t * 64 - t


@pytest.mark.parametrize("t", [1, 33])
@pytest.mark.parametrize("std,scale", [(1.0, 1e-6), (8.0, 1.0), (30.0, 4.0), (1.0, 1e-38)])
def test_scales(gpu, t, std, scale):
    """From nearly equal weights to a single one, and growing maxima."""
    q, k, v = inputs(2, t, 300, 2, 1, 64, torch.float16, 3, std)
    k = k * (1 + torch.arange(300)[:, None, None] / 100).half()
    check(gpu, q, k, v, scale=scale)


@pytest.mark.parametrize("t", [1, 20, 50])
def test_views(gpu, t):
    from thintnpu_amd import capi
    g = gen(t)
    for dtype in TYPES.values():
        states = torch.randn((2, 90, 2, 5, 41), generator=g).to(dtype)  # k and v in one tensor, odd strides
        q = torch.randn((2, 10, t, 43), generator=g).to(dtype)  # heads before tokens
        lengths = torch.tensor([90, 41], dtype=torch.int32)
        mask = torch.rand((90, 2, 3), generator=g) < 0.7
        ds, dq, dl, dm = states.to(gpu), q.to(gpu), torch.stack([lengths, lengths + 1], 1).to(gpu), mask.to(gpu)
        view = lambda st, qq, ll, mm: (qq[..., 3:43].permute(0, 2, 1, 3), st[:, :, 0, :, 1:], st[:, :, 1, :, :40], ll, mm[:, :, 1].t())  # noqa: E731
        host = view(states, q, lengths, mask)
        dev = view(ds, dq, dl[:, 0], dm)
        got = check(gpu, *host, views=dev)
        big = torch.zeros((2, t, 12, 47), dtype=dtype, device=gpu)
        out = big[:, :, 1:11, 4:44]
        assert capi.cross_attention(*dev, out=out) is out
        assert torch.equal(out, got)
        out.zero_()
        assert not big.any()
        # keys of every head alike, one state for the whole batch
        a = capi.cross_attention(dev[0], dev[1][:1, :, :1].expand(2, 90, 5, 40), dev[2])
        b = capi.cross_attention(dev[0], dev[1][:1, :, :1].repeat(2, 1, 5, 1), dev[2])
        assert torch.equal(a, b)


def test_equal_states(gpu):
    """Shared and separate heads, and a batch in any order, give the same bits."""
    from thintnpu_amd import capi
    q, k, v = (x.to(gpu) for x in inputs(6, 3, 700, 8, 2, 128, torch.bfloat16, 12))
    a = capi.cross_attention(q, k, v)
    order = torch.tensor([3, 0, 5, 1, 4, 2], device=gpu)
    assert torch.equal(capi.cross_attention(q[order], k[order], v[order]), a[order])


def test_no_rows_and_no_states(gpu):
    from thintnpu_amd import capi
    for t in (1, 50):
        q, k, v = (x.to(gpu) for x in inputs(2, t, 0, 2, 2, 32, torch.float16, 1))
        assert not capi.cross_attention(q, k, v, out=torch.ones_like(q)).any()
        assert not capi.cross_attention(q, k, v, mask=torch.ones((2, 0), dtype=torch.bool, device=gpu), out=torch.ones_like(q)).any()
    for shape in ((0, 3, 2, 32), (2, 0, 2, 32), (2, 3, 0, 32)):
        q = torch.empty(shape, dtype=torch.float16, device=gpu)
        k = torch.empty((shape[0], 5, 2, 32), dtype=torch.float16, device=gpu)
        assert capi.cross_attention(q, k, k).shape == shape


def test_beyond_32_bits(gpu):
    far = 2 ** 32 + 32  # from sample to sample; 2^25 - 8 from state to state
    base = torch.empty(far + 2 ** 27, dtype=torch.float16, device=gpu)
    for t in (1, 40):
        q, k, v = inputs(2, t, 3, 1, 1, 32, torch.float16, t)
        vk, vv = base.as_strided(k.shape, (far, 2 ** 25 - 8, 32, 1)), base.as_strided(v.shape, (far, 2 ** 25 - 8, 32, 1), 1024)
        vk.copy_(k)
        vv.copy_(v)
        check(gpu, q, k, v, views=(q.to(gpu), vk, vv, None, None))


@pytest.mark.parametrize("t", [1, 70])
def test_same_bits_streams_and_graphs(gpu, t):
    from thintnpu_amd import capi
    q, k, v = (x.to(gpu) for x in inputs(2, t, 3000, 4, 2, 64, torch.bfloat16, 8))
    ref = capi.cross_attention(q, k, v)
    for _ in range(3):
        assert torch.equal(capi.cross_attention(q, k, v), ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = capi.cross_attention(q, k, v, stream=side)
    side.synchronize()
    assert torch.equal(got, ref)
    qs, outs, graphs = [q.clone(), q.clone()], [], []
    for x in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(capi.cross_attention(x, k, v))
        graphs.append(graph)
    for step in range(3):
        for i, x in enumerate(qs):
            x.copy_(q * (0.5 + step + i))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for x, out in zip(qs, outs):
            assert torch.equal(out, capi.cross_attention(x, k, v))


@pytest.mark.parametrize("b", [70, 150])
def test_many_sequences(gpu, b):
    """Few rows of more sequences than a wavefront has lanes, some without states."""
    q, k, v = inputs(b, 2, 2100, 2, 1, 16, torch.float16, b)
    lengths = torch.randint(0, 2101, (b,), generator=gen(b), dtype=torch.int32)
    lengths[torch.arange(0, b, 7)] = 0
    lengths[63:66] = torch.tensor([0, 2100, 1], dtype=torch.int32)
    got = check(gpu, q, k, v, lengths)
    assert not got[::7].any()
    check(gpu, q, k, v, torch.zeros_like(lengths))


@pytest.mark.parametrize("d", [8, 24, 40, 64, 72])
def test_narrow_rows_split(gpu, d):
    for t in (33, 100):
        q, k, v = inputs(2, t, 2500, 2, 2, d, torch.bfloat16, d + t)
        check(gpu, q, k, v, torch.tensor([2500, 300], dtype=torch.int32), torch.rand((2, 2500), generator=gen(d)) < 0.9)


@pytest.mark.parametrize("t,s", [(1, 90), (40, 90), (1, 700), (40, 700)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_queries_that_are_not_finite(gpu, t, s, bad):
    """They touch their own row alone, and nothing where no state is seen."""
    from thintnpu_amd import capi
    q, k, v = inputs(2, t, s, 2, 2, 32, torch.float16, s)
    q[:, 0, 1, 3] = bad
    k[:, 0, 1, 3] = bad if math.isinf(bad) else 1.0  # a score of +inf, then a masked one of the other sign
    mask = torch.ones((2, s), dtype=torch.bool)
    mask[0] = False
    mask[1, 5:9] = False
    got = capi.cross_attention(*(x.to(gpu) for x in (q, k, v)), mask=mask.to(gpu)).cpu()
    assert not got[0].any()
    assert torch.isnan(got[1, 0, 1]).all() and torch.isfinite(got[1, 1:, 0]).all() and torch.isfinite(got[1, 0, 0]).all()


def test_many_heads(gpu):
    """One row of each of many heads: 2100 workgroups, the last of them in turn."""
    q, k, v = inputs(175, 1, 40, 12, 12, 32, torch.float16, 3)
    check(gpu, q, k, v, torch.randint(0, 41, (175,), generator=gen(4), dtype=torch.int32))


@pytest.mark.parametrize("d", [24, 128])
def test_many_rows_of_many_parts(gpu, d):
    """2400 rows whose states are split over 10 workgroups and more, some of them without any."""
    q, k, v = inputs(2, 300, 6000, 4, 4, d, torch.float16, d)
    check(gpu, q, k, v, torch.tensor([6000, 700], dtype=torch.int32), torch.rand((2, 6000), generator=gen(d)) < 0.8)
