"""thin_rotary_axes against the 64-bit definition.

With u = 2^-24: sine and cosine are off by 8 u (what is left of the angle within
an eighth turn is rounded twice, 2 * 0.79 u, and once with its constant; the
series leave out 2.5e-8 < u / 2, and add 3 roundings of values up to 1), the two
products and their sum by 3 u more, so an element by 11 u of |a| + |b|; then one
rounding to the type."""
import pytest
import torch

from oracle import rotary as oracle
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
U = 2.0 ** -24


def close(got, ref, size, dtype):
    allowed = 11 * U * size + torch.finfo(dtype).eps / 2 * 1.01 * ref.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    far = (got.cpu().double() - ref).abs() / allowed
    assert (far <= 1).all(), float(far.max())


def inputs(b, t, h, hk, d, pairs, axes, dtype, seed, wide=False, far=1 << 20):
    g = gen(seed)
    q, k = torch.randn((b, t, h, d), generator=g).to(dtype), torch.randn((b, t, hk, d), generator=g).to(dtype)
    positions = torch.randint(-far, far, (axes, b, t), generator=g, dtype=torch.int64 if wide else torch.int32)
    freqs = torch.rand(pairs, generator=g) ** 6
    return q, k, positions, freqs, torch.randint(0, axes, (pairs,), generator=g, dtype=torch.int32)


def check(gpu, q, k, positions, freqs, axes, interleaved, inverse=False):
    from thintnpu_amd import capi
    got = capi.rotary_axes(q.to(gpu), positions.to(gpu), freqs.to(gpu), axes.to(gpu), k=k.to(gpu), interleaved=interleaved, inverse=inverse)
    for y, x in zip(got, (q, k)):
        ref, size = oracle.rotary_axes(x, positions, freqs, axes, interleaved, inverse)
        close(y, ref, size, x.dtype)
        assert torch.equal(y.cpu()[..., 2 * freqs.numel():], x[..., 2 * freqs.numel():])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,pairs", [(2, 1), (8, 4), (16, 7), (22, 11), (64, 32), (80, 30), (128, 64), (130, 33), (256, 128), (9, 4), (5, 0)])
def test_widths(gpu, dtype, interleaved, d, pairs):
    check(gpu, *inputs(2, 5, 3, 2, d, pairs, 3, TYPES[dtype], d + pairs), interleaved)


@pytest.mark.parametrize("b,t,h,hk", [(1, 1, 1, 1), (64, 1, 32, 8), (3, 400, 7, 1), (1, 6400, 16, 16), (2, 5, 40, 3)])
def test_counts(gpu, b, t, h, hk):
    check(gpu, *inputs(b, t, h, hk, 64, 32, 2, torch.float16, b + t), False)


def test_many_heads_to_a_thread(gpu):
    """Work enough that a thread turns several heads: against one at a time."""
    from thintnpu_amd import capi
    for h, hk, inter in ((33, 5, False), (40, 8, True)):
        q, k, positions, freqs, axes = (x.to(gpu) for x in inputs(5, 4001, h, hk, 128, 64, 3, torch.bfloat16, h))
        got = capi.rotary_axes(q, positions, freqs, axes, k=k, interleaved=inter)
        for x, y in zip((q, k), got):
            for i in range(x.shape[2]):
                assert torch.equal(capi.rotary_axes(x[:, :, i:i + 1], positions, freqs, axes, interleaved=inter), y[:, :, i:i + 1])


def test_far_positions(gpu):
    """Angles up to 2^28 radians, positions of 64 bits."""
    for far, wide in ((1 << 28, False), ((1 << 31) - 1, True)):
        q, k, positions, freqs, axes = inputs(2, 300, 2, 1, 32, 16, 2, torch.float32, 3, wide, far)
        freqs *= min(1.0, (1 << 28) / far)
        freqs[0] = min(1.0, (1 << 28) / far)
        check(gpu, q, k, positions, freqs, axes, True)


def test_quarter_turns(gpu):
    """Angles at and next to multiples of an eighth turn."""
    n = torch.arange(-40, 41, dtype=torch.int32)
    base = float(torch.tensor(0.7853981633974483).float())
    freqs = torch.tensor([base, base * (1 + 2.0 ** -20), base * 2, base * 4])
    q = torch.tensor([1.0, 0.0]).repeat(4).view(1, 1, 1, 8).expand(1, 81, 2, 8).contiguous()
    q[:, :, 1] = torch.tensor([0.0, 1.0]).repeat(4)
    check(gpu, q, q, n.view(1, 1, 81), freqs, torch.zeros(4, dtype=torch.int32), True)


def test_inverse_and_gradient(gpu):
    """The inverse turn of a gradient is the turn's, also by differences."""
    from thintnpu_amd import capi
    q, k, positions, freqs, axes = inputs(2, 7, 3, 2, 32, 13, 3, torch.float32, 9, far=1000)
    check(gpu, q, k, positions, freqs, axes, False, inverse=True)
    dev = [x.to(gpu) for x in (positions, freqs, axes)]
    grad = torch.randn(q.shape, generator=gen(4))
    back = capi.rotary_axes(grad.to(gpu), *dev, inverse=True).cpu().double()
    step = torch.randn(q.shape, generator=gen(5)).double()
    ahead, behind = (oracle.rotary_axes(q.double() + s * 1e-3 * step, positions, freqs, axes)[0] for s in (1, -1))
    want = ((ahead - behind) / 2e-3 * grad.double()).sum()
    assert abs((back * step).sum() - want) <= 1e-4 * (grad.double() * step).abs().sum()
    turned = capi.rotary_axes(capi.rotary_axes(q.to(gpu), *dev), *dev, inverse=True)
    assert (turned.cpu() - q).abs().max() < 100 * U * q.abs().max()


def test_axes_outside_stay(gpu):
    q, k, positions, freqs, axes = inputs(1, 6, 2, 1, 20, 9, 2, torch.bfloat16, 2)
    axes[1], axes[4], axes[8] = -1, 2, 2 ** 31 - 1
    got = check(gpu, q, k, positions, freqs, axes, False)
    for i in (1, 4, 8):
        assert torch.equal(got[0].cpu()[..., [i, 9 + i]], q[..., [i, 9 + i]])


@pytest.mark.parametrize("interleaved", [False, True])
def test_views_and_in_place(gpu, interleaved):
    from thintnpu_amd import capi
    q, k, positions, freqs, axes = inputs(3, 11, 4, 4, 48, 23, 2, torch.float16, 6)
    packed = torch.cat([q, k, q], 2)
    base = torch.zeros((3, 11, 12, 51), dtype=q.dtype)
    base[..., 1:49] = packed
    dev = base.to(gpu)
    ref = capi.rotary_axes(q.to(gpu), positions.to(gpu), freqs.to(gpu), axes.to(gpu), k=k.to(gpu), interleaved=interleaved)
    views = dev[:, :, :4, 1:49], dev[:, :, 4:8, 1:49]
    wide = torch.zeros((2, 11, 2, 3), dtype=torch.int64, device=gpu)
    wide[:, :, 1] = positions.permute(0, 2, 1)
    tables = torch.zeros((23, 2), device=gpu), torch.zeros((23, 3), dtype=torch.int32, device=gpu)
    tables[0][:, 1], tables[1][:, 2] = freqs.to(gpu), axes.to(gpu)
    got = capi.rotary_axes(views[0], wide[:, :, 1].permute(0, 2, 1), tables[0][:, 1], tables[1][:, 2], k=views[1],
                           interleaved=interleaved, out=views)
    assert got[0] is views[0]
    assert all(torch.equal(a, b) for a, b in zip(views, ref))
    now = dev.cpu()
    assert torch.equal(now[:, :, 8:], base[:, :, 8:]) and not now[..., 0].any() and not now[..., 49:].any()
    # heads before tokens, one position for the whole batch
    heads = q.permute(0, 2, 1, 3).contiguous().to(gpu)
    one = positions[:, :1].to(gpu)
    a = capi.rotary_axes(heads.permute(0, 2, 1, 3), one.expand(2, 3, 11), freqs.to(gpu), axes.to(gpu), interleaved=interleaved)
    b = capi.rotary_axes(q.to(gpu), one.repeat(1, 3, 1), freqs.to(gpu), axes.to(gpu), interleaved=interleaved)
    assert torch.equal(a, b)


def test_special_values(gpu):
    """NaN and infinities stay in their pairs."""
    from thintnpu_amd import capi
    q, _, positions, freqs, axes = inputs(1, 4, 1, 1, 16, 8, 1, torch.float32, 8)
    q[0, 1, 0, 3], q[0, 2, 0, 9] = float("nan"), float("inf")
    y = capi.rotary_axes(q.to(gpu), positions.to(gpu), freqs.to(gpu), axes.to(gpu)).cpu()
    bad = ~torch.isfinite(y)
    assert bad[0, 1, 0, [3, 11]].all() and bad[0, 2, 0, [1, 9]].any() and int(bad.sum()) <= 4
    q[~torch.isfinite(q)] = 0
    ref, size = oracle.rotary_axes(q, positions, freqs, axes)
    bad[0, 1, 0, [3, 11]] = bad[0, 2, 0, [1, 9]] = True
    assert ((y.double() - ref).abs() <= (11 * size + ref.abs()) * U)[~bad].all()


def test_empty(gpu):
    from thintnpu_amd import capi
    freqs, axes = capi.rotary_tables((2, 2))
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        assert capi.rotary_axes(torch.empty(shape, device=gpu), torch.zeros((2, *shape[:2]), dtype=torch.int32, device=gpu), freqs, axes).shape == shape


def test_tables(gpu):
    from thintnpu_amd import capi
    freqs, axes = capi.rotary_tables((2, 3, 1), base=100.0)
    assert axes.tolist() == [0, 0, 1, 1, 1, 2] and freqs.dtype == torch.float32
    torch.testing.assert_close(freqs.cpu().double(), 100.0 ** (-torch.arange(6).double() / 6), rtol=U, atol=0)
    freqs, axes = capi.rotary_tables((2, 4), per_axis=True)
    torch.testing.assert_close(freqs.cpu().double(), 10000.0 ** -torch.tensor([0, 0.5, 0, 0.25, 0.5, 0.75]).double(), rtol=U, atol=0)


def test_beyond_32_bits(gpu):
    from thintnpu_amd import capi
    q, _, positions, freqs, axes = (x.to(gpu) for x in inputs(2, 3, 2, 1, 64, 32, 2, torch.float16, 4))
    far = 2 ** 32 + 64
    base = torch.empty(far + 4096, dtype=torch.float16, device=gpu)
    view = base.as_strided(q.shape, (far, 128, 64, 1))
    view.copy_(q)
    ref = capi.rotary_axes(q, positions, freqs, axes)
    assert torch.equal(capi.rotary_axes(view, positions, freqs, axes), ref)
    capi.rotary_axes(view, positions, freqs, axes, out=view)
    assert torch.equal(view, ref)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,pairs", [(26, 6), (54, 27), (72, 18), (90, 45), (128, 32), (200, 50), (77, 20), (47, 12), (300, 131), (21, 1)])
def test_pieces(gpu, dtype, interleaved, d, pairs):
    """Pairs that pieces of one, two, four and eight divide or leave a rest of, dims
    behind them in any number, NaN and infinities among those; in place too."""
    from thintnpu_amd import capi
    q, k, positions, freqs, axes = inputs(2, 3, 3, 2, d, pairs, 2, TYPES[dtype], d)
    got = check(gpu, q, k, positions, freqs, axes, interleaved)
    x, y = q.to(gpu), k.to(gpu)
    same = capi.rotary_axes(x, positions.to(gpu), freqs.to(gpu), axes.to(gpu), k=y, interleaved=interleaved, out=(x, y))
    assert torch.equal(same[0], got[0]) and torch.equal(same[1], got[1])
    q[..., 2 * pairs::3], q[..., 2 * pairs + 1::3] = torch.inf, torch.nan
    odd = capi.rotary_axes(q.to(gpu), positions.to(gpu), freqs.to(gpu), axes.to(gpu), interleaved=interleaved)
    assert torch.equal(odd[..., :2 * pairs], got[0][..., :2 * pairs])
    assert torch.equal(odd.cpu()[..., 2 * pairs:].nan_to_num(5.0), q[..., 2 * pairs:].nan_to_num(5.0))
