"""rotary_axes, cross_attention, cache_write, cache_attention and verify_drafts as
thin_fused operators of the npu device (the bits of the C ABI's calls, refusals,
capture and replay), on streams of any kind, and all of them in a row as a head
that answers with tokens about a feature map uses them, every step against the
64-bit definition on the inputs that it got."""
import ctypes

import pytest
import torch

from oracle import attend as oa
from oracle import cache as oc
from oracle import drafts as od
from oracle import rotary as orot
from tests.helpers import gen
from tests.test_gpu_rotary import close as rotary_close

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def npu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device visible")
    import thin_backend
    thin_backend.load_flow_libraries()
    return torch.device("npu:0")


def same(a, b):
    assert a.shape == b.shape and a.dtype == b.dtype
    assert torch.equal(a.cpu(), b.cpu())


def parts(b, t, heads, d, page, slots, seed, dtype=torch.bfloat16):
    g = gen(seed)
    pages = b * slots + 1
    codes = [torch.zeros((pages, heads, page, d), dtype=torch.uint8) for _ in range(2)]
    scales = [torch.ones((pages, heads)) for _ in range(2)]
    table = torch.randperm(pages, generator=g)[:b * slots].view(b, slots).int()
    k, v = (torch.randn((b, t, heads, d), generator=g).to(dtype) for _ in range(2))
    return codes + scales, table, k, v


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_npu_equals_the_c_abi(gpu, npu, dtype):
    from thintnpu_amd import capi
    g = gen(1)
    f = torch.ops.thin_fused
    with torch.inference_mode():
        q, k = torch.randn((2, 30, 4, 32), generator=g).to(dtype), torch.randn((2, 30, 2, 32), generator=g).to(dtype)
        positions = torch.randint(0, 500, (2, 2, 30), generator=g, dtype=torch.int32)
        freqs, axes = capi.rotary_tables((9, 5), device="cpu")
        for inter, inverse in ((False, False), (True, True)):
            got = f.rotary_axes(*(x.to(npu) for x in (q, positions, freqs, axes)), k.to(npu), inter, inverse)
            ref = capi.rotary_axes(*(x.to(gpu) for x in (q, positions, freqs, axes)), k=k.to(gpu), interleaved=inter, inverse=inverse)
            assert len(got) == 2
            for a, b in zip(got, ref):
                same(a, b)
        assert len(f.rotary_axes(*(x.to(npu) for x in (q, positions, freqs, axes)))) == 1
        for s in (50, 3000):
            kk, vv = (torch.randn((2, s, 2, 32), generator=g).to(dtype) for _ in range(2))
            lengths, mask = torch.tensor([s, s // 2], dtype=torch.int32), torch.rand((2, s), generator=g) < 0.8
            same(f.cross_attention(q.to(npu), kk.to(npu), vv.to(npu), lengths.to(npu), mask.to(npu), 0.2),
                 capi.cross_attention(q.to(gpu), kk.to(gpu), vv.to(gpu), lengths.to(gpu), mask.to(gpu), 0.2))
            same(f.cross_attention(q[:, :1].to(npu), kk.to(npu), vv.to(npu)), capi.cross_attention(q[:, :1].to(gpu), kk.to(gpu), vv.to(gpu)))
        cache, table, k, v = parts(2, 30, 2, 32, 16, 200, 3, dtype)
        there, here = [x.to(npu) for x in cache], [x.to(gpu) for x in cache]
        lengths, counts = torch.tensor([47, 30], dtype=torch.int32), torch.tensor([30, 11], dtype=torch.int32)
        f.cache_write(k.to(npu), v.to(npu), *there, table.to(npu), lengths.to(npu), counts.to(npu))
        capi.cache_write(k.to(gpu), v.to(gpu), *here, table.to(gpu), lengths.to(gpu), counts.to(gpu))
        for a, b in zip(there, here):
            same(a, b)
        same(f.cache_attention(q.to(npu), *there, table.to(npu), lengths.to(npu), counts.to(npu)),
             capi.cache_attention(q.to(gpu), *here, table.to(gpu), lengths.to(gpu), counts.to(gpu)))
        same(f.cache_attention(q[:, :2].to(npu), *there, table.to(npu), lengths.to(npu), scale=0.3),
             capi.cache_attention(q[:, :2].to(gpu), *here, table.to(gpu), lengths.to(gpu), scale=0.3))
        for vocab in (80, 9000):
            target, draft = (torch.softmax(torch.randn((5, n, vocab), generator=g), 2).to(dtype) for n in (4, 3))
            tokens, accept, sample = torch.randint(0, vocab, (5, 3), generator=g), torch.rand((5, 3), generator=g), torch.rand(5, generator=g)
            number = torch.tensor([3, 2, 1, 0, 3], dtype=torch.int32)
            for dr, n in ((draft, None), (None, number)):
                got = f.verify_drafts(target.to(npu), None if dr is None else dr.to(npu), tokens.to(npu), accept.to(npu), sample.to(npu), None if n is None else n.to(npu))
                ref = capi.verify_drafts(target.to(gpu), None if dr is None else dr.to(gpu), tokens.to(gpu), accept.to(gpu), sample.to(gpu), None if n is None else n.to(gpu))
                for a, b in zip(got, ref):
                    same(a, b)


def test_npu_refusals(npu):
    f = torch.ops.thin_fused
    q = torch.randn(2, 3, 4, 32).half().to(npu)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32).to(npu)  # noqa: E731
    codes, scales = torch.zeros(5, 4, 16, 32, dtype=torch.uint8).to(npu), torch.zeros(5, 4).to(npu)
    other = torch.zeros(5, 4, 16, 32, dtype=torch.uint8).to(npu), torch.zeros(5, 4).to(npu)
    cache = codes, other[0], scales, other[1]
    with torch.inference_mode():
        for call in (lambda: f.rotary_axes(q, i32(1, 2, 3), torch.zeros(17).to(npu), i32(17)),
                     lambda: f.rotary_axes(q.long(), i32(1, 2, 3), torch.zeros(4).to(npu), i32(4)),
                     lambda: f.rotary_axes(q[0], i32(1, 2, 3), torch.zeros(4).to(npu), i32(4)),
                     lambda: f.rotary_axes(q, torch.zeros(1, 2, 3, dtype=torch.int32), torch.zeros(4).to(npu), i32(4)),
                     lambda: f.cross_attention(q.float(), q.float(), q.float()),
                     lambda: f.cross_attention(q, q[:, :, :3], q[:, :, :3]),
                     lambda: f.cross_attention(q, q, q, scale=-1.0),
                     lambda: f.cross_attention(q, q, q, i32(3)),
                     lambda: f.cache_write(q, q, codes, codes, scales, other[1], i32(2, 2), i32(2)),
                     lambda: f.cache_write(q, q.float(), *cache, i32(2, 2), i32(2)),
                     lambda: f.cache_attention(q, *cache, i32(3, 2), i32(2)),
                     lambda: f.cache_attention(q[..., :16], *cache, i32(2, 2), i32(2)),
                     lambda: f.verify_drafts(q[0].float(), None, torch.zeros(3, 3, dtype=torch.int64).to(npu), torch.zeros(3, 3).to(npu), torch.zeros(3).to(npu)),
                     lambda: f.verify_drafts(q[..., 0].long(), None, i32(2, 2), torch.zeros(2, 2).to(npu), torch.zeros(2).to(npu))):
            with pytest.raises(Exception):
                call()
    with pytest.raises(RuntimeError, match="inference-only"):
        f.cross_attention(torch.randn(2, 3, 4, 32, requires_grad=True).half().to(npu), q, q)


def test_npu_captured(npu):
    """A captured step: positions, the cache's writing and reading, the map."""
    from thin_backend.graph import CapturedForward
    f = torch.ops.thin_fused
    cache, table, k, v = parts(2, 3, 2, 32, 16, 60, 5, torch.float16)
    with torch.inference_mode():
        table, k, v = table.to(npu), k.to(npu), v.to(npu)
        lengths = torch.tensor([800, 90], dtype=torch.int32).to(npu)
        positions = torch.arange(6, dtype=torch.int32).view(1, 2, 3).to(npu)
        freqs, axes = torch.rand(16).to(npu), torch.zeros(16, dtype=torch.int32).to(npu)
        states = torch.randn((2, 2500, 2, 32), generator=gen(3)).half().to(npu)

        def forward_on(state):
            def forward(q):
                q, kk = f.rotary_axes(q, positions, freqs, axes, k)
                f.cache_write(kk, v, *state, table, lengths)
                x = f.cache_attention(q, *state, table, lengths)
                return q, x, f.cross_attention(x, states, states)
            return forward

        one, two = [x.to(npu) for x in cache], [x.to(npu) for x in cache]
        first = torch.randn((2, 3, 4, 32), generator=gen(1)).half()
        graph = CapturedForward(forward_on(one), first.to(npu))
        for seed in (2, 3, 4):
            q = torch.randn((2, 3, 4, 32), generator=gen(seed)).half().to(npu)
            for a, b in zip(graph(q), forward_on(two)(q)):
                same(a, b)
            for a, b in zip(one, two):
                same(a, b)


def test_answering_head(gpu):
    """Six decode steps about a feature map, each with drafts: rotary positions
    (time, height, width), keys and values into the 8-bit cache, attention over it
    and over the map's states, a product, softmax, verification; what the target
    refuses is written over in the next step."""
    from thintnpu_amd import capi
    g = gen(20)
    b, t, h, hk, d, page, slots, states, vocab = 3, 4, 8, 2, 32, 16, 4, 130, 120
    dtype = torch.float16
    cache = [torch.zeros((b * slots, hk, page, d), dtype=torch.uint8) for _ in range(2)] + [torch.ones((b * slots, hk)) for _ in range(2)]
    dev = [x.to(gpu) for x in cache]
    table = torch.randperm(b * slots, generator=g).view(b, slots).int()
    freqs, axes = capi.rotary_tables((6, 5, 5))
    height, width = 10, 13
    map_positions = torch.stack([torch.zeros(states), torch.arange(states) // width, torch.arange(states) % width]).int()
    map_k = torch.randn((b, states, hk, d), generator=g).to(dtype)
    map_v = torch.randn((b, states, hk, d), generator=g).to(dtype)
    mask = torch.arange(states)[None] % width < torch.tensor([13, 9, 4])[:, None]
    where = map_positions[:, None].expand(3, b, states).to(gpu)
    map_kr = capi.rotary_axes(map_k.to(gpu), where, freqs, axes)
    ref, size = orot.rotary_axes(map_k, map_positions[:, None].expand(3, b, states), freqs.cpu(), axes.cpu())
    rotary_close(map_kr, ref, size, dtype)
    head = (torch.randn((1, h * d, vocab), generator=g) * 0.1).to(dtype)
    lengths = torch.zeros(b, dtype=torch.int32)
    assert height * width == states
    for step in range(6):
        counts = torch.tensor([t, 1 + step % t, t - step % 2], dtype=torch.int32)
        lengths = lengths + counts
        q, k, v = (torch.randn((b, t, n, d), generator=g).to(dtype) for n in (h, hk, hk))
        at = (lengths - counts)[:, None] + torch.arange(t)
        positions = torch.stack([at, at * 0 + 10, at * 0 + 13]).int()
        qr, kr = capi.rotary_axes(q.to(gpu), positions.to(gpu), freqs, axes, k=k.to(gpu))
        for got, x in ((qr, q), (kr, k)):
            ref, size = orot.rotary_axes(x, positions, freqs.cpu(), axes.cpu())
            rotary_close(got, ref, size, dtype)
        capi.cache_write(kr, v.to(gpu), *dev, table.to(gpu), lengths.to(gpu), counts.to(gpu))
        oc.write(kr.cpu(), v, *cache, table, lengths, counts)
        for x, y in zip(dev, cache):
            assert torch.equal(x.cpu(), y)
        x = capi.cache_attention(qr, *dev, table.to(gpu), lengths.to(gpu), counts.to(gpu))
        ref = oc.attention(qr.cpu(), *cache, table, lengths, counts)
        assert ((x.cpu().double() - ref[0]).abs() <= oa.allowed(q, ref, slots * page, 448 * float(cache[3].max()))).all()
        y = capi.cross_attention(x, map_kr, map_v.to(gpu), mask=mask.to(gpu))
        ref = oa.cross_attention(x.cpu(), map_kr.cpu(), map_v, mask=mask)
        assert ((y.cpu().double() - ref[0]).abs() <= oa.allowed(q, ref, states, 8.0)).all()
        scores = capi.bmm((y + x).reshape(1, b * t, h * d), head.to(gpu))
        target = capi.softmax(scores, 2, half_to_float=True).view(b, t, vocab)
        draft = torch.softmax(scores.float().view(b, t, vocab)[:, :-1] * 0.8, 2)
        tokens = draft.argmax(2)
        accept, sample = torch.rand((b, t - 1), generator=g), torch.rand(b, generator=g)
        kept, taken = capi.verify_drafts(target, draft, tokens, accept.to(gpu), sample.to(gpu), counts=(counts - 1).to(gpu))
        want = od.verify(target.cpu(), draft.cpu(), tokens.cpu(), accept, sample, counts - 1)
        assert torch.equal(kept.cpu(), want[0]) and torch.equal(taken.cpu(), want[1])
        lengths = lengths - (counts - 1 - taken.cpu())


def calls_of(gpu):
    """(name, call(stream) -> tensors) of every operator on fixed inputs."""
    from thintnpu_amd import capi
    g = gen(7)
    q, k = torch.randn((2, 300, 8, 64), generator=g).half().to(gpu), torch.randn((2, 300, 2, 64), generator=g).half().to(gpu)
    positions = torch.randint(0, 500, (2, 2, 300), generator=g, dtype=torch.int32).to(gpu)
    freqs, axes = capi.rotary_tables((16, 16))
    states = torch.randn((2, 4000, 2, 64), generator=g).half().to(gpu)
    cache, table, kk, vv = parts(2, 300, 2, 64, 32, 120, 3, torch.float16)
    cache, table, kk, vv = [x.to(gpu) for x in cache], table.to(gpu), kk.to(gpu), vv.to(gpu)
    lengths = torch.tensor([3800, 1000], dtype=torch.int32, device=gpu)
    target = torch.softmax(torch.randn((9, 4, 30000), generator=g), 2).to(gpu)
    draft, tokens = target[:, :3].flip(2).contiguous(), torch.randint(0, 30000, (9, 3), generator=g).to(gpu)
    accept, sample = torch.rand((9, 3), generator=g).to(gpu), torch.rand(9, generator=g).to(gpu)

    def write(s):
        capi.cache_write(kk, vv, *cache, table, lengths, stream=s)
        return cache

    return [lambda s: capi.rotary_axes(q, positions, freqs, axes, k=k, stream=s),
            lambda s: (capi.rotary_axes(q, positions, freqs, axes, stream=s),),
            lambda s: (capi.cross_attention(q, states, states, stream=s),),
            lambda s: (capi.cross_attention(q[:, :1], states, states, stream=s),),
            write,
            lambda s: (capi.cache_attention(q, *cache, table, lengths, stream=s),),
            lambda s: (capi.cache_attention(q[:, :2], *cache, table, lengths, stream=s),),
            lambda s: capi.verify_drafts(target, draft, tokens, accept, sample, stream=s)]


@pytest.mark.parametrize("raw", [False, True])
def test_calls_on_another_stream(gpu, raw):
    """Outputs and workspaces of a call on another stream are not blocks that the
    caller's stream still writes, and the outputs are not handed out again while
    it reads them."""
    busy = torch.zeros(1 << 28, device=gpu)
    side = torch.cuda.Stream()
    stream = side.cuda_stream if raw else side
    for call in calls_of(gpu):
        ref = [t.clone() for t in call(None)]
        torch.cuda.synchronize()
        for _ in range(20):
            busy.add_(1)  # the caller's stream is some milliseconds behind
        blocks = [torch.empty_like(t) for t in ref] + [torch.empty(1 << n, dtype=torch.uint8, device=gpu) for n in range(9, 24)]
        for x in blocks:
            x.fill_(77)
        del x, blocks
        got = call(stream)
        side.synchronize()
        kept = [t.clone() for t in got]
        del got
        again = call(stream)
        torch.cuda.synchronize()
        for a, b, c in zip(ref, kept, again):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_streams_of_any_kind(gpu):
    """The default stream's null handle, a c_void_p, the current and the default stream."""
    side = torch.cuda.Stream()
    for call in calls_of(gpu):
        ref = [t.clone() for t in call(None)]
        torch.cuda.synchronize()
        for stream in (0, ctypes.c_void_p(None), ctypes.c_void_p(side.cuda_stream), torch.cuda.current_stream(), torch.cuda.default_stream()):
            got = call(stream)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_wrappers_refuse(gpu):
    from thintnpu_amd import capi
    q = torch.zeros((2, 3, 4, 32), dtype=torch.float16, device=gpu)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731
    codes = [torch.zeros((5, 4, 16, 32), dtype=torch.float8_e4m3fn, device=gpu) for _ in range(2)]
    scales = [torch.zeros((5, 4), device=gpu) for _ in range(2)]
    with pytest.raises(ValueError):
        capi.rotary_axes(q, torch.zeros((1, 2, 3), dtype=torch.int32), torch.zeros(4, device=gpu), i32(4))
    with pytest.raises(ValueError):
        capi.cross_attention(q, q.cpu(), q)
    with pytest.raises(ValueError):
        capi.cache_write(q, q, codes[0].cpu(), codes[1], *scales, i32(2, 2), i32(2))
    with pytest.raises(ValueError):
        capi.cache_attention(q, *codes, *scales, i32(2, 2).cpu(), i32(2))
    with pytest.raises(capi.ThinError):
        capi.cache_attention(q.float(), *codes, *scales, i32(2, 2), i32(2))
    with pytest.raises(capi.ThinError):
        capi.cross_attention(q, q, q, out=q)
    long = torch.zeros((2, 9000, 4, 32), dtype=torch.float16, device=gpu)
    with pytest.raises(capi.ThinError):
        capi.cross_attention(q, long, long, workspace=torch.zeros(64, device=gpu))
    with pytest.raises(ValueError):
        capi.cross_attention(q, long, long, workspace=torch.zeros(1 << 20))
    need = capi.lib().thin_cross_attention_workspace(capi._packed(q), capi._packed(long))
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    assert torch.equal(capi.cross_attention(q, long, long, workspace=ws), capi.cross_attention(q, long, long))
