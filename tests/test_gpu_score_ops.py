"""group_norm, expert_route, expert_dispatch, expert_combine and token_logprobs
as thin_fused operators of the npu device (the bits of the C ABI's calls, their
refusals, capture and replay), and all of them in a row as a sparse expert head
on channels-last features uses them, every step against the 64-bit definition
on the inputs that it got."""
import pytest
import torch

from oracle import experts as ex
from oracle import logprobs as lp
from oracle import norm
from tests.helpers import gen
from tests.test_gpu_experts import U
from tests.test_gpu_group_norm import bound

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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_npu_equals_the_c_abi(gpu, npu, dtype):
    from thintnpu_amd import capi
    g = gen(1)
    f = torch.ops.thin_fused
    with torch.inference_mode():
        for shape in ((2, 6, 5, 32), (1, 120, 120, 64)):
            x, w, b = torch.randn(shape, generator=g).to(dtype), torch.randn(shape[-1], generator=g), torch.randn(shape[-1], generator=g)
            same(f.group_norm(x.to(npu), 4, w.to(npu), b.to(npu), silu=True),
                 capi.group_norm(x.to(gpu), 4, w.to(gpu), b.to(gpu), silu=True))
        x = torch.randn((2, 3, 4, 5, 16), generator=g).to(dtype)
        same(f.group_norm(x.to(npu), 5, channels=40), capi.group_norm_nc1hwc0(x.to(gpu), 5, channels=40))
        logits, bias = torch.randn((20, 64), generator=g).to(dtype), torch.randn(64, generator=g) * 0.1
        got = f.expert_route(logits.to(npu), 6, bias.to(npu), softmax=False, groups=8, top_groups=3, scale=2.0)
        ref = capi.expert_route(logits.to(gpu), 6, bias.to(gpu), "sigmoid", 8, 3, scale=2.0)
        for a, b in zip(got, ref):
            same(a, b)
        for t in (20, 3000):
            x = torch.randn((t, 24), generator=g).to(dtype)
            ids = torch.randint(0, 7, (t, 3), generator=g).int()
            moved = f.expert_dispatch(x.to(npu), ids.to(npu), 7)
            there = capi.expert_dispatch(x.to(gpu), ids.to(gpu), 7)
            for a, b in zip(moved, there):
                same(a, b)
            weights = torch.rand((t, 3), generator=g)
            same(f.expert_combine(moved[0], weights.to(npu), moved[2]), capi.expert_combine(there[0], weights.to(gpu), there[2]))
        for v in (80, 5000):
            x, tokens = torch.randn((30, v), generator=g).to(dtype), torch.randint(0, v, (30,), generator=g)
            for a, b in zip(f.token_logprobs(x.to(npu), tokens.to(npu), 7), capi.token_logprobs(x.to(gpu), tokens.to(gpu), 7)):
                same(a, b)


def test_npu_refusals(npu):
    f = torch.ops.thin_fused
    x = torch.randn(2, 4, 4, 16).half().to(npu)
    with torch.inference_mode():
        for call in (lambda: f.group_norm(x, 3), lambda: f.group_norm(x, 4, channels=16),
                     lambda: f.group_norm(x, 4, torch.ones(16)), lambda: f.group_norm(x.long(), 4),
                     lambda: f.expert_route(x, 2), lambda: f.expert_route(x[0, 0], 17), lambda: f.expert_route(x[0, 0], 0),
                     lambda: f.expert_dispatch(x[0, 0], torch.zeros(4, 1, dtype=torch.int64).to(npu), 3),
                     lambda: f.expert_dispatch(x[0, 0], torch.zeros(4, 1, dtype=torch.int32).to(npu), 0),
                     lambda: f.expert_combine(x[0, 0], torch.zeros(3, 1).to(npu), torch.zeros(4, 1, dtype=torch.int32).to(npu)),
                     lambda: f.token_logprobs(x[0, 0], torch.zeros(4, dtype=torch.int64).to(npu), 17),
                     lambda: f.token_logprobs(x[0, 0], torch.zeros(4, dtype=torch.int32).to(npu))):
            with pytest.raises(Exception):
                call()
    with pytest.raises(RuntimeError, match="inference-only"):
        f.token_logprobs(torch.randn(4, 16, requires_grad=True).to(npu), torch.zeros(4, dtype=torch.int64).to(npu))


def test_npu_captured(npu):
    """A captured forward of the norm, the routing and the log probabilities."""
    from thin_backend.graph import CapturedForward
    f = torch.ops.thin_fused

    def forward(x):
        y = f.group_norm(x, 8, silu=True)
        w, e = f.expert_route(y.view(-1, 64), 4, scale=1.5)
        return (y, w, e, *f.token_logprobs(y.view(-1, 64), tokens, 3))

    with torch.inference_mode():
        tokens = torch.arange(200).remainder(64).to(npu)
        first = torch.randn((2, 10, 10, 64), generator=gen(1)).half()
        graph = CapturedForward(forward, first.to(npu))
        for seed in (2, 3, 4):
            x = torch.randn((2, 10, 10, 64), generator=gen(seed)).half().to(npu)
            for a, b in zip(graph(x), forward(x)):
                same(a, b)
        graph.close() if hasattr(graph, "close") else None


def test_expert_head(gpu):
    """Features -> group norm + SiLU -> router -> experts -> back -> classes ->
    log probabilities; the products run through the library's own bmm."""
    from thintnpu_amd import capi
    g = gen(11)
    n, h, w, c, e, k, classes = 2, 9, 7, 64, 12, 3, 80
    x = torch.randn((n, h, w, c), generator=g).half()
    scale, shift = (torch.rand(c, generator=g) + 0.5).half(), (torch.randn(c, generator=g) * 0.2).half()
    router = (torch.randn((1, c, e), generator=g) * 0.3).half()
    bias = torch.randn(e, generator=g) * 0.05
    expert_w = (torch.randn((e, c, c), generator=g) * 0.15).half()
    head = (torch.randn((1, c, classes), generator=g) * 0.3).half()

    y = capi.group_norm(x.to(gpu), 8, scale.to(gpu), shift.to(gpu), silu=True)
    ref = norm.group_norm(x, 8, scale, shift, 1e-5, True)
    assert ((y.cpu().double() - ref["y"]).abs() <= bound(x, ref, shift, x.dtype, True)).all()
    tokens = y.view(1, -1, c)
    t = tokens.shape[1]

    logits = capi.bmm(tokens, router.to(gpu))[0]
    weights, experts = capi.expert_route(logits, k, bias=bias.to(gpu), scores="sigmoid", groups=4, top_groups=2)
    rw, re = ex.route(logits.cpu(), k, bias, "sigmoid", 4, 2)
    assert torch.equal(experts.cpu(), re)
    torch.testing.assert_close(weights.cpu().double(), rw, rtol=200 * U, atol=0)

    rows, offsets, slots = capi.expert_dispatch(tokens[0], experts, e)
    order, ro, rs = ex.dispatch(None, re, e)
    assert torch.equal(offsets.cpu(), ro) and torch.equal(slots.cpu(), rs)
    assert torch.equal(rows.cpu(), tokens[0].cpu()[order])
    ends = offsets.tolist()
    back = torch.empty_like(rows)
    for i in range(e):
        if ends[i] < ends[i + 1]:
            back[ends[i]:ends[i + 1]] = capi.bmm(rows[None, ends[i]:ends[i + 1]], expert_w[i:i + 1].to(gpu))[0]
    mixed = capi.expert_combine(back, weights, slots)
    sums, size = ex.combine(back.cpu(), weights.cpu(), rs)
    assert ((mixed.cpu().double() - sums).abs() <= size * k * U + 2.0 ** -11 * sums.abs() * 1.001 + 2.0 ** -24).all()
    # the same without moving a row
    dense = torch.zeros((t, c), dtype=torch.float64)
    for i in range(t):
        for j in range(k):
            out = (tokens[0, i].cpu().float() @ expert_w[re[i, j]].float()).half()
            dense[i] += weights[i, j].cpu().double() * out.double()
    # products summed in another order differ by half a step of fp16 here and there
    torch.testing.assert_close(mixed.cpu().double(), dense, rtol=4e-3, atol=4e-3)

    scores = capi.bmm(mixed[None], head.to(gpu))[0]
    given = torch.randint(0, classes, (t,), generator=g)
    got = capi.token_logprobs(scores, given.to(gpu), 5)
    want = lp.token_logprobs(scores.cpu(), given, 5)
    assert torch.equal(got[3].cpu(), want[3])
    for a, b in zip(got[:3], want[:3]):
        torch.testing.assert_close(a.cpu().double(), b, rtol=200 * U, atol=400 * U)


@pytest.mark.parametrize("raw", [False, True])
def test_calls_on_another_stream(gpu, raw):
    """Outputs and workspaces of a call on another stream are not blocks that the
    caller's stream still writes, and the outputs are not handed out again while
    it reads them."""
    from thintnpu_amd import capi
    g = gen(3)
    x = torch.randn((1, 160, 160, 64), generator=g).half().to(gpu)
    logits, rows = torch.randn((3000, 64), generator=g).to(gpu), torch.randn((3000, 40), generator=g).half().to(gpu)
    ids, weights = torch.randint(0, 64, (3000, 4), generator=g).int().to(gpu), torch.rand((3000, 4), generator=g).to(gpu)
    wide, tokens = torch.randn((40, 9000), generator=g).to(gpu), torch.randint(0, 9000, (40,), generator=g).to(gpu)
    moved, _, slots = capi.expert_dispatch(rows, ids, 64)
    calls = [lambda s: (capi.group_norm(x, 8, silu=True, stream=s),),
             lambda s: (capi.group_norm_nc1hwc0(x.view(1, 4, 160, 160, 16), 4, stream=s),),
             lambda s: capi.expert_route(logits, 4, groups=8, top_groups=3, stream=s),
             lambda s: capi.expert_dispatch(rows, ids, 64, stream=s),
             lambda s: (capi.expert_combine(moved, weights, slots, stream=s),),
             lambda s: capi.token_logprobs(wide, tokens, 5, stream=s)]
    busy = torch.zeros(1 << 28, device=gpu)
    side = torch.cuda.Stream()
    stream = side.cuda_stream if raw else side
    for call in calls:
        ref = [t.clone() for t in call(None)]
        torch.cuda.synchronize()
        for _ in range(20):
            busy.add_(1)  # the caller's stream is some milliseconds behind
        blocks = [torch.empty_like(t) for t in ref] + [torch.empty(1 << n, dtype=torch.uint8, device=gpu) for n in range(9, 21)]
        for b in blocks:
            b.fill_(77)
        del b, blocks
        got = call(stream)
        side.synchronize()
        kept = [t.clone() for t in got]
        del got
        again = call(stream)
        torch.cuda.synchronize()
        for a, b, c in zip(ref, kept, again):
            assert torch.equal(a, b) and torch.equal(a, c)
    out = torch.empty_like(x)
    assert capi.group_norm(x, 8, silu=True, out=out, stream=stream) is out
    side.synchronize()
    assert torch.equal(out, calls[0](None)[0])


def test_streams_of_any_kind(gpu):
    """The default stream's null handle, a c_void_p, and a stream that a capture
    takes in, with replays."""
    import ctypes

    from thintnpu_amd import capi
    x = torch.randn((1, 160, 160, 64), generator=gen(5)).half().to(gpu)
    logits = torch.randn((40, 9000), generator=gen(6)).to(gpu)
    tokens = torch.arange(40, device=gpu)
    side = torch.cuda.Stream()
    ref = capi.group_norm(x, 8), *capi.token_logprobs(logits, tokens, 3)
    torch.cuda.synchronize()
    for stream in (0, ctypes.c_void_p(None), ctypes.c_void_p(side.cuda_stream), torch.cuda.current_stream(),
                   torch.cuda.default_stream()):
        got = capi.group_norm(x, 8, stream=stream), *capi.token_logprobs(logits, tokens, 3, stream=stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        out = capi.group_norm(x, 8, stream=side), *capi.token_logprobs(logits, tokens, 3, stream=side)
        torch.cuda.current_stream().wait_stream(side)
    for step in range(3):
        x.copy_(torch.randn(x.shape, generator=gen(step)).half())
        logits.copy_(torch.randn(logits.shape, generator=gen(10 + step)))
        graph.replay()
        torch.cuda.synchronize()
        ref = capi.group_norm(x, 8), *capi.token_logprobs(logits, tokens, 3)
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
