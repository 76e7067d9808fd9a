"""Pins the oracles of group norm, expert routing and token log probabilities
(CPU only) to values worked out by hand and to PyTorch's own 64-bit operators."""
import math

import torch

from oracle import experts as ex
from oracle import logprobs as lp
from oracle import norm


def test_group_norm_against_torch():
    g = torch.Generator().manual_seed(3)
    x = torch.randn((2, 5, 7, 12), generator=g).double() * 2 + 1
    w, b = torch.randn(12, generator=g).double(), torch.randn(12, generator=g).double()
    ref = torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), 4, w, b, 1e-5).permute(0, 2, 3, 1)
    torch.testing.assert_close(norm.group_norm(x, 4, w, b)["y"], ref, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(norm.group_norm(x, 4, w, b, silu=True)["y"], torch.nn.functional.silu(ref), rtol=1e-12,
                               atol=1e-12)


def test_blocked_view():
    x = torch.arange(2 * 2 * 3 * 1 * 16).reshape(2, 2, 3, 1, 16)
    y = norm.blocked(x, 20)
    assert y.shape == (2, 3, 1, 20)
    assert y[1, 2, 0, 17] == x[1, 1, 2, 0, 1]


def test_best_order():
    nan, inf = math.nan, math.inf
    assert ex.best([1.0, nan, 3.0, 3.0, -inf, nan, -0.0, 0.0], 8) == [1, 5, 2, 3, 0, 6, 7, 4]


def test_route_by_hand():
    logits = torch.tensor([[0.0, math.log(3.0), 0.0, math.log(4.0)]], dtype=torch.float64)
    w, e = ex.route(logits, 2)
    assert e.tolist() == [[3, 1]]
    torch.testing.assert_close(w, torch.tensor([[4 / 7, 3 / 7]], dtype=torch.float64))
    w, e = ex.route(logits, 2, renormalize=False, scale=9.0)
    torch.testing.assert_close(w, torch.tensor([[4.0, 3.0]], dtype=torch.float64))
    # sigmoids 1/2, 3/4, 1/2, 4/5; the bias moves experts 0 and 2 to the front, not their weights
    w, e = ex.route(logits, 2, bias=torch.tensor([1.0, 0.0, 1.0, 0.0]), scores="sigmoid")
    assert e.tolist() == [[0, 2]]
    torch.testing.assert_close(w, torch.tensor([[0.5, 0.5]], dtype=torch.float64))
    # groups {0, 1} and {2, 3}: highest logits 3 against 4
    assert ex.route(logits, 2, groups=2, top_groups=1)[1].tolist() == [[3, 2]]
    # with a bias the two highest count: 1/2 + 3/4 + 0.1 against 1/2 + 4/5
    assert ex.route(logits, 1, bias=torch.tensor([0.1, 0.0, 0.0, 0.0]), scores="sigmoid", groups=2,
                    top_groups=1)[1].tolist() == [[1]]


def test_dispatch_and_combine_by_hand():
    experts = torch.tensor([[2, 0], [0, 0], [5, 2]], dtype=torch.int32)
    tokens, offsets, slots = ex.dispatch(None, experts, 3)
    assert tokens.tolist() == [0, 1, 1, 0, 2]
    assert offsets.tolist() == [0, 3, 3, 5]
    assert slots.tolist() == [[3, 0], [1, 2], [-1, 4]]
    y = torch.tensor([[1.0], [2.0], [4.0], [8.0], [16.0]])
    out, size = ex.combine(y, torch.tensor([[1.0, -2.0], [0.5, 0.25], [9.0, 1.0]]), slots)
    assert out.tolist() == [[6.0], [2.0], [16.0]] and size.tolist() == [[10.0], [2.0], [16.0]]


def test_logprobs_against_torch():
    g = torch.Generator().manual_seed(4)
    x = torch.randn((6, 50), generator=g).double() * 3
    x[2, 10:] = -math.inf
    tokens = torch.tensor([0, 49, 3, 50, -1, 7])
    got = lp.token_logprobs(x, tokens, 3)
    ref = torch.log_softmax(x, 1)
    assert torch.isnan(got[0][3:5]).all()
    for i in (0, 1, 2, 5):
        torch.testing.assert_close(got[0][i], ref[i, tokens[i]])
    torch.testing.assert_close(got[1], torch.distributions.Categorical(logits=x.clamp(min=-1e4)).entropy())
    top = torch.topk(ref, 3)
    assert torch.equal(got[3], top.indices)
    torch.testing.assert_close(got[2], top.values)
