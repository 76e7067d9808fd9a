"""Refusals of group norm, expert routing, dispatch, combine and token log
probabilities, before any device work: descriptors that do not fit, sizes
outside the limits, rows that are not adjacent, outputs that overlap operands,
workspaces too small.  Nothing here launches a kernel."""
import ctypes

import pytest
import torch

from thintnpu_amd import capi

P = ctypes.byref
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4


def desc(shape, dtype=capi.F16, data=None, strides=None, _next=[1 << 40]):
    """A descriptor at an address of its own, far from every other."""
    d = capi.ThinDesc()
    d.data, d.dtype, d.rank = data or _next[0], dtype, len(shape)
    _next[0] += 1 << 40
    if strides is None:
        strides, acc = [], 1
        for s in reversed(shape):
            strides.insert(0, acc)
            acc *= s
    for i, (s, st) in enumerate(zip(shape, strides)):
        d.sizes[i], d.strides[i] = s, st
    return d


def status(name, *args):
    args = [P(a) if isinstance(a, capi.ThinDesc) else a for a in args]
    code = getattr(capi.lib(), name)(*args)
    return code, capi.lib().thin_last_error().decode()


def refused(code, name, *args):
    got, message = status(name, *args)
    assert got == code and message, (got, message)


def norm(code, x=None, out=None, blocked=0, channels=64, groups=8, weight=None, bias=None, eps=1e-5, ws=None, nbytes=0):
    x = desc((2, 4, 4, 64)) if x is None else x
    out = desc(tuple(x.sizes[:x.rank]), x.dtype) if out is None else out
    refused(code, "thin_group_norm", x, blocked, channels, groups, weight, bias, eps, 0, out, ws, nbytes, None)


def test_group_norm_refusals():
    norm(INVALID, channels=60)
    norm(UNSUPPORTED, x=desc((2 ** 24, 64)))  # 2^32 threads
    norm(INVALID, groups=7)
    norm(INVALID, groups=0)
    norm(INVALID, groups=-8)
    norm(INVALID, eps=-1.0)
    norm(INVALID, eps=float("nan"))
    norm(INVALID, x=desc((64,)))
    norm(INVALID, x=desc((2, 4, 4, 64), capi.I32))
    norm(INVALID, out=desc((2, 4, 4, 64), capi.F32))
    norm(INVALID, out=desc((2, 4, 2, 64)))
    norm(INVALID, weight=desc((32,)))
    norm(INVALID, weight=desc((64,), capi.BF16))
    norm(INVALID, bias=desc((64, 1)))
    norm(INVALID, blocked=1)  # no [N, C1, H, W, 16]
    norm(INVALID, x=desc((2, 4, 3, 3, 16)), blocked=1, channels=48)
    norm(INVALID, x=desc((2, 4, 3, 3, 16)), blocked=1, channels=65)
    norm(UNSUPPORTED, x=desc((2, 4, 4, 64), strides=(4096, 1024, 128, 2)))
    norm(UNSUPPORTED, x=desc((2, 3, 4, 5, 64), strides=(99999, 9999, 999, 99, 1)))
    norm(UNSUPPORTED, x=desc((1, 2 ** 16, 2 ** 16, 64)))
    x = desc((2, 4, 4, 64))
    norm(INVALID, x=x, out=desc((2, 4, 4, 64), data=x.data + 2))  # overlaps without being x
    row = (4 * 4 * 96, 4 * 96, 96, 1)  # channel ranges of one tensor that share some channels
    x = desc((2, 4, 4, 64), strides=row)
    norm(INVALID, x=x, out=desc((2, 4, 4, 64), data=x.data + 2 * 32, strides=row))
    norm(INVALID, x=x, out=desc((2, 4, 4, 64), data=x.data + 2 * 63, strides=row))
    norm(INVALID, x=x, out=desc((2, 4, 4, 64), data=x.data + 2 * 64, strides=row))  # the next row's
    row = (4 * 4 * 128, 4 * 128, 128, 1)
    x = desc((2, 4, 4, 64), strides=row)
    norm(INVALID, x=x, out=desc((2, 4, 4, 64), data=x.data + 2 * 60, strides=row))
    norm(INVALID, x=x, out=desc((2, 4, 4, 64), data=x.data + 2 * (128 * 5 + 68), strides=row))
    norm(INVALID, out=desc((2, 4, 4, 64), strides=(0, 256, 64, 1)))
    norm(INVALID, x=desc((2, 4, 4, 64), data=1 << 30, strides=(0, 256, 64, 1)),
         out=desc((2, 4, 4, 64), data=1 << 30, strides=(0, 256, 64, 1)))
    norm(INVALID, x=x, weight=desc((64,), data=1 << 30), out=desc((2, 4, 4, 64), data=(1 << 30) + 64))
    big = desc((1, 200, 200, 64))
    need = capi.lib().thin_group_norm_workspace(P(big), P(big), 0, 64, 8)
    assert need > 0
    norm(WORKSPACE, x=big)
    norm(WORKSPACE, x=big, ws=1 << 30, nbytes=need - 1)
    norm(WORKSPACE, x=big, ws=(1 << 30) + 2, nbytes=need)
    assert capi.lib().thin_group_norm_workspace(P(big), P(big), 0, 64, 7) == 0
    assert capi.lib().thin_group_norm_workspace(None, P(big), 0, 64, 8) == 0


def route(code, logits=None, bias=None, groups=1, top=1, weights=None, experts=None, k=2):
    logits = desc((5, 16), capi.F32) if logits is None else logits
    weights = desc((5, k), capi.F32) if weights is None else weights
    experts = desc((5, k), capi.I32) if experts is None else experts
    refused(code, "thin_expert_route", logits, bias, 1, groups, top, 1, 1.0, weights, experts, None)


def test_route_refusals():
    route(INVALID, logits=desc((5, 16), capi.I64))
    route(INVALID, logits=desc((5, 4, 4), capi.F32))
    route(UNSUPPORTED, logits=desc((5, 1025), capi.F32))
    route(UNSUPPORTED, logits=desc((5, 0), capi.F32))
    route(UNSUPPORTED, logits=desc((5, 16), capi.F32, strides=(1, 5)))
    route(INVALID, k=17)
    route(INVALID, k=0)
    route(INVALID, logits=desc((5, 64), capi.F32), k=33)
    route(INVALID, groups=3)
    route(INVALID, groups=0)
    route(INVALID, groups=4, top=5)
    route(INVALID, groups=4, top=0)
    route(INVALID, groups=8, top=1, k=3)  # more than the kept groups hold
    route(INVALID, logits=desc((5, 130), capi.F32), groups=65)
    route(INVALID, bias=desc((15,), capi.F32))
    route(INVALID, bias=desc((16,)))
    route(INVALID, weights=desc((4, 2), capi.F32))
    route(INVALID, weights=desc((5, 2)))
    route(INVALID, weights=desc((5, 2), capi.F32, strides=(0, 1)))
    t = 2 ** 30  # 2^32 threads
    route(UNSUPPORTED, logits=desc((t, 16), strides=(0, 1)), weights=desc((t, 2), capi.F32),
          experts=desc((t, 2), capi.I32))
    route(INVALID, experts=desc((5, 2), capi.I64))
    route(INVALID, experts=desc((5, 3), capi.I32))
    logits = desc((5, 16), capi.F32)
    route(INVALID, logits=logits, weights=desc((5, 2), capi.F32, data=logits.data + 16))
    route(INVALID, weights=desc((5, 2), capi.F32, data=1 << 30), experts=desc((5, 2), capi.I32, data=(1 << 30) + 4))


def dispatch(code, x=None, experts=None, count=4, rows=None, offsets=None, slots=None, ws=None, nbytes=0, t=6, k=2):
    x = desc((t, 8)) if x is None else x
    experts = desc((t, k), capi.I32) if experts is None else experts
    rows = desc((t * k, 8)) if rows is None else rows
    offsets = desc((count + 1,), capi.I32) if offsets is None else offsets
    slots = desc((t, k), capi.I32) if slots is None else slots
    refused(code, "thin_expert_dispatch", x, experts, count, rows, offsets, slots, ws, nbytes, None)


def test_dispatch_refusals():
    dispatch(INVALID, x=desc((6, 8), capi.I32))
    dispatch(INVALID, x=desc((6, 8), capi.F32))  # rows of another type
    dispatch(INVALID, x=desc((5, 8)))
    dispatch(INVALID, experts=desc((6, 2), capi.I64))
    dispatch(INVALID, experts=desc((12,), capi.I32))
    dispatch(INVALID, rows=desc((11, 8)))
    dispatch(INVALID, rows=desc((12, 9)))
    dispatch(INVALID, offsets=desc((4,), capi.I32))
    dispatch(INVALID, offsets=desc((5,), capi.I64))
    dispatch(INVALID, slots=desc((6, 3), capi.I32))
    dispatch(INVALID, slots=desc((6, 2), capi.I32, strides=(0, 1)))
    dispatch(INVALID, rows=desc((12, 8), strides=(0, 1)))
    dispatch(UNSUPPORTED, count=1025)
    dispatch(UNSUPPORTED, count=0, offsets=desc((1,), capi.I32))
    dispatch(UNSUPPORTED, k=33)
    dispatch(UNSUPPORTED, k=0, rows=desc((0, 8)))
    dispatch(UNSUPPORTED, x=desc((6, 8), strides=(1, 6)))
    dispatch(UNSUPPORTED, rows=desc((12, 8), strides=(16, 2)))
    dispatch(UNSUPPORTED, t=2 ** 30, k=2)
    x = desc((6, 8))
    dispatch(INVALID, x=x, rows=desc((12, 8), data=x.data + 80))
    experts = desc((6, 2), capi.I32)
    dispatch(INVALID, experts=experts, slots=desc((6, 2), capi.I32, data=experts.data))
    need = capi.lib().thin_expert_dispatch_workspace(5000, 2, 4)
    assert need > 0 and capi.lib().thin_expert_dispatch_workspace(6, 2, 4) == 0
    dispatch(WORKSPACE, t=5000)
    dispatch(WORKSPACE, t=5000, ws=(1 << 30) + 2, nbytes=need)
    t = 2 ** 24  # 2^32 threads
    dispatch(UNSUPPORTED, t=t, k=1, x=desc((t, 2048)), rows=desc((t, 2048)), ws=1 << 30, nbytes=1 << 30)
    dispatch(UNSUPPORTED, x=desc((6, 1 << 28)), rows=desc((12, 1 << 28)))
    dispatch(WORKSPACE, t=5000, ws=1 << 30, nbytes=need - 1)


def combine(code, y=None, weights=None, slots=None, out=None):
    y = desc((9, 8)) if y is None else y
    weights = desc((4, 2), capi.F32) if weights is None else weights
    slots = desc((4, 2), capi.I32) if slots is None else slots
    out = desc((4, 8)) if out is None else out
    refused(code, "thin_expert_combine", y, weights, slots, out, None)


def test_combine_refusals():
    combine(INVALID, y=desc((9, 8), capi.U8))
    combine(INVALID, y=desc((9, 8), capi.F32))
    combine(INVALID, y=desc((9, 7)))
    combine(INVALID, weights=desc((4, 2)))
    combine(INVALID, weights=desc((4, 3), capi.F32))
    combine(INVALID, slots=desc((4, 2), capi.I64))
    combine(INVALID, out=desc((5, 8)))
    combine(INVALID, out=desc((4, 8), strides=(0, 1)))
    combine(UNSUPPORTED, y=desc((9, 8), strides=(1, 9)))
    combine(UNSUPPORTED, out=desc((4, 8), strides=(16, 2)))
    t = 2 ** 24  # 2^32 threads
    combine(UNSUPPORTED, y=desc((9, 2048)), weights=desc((t, 2), capi.F32), slots=desc((t, 2), capi.I32),
            out=desc((t, 2048)))
    y = desc((9, 8))
    combine(INVALID, y=y, out=desc((4, 8), data=y.data))


def logprobs(code, logits=None, tokens=None, lp=None, ent=None, tl=None, ti=None, ws=None, nbytes=0, r=3, v=50, top=4):
    logits = desc((r, v)) if logits is None else logits
    tokens = desc((r,), capi.I64) if tokens is None else tokens
    lp = desc((r,), capi.F32) if lp is None else lp
    ent = desc((r,), capi.F32) if ent is None else ent
    tl = desc((r, top), capi.F32) if tl is None else tl
    ti = desc((r, top), capi.I64) if ti is None else ti
    refused(code, "thin_token_logprobs", logits, tokens, lp, ent, tl, ti, ws, nbytes, None)


def test_logprobs_refusals():
    logprobs(INVALID, logits=desc((3, 50), capi.I32))
    logprobs(INVALID, logits=desc((50,)))
    logprobs(INVALID, tokens=desc((3,), capi.I32))
    logprobs(INVALID, tokens=desc((4,), capi.I64))
    logprobs(INVALID, lp=desc((3,)))
    logprobs(INVALID, ent=desc((2,), capi.F32))
    logprobs(INVALID, tl=desc((3, 5), capi.F32))
    logprobs(INVALID, ti=desc((3, 4), capi.I32))
    logprobs(INVALID, top=33)
    logprobs(INVALID, lp=desc((3,), capi.F32, strides=(0,)))
    logprobs(INVALID, v=3)
    logprobs(INVALID, v=0, top=0)
    logprobs(UNSUPPORTED, logits=desc((3, 50), strides=(1, 3)))
    logprobs(UNSUPPORTED, r=1, v=8388609)
    logprobs(UNSUPPORTED, r=2 ** 27, v=80000)
    logprobs(UNSUPPORTED, r=2 ** 26, v=1000)  # 2^32 threads
    logprobs(UNSUPPORTED, r=2 ** 25, v=5000)
    logits = desc((3, 50))
    logprobs(INVALID, logits=logits, lp=desc((3,), capi.F32, data=logits.data + 4))
    lp = desc((3,), capi.F32)
    logprobs(INVALID, lp=lp, ent=desc((3,), capi.F32, data=lp.data + 8))
    need = capi.lib().thin_token_logprobs_workspace(3, 600000, 4)
    assert need > 0 and capi.lib().thin_token_logprobs_workspace(3, 1024, 4) == 0
    logprobs(WORKSPACE, v=600000)
    logprobs(WORKSPACE, v=600000, ws=(1 << 30) + 2, nbytes=need)
    logprobs(WORKSPACE, v=600000, ws=1 << 30, nbytes=need - 1)


def test_wrappers_refuse_host_tensors():
    x = torch.zeros((2, 4, 4, 16))
    with pytest.raises(ValueError):
        capi.group_norm(x, 4)
    with pytest.raises(ValueError):
        capi.group_norm(x[0, 0, 0], 4)
    with pytest.raises(ValueError):
        capi.group_norm_nc1hwc0(x, 4)
    with pytest.raises(ValueError):
        capi.expert_route(torch.zeros((2, 8)), 2)
    with pytest.raises(ValueError):
        capi.expert_route(torch.zeros((2, 8)), 2, scores="tanh")
    with pytest.raises(ValueError):
        capi.expert_dispatch(torch.zeros((2, 8)), torch.zeros((2, 1), dtype=torch.int32), 3)
    with pytest.raises(ValueError):
        capi.expert_combine(torch.zeros((2, 8)), torch.zeros((2, 1)), torch.zeros((2, 1), dtype=torch.int32))
    with pytest.raises(ValueError):
        capi.token_logprobs(torch.zeros((2, 8)), torch.zeros(2, dtype=torch.int64))
