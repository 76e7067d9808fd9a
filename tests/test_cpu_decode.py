"""Refusals of rotary positions, cross attention, the 8-bit cache and the
verification of drafts, before any device work.  Nothing here launches a kernel."""
import pytest
import torch

from tests.test_cpu_scores import INVALID, UNSUPPORTED, WORKSPACE, P, desc, refused
from thintnpu_amd import capi

NAN, INF = float("nan"), float("inf")


def rotary(code, q=None, k=None, positions=None, freqs=None, axes=None, q_out=None, k_out=None, pairs=4):
    q = desc((2, 3, 4, 8)) if q is None else q
    positions = desc((2, 2, 3), capi.I32) if positions is None else positions
    freqs = desc((pairs,), capi.F32) if freqs is None else freqs
    axes = desc((pairs,), capi.I32) if axes is None else axes
    q_out = desc(tuple(q.sizes[:q.rank]), q.dtype) if q_out is None else q_out
    refused(code, "thin_rotary_axes", q, k, positions, freqs, axes, 0, 0, q_out, k_out, None)


def test_rotary_refusals():
    rotary(INVALID, q=desc((2, 3, 32)))
    rotary(INVALID, q=desc((2, 3, 4, 8), capi.I32))
    rotary(INVALID, q_out=desc((2, 3, 4, 8), capi.BF16))
    rotary(INVALID, q_out=desc((2, 3, 4, 9)))
    rotary(INVALID, k=desc((2, 3, 1, 8)))
    rotary(INVALID, k_out=desc((2, 3, 1, 8)))
    for k in (desc((2, 3, 1, 8), capi.F32), desc((2, 2, 1, 8)), desc((2, 3, 1, 10)), desc((1, 3, 1, 8)), desc((3, 1, 8))):
        rotary(INVALID, k=k, k_out=desc(tuple(k.sizes[:k.rank]), k.dtype))
    rotary(INVALID, k=desc((2, 3, 1, 8)), k_out=desc((2, 3, 2, 8)))
    for positions in (desc((2, 3), capi.I32), desc((2, 2, 3), capi.F32), desc((2, 2, 4), capi.I32), desc((2, 1, 3), capi.I32), desc((0, 2, 3), capi.I32)):
        rotary(INVALID, positions=positions)
    rotary(INVALID, freqs=desc((4,), capi.F16))
    rotary(INVALID, axes=desc((4,), capi.I64))
    rotary(INVALID, axes=desc((3,), capi.I32))
    rotary(INVALID, pairs=5)
    rotary(UNSUPPORTED, q=desc((2, 3, 4, 8), strides=(200, 60, 16, 2)))
    rotary(UNSUPPORTED, q_out=desc((2, 3, 4, 8), strides=(200, 60, 16, 2)))
    rotary(UNSUPPORTED, q=desc((1, 1, 1, 1 << 16)), positions=desc((1, 1, 1), capi.I32))
    rotary(UNSUPPORTED, q=desc((2 ** 16, 2 ** 16, 1, 8)), positions=desc((1, 2 ** 16, 2 ** 16), capi.I32))
    rotary(INVALID, q_out=desc((2, 3, 4, 8), strides=(0, 32, 8, 1)))
    q = desc((2, 3, 4, 8))
    rotary(INVALID, q=q, q_out=desc((2, 3, 4, 8), data=q.data + 16))
    rotary(INVALID, q=q, q_out=desc((2, 3, 4, 8), data=q.data, strides=(96, 8, 24, 1)))
    rotary(INVALID, q=q, k=desc((2, 3, 4, 8)), k_out=desc((2, 3, 4, 8), data=q.data))
    out = desc((2, 3, 4, 8))
    rotary(INVALID, q_out=out, k=desc((2, 3, 4, 8)), k_out=desc((2, 3, 4, 8), data=out.data + 320))
    freqs = desc((4,), capi.F32)
    rotary(INVALID, freqs=freqs, q_out=desc((2, 3, 4, 8), data=freqs.data))


def cross(code, q=None, k=None, v=None, lengths=None, mask=None, scale=1.0, out=None, ws=None, nbytes=0):
    q = desc((2, 3, 4, 64)) if q is None else q
    k = desc((2, 9, 2, 64), q.dtype) if k is None else k
    v = desc(tuple(k.sizes[:k.rank]), k.dtype) if v is None else v
    out = desc(tuple(q.sizes[:q.rank]), q.dtype) if out is None else out
    refused(code, "thin_cross_attention", q, k, v, lengths, mask, scale, out, ws, nbytes, None)


def test_cross_refusals():
    cross(INVALID, q=desc((2, 3, 4, 64), capi.F32))
    cross(INVALID, k=desc((2, 9, 2, 64), capi.BF16))
    cross(INVALID, v=desc((2, 9, 2, 64), capi.BF16))
    cross(INVALID, out=desc((2, 3, 4, 64), capi.F32))
    cross(INVALID, q=desc((2, 3, 256)))
    cross(INVALID, k=desc((2, 9, 128)))
    cross(INVALID, v=desc((2, 8, 2, 64)))
    cross(INVALID, out=desc((2, 3, 4, 32)))
    cross(INVALID, k=desc((1, 9, 2, 64)))
    cross(INVALID, k=desc((2, 9, 2, 32)))
    cross(INVALID, k=desc((2, 9, 3, 64)))
    cross(INVALID, k=desc((2, 9, 0, 64)))
    for d in (4, 12, 100, 264):
        cross(UNSUPPORTED, q=desc((2, 3, 4, d)), k=desc((2, 9, 2, d)))
    cross(INVALID, lengths=desc((3,), capi.I32))
    cross(INVALID, lengths=desc((2,), capi.I64))
    cross(INVALID, mask=desc((2, 8), capi.U8))
    cross(INVALID, mask=desc((2, 9), capi.F16))
    strided = (1536, 512, 128, 2)
    cross(UNSUPPORTED, q=desc((2, 3, 4, 64), strides=strided))
    cross(UNSUPPORTED, k=desc((2, 9, 2, 64), strides=strided))
    cross(UNSUPPORTED, v=desc((2, 9, 2, 64), strides=strided))
    cross(UNSUPPORTED, out=desc((2, 3, 4, 64), strides=strided))
    for scale in (0.0, -1.0, NAN, INF, 3e38, 1e-45):
        cross(INVALID, scale=scale)
    cross(UNSUPPORTED, q=desc((2, 2 ** 29, 4, 64)))
    cross(UNSUPPORTED, k=desc((2, 2 ** 30, 2, 64)))
    cross(UNSUPPORTED, q=desc((2 ** 14, 2 ** 17, 4, 64)), k=desc((2 ** 14, 9, 2, 64)))
    cross(INVALID, out=desc((2, 3, 4, 64), strides=(768, 256, 0, 1)))
    cross(UNSUPPORTED, k=desc((2, 9, 2, 64), strides=(64, 2 ** 25, 64, 1)))
    cross(UNSUPPORTED, v=desc((2, 9, 2, 64), strides=(64, 2 ** 25, 64, 1)))
    q, k = desc((2, 3, 4, 64)), desc((2, 9, 2, 64))
    cross(INVALID, q=q, out=desc((2, 3, 4, 64), data=q.data))
    cross(INVALID, k=k, out=desc((2, 3, 4, 64), data=k.data + 64))
    long = desc((2, 9000, 2, 64))
    need = capi.lib().thin_cross_attention_workspace(P(q), P(long))
    assert need > 0 and capi.lib().thin_cross_attention_workspace(P(q), P(k)) == 0
    assert capi.lib().thin_cross_attention_workspace(None, P(k)) == 0
    assert capi.lib().thin_cross_attention_workspace(P(q), P(desc((2, 9, 0, 64)))) == 0
    cross(WORKSPACE, k=long)
    cross(WORKSPACE, k=long, ws=1 << 30, nbytes=need - 1)
    cross(WORKSPACE, k=long, ws=(1 << 30) + 2, nbytes=need)


class Parts:
    """Descriptors of a call with one of them replaced."""

    def __init__(self, **given):
        self.q = desc((2, 3, 4, 32))
        self.k, self.v = desc((2, 3, 2, 32)), desc((2, 3, 2, 32))
        self.kc, self.vc = desc((7, 2, 16, 32), capi.U8), desc((7, 2, 16, 32), capi.U8)
        self.ks, self.vs = desc((7, 2), capi.F32), desc((7, 2), capi.F32)
        self.table, self.lengths, self.counts = desc((2, 3), capi.I32), desc((2,), capi.I32), None
        self.out = desc((2, 3, 4, 32))
        self.scale, self.ws, self.nbytes = 1.0, None, 0
        self.__dict__.update(given)

    def cache(self):
        return self.kc, self.vc, self.ks, self.vs, self.table, self.lengths, self.counts

    def write(self, code):
        refused(code, "thin_cache_write", self.k, self.v, *self.cache(), None)

    def attend(self, code):
        refused(code, "thin_cache_attention", self.q, *self.cache(), self.scale, self.out, self.ws, self.nbytes, None)


def test_cache_refusals():
    for code, given in (
            (INVALID, dict(kc=desc((7, 2, 16, 32)))),
            (INVALID, dict(kc=desc((7, 2, 512), capi.U8))),
            (INVALID, dict(vc=desc((7, 2, 32, 32), capi.U8))),
            (INVALID, dict(vc=desc((7, 2, 16, 32), capi.I16))),
            (INVALID, dict(kc=desc((7, 2, 16, 48), capi.U8), vc=desc((7, 2, 16, 48), capi.U8))),
            (INVALID, dict(ks=desc((7, 2), capi.F16))),
            (INVALID, dict(vs=desc((7, 3), capi.F32))),
            (INVALID, dict(ks=desc((14,), capi.F32))),
            (INVALID, dict(table=desc((2, 3), capi.I64))),
            (INVALID, dict(table=desc((3, 3), capi.I32))),
            (INVALID, dict(lengths=desc((2,), capi.I64))),
            (INVALID, dict(lengths=desc((1,), capi.I32))),
            (INVALID, dict(counts=desc((3,), capi.I32))),
            (INVALID, dict(counts=desc((2,), capi.F32))),
            (UNSUPPORTED, dict(kc=desc((7, 2, 24, 32), capi.U8), vc=desc((7, 2, 24, 32), capi.U8))),
            (UNSUPPORTED, dict(kc=desc((7, 2, 8, 32), capi.U8), vc=desc((7, 2, 8, 32), capi.U8))),
            (UNSUPPORTED, dict(kc=desc((7, 2, 2048, 32), capi.U8), vc=desc((7, 2, 2048, 32), capi.U8))),
            (UNSUPPORTED, dict(kc=desc((7, 2, 16, 32), capi.U8, strides=(2048, 1024, 64, 2)))),
            (UNSUPPORTED, dict(vc=desc((7, 2, 16, 32), capi.U8, strides=(2048, 1024, 64, 2)))),
            (UNSUPPORTED, dict(vc=desc((7, 2, 16, 32), capi.U8, strides=(64, 32, 2 ** 26, 1)))),
            (UNSUPPORTED, dict(table=desc((2, 2 ** 26), capi.I32)))):
        Parts(**given).write(code)
        Parts(**given).attend(code)
    for d in (8, 24, 40, 272):
        parts = Parts(q=desc((2, 3, 4, d)), out=desc((2, 3, 4, d)), k=desc((2, 3, 2, d)), v=desc((2, 3, 2, d)),
                      kc=desc((7, 2, 16, d), capi.U8), vc=desc((7, 2, 16, d), capi.U8))
        parts.write(UNSUPPORTED)
        parts.attend(UNSUPPORTED)


def test_write_refusals():
    Parts(k=desc((2, 3, 2, 32), capi.I32)).write(INVALID)
    Parts(v=desc((2, 3, 2, 32), capi.BF16)).write(INVALID)
    Parts(v=desc((2, 3, 2, 64))).write(INVALID)
    Parts(k=desc((6, 2, 32)), v=desc((6, 2, 32))).write(INVALID)
    Parts(k=desc((2, 3, 4, 32)), v=desc((2, 3, 4, 32))).write(INVALID)
    Parts(k=desc((2, 3, 2, 32), strides=(512, 128, 64, 2))).write(UNSUPPORTED)
    Parts(k=desc((2, 2 ** 30, 2, 32)), v=desc((2, 2 ** 30, 2, 32))).write(UNSUPPORTED)
    n = 2 ** 29
    Parts(k=desc((n, 3, 2, 32)), v=desc((n, 3, 2, 32)), table=desc((n, 3), capi.I32), lengths=desc((n,), capi.I32)).write(UNSUPPORTED)
    Parts(kc=desc((7, 2, 16, 32), capi.U8, strides=(0, 512, 32, 1))).write(INVALID)
    Parts(ks=desc((7, 2), capi.F32, strides=(1, 0))).write(INVALID)
    one = desc((7, 2, 16, 32), capi.U8)
    Parts(kc=one, vc=one).write(INVALID)
    Parts(kc=one, vs=desc((7, 2), capi.F32, data=one.data + 64)).write(INVALID)
    Parts(kc=one, k=desc((2, 3, 2, 32), data=one.data)).write(INVALID)
    Parts(kc=one, table=desc((2, 3), capi.I32, data=one.data + 7)).write(INVALID)
    scales = desc((7, 2), capi.F32)
    Parts(ks=scales, vs=desc((7, 2), capi.F32, data=scales.data + 4)).write(INVALID)
    Parts(ks=scales, lengths=desc((2,), capi.I32, data=scales.data + 8)).write(INVALID)


def test_attention_refusals():
    Parts(q=desc((2, 3, 4, 32), capi.F32), out=desc((2, 3, 4, 32), capi.F32)).attend(INVALID)
    Parts(out=desc((2, 3, 4, 32), capi.BF16)).attend(INVALID)
    Parts(out=desc((2, 4, 3, 32))).attend(INVALID)
    Parts(q=desc((2, 12, 32)), out=desc((2, 12, 32))).attend(INVALID)
    Parts(q=desc((2, 3, 5, 32)), out=desc((2, 3, 5, 32))).attend(INVALID)
    Parts(q=desc((2, 3, 4, 32), strides=(1024, 256, 64, 2))).attend(UNSUPPORTED)
    Parts(out=desc((2, 3, 4, 32), strides=(1024, 256, 64, 2))).attend(UNSUPPORTED)
    for scale in (0.0, -1.0, NAN, INF, 3e38, 1e-45):
        Parts(scale=scale).attend(INVALID)
    Parts(q=desc((2, 2 ** 29, 4, 32)), out=desc((2, 2 ** 29, 4, 32))).attend(UNSUPPORTED)
    Parts(out=desc((2, 3, 4, 32), strides=(0, 128, 32, 1))).attend(INVALID)
    q = desc((2, 3, 4, 32))
    Parts(q=q, out=desc((2, 3, 4, 32), data=q.data)).attend(INVALID)
    kc = desc((7, 2, 16, 32), capi.U8)
    Parts(kc=kc, out=desc((2, 3, 4, 32), data=kc.data + 3000)).attend(INVALID)
    table = desc((2, 600), capi.I32)
    need = capi.lib().thin_cache_attention_workspace(P(q), P(kc), P(table))
    assert need > 0 and capi.lib().thin_cache_attention_workspace(P(q), P(kc), P(desc((2, 3), capi.I32))) == 0
    assert capi.lib().thin_cache_attention_workspace(P(q), None, P(table)) == 0
    Parts(table=table).attend(WORKSPACE)
    Parts(table=table, ws=1 << 30, nbytes=need - 1).attend(WORKSPACE)
    Parts(table=table, ws=(1 << 30) + 2, nbytes=need).attend(WORKSPACE)


def verify(code, b=3, k=2, v=50, ws=None, nbytes=0, **given):
    parts = dict(target=desc((b, k + 1, v), capi.F32), draft=desc((b, k, v), capi.F32), tokens=desc((b, k), capi.I64), counts=None,
                 accept=desc((b, k), capi.F32), sample=desc((b,), capi.F32), out=desc((b, k + 1), capi.I64), taken=desc((b,), capi.I32))
    parts.update(given)
    refused(code, "thin_verify_drafts", *parts.values(), ws, nbytes, None)


def test_verify_refusals():
    verify(INVALID, target=desc((3, 3, 50), capi.I32))
    verify(INVALID, target=desc((3, 150), capi.F32))
    verify(INVALID, target=desc((3, 0, 50), capi.F32))
    verify(INVALID, draft=desc((3, 2, 50)))
    verify(INVALID, draft=desc((3, 3, 50), capi.F32))
    verify(INVALID, draft=desc((3, 2, 49), capi.F32))
    verify(INVALID, tokens=desc((3, 2), capi.I32))
    verify(INVALID, tokens=desc((3, 3), capi.I64))
    verify(INVALID, accept=desc((3, 2)))
    verify(INVALID, accept=desc((2, 2), capi.F32))
    verify(INVALID, sample=desc((3, 1), capi.F32))
    verify(INVALID, counts=desc((3,), capi.I64))
    verify(INVALID, out=desc((3, 2), capi.I64))
    verify(INVALID, out=desc((3, 3), capi.I32))
    verify(INVALID, taken=desc((3,), capi.I64))
    verify(INVALID, v=0)
    verify(UNSUPPORTED, k=65)
    verify(UNSUPPORTED, v=8388609)
    verify(UNSUPPORTED, target=desc((3, 3, 50), capi.F32, strides=(150, 1, 3)))
    verify(UNSUPPORTED, draft=desc((3, 2, 50), capi.F32, strides=(100, 1, 2)))
    verify(UNSUPPORTED, b=2 ** 24)
    verify(INVALID, out=desc((3, 3), capi.I64, strides=(0, 1)))
    verify(INVALID, taken=desc((3,), capi.I32, strides=(0,)))
    tokens, out = desc((3, 2), capi.I64), desc((3, 3), capi.I64)
    verify(INVALID, tokens=tokens, out=desc((3, 3), capi.I64, data=tokens.data))
    verify(INVALID, out=out, taken=desc((3,), capi.I32, data=out.data + 8))
    need = capi.lib().thin_verify_drafts_workspace(3, 5000)
    assert need > 0 and capi.lib().thin_verify_drafts_workspace(3, 50) == 0 and capi.lib().thin_verify_drafts_workspace(-1, 50) == 0
    verify(WORKSPACE, v=5000)
    verify(WORKSPACE, v=5000, ws=1 << 30, nbytes=need - 1)
    verify(WORKSPACE, v=5000, ws=(1 << 30) + 4, nbytes=need)


def test_null_operands():
    refused(INVALID, "thin_rotary_axes", None, None, None, None, None, 0, 0, None, None, None)
    refused(INVALID, "thin_cross_attention", None, None, None, None, None, 1.0, None, None, 0, None)
    refused(INVALID, "thin_cache_write", *[None] * 10)
    refused(INVALID, "thin_cache_attention", *[None] * 8, 1.0, None, None, 0, None)
    refused(INVALID, "thin_verify_drafts", *[None] * 9, 0, None)


def test_wrappers_refuse_host_tensors():
    q, codes, scales = torch.zeros((2, 3, 4, 32)).half(), torch.zeros((7, 4, 16, 32), dtype=torch.uint8), torch.zeros((7, 4))
    table, lengths = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: capi.rotary_axes(q, torch.zeros((1, 2, 3), dtype=torch.int32), torch.zeros(2), torch.zeros(2, dtype=torch.int32)),
                 lambda: capi.cross_attention(q, q, q),
                 lambda: capi.cache_write(q, q, codes, codes, scales, scales, table, lengths),
                 lambda: capi.cache_attention(q, codes, codes, scales, scales, table, lengths),
                 lambda: capi.verify_drafts(torch.zeros((2, 3, 9)), None, torch.zeros((2, 2), dtype=torch.int64), torch.zeros((2, 2)), torch.zeros(2))):
        with pytest.raises(ValueError):
            call()
