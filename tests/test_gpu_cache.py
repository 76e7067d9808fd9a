"""thin_cache_write against exact arithmetic (codes and scales equal, NaN by its
place), and thin_cache_attention against the 64-bit definition on the codes there
are, within oracle.attend.allowed()."""
import math

import pytest
import torch

from oracle import attend
from oracle import cache as oracle
from tests.helpers import gen

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALVES = {n: TYPES[n] for n in ("fp16", "bf16")}


class Cache:
    """The same cache on the host and on the device; codes of the host as bytes."""

    def __init__(self, gpu, b, slots, page, heads, d, seed, spare=2, filled=True):
        g = gen(seed)
        pages = b * slots + spare
        self.gpu, self.g, self.shape = gpu, g, (pages, heads, page, d)
        self.host = []
        for _ in range(2):
            codes = torch.randint(0, 256, self.shape, generator=g, dtype=torch.int64)
            codes = torch.where((codes & 0x7F) == 0x7F, codes - 1, codes).to(torch.uint8)
            self.host.append(codes if filled else torch.full(self.shape, 0x7F, dtype=torch.uint8))
        for _ in range(2):
            scales = torch.exp2(torch.randint(-8, 1, (pages, heads), generator=g).float())
            self.host.append(scales if filled else torch.full((pages, heads), math.nan))
        self.table = torch.randperm(pages, generator=g)[:b * slots].view(b, slots).int()
        self.dev = [x.to(gpu) for x in self.host]

    def write(self, k, v, lengths, counts=None, table=None):
        from thintnpu_amd import capi
        table = self.table if table is None else table
        to = lambda x: None if x is None else x.to(self.gpu)  # noqa: E731
        # (bytes and float8 codes are the same to it)
        codes = [x.view(torch.float8_e4m3fn) for x in self.dev[:2]] if k.shape[1] % 2 else self.dev[:2]
        capi.cache_write(to(k), to(v), *codes, *self.dev[2:], to(table), to(lengths), to(counts))
        oracle.write(k, v, *self.host, table, lengths, counts)
        self.same()

    def same(self):
        for a, b in zip(self.dev[:2], self.host[:2]):
            a = a.cpu()
            nan = (a & 0x7F) == 0x7F
            assert torch.equal(nan, (b & 0x7F) == 0x7F)
            assert torch.equal(a[~nan], b[~nan])
        for a, b in zip(self.dev[2:], self.host[2:]):
            a = a.cpu()
            assert torch.equal(a.nan_to_num(-1.0), b.nan_to_num(-1.0))

    def attend(self, q, lengths, counts=None, scale=None, table=None):
        from thintnpu_amd import capi
        table = self.table if table is None else table
        to = lambda x: None if x is None else x.to(self.gpu)  # noqa: E731
        got = capi.cache_attention(to(q), *self.dev, to(table), to(lengths), to(counts), scale)
        ref = oracle.attention(q, *self.host, table, lengths, counts, scale)
        close(got, ref, q, table.shape[1] * self.shape[2], self.host)
        return got


def close(got, ref, q, keys, host):
    got, out = got.cpu().double(), ref[0]
    assert torch.equal(torch.isnan(got), torch.isnan(out))
    # weights as multiples of the largest scale of the values: 448 * that is what 2^-33 counts
    top = float(host[3][torch.isfinite(host[3])].max()) * 448 * 2
    allowed = attend.allowed(q, ref, keys, top)
    over = torch.isinf(got)  # past the largest of the type
    assert (out.abs() + allowed >= torch.finfo(q.dtype).max)[over].all() and (got.sign() == out.sign())[over].all()
    far = ((got - out).abs() / allowed)[~torch.isnan(out) & ~over]
    assert far.numel() == 0 or far.max() <= 1, float(far.max())


def tokens(b, t, heads, d, dtype, seed, std=1.0):
    g = gen(seed)
    return tuple((torch.randn((b, t, heads, d), generator=g) * std * torch.exp2(torch.randn((b, t, 1, 1), generator=g))).to(dtype) for _ in range(2))


def queries(b, t, h, d, dtype, seed):
    return torch.randn((b, t, h, d), generator=gen(seed)).to(dtype)


# ------------------------------------------------------------------ write

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,page", [(16, 16), (32, 48), (64, 64), (80, 32), (128, 128), (208, 16), (256, 256)])
def test_write_widths_and_pages(gpu, dtype, d, page):
    c = Cache(gpu, 3, 3, page, 2, d, d + page)
    lengths = torch.tensor([page + 5, 3 * page, page // 2], dtype=torch.int32)
    c.write(*tokens(3, 1, 2, d, TYPES[dtype], 1), lengths)
    c.write(*tokens(3, page // 2, 2, d, TYPES[dtype], 2), lengths)
    c.write(*tokens(3, 2 * page, 2, d, TYPES[dtype], 3), torch.full((3,), 3 * page - 1, dtype=torch.int32),
            torch.tensor([2 * page, 1, page + 1], dtype=torch.int32))


def test_write_one_after_another(gpu):
    """Tokens one by one, the larger ones raising their page's scale."""
    c = Cache(gpu, 2, 3, 16, 3, 32, 7, filled=False)
    for i in range(40):
        k, v = tokens(2, 1, 3, 32, torch.bfloat16, 100 + i, 2.0 ** (i % 5))
        c.write(k, v, torch.tensor([i + 1, i // 2 + 1], dtype=torch.int32), torch.tensor([1, i % 2], dtype=torch.int32))


def test_write_drafts_given_up(gpu):
    """A lower length gives tokens up; their places are written anew, and a page
    begun anew has a scale of its own."""
    c = Cache(gpu, 1, 4, 16, 2, 16, 9, filled=False)
    length = 0
    for i, keep in enumerate((16, 3, 5, 0, 2, 6, 4)):
        n = 16 if i == 0 else 6
        k, v = tokens(1, n, 2, 16, torch.float16, i, 1.0 if i % 2 else 50.0)
        c.write(k, v, torch.tensor([length + n], dtype=torch.int32))
        length += keep
    assert length == 36


@pytest.mark.parametrize("dtype", TYPES)
def test_write_special_values(gpu, dtype):
    t = TYPES[dtype]
    c = Cache(gpu, 1, 2, 16, 1, 64, 3)
    k = torch.zeros((1, 12, 1, 64), dtype=t)
    v = torch.randn((1, 12, 1, 64), generator=gen(1)).to(t)
    v[0, 0, 0, :6] = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1.0]).to(t)
    v[0, 3] = math.nan
    c.write(k, v, torch.tensor([12], dtype=torch.int32))          # zeros: a scale of 1
    assert c.dev[2][c.table[0, 0], 0] == 1.0
    c.write(v[:, :2], k[:, :2], torch.tensor([14], dtype=torch.int32))
    c.write(k[:, :1], k[:, :1], torch.tensor([15], dtype=torch.int32))  # nothing to raise it
    low = torch.full((1, 4, 1, 64), torch.finfo(t).max, dtype=t)
    c.write(low, -low, torch.tensor([20], dtype=torch.int32))
    tiny = torch.full((1, 2, 1, 64), torch.finfo(t).smallest_normal * torch.finfo(t).eps, dtype=t)
    c.write(tiny, v[:, :2] * 0 + math.inf, torch.tensor([18], dtype=torch.int32))
    c.write(v[:, 3:4], v[:, 3:4], torch.tensor([17], dtype=torch.int32))  # NaN alone


def test_write_codes_of_every_size(gpu):
    """Every half in the range of the codes, ties and subnormals among them."""
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    x = torch.cat([x, torch.zeros(-x.numel() % 256).half()]).view(1, -1, 1, 256)
    n = x.shape[1]
    c = Cache(gpu, 1, -(-n // 256), 256, 1, 256, 4)
    x[0, ::256, 0, 0] = 448.0
    c.write(x, -x, torch.tensor([n], dtype=torch.int32))
    assert (c.dev[2][c.table[0, :-1].long()] == 1).all()


def test_write_many(gpu):
    """Against the attention's reading: the values that come back are the tokens'."""
    from thintnpu_amd import capi
    b, t, heads, d, page = 5, 700, 4, 64, 32
    c = Cache(gpu, b, 24, page, heads, d, 2)
    k, v = tokens(b, t, heads, d, torch.float16, 1)
    counts, lengths = torch.tensor([700, 1, 333, 64, 0], dtype=torch.int32), torch.tensor([700, 768, 700, 65, 5], dtype=torch.int32)
    before = [x.clone() for x in c.dev]
    capi.cache_write(k.to(gpu), v.to(gpu), *c.dev, c.table.to(gpu), lengths.to(gpu), counts.to(gpu))
    touched = torch.zeros(c.shape[0], page, dtype=torch.bool)
    for i in range(b):
        begin = int(lengths[i] - counts[i])
        for j in range(int(counts[i])):
            touched[int(c.table[i, (begin + j) // page]), (begin + j) % page] = True
        for x, codes, scales in ((k, c.dev[0], c.dev[2]), (v, c.dev[1], c.dev[3])):
            where = torch.arange(begin, int(lengths[i]))
            ids = c.table[i].long()[where // page]
            s = scales.cpu()[ids].double()
            back = oracle.decode(codes.cpu()[ids, :, where % page]) * s[..., None]
            want = x[i, :int(counts[i])].double()
            # half a step of 3 bits, or of the smallest exponent's
            assert ((back - want).abs() <= want.abs() / 16 + s[..., None] * 2.0 ** -10).all()
    pages = touched.any(1)
    for a, x in zip(c.dev[:2], before[:2]):
        # what lies behind a sequence's end, and pages of nobody, stay
        assert torch.equal(a.cpu()[~pages], x.cpu()[~pages])
    assert torch.equal(c.dev[2].cpu()[~pages], before[2].cpu()[~pages])


def test_write_nowhere(gpu):
    """Pages that do not exist, lengths beyond the table or below the tokens, no tokens."""
    c = Cache(gpu, 5, 3, 16, 2, 32, 5)
    table = c.table.clone()
    table[0, 1], table[1, 0], table[2] = -1, c.shape[0], 2 ** 31 - 1
    k, v = tokens(5, 20, 2, 32, torch.float16, 6)
    c.write(k, v, torch.tensor([40, 21, 20, 55, 7], dtype=torch.int32), table=table)
    c.write(k, v, torch.tensor([-4, 0, 2 ** 31 - 1, 1, 48], dtype=torch.int32), torch.tensor([20, 3, 20, -1, 2 ** 31 - 1], dtype=torch.int32))
    c.write(k[:, :0], v[:, :0], torch.tensor([5] * 5, dtype=torch.int32))


def test_write_views(gpu):
    from thintnpu_amd import capi
    g = gen(8)
    pages, heads, page, d, b, t = 7, 3, 16, 32, 2, 9
    x = torch.randn((b, t, 2, heads, d + 1), generator=g).to(torch.bfloat16)
    k, v = x[:, :, 0, :, 1:], x[:, :, 1, :, :d]
    table = torch.tensor([[5, 1], [0, 3]], dtype=torch.int32)
    lengths = torch.tensor([20, 9], dtype=torch.int32)
    host = [torch.full((pages, heads, page, d), 0x38, dtype=torch.uint8) for _ in range(2)] + [torch.ones((pages, heads)) for _ in range(2)]
    both = torch.full((pages, page, 2, heads, d + 5), 0x38, dtype=torch.uint8, device=gpu)  # tokens before heads, odd strides
    scales = torch.ones((heads, pages, 2), device=gpu)
    kc, vc = (both[:, :, i, :, 3:3 + d].permute(0, 2, 1, 3) for i in range(2))
    ks, vs = (scales[:, :, i].t() for i in range(2))
    dx = x.to(gpu)
    wide = torch.zeros((4, 2, 2), dtype=torch.int32, device=gpu)
    wide[::2, :, 1] = table.to(gpu)
    capi.cache_write(dx[:, :, 0, :, 1:], dx[:, :, 1, :, :d], kc, vc, ks, vs, wide[::2, :, 1], lengths.to(gpu))
    oracle.write(k, v, *host, table, lengths)
    assert all(torch.equal(a.cpu(), b) for a, b in zip((kc, vc, ks, vs), host))
    rest = both.clone()
    rest[..., 3:3 + d] = 0x38
    assert (rest == 0x38).all()
    q = queries(b, t, 6, d, torch.bfloat16, 3)
    got = capi.cache_attention(q.to(gpu), kc, vc, ks, vs, wide[::2, :, 1], lengths.to(gpu))
    close(got, oracle.attention(q, *host, table, lengths), q, 32, host)


# ------------------------------------------------------------------ attention

@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128, 144, 192, 208, 256])
def test_attention_widths(gpu, dtype, d):
    c = Cache(gpu, 2, 5, 32, 2, d, d)
    lengths = torch.tensor([159, 70], dtype=torch.int32)
    for t, h in ((1, 4), (5, 10), (40, 4)):  # 2, 25 and 80 rows of a head
        c.attend(queries(2, t, h, d, HALVES[dtype], t), lengths)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 1024])
def test_attention_pages(gpu, page):
    slots = max(2, 300 // page)
    c = Cache(gpu, 3, slots, page, 2, 64, page)
    for t, h in ((1, 8), (9, 6), (50, 4)):
        c.attend(queries(3, t, h, 64, torch.float16, t), torch.tensor([slots * page, slots * page - 17, max(t, 33)], dtype=torch.int32))


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 128, 129, 255, 256, 257])
def test_attention_lengths(gpu, length):
    c = Cache(gpu, 2, 17, 16, 1, 64, length)
    for t, h in ((1, 5), (4, 8), (70, 2)):
        c.attend(queries(2, t, h, 64, torch.bfloat16, t), torch.tensor([max(length, t), 270], dtype=torch.int32))


@pytest.mark.parametrize("b,t,h,heads,slots,page", [(1, 1, 1, 1, 500, 16), (2, 6, 20, 4, 200, 48), (1, 40, 4, 2, 100, 64), (3, 1, 32, 1, 60, 128)])
def test_attention_split(gpu, b, t, h, heads, slots, page):
    """Long contexts of few rows: their tokens are split and joined, also where
    lengths differ much and a split has none."""
    c = Cache(gpu, b, slots, page, heads, 64, slots)
    lengths = torch.tensor([slots * page, 300, 40][:b], dtype=torch.int32)
    c.attend(queries(b, t, h, 64, torch.float16, 1), lengths)
    c.attend(queries(b, t, h, 64, torch.bfloat16, 2), lengths, torch.tensor([1, t, 0][:b], dtype=torch.int32))


@pytest.mark.parametrize("t,h", [(1, 4), (7, 4), (30, 8)])
def test_attention_counts(gpu, t, h):
    """Ragged counts, none at all, lengths of zero, below the tokens and beyond the table."""
    c = Cache(gpu, 8, 3, 16, 2, 32, 4)
    lengths = torch.tensor([48, 30, 0, 5, 48, 60, 2 ** 31 - 1, -7], dtype=torch.int32)
    counts = torch.tensor([t, 1, t, t, 0, t, -2, 2 ** 31 - 1], dtype=torch.int32)
    q = queries(8, t, h, 32, torch.float16, 5)
    got = c.attend(q, lengths, counts)
    assert not got[2].any() and not got[4].any() and not got[6].any() and not got[7].any() and not got[1, 1:].any()
    c.attend(q, lengths)


@pytest.mark.parametrize("t,h", [(1, 4), (5, 6), (40, 4)])
def test_attention_bad_pages(gpu, t, h):
    """Tokens of pages that do not exist are not seen."""
    c = Cache(gpu, 3, 6, 16, 2, 64, 6)
    table = c.table.clone()
    table[0, 2], table[0, 5], table[1], table[2, 0] = -1, c.shape[0], 2 ** 31 - 1, -2 ** 31
    got = c.attend(queries(3, t, h, 64, torch.bfloat16, t), torch.tensor([96, 96, 50], dtype=torch.int32), table=table)
    assert not got[1].any()


@pytest.mark.parametrize("t,h", [(1, 4), (9, 4), (33, 6)])
@pytest.mark.parametrize("dtype", HALVES)
def test_attention_does_not_see_ahead(gpu, t, h, dtype):
    """NaN codes, and scales of NaN and infinity, of later tokens and behind the
    end reach no earlier row; seen ones reach the rows that see them."""
    q = queries(3, t, h, 64, HALVES[dtype], 2)
    for page, at, which in ((16, 41, 0), (16, 41, 1), (48, 60, 1), (64, 3, 0), (64, 64, 1)):
        c = Cache(gpu, 3, 6, page, 2, 64, page + at)
        lengths = torch.tensor([at + 1, at + t, at + t + 1], dtype=torch.int32)  # the last, the first and none of the call's own
        lengths = torch.maximum(lengths, torch.tensor(t, dtype=torch.int32))
        for i in range(3):
            c.host[which][c.table[i, at // page].long(), 1, at % page, 5] = 0x7F
            n = int(lengths[i])
            c.host[0][c.table[i, n // page].long(), :, n % page:] = 0xFF  # behind the end
            c.host[1][c.table[i, n // page].long(), :, n % page:] = 0x7F
            for s in range(n // page + 1, 6):
                for x, bad in ((2, math.nan), (3, math.inf)):
                    c.host[x][c.table[i, s].long()] = bad
        c.dev = [x.to(gpu) for x in c.host]
        c.attend(q, lengths)
        # an infinite scale of the page of the last token, seen by that token's row alone
        edge = torch.full((3,), 2 * page + 1, dtype=torch.int32)
        if t <= page:
            for i in range(3):
                c.host[3][c.table[i, 2].long()] = math.nan
            c.dev = [x.to(gpu) for x in c.host]
            got = c.attend(q, edge)
            assert torch.isnan(got[:, -1]).all()


@pytest.mark.parametrize("t", [1, 40])
def test_attention_scales_of_any_size(gpu, t):
    """Pages whose scales lie far apart, in either order; scales that are no
    powers of two; zeros."""
    for i, low in enumerate((-20.0, 20.0, -3.0)):
        c = Cache(gpu, 2, 8, 16, 2, 64, 30 + i)
        c.host[3] = torch.exp2(torch.linspace(0, low, c.shape[0]))[:, None].repeat(1, 2) * 1.3
        c.host[2] = c.host[2] * 0.7
        if i == 2:
            c.host[3][c.table[0, :3].long()] = 0.0
            c.host[3][c.table[1].long()] = 0.0
        c.dev = [x.to(gpu) for x in c.host]
        for dtype in HALVES.values():
            c.attend(queries(2, t, 4, 64, dtype, i), torch.tensor([128, 100], dtype=torch.int32))


def test_attention_rows_in_any_number(gpu):
    c = Cache(gpu, 1, 10, 32, 1, 64, 1)
    for t, h in ((1, 1), (1, 16), (1, 17), (1, 32), (1, 33), (2, 16), (3, 11), (129, 1), (64, 2), (1, 128), (100, 3)):
        c.attend(queries(1, t, h, 64, torch.float16, t + h), torch.tensor([300], dtype=torch.int32))


def test_no_tokens_and_no_pages(gpu):
    from thintnpu_amd import capi
    q = torch.ones((2, 3, 4, 32), dtype=torch.float16, device=gpu)
    codes, scales = torch.zeros((0, 2, 16, 32), dtype=torch.uint8, device=gpu), torch.zeros((0, 2), device=gpu)
    lengths = torch.tensor([3, 9], dtype=torch.int32, device=gpu)
    for slots in (0, 2):
        table = torch.zeros((2, slots), dtype=torch.int32, device=gpu)
        assert not capi.cache_attention(q, codes, codes, scales, scales, table, lengths, out=torch.ones_like(q)).any()
        capi.cache_write(q[:, :, :2], q[:, :, :2], codes, codes, scales, scales, table, lengths)
    assert capi.cache_attention(q[:, :0], codes, codes, scales, scales, table, lengths).shape == (2, 0, 4, 32)


def test_beyond_32_bits(gpu):
    """A cache of more than 4 GB, and pages at both ends of it."""
    from thintnpu_amd import capi
    per = 2 * 16 * 64
    pages = 2 ** 32 // per + 5
    big = [torch.zeros((pages, 2, 16, 64), dtype=torch.uint8, device=gpu) for _ in range(2)]
    scales = [torch.ones((pages, 2), device=gpu) for _ in range(2)]
    small = Cache(gpu, 1, 3, 16, 2, 64, 1)
    ids = torch.tensor([pages - 1, 0, pages - 3])
    table = ids.int().view(1, 3).to(gpu)
    k, v = tokens(1, 40, 2, 64, torch.float16, 4)
    lengths = torch.tensor([44], dtype=torch.int32)
    for a, b in zip(big + scales, small.host):
        a[ids.to(gpu)] = b[small.table[0].long()].to(gpu)
    capi.cache_write(k.to(gpu), v.to(gpu), *big, *scales, table, lengths.to(gpu))
    small.write(k, v, lengths)
    for a, b in zip(big + scales, small.host):
        assert torch.equal(a[ids.to(gpu)].cpu(), b[small.table[0].long()])
    for t, h in ((1, 4), (40, 4)):
        q = queries(1, t, h, 64, torch.float16, t)
        got = capi.cache_attention(q.to(gpu), *big, *scales, table, lengths.to(gpu))
        assert torch.equal(got, small.attend(q, lengths))


@pytest.mark.parametrize("t", [1, 60])
def test_same_bits_streams_and_graphs(gpu, t):
    from thintnpu_amd import capi
    b, heads, d, page = 3, 2, 64, 32
    c = Cache(gpu, b, 40, page, heads, d, 3)
    table = c.table.to(gpu)
    lengths = torch.tensor([1000, 400, 64], dtype=torch.int32, device=gpu)
    k, v = (x.to(gpu) for x in tokens(b, t, heads, d, torch.bfloat16, 4))
    q = queries(b, t, 8, d, torch.bfloat16, 5).to(gpu)

    def step(cache, stream=None):
        capi.cache_write(k, v, *cache, table, lengths, stream=stream)
        return capi.cache_attention(q, *cache, table, lengths, stream=stream)

    def fresh():
        return [x.to(gpu) for x in c.host]

    one, two = fresh(), fresh()
    ref = step(one)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(two, side)
    side.synchronize()
    assert torch.equal(got, ref) and all(torch.equal(x, y) for x, y in zip(one, two))
    caches, outs, graphs = [fresh(), fresh()], [], []
    for cache in caches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(cache))
        graphs.append(graph)
    eager = fresh()
    for _ in range(4):
        lengths.add_(1)
        k.mul_(1.3)
        for graph in graphs:
            graph.replay()
        want = step(eager)
        torch.cuda.synchronize()
        for cache, out in zip(caches, outs):
            assert torch.equal(out, want) and all(torch.equal(x, y) for x, y in zip(cache, eager))


@pytest.mark.parametrize("b", [70, 150])
def test_attention_many_sequences(gpu, b):
    """Few rows of more sequences than a wavefront has lanes, some without tokens."""
    c = Cache(gpu, b, 9, 64, 1, 16, b)
    lengths = torch.randint(3, 577, (b,), generator=c.g, dtype=torch.int32)
    counts = torch.randint(0, 4, (b,), generator=c.g, dtype=torch.int32)
    lengths[::7] = 0
    lengths[63:66] = torch.tensor([0, 576, 1], dtype=torch.int32)
    got = c.attend(queries(b, 3, 4, 16, torch.bfloat16, b), lengths, counts)
    assert not got[::7].any()


@pytest.mark.parametrize("b,heads,t,h,d,length", [(32, 32, 5, 128, 144, 4300), (16, 16, 40, 16, 32, 9000), (16, 16, 130, 16, 64, 5000)])
@pytest.mark.parametrize("dtype", HALVES)
def test_attention_long(gpu, b, heads, t, h, d, length, dtype):
    """Many sequences that read the same long context: a workgroup walks far enough
    to look its pages up again.  All get the same bits, the first is checked."""
    from thintnpu_amd import capi
    c = Cache(gpu, 1, -(-length // 16), 16, heads, d, length)
    c.host[3][c.table[0].long()] *= torch.exp2(torch.arange(c.table.shape[1]) // 48 % 5 * 2.0)[:, None]  # in steps, up and down
    c.host[1][c.table[0, 70].long(), 0, 3, 2] = 0x7F
    bad = c.table.clone()
    bad[0, 100:103] = -1
    c.dev = [x.to(gpu) for x in c.host]
    q = queries(1, t, h, d, HALVES[dtype], t)
    lengths = torch.tensor([length], dtype=torch.int32)
    got = capi.cache_attention(q.repeat(b, 1, 1, 1).to(gpu), *c.dev, bad.repeat(b, 1).to(gpu), lengths.repeat(b).to(gpu))
    assert torch.equal(got.view(torch.int16), got[:1].expand_as(got).contiguous().view(torch.int16))
    close(got[:1], oracle.attention(q, *c.host, bad, lengths), q, length, c.host)


@pytest.mark.parametrize("t", [1, 6, 40])
@pytest.mark.parametrize("dtype", HALVES)
def test_attention_scales_of_zero(gpu, t, dtype):
    """Keys and values of scale 0 beside places that are not seen."""
    for which in (2, 3):
        c = Cache(gpu, 2, 4, 16, 2, 32, t)
        c.host[which][c.table[:, 1:].long()] = 0.0
        c.dev = [x.to(gpu) for x in c.host]
        for length in (41, 57, 60):
            got = c.attend(queries(2, t, 4, 32, HALVES[dtype], t), torch.tensor([length, max(t, 20)], dtype=torch.int32))
            assert torch.isfinite(got).all()
