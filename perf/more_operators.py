"""The measured work of a head that answers with tokens about a feature map.

Five operators, through the C ABI as `thintnpu_amd.capi` binds it, on torch
device tensors: rotary positions with several axes, cross attention to an
encoder's states, new keys and values into a cache held in 8 bits (e4m3, a
power-of-two scale for each page of tokens and head), attention over that cache,
and the verification of drafted tokens.  The plain forms are elementary torch
operations in 32 bits (64 for angles, for the products that accept a draft and
for sums of probabilities, where 32 lose the order near a border).

Maps have the sizes of a 640-pixel detector's; token counts, heads, widths,
context lengths and vocabularies are generic.
"""
import math

import torch

own = False

KINDS = ("rotary", "cross", "write", "cache", "verify")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
TOP = 448.0  # the largest e4m3 value


def listed():
    return [
        # One serving step's queries and keys, three axes over the frequencies of one table: latency.
        {"name": "rotary_step", "kind": "rotary", "type": "bf16", "b": 64, "t": 1, "h": 32, "hk": 8, "d": 128, "axes": 3, "rotated": 128, "pairs": "halves"},
        # The 80 x 80 tokens of a batch of maps, two axes with frequencies of their own, adjacent pairs.
        {"name": "rotary_map", "kind": "rotary", "type": "fp16", "b": 8, "t": 6400, "h": 16, "hk": 16, "d": 64, "axes": 2, "rotated": 64, "pairs": "adjacent"},
        # 300 object queries to the 8400 tokens of three maps, padded images masked.
        {"name": "cross_queries", "kind": "cross", "type": "fp16", "b": 8, "t": 300, "s": 8400, "h": 8, "hk": 8, "d": 32, "masked": "mask"},
        # One token of each of 64 answers to its own 1500 states at most.
        {"name": "cross_step", "kind": "cross", "type": "bf16", "b": 64, "t": 1, "s": 1500, "h": 16, "hk": 16, "d": 64, "masked": "lengths"},
        # Prompts to long states, shared heads: the largest products.
        {"name": "cross_prompt", "kind": "cross", "type": "bf16", "b": 4, "t": 2048, "s": 4096, "h": 32, "hk": 8, "d": 128, "masked": "none"},
        # One token and four drafts of 48 answers into their pages.
        {"name": "write_step", "kind": "write", "type": "bf16", "b": 48, "t": 5, "hk": 8, "d": 128, "page": 64, "len": 1000, "ragged": False},
        # Prompts of up to 2048 tokens into pages, ragged.
        {"name": "write_prompt", "kind": "write", "type": "fp16", "b": 6, "t": 2048, "hk": 8, "d": 128, "page": 32, "len": 2500, "ragged": True},
        # One token of a serving batch over contexts of up to 8192.
        {"name": "cache_step", "kind": "cache", "type": "bf16", "b": 32, "t": 1, "h": 32, "hk": 8, "d": 128, "page": 64, "len": 8192, "ragged": False},
        # A token and up to five drafts of two long contexts, small pages.
        {"name": "cache_drafts", "kind": "cache", "type": "fp16", "b": 2, "t": 6, "h": 20, "hk": 4, "d": 128, "page": 16, "len": 60001, "ragged": True},
        # Chunks of prompts behind a cached beginning.
        {"name": "cache_prompt", "kind": "cache", "type": "bf16", "b": 3, "t": 1024, "h": 24, "hk": 4, "d": 64, "page": 32, "len": 8000, "ragged": True},
        # Four drafts of each of 48 answers.
        {"name": "verify_step", "kind": "verify", "type": "fp32", "b": 48, "k": 4, "v": 128000, "draft": True},
        # Two answers whose drafts come without probabilities, a ragged vocabulary.
        {"name": "verify_few", "kind": "verify", "type": "fp16", "b": 2, "k": 7, "v": 50001, "draft": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    hk = rng.choice([1, 2, 3, 4, 8, 8, 16])
    return hk * rng.choice([1, 1, 2, 3, 4, 5, 8]), hk


def draw(rng):
    kind = rng.choice(KINDS)
    half = rng.choice(["fp16", "bf16"])
    h, hk = _heads(rng)
    if kind == "rotary":
        while True:
            d = 2 * _log(rng, 8, 128)
            axes = rng.randint(1, 3)
            rotated = rng.choice([d, d, d // 4 * 2])
            c = {"kind": kind, "type": rng.choice([half, half, "fp32"]), "b": _log(rng, 1, 32), "t": _log(rng, 1, 20000), "h": h, "hk": hk, "d": d,
                 "axes": axes, "rotated": rotated, "pairs": rng.choice(["halves", "adjacent"])}
            if rotated >= 2 * axes and c["b"] * c["t"] * (h + hk) * d * (2 if c["type"] == "fp32" else 1) <= 8 * 6400 * 32 * 64:
                return c
    if kind == "cross":
        while True:
            d = 8 * _log(rng, 2, 32)
            c = {"kind": kind, "type": half, "b": _log(rng, 1, 64), "t": rng.choice([1, _log(rng, 1, 4096)]), "s": _log(rng, 1, 20000), "h": h, "hk": hk, "d": d,
                 "masked": rng.choice(["none", "lengths", "mask"])}
            if c["b"] * h * c["t"] * c["s"] <= 4 * 32 * 2048 * 4096 // 2 and c["b"] * h * c["t"] * c["s"] * d <= 4 * 32 * 2048 * 4096 * 128 // 2 and c["b"] * c["s"] * hk * d <= 1 << 27:
                return c
    if kind in ("write", "cache"):
        while True:
            d, length = 16 * _log(rng, 2, 16), _log(rng, 2, 20000)
            c = {"kind": kind, "type": half, "b": _log(rng, 1, 64), "t": min(length, rng.choice([1, rng.randint(2, 8), _log(rng, 2, 2048)])), "hk": hk, "d": d,
                 "page": rng.choice([16, 32, 48, 64, 128]), "len": length, "ragged": rng.random() < 0.5}
            if kind == "cache":
                c["h"] = h
            tokens = c["b"] * length * hk * d
            if kind == "write" and tokens <= 6 * 2500 * 8 * 128 and c["b"] * c["t"] * hk * d <= 6 * 2048 * 8 * 128:
                return c
            if kind == "cache" and tokens <= 32 * 8192 * 8 * 128 // 2 and c["b"] * h * c["t"] * length <= 3 * 24 * 1024 * 8000 // 2:
                return c
    while True:
        c = {"kind": kind, "type": rng.choice(["fp32", "fp32", half]), "b": _log(rng, 1, 128), "k": rng.randint(1, 8), "v": _log(rng, 2, 200000), "draft": rng.random() < 0.7}
        if c["b"] * (c["k"] + 1) * c["v"] <= 48 * 5 * 128000:
            return c


# ------------------------------------------------------------------ inputs

def _tables(case):
    """(freqs, axes): the frequency and the axis of each rotated pair."""
    pairs, n = case["rotated"] // 2, case["axes"]
    parts = [pairs // n + (1 if i < pairs % n else 0) for i in range(n)]
    axes = torch.tensor([a for a, p in enumerate(parts) for _ in range(p)], dtype=torch.int32, device="cuda")
    if case["pairs"] == "halves":  # one run of frequencies over all axes
        steps = [i / pairs for i in range(pairs)]
    else:  # each axis with frequencies of its own
        steps = [i / p for p in parts for i in range(p)]
    return torch.tensor([10000.0 ** -s for s in steps], dtype=torch.float64).float().cuda(), axes


def _paged(values, page):
    """(codes, scales) of [pages, heads, page, d] values."""
    amax = values.abs().amax((2, 3))
    scales = _scale_of(amax)
    return (values / scales[..., None, None]).to(E4M3), scales


def _scale_of(amax):
    """2^e, the least with amax <= 448 * 2^e (exact: 448 = 0.875 * 2^9); 1 for 0."""
    mantissa, exponent = torch.frexp(amax)
    e = exponent - 9 + (mantissa > 0.875).int()
    return torch.where(amax == 0, torch.ones_like(amax), ((e + 127) << 23).view(torch.float32))


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["type"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * std

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=gen, device="cuda", dtype=torch.int32)

    kind = case["kind"]
    if kind == "rotary":  # positions of a map's tokens, or of tokens far into a context
        b, t = case["b"], case["t"]
        width = max(1, int(math.sqrt(t)))
        index = torch.arange(t, device="cuda", dtype=torch.int32)
        grid = torch.stack([index // width, index % width, index // (width * 4)][:case["axes"]])
        positions = grid[:, None, :] + whole(0, 100000, case["axes"], b, 1)
        freqs, axes = _tables(case)
        return {"q": normal(b, t, case["h"], case["d"]).to(dtype), "k": normal(b, t, case["hk"], case["d"]).to(dtype),
                "positions": positions, "freqs": freqs, "axes": axes}
    if kind == "cross":
        b, t, s, d = case["b"], case["t"], case["s"], case["d"]
        data = {"q": normal(b, t, case["h"], d, std=1.5).to(dtype), "k": (normal(b, s, case["hk"], d) + normal(case["hk"], d, std=0.5)).to(dtype),
                "v": normal(b, s, case["hk"], d).to(dtype), "lengths": None, "mask": None}
        if case["masked"] == "lengths":
            data["lengths"] = whole(max(1, s // 4), s + 1, b)
        elif case["masked"] == "mask":  # the left columns of each map are image
            width = min(s, 80)
            data["mask"] = (torch.arange(s, device="cuda", dtype=torch.int32) % width)[None] < whole(max(1, width // 2), width + 1, b, 1)
        return data
    if kind in ("write", "cache"):
        b, t, hk, d, page = case["b"], case["t"], case["hk"], case["d"], case["page"]
        per = -(-case["len"] // page)
        pages = b * per + 3
        spread = normal(hk, d).abs() + 0.3  # channels of unequal size
        stored = {}
        for name in ("k", "v"):
            stored[name + "_cache"], stored[name + "_scales"] = _paged((normal(pages, hk, page, d) * spread[:, None]), page)
        table = torch.randperm(pages, generator=gen, device="cuda")[:b * per].view(b, per).int()
        counts = whole(1, t + 1, b) if case["ragged"] else torch.full((b,), t, dtype=torch.int32, device="cuda")
        lengths = whole(max(t, case["len"] // 4), case["len"] + 1, b)
        counts[0], lengths[0] = t, case["len"]
        data = {**stored, "table": table, "lengths": lengths, "counts": counts if case["ragged"] else None}
        if kind == "write":
            grown = torch.exp2(normal(b, t, 1, 1, std=0.7))  # now and then a token larger than its page's
            data["k"], data["v"] = ((normal(b, t, hk, d) * spread * grown).to(dtype) for _ in range(2))
        else:
            data["q"] = normal(b, t, case["h"], d, std=1.5).to(dtype)
        return data
    b, k, v = case["b"], case["k"], case["v"]  # a target and a draft model that mostly agree
    logits = normal(b, k + 1, v, std=2.0)
    likely = torch.randint(0, v, (b, k + 1, 8), generator=gen, device="cuda")
    logits.scatter_(2, likely, 8.0 + 5.0 * torch.rand((b, k + 1, 8), generator=gen, device="cuda"))
    target = torch.softmax(logits, 2).to(dtype)
    near = logits[:, :k] + normal(b, k, v, std=0.5)
    guess = torch.softmax(near, 2)
    drawn = torch.rand((b, k, 1), generator=gen, device="cuda", dtype=torch.float64)
    tokens = (guess.double().cumsum(2) < drawn).sum(2).clamp(max=v - 1)
    return {"target": target, "draft": guess.to(dtype) if case["draft"] else None, "tokens": tokens,
            "accept": torch.rand((b, k), generator=gen, device="cuda"), "sample": torch.rand((b,), generator=gen, device="cuda")}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ------------------------------------------------------------------ calls

def run(state):
    return (_own if own else _plain)(state)


def _own(state):
    from thintnpu_amd import capi
    case = state["case"]
    kind = case["kind"]
    if kind == "rotary":
        return capi.rotary_axes(state["q"], state["positions"], state["freqs"], state["axes"], k=state["k"], interleaved=case["pairs"] == "adjacent")
    if kind == "cross":
        return capi.cross_attention(state["q"], state["k"], state["v"], lengths=state["lengths"], mask=state["mask"])
    cache = [state.get(n) for n in ("k_cache", "v_cache", "k_scales", "v_scales", "table", "lengths")]
    if kind == "write":
        capi.cache_write(state["k"], state["v"], *cache, counts=state["counts"])
        return cache[:4]
    if kind == "cache":
        return capi.cache_attention(state["q"], *cache, counts=state["counts"])
    return capi.verify_drafts(state["target"], state["draft"], state["tokens"], state["accept"], state["sample"])


def _plain(state):
    return {"rotary": _plain_rotary, "cross": _plain_cross, "write": _plain_write, "cache": _plain_cache, "verify": _plain_verify}[state["case"]["kind"]](state)


def _plain_rotary(state):
    case = state["case"]
    p = case["rotated"] // 2
    angle = state["positions"][state["axes"].long()].permute(1, 2, 0).double() * state["freqs"].double()
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]

    def turn(x):
        f = x.float()
        r = f[..., :2 * p]
        if case["pairs"] == "halves":
            first, second = r[..., :p], r[..., p:]
            turned = torch.cat([first * cos - second * sin, second * cos + first * sin], -1)
        else:
            first, second = r[..., 0::2], r[..., 1::2]
            turned = torch.stack([first * cos - second * sin, second * cos + first * sin], -1).flatten(-2)
        return torch.cat([turned, f[..., 2 * p:]], -1).to(x.dtype)

    return turn(state["q"]), turn(state["k"])


def _attend(q, k, v, seen, dtype):
    """q [b, t, h, d], k and v [b, hk, s, d] and seen [b, 1 or t, s] -> [b, t, h, d]."""
    b, t, h, d = q.shape
    hk, s = k.shape[1], k.shape[2]
    rows = q.float().view(b, t, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    scores = torch.matmul(rows, k.transpose(2, 3)) / math.sqrt(d)
    scores = scores.view(b, hk, h // hk, t, s)
    if seen is not None:
        scores = torch.where(seen[:, None, None], scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.view(b, hk, -1, s), v).view(b, hk, h // hk, t, d)
    out = torch.where(total == 0, torch.zeros_like(out), out / total)
    return out.permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(dtype)


def _plain_cross(state):
    s = state["case"]["s"]
    seen = None
    if state["lengths"] is not None:
        seen = (torch.arange(s, device="cuda") < state["lengths"][:, None])[:, None]
    elif state["mask"] is not None:
        seen = state["mask"][:, None]
    k, v = state["k"].float().permute(0, 2, 1, 3), state["v"].float().permute(0, 2, 1, 3)
    return _attend(state["q"], k.contiguous(), v.contiguous(), seen, state["q"].dtype)


def _counts(state):
    return state["counts"] if state["counts"] is not None else torch.full_like(state["lengths"], state["case"]["t"])


def _plain_cache(state):
    case, table = state["case"], state["table"].long()
    counts = _counts(state)
    b, t, hk, d = case["b"], case["t"], case["hk"], case["d"]

    def gathered(name):
        x = state[name + "_cache"].view(torch.uint8)[table].view(E4M3).float() * state[name + "_scales"][table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)

    k, v = gathered("k"), gathered("v")
    row = torch.arange(t, device="cuda")
    limit = (state["lengths"] - counts)[:, None] + row + 1
    limit = torch.where(row < counts[:, None], limit, torch.zeros_like(limit))
    return _attend(state["q"], k, v, torch.arange(k.shape[2], device="cuda") < limit[..., None], state["q"].dtype)


def _plain_write(state):
    case = state["case"]
    b, t, page = case["b"], case["t"], case["page"]
    counts = _counts(state)
    begin = (state["lengths"] - counts).long()
    spans = (t + page - 2) // page + 1
    first = begin // page
    slot = first[:, None] + torch.arange(spans, device="cuda")
    place = slot[..., None] * page + torch.arange(page, device="cuda")  # [b, spans, page]
    token = place - begin[:, None, None]
    new = (token >= 0) & (token < counts[:, None, None])
    old = token < 0
    touched = new.any(2)
    ids = state["table"].long().gather(1, slot.clamp(max=state["table"].shape[1] - 1))
    ids, new, old, token = ids[touched], new[touched], old[touched], token[touched]
    owner = torch.arange(b, device="cuda")[:, None].expand(b, spans)[touched]
    for name in ("k", "v"):
        x = state[name].float()[owner[:, None], token.clamp(0, t - 1)].permute(0, 2, 1, 3)  # [n, heads, page, d]
        fresh = new[:, None, :, None]
        amax = torch.where(fresh, x.abs(), torch.zeros_like(x)).amax((2, 3))
        before = state[name + "_scales"][ids]
        scale = _scale_of(amax)
        scale = torch.where(old.any(1)[:, None], torch.maximum(before, torch.where(amax == 0, torch.zeros_like(scale), scale)), scale)
        there = state[name + "_cache"].view(torch.uint8)[ids]
        moved = (there.view(E4M3).float() * before[..., None, None] / scale[..., None, None]).to(E4M3).view(torch.uint8)
        codes = (x / scale[..., None, None]).clamp(-TOP, TOP).to(E4M3).view(torch.uint8)
        state[name + "_cache"].view(torch.uint8)[ids] = torch.where(fresh, codes, torch.where(old[:, None, :, None], moved, there))
        state[name + "_scales"][ids] = scale
    return [state[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales")]


def _plain_verify(state):
    target, draft, tokens = state["target"], state["draft"], state["tokens"]
    b, k = tokens.shape
    v = target.shape[2]
    p = target[:, :k].gather(2, tokens[..., None])[..., 0].double()
    q = draft.gather(2, tokens[..., None])[..., 0].double() if draft is not None else torch.ones_like(p)
    taken = (state["accept"].double() * q < p).long().cumprod(1).sum(1)
    row = target.gather(1, taken[:, None, None].expand(b, 1, v))[:, 0].double()
    refused = taken < k
    at = taken.clamp(max=k - 1)
    if draft is not None:
        other = draft.gather(1, at[:, None, None].expand(b, 1, v))[:, 0].double()
    else:  # certain of its token
        other = torch.zeros_like(row).scatter_(1, tokens.gather(1, at[:, None]), math.inf)
    rest = torch.where(refused[:, None], (row - other).clamp(min=0), row)
    rest = torch.where((rest.sum(1) > 0)[:, None], rest, row)
    edge = state["sample"].double() * rest.sum(1)
    total = rest.cumsum(1)
    found = ((total <= edge[:, None]) & (torch.arange(v, device="cuda") < v - 1)).sum(1)
    place = torch.arange(k + 1, device="cuda")
    given = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(place < taken[:, None], given, torch.where(place == taken[:, None], found[:, None], torch.full_like(given, -1)))
    return out, taken.int()


# ------------------------------------------------------------------ work

def work(case):
    size = 4 if case["type"] == "fp32" else 2
    kind = case["kind"]
    if kind == "rotary":
        b, t, h = case["b"], case["t"], case["h"] + case["hk"]
        return {"bytes": 2 * b * t * h * case["d"] * size + case["axes"] * b * t * 4, "flops": 3 * b * t * h * case["rotated"]}
    if kind == "cross":
        b, t, s, h, d = case["b"], case["t"], case["s"], case["h"], case["d"]
        share = {"none": 1.0, "lengths": 0.625, "mask": 0.75}[case["masked"]] if s > 1 else 1.0
        return {"bytes": 2 * b * t * h * d * size + 2 * b * s * share * case["hk"] * d * size, "flops": 4 * b * h * t * s * share * d}
    if kind == "write":
        n = case["b"] * case["t"] * case["hk"] * case["d"] * (0.5 if case["ragged"] else 1.0)
        return {"bytes": 2 * n * (size + 1), "flops": 4 * n}
    if kind == "cache":
        b, t, h, d = case["b"], case["t"], case["h"], case["d"]
        live = 0.625 * b * case["len"] + 0.375 * case["len"]
        tokens = t * (0.5 if case["ragged"] and t > 1 else 1.0)
        return {"bytes": 2 * live * case["hk"] * d + 2 * b * t * h * d * size, "flops": 4 * live * tokens * h * d}
    return {"bytes": case["b"] * case["v"] * size * (2 if case["draft"] else 1), "flops": case["b"] * case["v"] * 3}


# ------------------------------------------------------------------ exact

def exact(case, seed):
    """The outputs of `run` from the definitions in 64 bits, one sample, page or
    rank at a time where the plain form works on whole tensors."""
    data = _inputs(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _exact_rotary(case, data)
    if kind == "cross":
        out = []
        for i in range(case["b"]):
            seen = torch.ones(case["s"], dtype=torch.bool, device="cuda")
            if data["mask"] is not None:
                seen = data["mask"][i]
            if data["lengths"] is not None:
                seen = torch.arange(case["s"], device="cuda") < data["lengths"][i]
            out.append(_exact_heads(data["q"][i], data["k"][i][seen].double(), data["v"][i][seen].double(), None))
        return torch.stack(out)
    if kind == "cache":
        out = []
        for i in range(case["b"]):
            length, t = int(data["lengths"][i]), case["t"]
            n = t if data["counts"] is None else int(data["counts"][i])
            pages = data["table"][i, :-(-length // case["page"])].tolist()
            k, v = (torch.cat([data[x + "_cache"][j].double() * data[x + "_scales"][j].double()[:, None, None] for j in pages], 1).transpose(0, 1)[:length] for x in "kv")
            part = _exact_heads(data["q"][i, :n], k, v, length - n)
            out.append(torch.cat([part, part.new_zeros(t - n, *part.shape[1:])]))
        return torch.stack(out)
    if kind == "write":
        return _exact_write(case, data)
    return _exact_verify(case, data)


def _exact_rotary(case, data):
    p = case["rotated"] // 2
    outs = []
    for x in (data["q"], data["k"]):
        y = x.double()
        z = y.clone()
        for i in range(p):
            one, two = (i, i + p) if case["pairs"] == "halves" else (2 * i, 2 * i + 1)
            angle = (data["positions"][int(data["axes"][i])].double() * float(data["freqs"][i]))[..., None]
            z[..., one] = y[..., one] * torch.cos(angle) - y[..., two] * torch.sin(angle)
            z[..., two] = y[..., one] * torch.sin(angle) + y[..., two] * torch.cos(angle)
        outs.append(z)
    return tuple(outs)


def _exact_heads(q, k, v, before):
    """q [t, h, d] over k, v [s, hk, d]; query i sees before + i + 1 keys (all for None)."""
    t, h, d = q.shape
    per = h // k.shape[1]
    out = torch.zeros((t, h, d), dtype=torch.float64, device="cuda")
    for j in range(h):
        s = q[:, j].double() @ k[:, j // per].t() * d ** -0.5
        if before is not None:
            s = s.masked_fill(torch.arange(k.shape[0], device="cuda")[None] > before + torch.arange(t, device="cuda")[:, None], -math.inf)
        if k.shape[0]:
            out[:, j] = torch.softmax(s, 1) @ v[:, j // per]
    return out


def _power(exponent):
    """2^exponent in 64 bits."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(x):
    """The nearest e4m3 value, ties to the even one (steps of 2^(e-3), e >= -6)."""
    exponent = (torch.frexp(x.abs())[1] - 1).clamp(min=-6)
    step = _power(exponent - 3)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def _exact_write(case, data):
    outs = [data["k_cache"].double(), data["v_cache"].double(), data["k_scales"].double(), data["v_scales"].double()]
    page = case["page"]
    for i in range(case["b"]):
        n = case["t"] if data["counts"] is None else int(data["counts"][i])
        length = int(data["lengths"][i])
        begin = length - n
        for slot in range(begin // page, -(-length // page)):
            at = int(data["table"][i, slot])
            low, high = max(begin, slot * page), min(length, (slot + 1) * page)
            off = low - slot * page
            for which, name in enumerate("kv"):
                x = data[name][i, low - begin:high - begin].double().transpose(0, 1)
                amax = x.abs().amax((1, 2))
                scale = _power(torch.ceil(torch.log2(amax.clamp(min=1e-30) / TOP)))
                scale = torch.where(amax > TOP * scale, scale * 2, torch.where(amax <= TOP * scale / 2, scale / 2, scale))
                scale = torch.where(amax == 0, torch.ones_like(scale) if off == 0 else torch.zeros_like(scale), scale)
                if off:
                    was = outs[2 + which][at].clone()
                    scale = torch.maximum(scale, was)
                    outs[which][at, :, :off] = _round_e4m3(outs[which][at, :, :off] * (was / scale)[:, None, None])
                outs[which][at, :, off:off + high - low] = _round_e4m3(x / scale[:, None, None])
                outs[2 + which][at] = scale
    return outs


def _exact_verify(case, data):
    b, k, v = case["b"], case["k"], case["v"]
    out, taken = torch.full((b, k + 1), -1, dtype=torch.int64), torch.zeros(b, dtype=torch.int32)
    for i in range(b):
        n = 0
        rest = None
        while n < k:
            x = int(data["tokens"][i, n])
            p = data["target"][i, n].double()
            q = data["draft"][i, n].double() if data["draft"] is not None else torch.nn.functional.one_hot(torch.tensor(x, device="cuda"), v).double()
            if not float(data["accept"][i, n]) * float(q[x]) < float(p[x]):
                rest = torch.relu(p - q)
                if data["draft"] is None:
                    rest[x] = 0.0
                rest = rest if float(rest.sum()) > 0 else p
                break
            out[i, n] = x
            n += 1
        rest = data["target"][i, k].double() if rest is None else rest
        total = torch.cumsum(rest, 0)
        out[i, n] = min(v - 1, int(torch.searchsorted(total, float(data["sample"][i]) * float(rest.sum()), right=True)))
        taken[i] = n
    return out.cuda(), taken.cuda()
