"""The measured work of the expert block and of the scores a model answers with.

Four operators, through the C ABI as `thintnpu_amd.capi` binds it, on torch
device tensors: group norm with an activation (channels last and NC1HWC0),
routing to experts, moving rows to their experts and back (dispatch and
combine), and log probabilities of given tokens with entropy and top
alternatives.  The plain forms are elementary torch operations in 32 bits (64
for long sums and for the choice scores, whose order near a tie 32 bits lose).

Feature maps have the sizes of a 640-pixel detector's layers; token counts,
row lengths, expert counts and vocabularies are generic.
"""
import math

import torch

own = False

KINDS = ("norm", "route", "dispatch", "combine", "logprobs")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # One frame's feature map between two convolutions in the blocked layout: a small
        # call, where the launch and the host's share count.
        {"name": "norm_frame", "kind": "norm", "layout": "blocked", "type": "fp16", "n": 1, "h": 80, "w": 80, "c": 128, "g": 32, "silu": True, "half": False},
        # The neck's maps of a batch, channels last.
        {"name": "norm_batch", "kind": "norm", "layout": "last", "type": "fp16", "n": 32, "h": 80, "w": 80, "c": 128, "g": 32, "silu": True, "half": False},
        # Token rows of a residual stream without an activation, the half of a wider
        # tensor's channels (as a split leaves them), groups of an odd number of channels.
        {"name": "norm_half", "kind": "norm", "layout": "last", "type": "bf16", "n": 5, "h": 61, "w": 83, "c": 648, "g": 24, "silu": False, "half": True},
        # One step of a serving batch through a router with a bias for balance and groups.
        {"name": "route_step", "kind": "route", "type": "bf16", "t": 48, "e": 256, "k": 8, "scores": "sigmoid", "bias": True, "groups": 8, "top": 4},
        # Prompts through the same router, its logits in 32 bits.
        {"name": "route_prompt", "kind": "route", "type": "fp32", "t": 16384, "e": 256, "k": 8, "scores": "sigmoid", "bias": True, "groups": 8, "top": 4},
        # Softmax routing of a feature map's pixels to few experts.
        {"name": "route_pixels", "kind": "route", "type": "fp16", "t": 51200, "e": 60, "k": 4, "scores": "softmax", "bias": False, "groups": 1, "top": 1},
        # Rows of one serving step to their experts.
        {"name": "dispatch_step", "kind": "dispatch", "type": "bf16", "t": 48, "e": 256, "k": 8, "hidden": 4096},
        # Rows of prompts to their experts: the largest movement.
        {"name": "dispatch_prompt", "kind": "dispatch", "type": "bf16", "t": 16384, "e": 256, "k": 8, "hidden": 2048},
        # The weighted sum of the experts' rows, one step and prompts.
        {"name": "combine_step", "kind": "combine", "type": "bf16", "t": 48, "e": 256, "k": 8, "hidden": 4096},
        {"name": "combine_prompt", "kind": "combine", "type": "fp16", "t": 16384, "e": 256, "k": 8, "hidden": 2048},
        # What a server returns with each sampled token: its log probability, the
        # entropy and twenty alternatives, for one step's rows.
        {"name": "logprobs_step", "kind": "logprobs", "type": "bf16", "r": 48, "v": 128000, "top": 20},
        # Scoring of a prompt (ragged vocabulary).
        {"name": "logprobs_prompt", "kind": "logprobs", "type": "fp16", "r": 4001, "v": 50001, "top": 5},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(KINDS)
    dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"])
    if kind == "norm":
        while True:
            layout = rng.choice(["last", "blocked"])
            per, g = _log(rng, 1, 64), rng.choice([1, 2, 4, 8, 16, 24, 32, 32, 48])
            c = {"kind": kind, "layout": layout, "type": dtype, "n": _log(rng, 1, 32), "h": _log(rng, 1, 160), "w": _log(rng, 1, 160),
                 "c": per * g, "g": g, "silu": rng.random() < 0.7, "half": rng.random() < 0.3}
            if c["c"] <= 2048 and c["n"] * c["h"] * c["w"] * (c["c"] + 15) * (2 if dtype == "fp32" else 1) <= 32 * 80 * 80 * 128:
                return c
    if kind == "route":
        while True:
            e = _log(rng, 4, 512)
            groups = rng.choice([v for v in (1, 1, 2, 4, 8, 16) if e % v == 0])
            top = rng.randint(1, groups)
            c = {"kind": kind, "type": dtype, "t": _log(rng, 1, 32768), "e": e, "k": rng.randint(1, min(16, e // groups * top)),
                 "scores": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups, "top": top}
            if c["t"] * e <= 16384 * 256:
                return c
    if kind in ("dispatch", "combine"):
        while True:
            e = _log(rng, 4, 512)
            c = {"kind": kind, "type": dtype, "t": _log(rng, 1, 32768), "e": e, "k": rng.randint(1, min(8, e)), "hidden": _log(rng, 64, 8192)}
            if c["t"] * c["k"] * c["hidden"] * (2 if dtype == "fp32" else 1) <= 16384 * 8 * 2048:
                return c
    while True:
        c = {"kind": "logprobs", "type": dtype, "r": _log(rng, 1, 70000), "v": _log(rng, 2, 200000), "top": rng.choice([0, 1, 5, 20, rng.randint(0, 32)])}
        c["top"] = min(c["top"], c["v"])
        if c["r"] * c["v"] * (2 if dtype == "fp32" else 1) <= 4001 * 50001:
            return c


# ------------------------------------------------------------------ inputs

def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["type"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * std

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    kind = case["kind"]
    if kind == "norm":  # a convolution's output: every channel with a mean and a spread of its own
        n, h, w, c = case["n"], case["h"], case["w"], case["c"]
        x = (normal(n, h, w, c) * (uniform(c) + 0.5) + normal(c, std=0.5)).to(dtype)
        weight, bias = (uniform(c) + 0.5).to(dtype), normal(c, std=0.2).to(dtype)
        if case["layout"] == "blocked":
            c1 = (c + 15) // 16
            full = torch.zeros((n, h, w, c1 * 16), dtype=dtype, device="cuda")
            full[..., :c] = x
            x = full.view(n, h, w, c1, 16).permute(0, 3, 1, 2, 4).contiguous()
        if case["half"]:  # the second half of a tensor of twice the channels
            x = torch.cat([x, x], 1 if case["layout"] == "blocked" else 3).chunk(2, 1 if case["layout"] == "blocked" else 3)[1]
        return {"x": x, "weight": weight, "bias": bias}
    if kind == "route":  # some experts are asked for more often than others
        t, e = case["t"], case["e"]
        logits = (normal(t, e, std=1.5) + normal(e, std=0.5)).to(dtype)
        return {"logits": logits, "bias": normal(e, std=0.05) if case["bias"] else None}
    if kind in ("dispatch", "combine"):
        t, e, k, hidden = case["t"], case["e"], case["k"], case["hidden"]
        experts = (normal(t, e) + normal(e, std=0.7)).topk(k, 1).indices.int()
        if kind == "dispatch":
            return {"x": normal(t, hidden).to(dtype), "experts": experts}
        weights = uniform(t, k) + 0.1
        slots = _places(experts, e)[0]
        return {"y": normal(t * k, hidden).to(dtype), "weights": weights / weights.sum(1, keepdim=True), "slots": slots}
    r, v = case["r"], case["v"]  # scores with a few likely tokens; half of the tokens given are the likeliest
    logits = normal(r, v, std=2.0)
    likely = torch.randint(0, v, (r, 8), generator=gen, device="cuda")
    logits.scatter_(1, likely, 6.0 + 5.0 * uniform(r, 8))
    logits = logits.to(dtype)
    tokens = torch.where(uniform(r) < 0.5, logits.argmax(1), torch.randint(0, v, (r,), generator=gen, device="cuda"))
    return {"logits": logits, "tokens": tokens}


def prepare(case, seed):
    return {"case": case, **_inputs(case, seed)}


# ------------------------------------------------------------------ calls

def run(state):
    return (_own if own else _plain)(state)


def _own(state):
    from thintnpu_amd import capi
    case = state["case"]
    kind = case["kind"]
    if kind == "norm":
        if case["layout"] == "blocked":
            return capi.group_norm_nc1hwc0(state["x"], case["g"], state["weight"], state["bias"], eps=EPS, silu=case["silu"], channels=case["c"])
        return capi.group_norm(state["x"], case["g"], state["weight"], state["bias"], eps=EPS, silu=case["silu"])
    if kind == "route":
        return capi.expert_route(state["logits"], case["k"], bias=state["bias"], scores=case["scores"], groups=case["groups"], top_groups=case["top"], scale=2.5)
    if kind == "dispatch":
        return capi.expert_dispatch(state["x"], state["experts"], case["e"])
    if kind == "combine":
        return capi.expert_combine(state["y"], state["weights"], state["slots"])
    return capi.token_logprobs(state["logits"], state["tokens"], top=case["top"])


def _plain(state):
    return {"norm": _plain_norm, "route": _plain_route, "dispatch": _plain_dispatch, "combine": _plain_combine, "logprobs": _plain_logprobs}[state["case"]["kind"]](state)


def _plain_norm(state):
    case, x = state["case"], state["x"]
    n, h, w, c, g = case["n"], case["h"], case["w"], case["c"], case["g"]
    blocked = case["layout"] == "blocked"
    v = x.float()
    if blocked:
        v = v.permute(0, 2, 3, 1, 4).reshape(n, h, w, -1)[..., :c]
    v = v.reshape(n, h * w, g, c // g)
    mean = v.mean((1, 3), keepdim=True)
    d = v - mean
    var = (d * d).mean((1, 3), keepdim=True)
    y = (d / torch.sqrt(var + EPS)).reshape(n, h, w, c) * state["weight"].float() + state["bias"].float()
    if case["silu"]:
        y = y / (1.0 + torch.exp(-y))
    y = y.to(x.dtype)
    if blocked:
        full = torch.zeros((n, h, w, x.shape[1] * 16), dtype=x.dtype, device=x.device)
        full[..., :c] = y
        y = full.view(n, h, w, -1, 16).permute(0, 3, 1, 2, 4).contiguous()
    return y


def _plain_route(state):
    case, logits = state["case"], state["logits"]
    t, e, k, groups = case["t"], case["e"], case["k"], case["groups"]
    # choice scores in 64 bits: their order decides; without a bias it is that of the logits
    x = logits.double()
    if case["scores"] == "softmax":
        ex = torch.exp(x - x.amax(1, keepdim=True))
        s = ex / ex.sum(1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-x))
    choice = s + state["bias"].double() if case["bias"] else x
    if case["top"] < groups:
        parts = choice.view(t, groups, e // groups)
        best = parts.sort(dim=2, descending=True, stable=True).values
        score = best[..., :2].sum(2) if case["bias"] else best[..., 0]
        kept = score.sort(dim=1, descending=True, stable=True).indices[:, :case["top"]]
        mask = torch.zeros((t, groups), dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        choice = torch.where(mask.repeat_interleave(e // groups, 1), choice, torch.full_like(choice, -math.inf))
    experts = choice.sort(dim=1, descending=True, stable=True).indices[:, :k]
    weights = s.gather(1, experts)
    weights = weights / weights.sum(1, keepdim=True) * 2.5
    return weights.float(), experts.int()


def _places(experts, e):
    """Slot of each assignment in the order (expert, assignment), and that order."""
    flat = experts.reshape(-1).long()
    order = flat.sort(stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=order.device)
    return slots.view(experts.shape).int(), order


def _plain_dispatch(state):
    case, experts = state["case"], state["experts"]
    slots, order = _places(experts, case["e"])
    counts = torch.zeros(case["e"], dtype=torch.int64, device=experts.device)
    counts.scatter_add_(0, experts.reshape(-1).long(), torch.ones_like(order))
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    return state["x"][order // case["k"]], offsets, slots


def _plain_combine(state):
    y, weights, slots = state["y"], state["weights"], state["slots"]
    rows = y[slots.reshape(-1).long()].view(*slots.shape, -1).float()
    return (rows * weights[..., None]).sum(1).to(y.dtype)


def _order_keys(values):
    """Whole numbers in the order of float32 values, the lower index first among equals."""
    bits = (values + 0.0).view(torch.int32)
    bits = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    return bits * 2 ** 32 + (2 ** 31 - torch.arange(values.shape[-1], device=values.device))


def _plain_logprobs(state):
    case, x = state["case"], state["logits"].float()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, dtype=torch.float64)
    lse = top[:, 0].double() + torch.log(total)
    mean = (e * (x - top)).sum(1, dtype=torch.float64) / total
    entropy = torch.log(total) - mean
    token = x.gather(1, state["tokens"][:, None])[:, 0].double() - lse
    ids = _order_keys(x).topk(case["top"], 1).indices
    alternatives = x.gather(1, ids).double() - lse[:, None]
    return token.float(), entropy.float(), alternatives.float(), ids


# ------------------------------------------------------------------ work

def work(case):
    size = 4 if case["type"] == "fp32" else 2
    kind = case["kind"]
    if kind == "norm":
        c = case["c"] if case["layout"] == "last" else (case["c"] + 15) // 16 * 16
        elements = case["n"] * case["h"] * case["w"] * c
        return {"bytes": 2 * elements * size + 2 * case["c"] * size, "flops": elements * (12 if case["silu"] else 7)}
    if kind == "route":
        t, e, k = case["t"], case["e"], case["k"]
        return {"bytes": t * e * size + t * k * 8 + (e * 4 if case["bias"] else 0), "flops": t * e * 6}
    if kind == "dispatch":
        t, e, k, hidden = case["t"], case["e"], case["k"], case["hidden"]
        return {"bytes": t * hidden * size * (1 + k) + t * k * 8 + (e + 1) * 4, "flops": t * k}
    if kind == "combine":
        t, k, hidden = case["t"], case["k"], case["hidden"]
        return {"bytes": t * hidden * size * (1 + k) + t * k * 8, "flops": 2 * t * k * hidden}
    r, v, top = case["r"], case["v"], case["top"]
    return {"bytes": r * v * size + r * 16 + r * top * 12, "flops": r * v * 6}


# ------------------------------------------------------------------ exact

def exact(case, seed):
    """The outputs of `run` from the definitions in 64 bits, one sample, group or
    rank at a time where the plain form works on whole tensors."""
    data = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        return _exact_norm(case, data)
    if kind == "route":
        return _exact_route(case, data)
    if kind == "dispatch":
        return _exact_dispatch(case, data)
    if kind == "combine":
        out = torch.zeros((case["t"], case["hidden"]), dtype=torch.float64, device="cuda")
        for j in range(case["k"]):
            out += data["weights"][:, j:j + 1].double() * data["y"].index_select(0, data["slots"][:, j].long()).double()
        return out
    rows = max(1, (1 << 26) // case["v"])
    parts = [_exact_logprobs(data["logits"][i:i + rows].double(), data["tokens"][i:i + rows], case["top"]) for i in range(0, case["r"], rows)]
    return tuple(torch.cat(p) for p in zip(*parts))


def _exact_norm(case, data):
    n, h, w, c, g = case["n"], case["h"], case["w"], case["c"], case["g"]
    x = data["x"]
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for i in range(n):
        if case["layout"] == "blocked":
            v = x[i].double().permute(1, 2, 0, 3).reshape(h * w, -1)[:, :c]
        else:
            v = x[i].double().reshape(h * w, c)
        v = v.reshape(h * w, g, c // g).transpose(0, 1).reshape(g, -1)
        var, mean = torch.var_mean(v, 1, correction=0, keepdim=True)
        y = ((v - mean) * torch.rsqrt(var + EPS)).view(g, h * w, c // g).transpose(0, 1).reshape(h * w, c)
        y = y * data["weight"].double() + data["bias"].double()
        if case["silu"]:
            y = y * torch.sigmoid(y)
        if case["layout"] == "blocked":
            full = torch.zeros((h * w, x.shape[1] * 16), dtype=torch.float64, device="cuda")
            full[:, :c] = y
            out[i] = full.view(h, w, -1, 16).permute(2, 0, 1, 3)
        else:
            out[i] = y.view(h, w, c)
    return out


def _exact_route(case, data):
    t, e, groups = case["t"], case["e"], case["groups"]
    x = data["logits"].double()
    s = torch.softmax(x, 1) if case["scores"] == "softmax" else torch.sigmoid(x)
    choice = s + data["bias"].double() if case["bias"] else x
    size = e // groups
    kept = torch.ones((t, groups), dtype=torch.bool, device="cuda")
    if case["top"] < groups:
        score = torch.stack([choice[:, i * size:(i + 1) * size].topk(min(2, size) if case["bias"] else 1, 1).values.sum(1) for i in range(groups)], 1)
        # a group stays if fewer than `top` groups lie before it
        before = (score[:, None, :] > score[:, :, None]).sum(2)
        index = torch.arange(groups, device="cuda")
        before += ((score[:, None, :] == score[:, :, None]) & (index[None, :] < index[:, None])).sum(2)
        kept = before < case["top"]
    left = choice.masked_fill(~kept.repeat_interleave(size, 1), -math.inf)
    chosen = []
    index = torch.arange(e, device="cuda").expand(t, e)
    for _ in range(case["k"]):
        best = left.amax(1, keepdim=True)
        first = torch.where(left == best, index, e).amin(1, keepdim=True)
        chosen.append(first)
        left = left.scatter(1, first, -math.inf)
    experts = torch.cat(chosen, 1)
    weights = s.gather(1, experts)
    return 2.5 * weights / weights.sum(1, keepdim=True), experts


def _exact_dispatch(case, data):
    t, e, k = case["t"], case["e"], case["k"]
    flat = data["experts"].reshape(-1).long()
    slots = torch.full((t * k,), -1, dtype=torch.int64, device="cuda")
    offsets = [0]
    tokens = []
    for i in range(e):
        mine = torch.nonzero(flat == i)[:, 0]
        slots[mine] = offsets[-1] + torch.arange(mine.numel(), device="cuda")
        tokens.append(torch.div(mine, k, rounding_mode="floor"))
        offsets.append(offsets[-1] + mine.numel())
    return data["x"].index_select(0, torch.cat(tokens)).double(), torch.tensor(offsets, device="cuda"), slots.view(t, k)


def _exact_logprobs(x, tokens, top):
    logp = torch.log_softmax(x, 1)
    entropy = -(torch.exp(logp) * logp).sum(1)
    ids = x.sort(dim=1, descending=True, stable=True).indices[:, :top]
    return logp.gather(1, tokens[:, None])[:, 0], entropy, logp.gather(1, ids), ids
