"""Serving operators around the quantised projections of an attention layer: what is measured, and their plain forms.

Between the QKV projection and the output projection of a decoder (or diffusion-transformer) block:

* ``rope``: RMS norm of each query and key head and the position rotation, with one or several position axes;
* ``append``: keys and values written into a paged cache that holds 4-bit codes, and read back from it;
* ``attention``: attention over that cache, for single tokens, a few tokens to verify, and prompts.

A case is a dict of plain values.  ``prepare`` makes its inputs from the seed, ``run`` makes one pass: in elementary torch operations
where ``own`` is false, through the framework's public entry points where it is true.  ``exact`` gives the same outputs
in 64 bits from the definitions.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- cases

def _rope(name, tokens, q_heads, k_heads, dim, **more):
    return {"name": name, "op": "rope", "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "dtype": "bf16", "rotary": dim,
            "axes": 1, "interleaved": False, "norm": True, "first": 0, **more}


def _append(name, tokens, k_heads, dim, **more):
    return {"name": name, "op": "append", "tokens": tokens, "k_heads": k_heads, "dim": dim, "dtype": "bf16", "page": 64, **more}


def _attention(name, batch, context, q_heads, k_heads, dim, **more):
    return {"name": name, "op": "attention", "batch": batch, "context": context, "queries": 1, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "dtype": "bf16", "page": 64, "window": 0, "ragged": 0, **more}


def listed():
    return [
        # one token of one sequence, far into a long context: the q and k heads of a 4096-wide decoder layer
        _rope("rope_token", 1, 32, 8, 128, first=100_000),
        # a prompt of that decoder
        _rope("rope_prompt", 8191, 32, 8, 128),
        # picture and text tokens of a model that reads both: one ladder of frequencies whose pairs belong to time, height, width; no norm
        _rope("rope_sections", 1777, 28, 4, 128, axes=3, norm=False, dtype="fp16", first=5000),
        # the latent tokens of a video in a diffusion transformer: a ladder per axis, neighbouring channels as pairs
        _rope("rope_video", 32_760, 20, 20, 128, axes=3, interleaved=True),
        # one new token for each of 64 sequences
        _append("append_tokens", 64, 8, 128),
        # a long prompt
        _append("append_prompt", 16_001, 8, 128, dtype="fp16"),
        # one sequence, a short context: latency
        _attention("attend_token", 1, 777, 32, 8, 128),
        # a serving batch of unequal lengths
        _attention("attend_batch", 64, 8192, 32, 8, 128, ragged=1),
        # two long documents
        _attention("attend_long", 2, 131_071, 64, 8, 128),
        # five drafted tokens of each sequence to verify, small heads, small pages, a sliding window
        _attention("attend_verify", 16, 3000, 24, 4, 64, queries=5, dtype="fp16", page=16, window=1024, ragged=1),
        # a whole prompt
        _attention("attend_prompt", 1, 8192, 32, 8, 128, queries=8192),
        # chunks of prompts behind cached prefixes, unequal ones, one of them a single token
        _attention("attend_chunks", 4, 9001, 40, 8, 128, queries=2047, page=128, ragged=2),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "rope":
        dim = rng.choice([64, 96, 128, 256])
        heads = rng.choice([1, 2, 4, 5, 8])
        each = rng.choice([1, 3, 4, 7])
        axes = rng.choice([1, 2, 3])
        case = _rope("", 1, heads * each, heads, dim, dtype=dtype, axes=axes, interleaved=rng.random() < 0.5, norm=rng.random() < 0.7,
                     rotary=dim if axes > 1 or rng.random() < 0.7 else dim // 2, first=_spread(rng, 1, 1_000_000))
        case["tokens"] = _spread(rng, 1, min(40_000, 160_000_000 // (heads * (each + 1) * dim)))
    elif op == "append":
        case = _append("", _spread(rng, 1, 16_000), rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), dtype=dtype, page=rng.choice([16, 32, 64, 128]))
    else:
        heads, each, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), rng.choice([64, 128, 256])
        case = _attention("", 1, 1, heads * each, heads, dim, dtype=dtype, page=rng.choice([16, 32, 64, 128]))
        if rng.random() < 0.6:      # single tokens, or a few to verify
            case["batch"] = _spread(rng, 1, 128)
            case["context"] = _spread(rng, 1, max(2, min(100_000, 60_000_000 // (case["batch"] * heads * dim))))
            case["queries"] = rng.choice([1, 1, 1, 2, 4, 7])
            case["ragged"] = rng.choice([0, 1])
        else:                       # prompts, and chunks of them
            case["batch"] = rng.choice([1, 1, 2, 3])
            case["queries"] = _spread(rng, 9, 3000)
            case["context"] = case["queries"] + (0 if rng.random() < 0.5 else _spread(rng, 1, 5000))
            case["ragged"] = rng.choice([0, 2])
        case["context"] = max(case["context"], case["queries"])
        if rng.random() < 0.25:
            case["window"] = _spread(rng, 1, 4096)
    case.pop("name")
    return case


def _lengths(case):
    """Keys and queries of each sequence: whole numbers that follow from the case alone."""

    rng = random.Random(case["batch"] * 1_000_003 + case["context"])
    keys, queries = [case["context"]] * case["batch"], [case["queries"]] * case["batch"]
    if case["ragged"]:
        for b in range(1, case["batch"]):       # the first sequence keeps the largest lengths
            queries[b] = queries[b] if case["ragged"] == 1 else max(1, _spread(rng, 1, case["queries"]))
            keys[b] = rng.randint(min(case["context"], max(1, queries[b])), case["context"])
        if case["ragged"] == 2 and case["batch"] > 1:
            queries[-1] = 1
    return keys, queries


def _pairs_seen(case):
    """(query, key) pairs that the masks leave, over all sequences."""

    total = 0
    for keys, queries in zip(*_lengths(case)):
        first = keys - queries + 1               # keys that the first query sees
        width = case["window"] or keys
        full = max(0, min(queries, keys - max(first, width) + 1)) if width < keys else 0
        rest = queries - full                    # queries that see all keys up to their own
        total += full * width + rest * first + rest * (rest - 1) // 2
    return total


def _keys_seen(case):
    return sum(min(keys, (case["window"] or keys) + queries - 1) for keys, queries in zip(*_lengths(case)))


def work(case):
    dim = case["dim"]
    if case["op"] == "rope":
        values = case["tokens"] * (case["q_heads"] + case["k_heads"]) * dim
        return {"bytes": 4 * values + 8 * case["axes"] * case["tokens"], "flops": 8 * values}
    if case["op"] == "append":
        vectors = 2 * case["tokens"] * case["k_heads"]       # keys and values: read, held (written, read), read back
        return {"bytes": vectors * (2 * dim + 2 * (dim // 2 + 4) + 2 * dim) + 16 * case["tokens"], "flops": 8 * vectors * dim}
    rows = sum(_lengths(case)[1]) * case["q_heads"]
    return {"bytes": _keys_seen(case) * case["k_heads"] * (dim + 8) + 4 * rows * dim, "flops": 4 * _pairs_seen(case) * case["q_heads"] * dim}


# ---------------------------------------------------------------- inputs

def _frequencies(case):
    """Radians per position of each pair of channels, and the axis of each pair."""

    pairs, axes = case["rotary"] // 2, case["axes"]
    theta = 1_000_000.0 if case["norm"] else 10_000.0
    if axes == 1:
        return [theta ** (-j / pairs) for j in range(pairs)], [0] * pairs
    share = [pairs // (axes + 1)] + [0] * (axes - 1)          # a smaller first axis (time), as such models have it
    for i in range(1, axes):
        share[i] = (pairs - share[0]) // (axes - 1) + (1 if i <= (pairs - share[0]) % (axes - 1) else 0)
    owner = [a for a in range(axes) for _ in range(share[a])]
    if case["interleaved"]:                                    # a ladder for each axis
        return [10_000.0 ** (-j / share[a]) for a in range(axes) for j in range(share[a])], owner
    return [theta ** (-j / pairs) for j in range(pairs)], owner   # one ladder, sections of it for the axes


def _quantized(x, dtype):
    """4-bit codes, scales and minima of the vectors along the last axis."""

    x = x.float()
    low = x.amin(-1)
    scale = ((x.amax(-1) - low) / 15).to(dtype).float()
    scale = torch.where(scale == 0, 1.0, scale)
    codes = ((x - low[..., None]) / scale[..., None]).round().clamp(0, 15)
    return codes.to(torch.uint8), scale, low


def _packed(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpacked(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def prepare(case, seed):
    device, dtype, dim = torch.device("cuda"), DTYPES[case["dtype"]], case["dim"]
    gen = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=device, dtype=torch.float32)

    state = {"case": case}
    if case["op"] == "rope":
        tokens, heads_q, heads_k = case["tokens"], case["q_heads"], case["k_heads"]
        # the output of a fused projection: queries, keys and values side by side
        fused = (normal(tokens, heads_q + 2 * heads_k, dim) * 1.5).to(dtype)
        state["q"], state["k"] = fused[:, :heads_q], fused[:, heads_q:heads_q + heads_k]
        frequencies, owner = _frequencies(case)
        state["frequencies"] = torch.tensor(frequencies, dtype=torch.float64, device=device)
        state["axes"] = torch.tensor(owner, dtype=torch.int32, device=device) if case["axes"] > 1 else None
        steps = torch.arange(tokens, device=device) + case["first"]
        if case["axes"] > 1:        # frames, rows and columns of a grid of 52 x 30 tokens
            state["positions"] = torch.stack((steps // 1560, steps // 52 % 30, steps % 52)[:case["axes"]])
        else:
            state["positions"] = steps
        state["q_weight"] = (1 + 0.2 * normal(dim)).to(dtype) if case["norm"] else None
        state["k_weight"] = (1 + 0.2 * normal(dim)).to(dtype) if case["norm"] else None
        return state
    page, heads = case["page"], case["k_heads"]
    if case["op"] == "append":
        tokens = case["tokens"]
        pages = tokens // page + 9
        fused = normal(tokens, 2 * heads, dim).to(dtype)
        state["k"], state["v"] = fused[:, :heads], fused[:, heads:]
        state["codes"] = torch.zeros((pages, 2, heads, page, dim // 2), dtype=torch.uint8, device=device)
        state["params"] = torch.zeros((pages, 2, heads, page, 2), dtype=dtype, device=device)
        state["slots"] = torch.randperm(pages * page, generator=gen, device=device)[:tokens].sort().values
        return state
    keys, queries = _lengths(case)
    per = [-(-n // page) for n in keys]
    pages = sum(per) + 3
    codes = torch.empty((pages, 2, heads, page, dim // 2), dtype=torch.uint8, device=device)
    params = torch.empty((pages, 2, heads, page, 2), dtype=dtype, device=device)
    step = max(1, (1 << 27) // (2 * heads * page * dim))
    for at in range(0, pages, step):
        some = normal(min(step, pages - at), 2, heads, page, dim)
        c, s, m = _quantized(some.to(dtype), dtype)
        codes[at:at + step] = _packed(c)
        params[at:at + step] = torch.stack((s, m), -1).to(dtype)
    order = torch.randperm(pages, generator=gen, device=device).to(torch.int32)
    table = torch.full((case["batch"], max(per)), -1, dtype=torch.int32, device=device)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    total = sum(queries)
    starts = [sum(queries[:b]) for b in range(len(queries) + 1)]
    state.update(codes=codes, params=params, table=table, q=normal(total, case["q_heads"], dim).to(dtype), keys=keys, queries=queries,
                 seq_lens=torch.tensor(keys, dtype=torch.int32, device=device),
                 query_starts=None if all(n == 1 for n in queries) else torch.tensor(starts, dtype=torch.int32, device=device))
    return state


# ---------------------------------------------------------------- the plain forms

def _rope_plain(state):
    case = state["case"]
    positions = state["positions"].reshape(case["axes"], -1).double()
    of_pair = positions[0][:, None] if state["axes"] is None else positions[state["axes"].long()].t()
    angle = of_pair * state["frequencies"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = case["rotary"] // 2

    def one(x, weight):
        y = x.float()
        if weight is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
        r, rest = y[..., :case["rotary"]], y[..., case["rotary"]:]
        if case["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        else:
            a, b = r[..., :half], r[..., half:]
            turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        return torch.cat((turned, rest), -1).to(x.dtype)

    return one(state["q"], state["q_weight"]), one(state["k"], state["k_weight"])


def _append_plain(state):
    codes, params, slots, page = state["codes"], state["params"], state["slots"], state["case"]["page"]
    both = torch.stack((state["k"], state["v"]), 1)                      # [tokens, 2, heads, dim]
    c, s, m = _quantized(both, params.dtype)
    at, row = slots // page, slots % page
    codes[at, :, :, row] = _packed(c)
    params[at, :, :, row] = torch.stack((s, m), -1).to(params.dtype)
    held, scale = _unpacked(codes[at, :, :, row]).float(), params[at, :, :, row].float()
    values = (held * scale[..., :1] + scale[..., 1:]).to(params.dtype)
    return values[:, 0], values[:, 1]


def _attention_plain(state):
    case, table, q = state["case"], state["table"].long().clamp(min=0), state["q"]
    page, heads, each, dim = case["page"], case["k_heads"], case["q_heads"] // case["k_heads"], case["dim"]
    batch, span, most = case["batch"], table.shape[1] * page, max(state["queries"])
    keys = state["seq_lens"].long()
    counts = torch.ones_like(keys) if state["query_starts"] is None else state["query_starts"].long().diff()
    starts = counts.cumsum(0) - counts
    scale = state["params"][table].float()                                # [batch, pages, 2, heads, page, 2]
    held = _unpacked(state["codes"][table]).float().mul_(scale[..., :1]).add_(scale[..., 1:])
    held = held.permute(2, 0, 3, 1, 4, 5).reshape(2, batch, heads, span, dim)
    local = torch.arange(most, device=q.device)
    real = local < counts[:, None]                                        # [batch, most]
    rows = (starts[:, None] + local).clamp(max=q.shape[0] - 1)
    padded = q[rows].float().reshape(batch, most, heads, each, dim).permute(0, 2, 1, 3, 4).reshape(batch, heads, most * each, dim)
    scores = (padded @ held[0].transpose(-1, -2)).mul_(dim ** -0.5)
    at = (keys - counts)[:, None] + local                                 # the position of each query
    key = torch.arange(span, device=q.device)
    seen = key <= at[..., None]
    if case["window"]:
        seen &= key > at[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(batch, 1, most, each, span).reshape(batch, 1, most * each, span)
    scores = scores.masked_fill_(~seen, -math.inf)
    scores = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores @ held[1]).div_(torch.where(total == 0, 1.0, total))
    out = out.reshape(batch, heads, most, each, dim).permute(0, 2, 1, 3, 4).reshape(batch, most, heads * each, dim)
    return out[real].to(q.dtype)


def run(state):
    case = state["case"]
    if own:
        from xqt_b200.ops.kv4 import kv4_append, kv4_attention, kv4_gather
        from xqt_b200.ops.rotary import qk_norm_rope

        if case["op"] == "rope":
            return qk_norm_rope(state["q"], state["k"], state["positions"], state["frequencies"], axes=state["axes"], q_weight=state["q_weight"],
                                k_weight=state["k_weight"], eps=1e-6, interleaved=case["interleaved"])
        if case["op"] == "append":
            kv4_append(state["k"], state["v"], state["codes"], state["params"], state["slots"])
            return kv4_gather(state["codes"], state["params"], state["slots"])
        return kv4_attention(state["q"], state["codes"], state["params"], state["table"], state["seq_lens"], query_starts=state["query_starts"],
                             window=case["window"] or None)
    return {"rope": _rope_plain, "append": _append_plain, "attention": _attention_plain}[case["op"]](state)


# ---------------------------------------------------------------- 64 bits, from the definitions

def _turned(x, weight, angle, case):
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
    n = case["rotary"]
    first = torch.arange(0, n, 2, device=x.device) if case["interleaved"] else torch.arange(n // 2, device=x.device)
    second = first + (1 if case["interleaved"] else n // 2)
    spun = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    x = x.clone()
    x[..., first], x[..., second] = spun.real, spun.imag
    return x


def _vectors(codes, params):
    """The values that a run of the cache stands for, in 64 bits."""

    values = torch.empty((*codes.shape[:-1], codes.shape[-1] * 2), dtype=torch.float64, device=codes.device)
    values[..., 0::2], values[..., 1::2] = (codes % 16).double(), (codes // 16).double()
    return values * params[..., 0:1].double() + params[..., 1:2].double()


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rope":
        positions = state["positions"].reshape(case["axes"], -1)
        owner = [0] * (case["rotary"] // 2) if state["axes"] is None else state["axes"].tolist()
        turns = state["frequencies"] / (2 * math.pi)
        angle = torch.stack([positions[a] * turns[j] for j, a in enumerate(owner)], -1)
        angle = (angle - angle.round()) * (2 * math.pi)
        return _turned(state["q"], state["q_weight"], angle, case), _turned(state["k"], state["k_weight"], angle, case)
    if case["op"] == "append":
        done = []
        for x in (state["k"], state["v"]):
            x = x.double()
            low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
            scale = ((high - low) / 15).to(DTYPES[case["dtype"]]).double()
            scale[scale == 0] = 1
            done.append(((x - low) / scale).round().clamp(0, 15) * scale + low)
        return tuple(done)
    keys, queries, each, dim = state["keys"], state["queries"], case["q_heads"] // case["k_heads"], case["dim"]
    out, at = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b, (n, m) in enumerate(zip(keys, queries)):
        pages = state["table"][b, : -(-n // case["page"])].long()
        place = torch.arange(n, device="cuda")
        for h in range(case["k_heads"]):
            k, v = (_vectors(state["codes"][pages, i, h], state["params"][pages, i, h]).reshape(-1, dim)[:n] for i in (0, 1))
            for r in range(0, m, 2048):
                some = state["q"][at + r:at + min(r + 2048, m), h * each:(h + 1) * each].double()
                mine = n - m + r + torch.arange(some.shape[0], device="cuda")
                hidden = place[None] > mine[:, None]
                if case["window"]:
                    hidden |= place[None] <= mine[:, None] - case["window"]
                score = torch.einsum("mgd,nd->mgn", some, k) / math.sqrt(dim)
                score = score.masked_fill(hidden[:, None], -math.inf)
                out[at + r:at + r + some.shape[0], h * each:(h + 1) * each] = torch.einsum("mgn,nd->mgd", score.softmax(-1), v)
        at += m
    return out
