"""Long generation over a paged cache that stays small, as cases that can be timed: features rotated by positions of several axes
(images, video, tokens that others were dropped before), keys and values appended so, one new token of every sequence attending and
adding its attention weights to what every token got so far, and the tokens that got least dropped.

The cache is ``pages`` pages of ``page`` tokens, (pages, kv_heads, page, dim) for the keys and the same for the values; a table names the
pages of every sequence; an 8-bit cache holds e4m3 codes and one exponent (a power of two, biased by 127) per token and head.  The weights are
(sequences, kv_heads, tokens that the table can hold) in 32 bits.  ``listed()`` names twelve cases, ``draw()`` gives more of the same ranges.
Where ``own`` is false ``run`` computes the operators by elementary torch operations.
"""
import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # training: the queries of a short picture, heads of 64, rows and columns as positions; forward and backward
        {"name": "rotate_300", "kind": "rotate", "type": "bf16", "layout": "tokens", "tokens": 300, "heads": 16, "dim": 64, "rotary": 64,
         "sections": "16 16", "in_turn": False, "interleaved": False, "train": True},
        # the decoder layer's 16 x 512 tokens as its projections leave them (features x tokens), one position per token
        {"name": "rotate_8192_features", "kind": "rotate", "type": "fp16", "layout": "features", "tokens": 8192, "heads": 32, "dim": 128, "rotary": 128,
         "sections": "64", "in_turn": False, "interleaved": False, "train": True},
        # a long video: time, height and width in turn over the planes, half of the features turned
        {"name": "rotate_30001_video", "kind": "rotate", "type": "bf16", "layout": "tokens", "tokens": 30001, "heads": 32, "dim": 128, "rotary": 64,
         "sections": "12 10 10", "in_turn": True, "interleaved": False, "train": True},
        # a decoder layer of 32 heads of 128 generating for one user, some of whose tokens were dropped
        {"name": "append_one_token", "kind": "append", "type": "fp16", "cache": "16", "layout": "features", "heads": 32, "kv_heads": 32, "dim": 128,
         "page": 64, "seqs": 1, "longest": 700, "shortest": 700, "new": 1, "rotary": 128, "sections": "64", "in_turn": False, "interleaved": False},
        # a step of generation for 64 users behind pictures: time, height and width
        {"name": "append_64", "kind": "append", "type": "bf16", "cache": "16", "layout": "tokens", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "seqs": 64, "longest": 8192, "shortest": 100, "new": 1, "rotary": 128, "sections": "16 24 24", "in_turn": False, "interleaved": False},
        # four videos as prompts
        {"name": "append_videos", "kind": "append", "type": "bf16", "cache": "16", "layout": "tokens", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "seqs": 4, "longest": 5001, "shortest": 2200, "new": 5001, "rotary": 128, "sections": "16 24 24", "in_turn": False, "interleaved": False},
        # the layer attending for one user and keeping account
        {"name": "weigh_700", "kind": "weigh", "type": "fp16", "cache": "16", "layout": "features", "heads": 32, "kv_heads": 32, "dim": 128,
         "page": 64, "seqs": 1, "longest": 700, "shortest": 700},
        # a full server whose sequences are kept between 2048 and 4224 tokens, shared key heads
        {"name": "weigh_64x4224", "kind": "weigh", "type": "bf16", "cache": "16", "layout": "tokens", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "seqs": 64, "longest": 4224, "shortest": 2049},
        # one very long document in 8 bits, eight query heads to a key head
        {"name": "weigh_131071_e4m3", "kind": "weigh", "type": "bf16", "cache": "e4m3", "layout": "tokens", "heads": 64, "kv_heads": 8, "dim": 128,
         "page": 64, "seqs": 1, "longest": 131071, "shortest": 131071},
        # the layer's user over a budget of 512
        {"name": "evict_700", "kind": "evict", "type": "fp16", "cache": "16", "kv_heads": 32, "dim": 128, "page": 64, "seqs": 1, "longest": 700, "shortest": 700,
         "keep": 512, "recent": 128, "first": 4},
        # the full server, every sequence beyond its budget by another number of tokens, some not
        {"name": "evict_64x4224", "kind": "evict", "type": "bf16", "cache": "16", "kv_heads": 8, "dim": 128, "page": 64, "seqs": 64, "longest": 4224, "shortest": 1500,
         "keep": 2048, "recent": 512, "first": 4},
        # a very long document, a quarter of it kept
        {"name": "evict_131071", "kind": "evict", "type": "bf16", "cache": "16", "kv_heads": 8, "dim": 128, "page": 64, "seqs": 1, "longest": 131071, "shortest": 131071,
         "keep": 32768, "recent": 4096, "first": 16},
    ]


def _between(rng, low, high):
    """A size, its logarithm spread over the range."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _split(rng, planes, axes):
    """planes in ``axes`` parts, none empty."""
    cuts = sorted(rng.sample(range(1, planes), axes - 1))
    return " ".join(str(b - a) for a, b in zip([0] + cuts, cuts + [planes]))


def _sections(case):
    """How many planes every axis has."""
    return [int(n) for n in case["sections"].split()]


def draw(rng):
    kind = rng.choice(("rotate", "append", "weigh", "evict"))
    dim = rng.choice((64, 128, 128, 128, 256))
    case = {"kind": kind, "type": rng.choice(("fp16", "bf16")), "layout": rng.choice(("tokens", "features")), "dim": dim}
    if kind in ("rotate", "append"):
        case["rotary"] = rng.choice((32, dim // 2, dim, dim))
        case["sections"] = _split(rng, case["rotary"] // 2, rng.choice((1, 1, 2, 3, 3, 4)))
        case["in_turn"] = rng.random() < 0.4
        case["interleaved"] = rng.random() < 0.4
    if kind == "rotate":
        case["type"] = rng.choice(("fp16", "bf16", "bf16", "fp32"))
        case["heads"] = rng.choice((1, 2, 5, 8, 16, 32, 40))
        case["tokens"] = _between(rng, 1, min(65536, (1 << 25) // (case["heads"] * dim)))
        case["train"] = rng.random() < 0.7
        return case
    case["cache"] = rng.choice(("16", "16", "e4m3"))
    case["kv_heads"] = rng.choice((1, 2, 4, 5, 8, 16, 32))
    case["page"] = rng.choice((16, 32, 64, 64, 128, 256))
    width = case["kv_heads"] * dim
    if kind != "evict":
        case["heads"] = case["kv_heads"] * rng.choice([g for g in (1, 2, 3, 4, 6, 8, 16) if g * case["kv_heads"] <= 64])
    # (an 8-bit cache that is an output is returned as the values it stands for, which should not be what is measured)
    room = 1 << (27 if kind == "weigh" else 24 if case["cache"] == "e4m3" else 26)
    if kind == "append":
        tokens = _between(rng, 1, min(20000, (1 << 25) // (case["heads"] * dim)))
        case["new"] = 1 if rng.random() < 0.4 else _between(rng, 2, 5001)
        case["seqs"] = max(1, min(256, tokens // case["new"]))
        case["longest"] = max(case["new"], _between(rng, 1, max(64, min(20000, room // (width * case["seqs"])))))
        case["shortest"] = rng.randint(1, min(100, case["longest"]))
        return case
    tokens = _between(rng, 1 if kind == "weigh" else 64, room // width)
    case["seqs"] = min(128, _between(rng, 1, tokens))
    case["longest"] = min(131072, max(1, tokens // case["seqs"]))
    case["shortest"] = rng.randint(1, case["longest"])
    if kind == "evict":
        del case["layout"]
        case["keep"] = _between(rng, 1, case["longest"])
        case["recent"] = rng.randint(0, case["keep"] // 2)
        case["first"] = rng.randint(0, min(16, case["keep"] - case["recent"]))
    return case


def _lengths(case):
    """The sequences' lengths, new tokens among them: spread over the logarithm between shortest and longest, in no order."""
    n, low, high = case["seqs"], case["shortest"], case["longest"]
    lengths = [high] if n == 1 else [round(low * (high / low) ** (i / (n - 1))) for i in range(n)]
    random.Random(7).shuffle(lengths)
    return lengths


def _new(case):
    """How many tokens of each sequence the call appends: the whole of it or the newest ``new``."""
    return [min(case["new"], n) for n in _lengths(case)]


def _pages(length, page):
    return -(-length // page)


def _positions(axes, tokens, rng):
    """(axes, tokens) of one sequence: text and, with more axes than one, pictures or videos between it (rows and columns; frames first; with a
    fourth axis the number of the video).  Text counts on where the largest position so far ended."""
    parts, count, at = [], 0, rng.randint(0, 200)
    while count < tokens:
        text = tokens if axes == 1 else rng.randint(1, 60)
        parts.append(torch.arange(at, at + text).expand(axes, -1))
        count, at = count + text, at + text
        if axes > 1:
            shape = [1] * (axes - 3) + [rng.randint(1, 30)] * (axes > 2) + [rng.randint(4, 40), rng.randint(4, 40)]
            grid = torch.meshgrid(*(torch.arange(n) for n in shape), indexing="ij")
            parts.append(at + torch.stack([g.flatten() for g in grid]))
            count, at = count + parts[-1].shape[1], at + max(shape)
    return torch.cat(parts, 1)[:, :tokens]


def _rotation(case, rows):
    """cos and sin of position / 10000^(2 j / r), side by side; the angles in 64 bits."""
    r = case["rotary"]
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(r // 2, dtype=torch.float64) / r)
    return torch.cat([angle.cos(), angle.sin()], 1).to(device="cuda", dtype=torch.float32)


def _axes(case):
    """The axis of every plane: stretches, or in turn as long as an axis has planes left."""
    if not case["in_turn"]:
        return [a for a, n in enumerate(_sections(case)) for _ in range(n)]
    left, out = _sections(case), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def prepare(case, seed):
    d = torch.device("cuda")
    gen = torch.Generator(device=d).manual_seed(seed)
    rng = random.Random(seed)
    dtype, dim = TYPES[case["type"]], case["dim"]
    state = {"case": case}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=d, dtype=dtype)

    def tokens_heads(count, heads):
        if case["layout"] == "features":   # as a projection W @ X leaves it
            return normal(heads * dim, count).view(heads, dim, count).permute(2, 0, 1)
        return normal(count, heads, dim)

    if case["kind"] in ("rotate", "append"):
        axes, counts = len(_sections(case)), [case["tokens"]] if case["kind"] == "rotate" else _new(case)
        places = torch.cat([_positions(axes, n, rng) for n in counts], 1)
        if case["kind"] == "append" and case["new"] == 1:   # behind all that there has been
            places = torch.tensor([[rng.randint(n, 3 * n) for n in _lengths(case)] for _ in range(axes)])
        state["rotation"] = _rotation(case, int(places.max()) + 1)
        state["positions"] = places.to(device=d, dtype=torch.int32)
        state["sections"], state["axes"] = _sections(case), torch.tensor(_axes(case), device=d)
    if case["kind"] == "rotate":
        state["x"], state["grad"] = tokens_heads(case["tokens"], case["heads"]), tokens_heads(case["tokens"], case["heads"])
        return state

    page, kv, lengths = case["page"], case["kv_heads"], _lengths(case)
    counts = [_pages(n, page) for n in lengths]
    total, width = sum(counts), max(counts)
    pages = total + 3
    # the pages of a cache that has been in use for a while lie in no order
    order = torch.randperm(pages, generator=gen, device=d)[:total].to(torch.int32)
    n_pages = torch.tensor(counts, device=d)
    column = torch.arange(width, device=d)
    at = (torch.cumsum(n_pages, 0) - n_pages)[:, None] + column
    state["table"] = torch.where(column < n_pages[:, None], order[at.clamp(max=total - 1)], -1).to(torch.int32)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=d)
    keys, values = normal(pages, kv, page, dim), normal(pages, kv, page, dim)
    if case["cache"] == "e4m3":
        keys, state["key_exponents"] = _to_e4m3(keys)
        values, state["value_exponents"] = _to_e4m3(values)
    state["keys"], state["values"] = keys, values
    if case["kind"] == "append":
        tokens = sum(_new(case))
        state["q"], state["k"], state["v"] = tokens_heads(tokens, case["heads"]), tokens_heads(tokens, kv), tokens_heads(tokens, kv)
        state["offsets"] = None
        if case["new"] > 1:
            state["offsets"] = torch.tensor([0] + _new(case), device=d).cumsum(0).to(torch.int32)
        return state
    # what tokens got so far: a few a lot, many next to nothing, some nothing at all
    got = torch.randn((case["seqs"], kv, width * page), generator=gen, device=d).mul_(3.0).exp_()
    there = torch.arange(width * page, device=d) < state["lengths"][:, None]
    state["weights"] = torch.where(there[:, None] & (got > 0.02), got / case["longest"], 0.0)   # (as some passes leave it, not more than one adds)
    if case["kind"] == "weigh":
        state["q"] = tokens_heads(case["seqs"], case["heads"])
        state["scale"] = 1.0 / math.sqrt(dim)
    return state


def _to_e4m3(x):
    """Codes and exponents of the last dimension's rows: the least power of two that brings the row's largest magnitude to 448."""
    x = x.float()
    exponent = ((x.abs().amax(-1).view(torch.int32) + 0x1FFFFF) >> 23).sub(8).clamp(1, 254)
    codes = (x * _power(254 - exponent)[..., None]).to(torch.float8_e4m3fn)
    return codes, exponent.to(torch.uint8)


def _power(exponent):
    """2 ** (exponent - 127), exactly."""
    return (exponent.to(torch.int32) << 23).view(torch.float32)


def _values(rows, exponents):
    """What cache rows stand for, in 32 bits."""
    return rows.float() if exponents is None else rows.float().mul_(_power(exponents)[..., None])


def _cache(state):
    """The cache as an output."""
    if state["case"]["cache"] == "16":
        return {"keys": state["keys"], "values": state["values"]}
    return {"keys": _values(state["keys"], state["key_exponents"]), "values": _values(state["values"], state["value_exponents"])}


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        import intrasm_engine_amd  # noqa: F401
        ops = torch.ops.iex_ops
    exponents = state.get("key_exponents"), state.get("value_exponents")
    if kind == "rotate":
        if not own:
            out = {"out": _turn(state, state["x"], False)}
            if case["train"]:
                out["grad"] = _turn(state, state["grad"], True)
            return out
        turn = (state["rotation"], state["positions"], state["sections"], case["in_turn"], case["interleaved"])
        if not case["train"]:
            return {"out": ops.rotate(state["x"], *turn)}
        x = state["x"].detach().requires_grad_()
        out = ops.rotate(x, *turn)
        return {"out": out.detach(), "grad": torch.autograd.grad(out, x, state["grad"])[0]}
    if kind == "append":
        if own:
            q = ops.kv_append_(state["k"], state["v"], state["keys"], state["values"], state["table"], state["lengths"], state["offsets"], state["q"],
                               state["rotation"], case["interleaved"], None, *exponents, state["positions"], state["sections"], case["in_turn"])
        else:
            q = _plain_append(state)
        return {"q": q, **_cache(state)}
    if kind == "weigh":
        if own:
            out = ops.paged_attention_accumulate_(state["q"], state["keys"], state["values"], state["table"], state["lengths"], state["weights"], state["scale"],
                                                  *exponents)
        else:
            out = _plain_weigh(state)
        return {"out": out, "weights": state["weights"]}
    # (a program drops tokens once: a pass that can be run again has lengths and weights of its own)
    lengths, weights = state["lengths"].clone(), state["weights"].clone()
    if own:
        kept = ops.evict_tokens_(state["keys"], state["values"], state["table"], lengths, weights, case["keep"], case["recent"], case["first"], None, *exponents)
    else:
        kept = _plain_evict(state, lengths, weights)
    return {"kept": kept, "lengths": lengths, "weights": weights, **_cache(state)}


def _turn(state, x, back):
    """x (tokens, heads, dim) turned by its positions, the other way where ``back``; as x lies."""
    case, dtype, r = state["case"], x.dtype, state["case"]["rotary"]
    place = state["positions"].long()[state["axes"]].T                            # (tokens, r / 2)
    plane = torch.arange(r // 2, device=x.device)
    c, s = state["rotation"][place, plane][:, None], state["rotation"][place, plane + r // 2][:, None]
    s = -s if back else s
    first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., first].float(), x[..., second].float()
    out = x.clone()
    out[..., first], out[..., second] = (a * c - b * s).to(dtype), (b * c + a * s).to(dtype)
    return out


def _plain_append(state):
    case, table, page = state["case"], state["table"], state["case"]["page"]
    lengths, v = state["lengths"].long(), state["v"]
    token = torch.arange(v.shape[0], device=v.device)
    if state["offsets"] is None:
        seq, slot = token, lengths - 1
    else:
        ends = state["offsets"][1:].long()
        seq = torch.searchsorted(ends, token, right=True)
        slot = lengths[seq] - ends[seq] + token
    row, slot = table[seq, slot // page].long(), slot % page
    if case["cache"] == "e4m3":   # (from 32 bits: a key is rounded once)
        for name, exponents, x in (("keys", "key_exponents", _turn(state, state["k"].float(), False)), ("values", "value_exponents", v)):
            codes, exponent = _to_e4m3(x)
            state[name].view(torch.uint8)[row, :, slot] = codes.view(torch.uint8)
            state[exponents][row, :, slot] = exponent
    else:
        state["keys"][row, :, slot], state["values"][row, :, slot] = _turn(state, state["k"], False), v
    return _turn(state, state["q"], False)


def _plain_weigh(state):
    case, table, lengths = state["case"], state["table"], state["lengths"]
    seqs, kv, dim, page = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    index = table.clamp(min=0).long()                                             # (seqs, width)

    def taken(name, exponents):
        rows = state[name]
        x = rows[index] if exponents is None else _values(rows.view(torch.uint8)[index].view(rows.dtype), exponents[index])
        return x.float().transpose(1, 2).reshape(seqs, kv, -1, dim)

    there = (torch.arange(table.shape[1] * page, device=table.device) < lengths[:, None])[:, None, None]
    q = state["q"].float().reshape(seqs, kv, -1, dim)
    score = torch.matmul(q, taken("keys", state.get("key_exponents")).transpose(2, 3).contiguous()) * state["scale"]
    score = torch.where(there, score, -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    weight = weight / weight.sum(-1, keepdim=True)
    state["weights"].add_(weight.sum(2))
    out = torch.matmul(weight, taken("values", state.get("value_exponents")))
    return out.reshape(seqs, case["heads"], dim).to(TYPES[case["type"]])


def _plain_evict(state, lengths, weights):
    case, table, page, keep = state["case"], state["table"].long(), state["case"]["page"], state["case"]["keep"]
    seqs, kv, room = weights.shape
    token = torch.arange(room, device=table.device)
    n = lengths[:, None, None].long()
    score = torch.where((token < case["first"]) | (token >= n - case["recent"]) | (n <= keep), math.inf, weights)
    score = torch.where(token < n, score, -math.inf)
    kept = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :keep]         # (ties: the earlier token first)
    kept = torch.where(kept < n, kept, room).sort(-1)[0]                                  # (seqs, kv, keep), what is not there last
    there = kept < room
    s, h, to = (x.expand_as(kept)[there] for x in (torch.arange(seqs, device=kept.device)[:, None, None], torch.arange(kv, device=kept.device)[:, None],
                                                   torch.arange(kept.shape[-1], device=kept.device)))
    at = kept[there]
    source, target = (table[s, at // page], h, at % page), (table[s, to // page], h, to % page)
    for name in ("keys", "values", "key_exponents", "value_exponents"):
        if name in state:
            rows = state[name].view(torch.uint8) if state[name].dtype == torch.float8_e4m3fn else state[name]
            rows[target] = rows[source]
    moved = torch.zeros_like(weights)
    moved[s, h, to] = weights[s, h, at]
    weights.copy_(moved)
    lengths.clamp_(max=keep)
    kept = torch.where(there, kept, -1).to(torch.int32)
    return torch.nn.functional.pad(kept, (0, keep - kept.shape[-1]), value=-1)


def work(case):
    dim = case["dim"]
    if case["kind"] == "rotate":
        size = 4 if case["type"] == "fp32" else 2
        passes, n = 2 if case["train"] else 1, case["tokens"]
        cells = n * case["heads"] * dim
        return {"bytes": passes * (2 * cells * size + n * (4 * case["rotary"] + 4 * len(_sections(case)))),
                "flops": passes * n * case["heads"] * case["rotary"] * 3}
    size = 1 if case["cache"] == "e4m3" else 2
    kv, page, seqs = case["kv_heads"], case["page"], case["seqs"]
    row = dim * size + (1 if size == 1 else 0)                 # one token's key (or value) of one head in the cache
    lengths = _lengths(case)
    if case["kind"] == "append":
        n, heads = sum(_new(case)), case["heads"]
        touched = sum(_pages(a, page) - (a - b) // page for a, b in zip(lengths, _new(case)))
        return {"bytes": n * (2 * kv * dim * 2 + 2 * heads * dim * 2 + 2 * kv * row + 4 * case["rotary"] + 4 * len(_sections(case))) + touched * 4,
                "flops": n * (heads + kv) * case["rotary"] * 3}
    if case["kind"] == "weigh":
        attended, heads = sum(lengths), case["heads"]
        return {"bytes": attended * kv * (2 * row + 8) + 2 * seqs * heads * dim * 2 + sum(_pages(n, page) for n in lengths) * 4,
                "flops": attended * heads * (4 * dim + 1)}
    over = [n for n in lengths if n > case["keep"]]            # every kept token read and written, the weights of all of them too
    return {"bytes": kv * (sum(over) * 8 + len(over) * case["keep"] * 2 * 2 * row + seqs * case["keep"] * 4), "flops": kv * sum(over)}


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence."""
    state = prepare(case, seed)
    f64, dim = torch.float64, case["dim"]

    def turned(x, sign):
        """x (tokens, heads, dim) in 64 bits, in complex numbers."""
        r = case["rotary"]
        x = x.to(f64).clone()
        frequency = torch.exp(torch.arange(0, r, 2, dtype=f64, device=x.device) * (-math.log(10000.0) / r))
        angle = torch.stack([state["positions"][a].to(f64) * frequency[j] for j, a in enumerate(_axes(case))], 1) * sign
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    if case["kind"] == "rotate":
        out = {"out": turned(state["x"], 1.0)}
        if case["train"]:
            out["grad"] = turned(state["grad"], -1.0)
        return out

    kv, page, lengths, table = case["kv_heads"], case["page"], _lengths(case), state["table"].long()

    def stands_for(name, rows):
        """(rows, kv, page, dim) of the cache's pages ``rows``."""
        if case["cache"] == "16":
            return state[name][rows].to(f64)
        codes = state[name].view(torch.uint8)[rows].view(torch.float8_e4m3fn).float().to(f64)
        return codes * 2.0 ** (state[{"keys": "key_exponents", "values": "value_exponents"}[name]][rows].to(f64) - 127.0)[..., None]

    every = torch.arange(state["keys"].shape[0], device=table.device)
    if case["kind"] == "append":
        out = {"q": turned(state["q"], 1.0), "keys": None, "values": None}
        if case["cache"] == "16":   # (in 8 bits what is stored is a choice, not a value)
            k, v, at = turned(state["k"], 1.0), state["v"].to(f64), 0
            out["keys"], out["values"] = stands_for("keys", every), stands_for("values", every)
            for s, (length, n) in enumerate(zip(lengths, _new(case))):
                slot = torch.arange(length - n, length, device=table.device)
                where = table[s][slot // page]
                out["keys"][where, :, slot % page], out["values"][where, :, slot % page] = k[at:at + n], v[at:at + n]
                at += n
        return out

    if case["kind"] == "weigh":
        q, group = state["q"].to(f64), case["heads"] // kv
        out, weights = torch.zeros_like(q), state["weights"].to(f64)
        for s, length in enumerate(lengths):
            rows = table[s, :_pages(length, page)]
            k, v = (stands_for(name, rows).transpose(0, 1).reshape(kv, -1, dim)[:, :length] for name in ("keys", "values"))
            score = torch.matmul(q[s].reshape(kv, group, dim), k.transpose(1, 2).contiguous()) * state["scale"]
            weight = torch.softmax(score, -1)
            out[s] = torch.matmul(weight, v).reshape(-1, dim)
            weights[s, :, :length] += weight.sum(1)
        return {"out": out, "weights": weights}

    keep, recent, first = case["keep"], case["recent"], case["first"]
    keys, values = stands_for("keys", every), stands_for("values", every)
    kept = torch.full((case["seqs"], kv, keep), -1, dtype=torch.int32, device=table.device)
    weights, heads = torch.zeros_like(state["weights"]), torch.arange(kv, device=table.device)[:, None]
    for s, length in enumerate(lengths):
        mine = min(length, keep)
        chosen = torch.arange(mine, device=table.device).expand(kv, -1)
        if length > keep:
            middle = state["weights"][s, :, first:length - recent]
            most = torch.argsort(-middle.to(f64), dim=-1, stable=True)[:, :keep - first - recent] + first
            ends = torch.cat([torch.arange(first, device=table.device), torch.arange(length - recent, length, device=table.device)]).expand(kv, -1)
            chosen = torch.cat([most, ends], 1).sort(1)[0]
        kept[s, :, :mine] = chosen
        weights[s, :, :mine] = torch.gather(state["weights"][s], 1, chosen)
        to = torch.arange(mine, device=table.device)
        for x in (keys, values):
            x[table[s][to // page][None], heads, (to % page)[None]] = x[table[s][chosen // page], heads, chosen % page]
    return {"kept": kept, "lengths": torch.tensor([min(n, keep) for n in lengths], dtype=torch.int32, device=table.device), "weights": weights, "keys": keys, "values": values}
