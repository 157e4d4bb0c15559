"""Serving a layer token by token, as cases that can be timed: keys and values appended to a paged cache, one new token of every
sequence attending to it, and the same over the pages that a cheap score selects.

The cache is ``pages`` pages of ``page`` tokens, (pages, kv_heads, page, dim) for the keys and the same for the values; a table names
the pages of every sequence.  An 8-bit cache holds e4m3 codes and one exponent (a power of two, biased by 127) per token and head.
``listed()`` names twelve cases, ``draw()`` gives more of the same ranges.  Where ``own`` is false ``run`` computes the operators by
elementary torch operations.
"""
import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decoder layer of 32 heads of 128 generating for one user: the smallest calls, where latency counts
        {"name": "append_one_token", "kind": "append", "type": "fp16", "cache": "16", "layout": "features", "heads": 32, "kv_heads": 32, "dim": 128,
         "page": 64, "seqs": 1, "longest": 700, "shortest": 700, "new": 1, "rotary": 128, "interleaved": False, "bounds": False},
        # a step of generation for 64 users of a model with shared key heads, bounds kept for selection
        {"name": "append_64", "kind": "append", "type": "bf16", "cache": "16", "layout": "tokens", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "seqs": 64, "longest": 8192, "shortest": 100, "new": 1, "rotary": 128, "interleaved": False, "bounds": True},
        # the layer's prompts, 16 x 512 tokens, as its projections leave them (features x tokens)
        {"name": "append_prompts_features", "kind": "append", "type": "fp16", "cache": "16", "layout": "features", "heads": 32, "kv_heads": 32, "dim": 128,
         "page": 64, "seqs": 16, "longest": 512, "shortest": 512, "new": 512, "rotary": 128, "interleaved": False, "bounds": False},
        # prompts of ragged lengths into an 8-bit cache, small pages, pairs of neighbours rotated in half of the features, bounds
        {"name": "append_prompts_e4m3", "kind": "append", "type": "bf16", "cache": "e4m3", "layout": "tokens", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "seqs": 23, "longest": 5001, "shortest": 3, "new": 4096, "rotary": 64, "interleaved": True, "bounds": True},
        # the layer attending for one user
        {"name": "attend_700", "kind": "attend", "type": "fp16", "cache": "16", "layout": "features", "heads": 32, "kv_heads": 32, "dim": 128,
         "page": 64, "seqs": 1, "longest": 700, "shortest": 700},
        # ... for the 16 sequences of its prompts, some way on
        {"name": "attend_16x800", "kind": "attend", "type": "fp16", "cache": "16", "layout": "features", "heads": 32, "kv_heads": 32, "dim": 128,
         "page": 64, "seqs": 16, "longest": 1023, "shortest": 600},
        # one very long document, eight query heads to a key head
        {"name": "attend_131071", "kind": "attend", "type": "bf16", "cache": "16", "layout": "tokens", "heads": 64, "kv_heads": 8, "dim": 128,
         "page": 64, "seqs": 1, "longest": 131071, "shortest": 131071},
        # many users of very different lengths, small heads, small pages
        {"name": "attend_ragged_d64", "kind": "attend", "type": "bf16", "cache": "16", "layout": "tokens", "heads": 16, "kv_heads": 16, "dim": 64,
         "page": 16, "seqs": 128, "longest": 4096, "shortest": 1},
        # a full server, 8-bit cache
        {"name": "attend_64_e4m3", "kind": "attend", "type": "bf16", "cache": "e4m3", "layout": "tokens", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "seqs": 64, "longest": 16384, "shortest": 4000},
        # 64 of the 512 pages of one long document
        {"name": "select_32768", "kind": "select", "type": "bf16", "cache": "16", "layout": "tokens", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "seqs": 1, "longest": 32768, "shortest": 32768, "count": 64, "first": 1, "last": 2},
        # many long contexts at once
        {"name": "select_32_ragged", "kind": "select", "type": "fp16", "cache": "16", "layout": "tokens", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "seqs": 32, "longest": 65536, "shortest": 1500, "count": 32, "first": 1, "last": 1},
        # small pages of an 8-bit cache
        {"name": "select_8_e4m3", "kind": "select", "type": "bf16", "cache": "e4m3", "layout": "tokens", "heads": 64, "kv_heads": 8, "dim": 128,
         "page": 32, "seqs": 8, "longest": 131072, "shortest": 90000, "count": 129, "first": 1, "last": 4},
    ]


def _between(rng, low, high):
    """A size, its logarithm spread over the range."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "select"))
    dim = rng.choice((64, 128, 128, 128, 256))
    case = {"kind": kind, "type": rng.choice(("fp16", "bf16")), "cache": rng.choice(("16", "16", "e4m3")), "layout": rng.choice(("tokens", "features")), "dim": dim}
    case["kv_heads"] = rng.choice((1, 2, 4, 5, 8, 16, 32))
    case["heads"] = case["kv_heads"] * rng.choice([g for g in (1, 2, 3, 4, 6, 8, 16) if g * case["kv_heads"] <= 64])
    case["page"] = rng.choice((16, 32, 64, 64, 128, 256))
    width = case["kv_heads"] * dim
    if kind == "append":
        # tokens of the call x features, held to what the prompts above come to
        tokens = _between(rng, 1, min(30000, (1 << 25) // (case["heads"] * dim)))
        case["new"] = 1 if rng.random() < 0.4 else _between(rng, 2, 4096)
        case["seqs"] = max(1, min(256, tokens // case["new"]))
        # (an 8-bit cache is returned as the values it stands for, which should not be what is measured)
        most = max(64, (1 << (24 if case["cache"] == "e4m3" else 27)) // (width * case["seqs"]))
        case["longest"] = max(case["new"], _between(rng, 1, min(20000, most)))
        case["shortest"] = rng.randint(1, min(100, case["longest"]))
        case["rotary"] = rng.choice((0, 32, dim // 2, dim, dim))
        case["interleaved"] = rng.random() < 0.4
        case["bounds"] = rng.random() < 0.5
    elif kind == "attend":
        tokens = _between(rng, 1, (1 << 28) // width)
        case["seqs"] = min(256, _between(rng, 1, tokens))
        case["longest"] = min(131072, max(1, tokens // case["seqs"]))
        case["shortest"] = rng.randint(1, case["longest"])
    else:
        tokens = _between(rng, 512, (1 << 28) // width)
        case["seqs"] = min(64, _between(rng, 1, tokens // 256))
        case["longest"] = min(131072, tokens // case["seqs"])
        case["shortest"] = rng.randint(1, case["longest"])
        pages = -(-case["longest"] // case["page"])
        case["count"] = _between(rng, 2, max(3, pages // 4))
        case["first"] = rng.randint(0, 1)
        case["last"] = rng.randint(0, 1)
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


def prepare(case, seed):
    d = torch.device("cuda")
    gen = torch.Generator(device=d).manual_seed(seed)
    dtype, page, kv, dim = TYPES[case["type"]], case["page"], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    counts = [_pages(n, page) for n in lengths]
    total, width = sum(counts), max(counts)
    pages = total + 3
    # the pages of a cache that has been in use for a while lie in no order
    order = torch.randperm(pages, generator=gen, device=d)[:total].to(torch.int32)
    n_pages = torch.tensor(counts, device=d)
    column = torch.arange(width, device=d)
    there = column < n_pages[:, None]
    at = (torch.cumsum(n_pages, 0) - n_pages)[:, None] + column
    table = torch.where(there, order[at.clamp(max=total - 1)], -1).to(torch.int32)
    state = {"case": case, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=d), "scale": 1.0 / math.sqrt(dim)}

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=d, dtype=dtype)

    def tokens_heads(count, heads):
        if case["layout"] == "features":   # as a projection W @ X leaves it
            return normal(heads * dim, count).view(heads, dim, count).permute(2, 0, 1)
        return normal(count, heads, dim)

    keys = normal(pages, kv, page, dim)
    if case["kind"] == "select":   # what a page holds hangs together
        keys.mul_(0.8).add_(normal(pages, kv, 1, dim), alpha=0.6)
    values = normal(pages, kv, page, dim)
    if case["cache"] == "e4m3":
        keys, state["key_exponents"] = _to_e4m3(keys)
        values, state["value_exponents"] = _to_e4m3(values)
    state["keys"], state["values"] = keys, values
    new = sum(_new(case)) if case["kind"] == "append" else case["seqs"]
    state["q"] = tokens_heads(new, case["heads"])
    if case["kind"] == "append":
        state["k"], state["v"] = tokens_heads(new, kv), tokens_heads(new, kv)
        state["offsets"] = None
        if case["new"] > 1:
            state["offsets"] = torch.tensor([0] + _new(case), device=d).cumsum(0).to(torch.int32)
        if case["rotary"]:
            state["rotation"] = _rotation(width * page, case["rotary"]).to(device=d, dtype=torch.float32)
    if case["kind"] == "select" or case.get("bounds"):
        used = torch.zeros(pages, dtype=torch.int64, device=d)
        full = torch.where(column < n_pages[:, None] - 1, page, state["lengths"][:, None] - (n_pages[:, None] - 1) * page)
        used[table[there].long()] = full[there]
        state["bounds"] = _bounds(keys, state.get("key_exponents"), used, dtype)
    return state


def _rotation(positions, r):
    """cos and sin of position / 10000^(2 j / r), side by side; the angles in 64 bits."""
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(r // 2, dtype=torch.float64) / r)
    return torch.cat([angle.cos(), angle.sin()], 1)


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


def _take(rows, index):
    """rows[index] (8-bit types as bytes)."""
    return rows.view(torch.uint8)[index].view(rows.dtype) if rows.dtype == torch.float8_e4m3fn else rows[index]


def _bounds(keys, exponents, used, dtype):
    """Smallest and largest key per page, head and feature over the page's first ``used`` tokens."""
    out = torch.zeros(keys.shape[0], keys.shape[1], 2, keys.shape[3], dtype=dtype, device=keys.device)
    step = max(1, (1 << 26) // keys[0].numel())
    for a in range(0, keys.shape[0], step):
        x = _values(keys[a:a + step], None if exponents is None else exponents[a:a + step])
        there = (torch.arange(keys.shape[2], device=keys.device) < used[a:a + step, None])[:, None, :, None]
        out[a:a + step, :, 0] = torch.where(there, x, math.inf).amin(2).to(dtype)
        out[a:a + step, :, 1] = torch.where(there, x, -math.inf).amax(2).to(dtype)
    return out


def run(state):
    case = state["case"]
    if own:
        import intrasm_engine_amd  # noqa: F401
        ops = torch.ops.iex_ops
    exponents = state.get("key_exponents"), state.get("value_exponents")
    if case["kind"] == "append":
        if own:
            q = ops.kv_append_(state["k"], state["v"], state["keys"], state["values"], state["table"], state["lengths"], state["offsets"],
                               state["q"], state.get("rotation"), case["interleaved"], state.get("bounds"), *exponents)
        else:
            q = _plain_append(state)
        out = {"q": q}
        if exponents[0] is None:
            out.update(keys=state["keys"], values=state["values"])
        else:   # 8 bits: as the values they stand for
            out.update(keys=_values(state["keys"], exponents[0]), values=_values(state["values"], exponents[1]))
        if "bounds" in state:
            out["bounds"] = state["bounds"]
        return out
    if case["kind"] == "attend":
        if own:
            return ops.paged_attention(state["q"], state["keys"], state["values"], state["table"], state["lengths"], state["scale"], None, *exponents)
        return _plain_attend(state, None)
    if own:
        pages = ops.select_pages(state["q"], state["bounds"], state["table"], state["lengths"], case["page"], case["count"], case["first"], case["last"])
        out = ops.paged_attention(state["q"], state["keys"], state["values"], state["table"], state["lengths"], state["scale"], pages, *exponents)
    else:
        pages = _plain_select(state)
        out = _plain_attend(state, pages)
    return {"pages": pages, "out": out}


def _plain_append(state):
    case, k, v, q = state["case"], state["k"].float(), state["v"].float(), state["q"].float()
    lengths, table, page = state["lengths"].long(), state["table"], case["page"]
    token = torch.arange(k.shape[0], device=k.device)
    if state["offsets"] is None:
        seq, position = token, lengths - 1
    else:
        ends = state["offsets"][1:].long()
        seq = torch.searchsorted(ends, token, right=True)
        position = lengths[seq] - ends[seq] + token
    row, slot = table[seq, position // page].long(), position % page
    if case["rotary"]:
        r = case["rotary"]
        c, s = state["rotation"][position, None, :r // 2], state["rotation"][position, None, r // 2:]

        def rotate(x):
            if case["interleaved"]:
                a, b = x[..., 0:r:2], x[..., 1:r:2]
                y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
            else:
                a, b = x[..., :r // 2], x[..., r // 2:r]
                y = torch.cat([a * c - b * s, b * c + a * s], -1)
            return torch.cat([y, x[..., r:]], -1)

        q, k = rotate(q), rotate(k)
    dtype = TYPES[case["type"]]
    if case["cache"] == "e4m3":
        codes, exponent = _to_e4m3(k)
        stored = _values(codes, exponent).to(dtype).float()
        state["keys"].view(torch.uint8)[row, :, slot] = codes.view(torch.uint8)
        state["key_exponents"][row, :, slot] = exponent
        codes, exponent = _to_e4m3(v)
        state["values"].view(torch.uint8)[row, :, slot] = codes.view(torch.uint8)
        state["value_exponents"][row, :, slot] = exponent
    else:
        stored = k.to(dtype)
        state["keys"][row, :, slot] = stored
        state["values"][row, :, slot] = state["v"]
        stored = stored.float()
    if "bounds" in state:
        begun = torch.zeros(state["keys"].shape[0], dtype=torch.int32, device=k.device).index_reduce_(0, row, (slot == 0).int(), "amax")
        fresh = (begun > 0)[:, None, None]
        low, high = state["bounds"][:, :, 0].float(), state["bounds"][:, :, 1].float()
        low = torch.where(fresh, math.inf, low).index_reduce_(0, row, stored, "amin")
        high = torch.where(fresh, -math.inf, high).index_reduce_(0, row, stored, "amax")
        state["bounds"][:, :, 0], state["bounds"][:, :, 1] = low.to(dtype), high.to(dtype)
    return q.to(dtype)


def _plain_select(state):
    case, table, lengths = state["case"], state["table"], state["lengths"]
    kv, dim = case["kv_heads"], case["dim"]
    q = state["q"].double().reshape(case["seqs"], kv, -1, dim)
    weights = torch.cat([q.clamp(max=0).sum(2), q.clamp(min=0).sum(2)], -1)                      # (seqs, kv, 2 dim): of the smallest, of the largest
    bounds = state["bounds"][table.clamp(min=0).long()].double().flatten(3)                      # (seqs, width, kv, 2 dim)
    score = (bounds * weights[:, None]).sum(-1).float().transpose(1, 2)                          # rounded once
    number = torch.arange(table.shape[1], device=table.device)
    used = ((lengths + case["page"] - 1) // case["page"])[:, None]
    kept = (number < case["first"]) | (number >= used - case["last"])
    score = torch.where(kept[:, None], math.inf, score)
    score = torch.where((number < used)[:, None], score, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :case["count"]]       # (ties: the lower page first)
    best = torch.where(best < used[..., None], best, table.shape[1]).sort(-1)[0]
    best = torch.where(best < table.shape[1], best, -1).to(torch.int32)
    missing = case["count"] - best.shape[-1]
    return torch.nn.functional.pad(best, (0, missing), value=-1) if missing > 0 else best


def _plain_attend(state, pages):
    case, table, lengths, page = state["case"], state["table"], state["lengths"], state["case"]["page"]
    seqs, kv, dim = case["seqs"], case["kv_heads"], case["dim"]
    slot = torch.arange(page, device=table.device)
    if pages is None:
        index = table.clamp(min=0).long()                                                        # (seqs, width)
        position = torch.arange(table.shape[1], device=table.device)[:, None] * page + slot
        there = (position < lengths[:, None, None])[:, None]                                     # (seqs, 1, width, page)

        def taken(rows, exponents):
            x = _values(_take(rows, index), None if exponents is None else exponents[index])
            return x.transpose(1, 2).reshape(seqs, kv, -1, dim)
    else:
        listed_page = pages.clamp(min=0).long()                                                  # (seqs, kv, count)
        index = torch.gather(table[:, None].expand(-1, kv, -1), 2, listed_page).clamp(min=0).long()
        head = torch.arange(kv, device=table.device)[:, None]
        there = (listed_page[..., None] * page + slot < lengths[:, None, None, None]) & (pages >= 0)[..., None]

        def taken(rows, exponents):
            x = rows.view(torch.uint8)[index, head].view(rows.dtype) if exponents is not None else rows[index, head]
            return _values(x, None if exponents is None else exponents[index, head]).reshape(seqs, kv, -1, dim)

    q = state["q"].float().reshape(seqs, kv, -1, dim)
    score = torch.matmul(q, taken(state["keys"], state.get("key_exponents")).transpose(2, 3).contiguous()) * state["scale"]
    there = there.flatten(2)[:, :, None]
    score = torch.where(there, score, -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    weight = weight / weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, taken(state["values"], state.get("value_exponents")))
    return out.reshape(seqs, case["heads"], dim).to(TYPES[case["type"]])


def work(case):
    size = 1 if case["cache"] == "e4m3" else 2
    kv, dim, heads, page, seqs = case["kv_heads"], case["dim"], case["heads"], case["page"], case["seqs"]
    row = dim * size + (1 if size == 1 else 0)                 # one token's key (or value) of one head in the cache
    lengths = _lengths(case)
    if case["kind"] == "append":
        new = _new(case)
        n = sum(new)
        touched = sum(_pages(a, page) - (a - b) // page for a, b in zip(lengths, new))
        moved = n * (2 * kv * dim * 2 + 2 * heads * dim * 2 + 2 * kv * row) + touched * 4
        if case["rotary"]:
            moved += n * case["rotary"] * 4
        if case["bounds"]:
            begun = sum(_pages(a, page) - _pages(a - b, page) for a, b in zip(lengths, new))
            moved += (2 * touched - begun) * kv * 2 * dim * 2   # written, and read where a page had tokens
        return {"bytes": moved, "flops": n * (heads + kv) * case["rotary"] * 3 + n * kv * dim * 2}
    q = 2 * seqs * heads * dim * 2
    if case["kind"] == "attend":
        attended = sum(lengths)
        return {"bytes": attended * kv * 2 * row + q + sum(_pages(n, page) for n in lengths) * 4, "flops": 4 * attended * heads * dim}
    pages = sum(_pages(n, page) for n in lengths)
    attended = sum(n if _pages(n, page) <= case["count"] else case["count"] * page for n in lengths)
    listed_pages = seqs * kv * case["count"] * 4
    return {"bytes": pages * (4 + kv * 2 * dim * 2) + attended * kv * 2 * row + q + 2 * listed_pages,
            "flops": pages * kv * 4 * dim + 4 * attended * heads * dim}


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence."""
    state = prepare(case, seed)
    f64 = torch.float64
    kv, dim, page, group = case["kv_heads"], case["dim"], case["page"], case["heads"] // case["kv_heads"]
    lengths, table = _lengths(case), state["table"].long()
    q = state["q"].to(f64)

    def cached(name, rows):
        """(rows, kv, page, dim) of the cache's pages ``rows``."""
        codes = state[name][rows] if case["cache"] == "16" else state[name].view(torch.uint8)[rows].view(torch.float8_e4m3fn).float()
        x = codes.to(f64)
        return x if case["cache"] == "16" else x * 2.0 ** (state[{"keys": "key_exponents", "values": "value_exponents"}[name]][rows].to(f64) - 127.0)[..., None]

    if case["kind"] == "append":
        r, at, turned_q, new = case["rotary"], 0, q.clone(), _new(case)
        keys, values = (state["keys"].to(f64), state["values"].to(f64)) if case["cache"] == "16" else (None, None)
        bounds = state["bounds"].to(f64) if "bounds" in state and keys is not None else None
        for s, (length, n) in enumerate(zip(lengths, new)):
            position = torch.arange(length - n, length, device=q.device)
            k = state["k"][at:at + n].to(f64)
            if r:
                frequency = torch.exp(torch.arange(0, r, 2, dtype=f64, device=q.device) * (-math.log(10000.0) / r))
                turn = torch.polar(torch.ones(n, r // 2, dtype=f64, device=q.device), position.to(f64)[:, None] * frequency)[:, None]
                first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
                for x in (k, turned_q[at:at + n]):
                    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
                    x[..., first], x[..., second] = z.real, z.imag
            if keys is not None:
                where = table[s][position // page]
                keys[where, :, position % page] = k
                values[where, :, position % page] = state["v"][at:at + n].to(f64)
                if bounds is not None:
                    for p in range(int(position[0]) // page, (length - 1) // page + 1):
                        mine = k[max(0, p * page - (length - n)):(p + 1) * page - (length - n)]
                        low, high, b = mine.amin(0), mine.amax(0), bounds[table[s, p]]
                        started = p * page >= length - n
                        bounds[table[s, p]] = torch.stack([low if started else torch.minimum(low, b[:, 0]), high if started else torch.maximum(high, b[:, 1])], 1)
            at += n
        out = {"q": turned_q, "keys": keys, "values": values}
        if "bounds" in state:
            out["bounds"] = bounds
        return out

    out = torch.zeros_like(q)
    for s, length in enumerate(lengths):
        used = _pages(length, page)
        query = q[s].reshape(kv, group, dim)
        rows = table[s, :used]
        position = torch.arange(used * page, device=q.device)
        if case["kind"] == "select" and used > case["count"]:
            low, high = state["bounds"][rows].to(f64).unbind(2)                                   # (used, kv, dim)
            score = torch.zeros(used, kv, dtype=f64, device=q.device)
            for g in range(group):
                score += torch.maximum(query[:, g] * low, query[:, g] * high).sum(-1)
            score[:case["first"]] = math.inf
            score[used - case["last"]:] = math.inf
            chosen = torch.argsort(score.float(), dim=0, descending=True, stable=True)[:case["count"]].sort(0)[0]     # (count, kv)
            heads = torch.arange(kv, device=q.device)
            k, v = (cached(name, rows[chosen.flatten()]).view(case["count"], kv, kv, page, dim)[:, heads, heads] for name in ("keys", "values"))
            position = (chosen.T[..., None] * page + torch.arange(page, device=q.device)).reshape(kv, -1)
        else:
            k, v = cached("keys", rows), cached("values", rows)
        k, v = (x.transpose(0, 1).reshape(kv, -1, dim) for x in (k, v))
        score = torch.matmul(query, k.transpose(1, 2).contiguous()) * state["scale"]
        score = score.masked_fill((position >= length).view(-1, 1, position.shape[-1]), -math.inf)
        out[s] = torch.matmul(torch.softmax(score, -1), v).reshape(-1, dim)
    return out if case["kind"] == "attend" else {"pages": None, "out": out}
