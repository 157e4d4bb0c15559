"""Appending to a paged cache, attention of single tokens over it and selection of its pages, against plain forms in 64 bits."""
import math

import pytest
import torch

from _paged import E4M3, HALF_STEP, Cache, feature_major, rotated, rotation_table, to_e4m3

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(dev):
    return torch.ops.iex_ops


def within(got, want, allowed, what=""):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    off = torch.where(want.isfinite(), (got - want).abs() - allowed, 0.0)
    assert torch.equal(got[~want.isfinite() & ~want.isnan()], want[~want.isfinite() & ~want.isnan()]), what
    assert not (off > 0).any(), f"{what}: {float(off.max())} beyond what is allowed, at {torch.nonzero(off == off.max())[0].tolist()}"


# ---- appending ------------------------------------------------------------------------------------------------------
def append(ops, c, k, v, offsets=None, q=None, rotation=None, interleaved=False):
    return ops.kv_append_(k, v, c.keys, c.values, c.table, c.lengths, offsets, q, rotation, interleaved, c.bounds, *c.exponents())


def check_append(ops, dev, new, before, kv_heads, heads, dim, page, dtype, e8, rotary, interleaved, bounds, layout, seed=1, extra=0, single=False, strided=False):
    lengths = [a + b for a, b in zip(new, before)]
    c = Cache(dev, lengths, kv_heads, dim, page, dtype, e8=e8, bounds=bounds, seed=seed, poison=False, strided=strided)
    n = sum(new) + extra
    gen = torch.Generator(device=dev).manual_seed(seed + 100)
    k, v, q = (torch.randn(n, h, dim, generator=gen, device=dev).to(dtype) * 3 for h in (kv_heads, kv_heads, heads))
    if bounds:   # as they were before the call
        for s, b in enumerate(before):
            for i in range(-(-lengths[s] // page)):
                if i * page < b:
                    c.set_bounds(int(c.table[s, i]), min(page, b - i * page))
    rotation = rotation_table(c.width * page, rotary, dev) if rotary else None
    old = {name: getattr(c, name).clone() for name in ("keys", "values", "key_exponents", "value_exponents", "bounds") if getattr(c, name) is not None}
    offsets = None if single else torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    shape = feature_major if layout == "features" else lambda x: x
    got_q = append(ops, c, shape(k), shape(v), offsets, shape(q), rotation, interleaved)
    assert got_q.shape == q.shape and got_q.stride() == shape(q).stride()

    places, token = [], 0
    positions = torch.zeros(n, dtype=torch.int64, device=dev)
    for s in range(len(new)):
        for i in range(new[s]):
            at = before[s] + i
            places.append((int(c.table[s, at // page]), at % page))
            positions[token] = at
            token += 1
    total = token
    pages = torch.tensor([p for p, _ in places], dtype=torch.int64, device=dev)
    slots = torch.tensor([x for _, x in places], dtype=torch.int64, device=dev)
    want_q, slack = rotated(q, positions, rotation, interleaved)
    tiny = 2.0 ** -25
    within(got_q[:total], want_q[:total], want_q[:total].abs() * HALF_STEP[dtype] + 2 * slack[:total] + tiny, "q")
    assert (got_q[total:] == 0).all()
    want_k, slack = rotated(k[:total], positions[:total], rotation, interleaved)
    if total:
        for name, want, loose in (("keys", want_k, slack), ("values", v[:total].double(), torch.zeros_like(slack))):
            now = c.stored(name, pages)[torch.arange(total, device=dev), :, slots]
            if e8:
                # half a step of a normal code (2^-4 of it), or of the least exponent's: 2^-10 of the row's scale, which is at most the row's largest / 224
                scale = want.abs().amax(-1, keepdim=True) / 224
                within(now, want, want.abs() * HALF_STEP[E4M3] + 2.0 ** -10 * scale + 2 * loose, name)
            else:
                within(now, want, want.abs() * HALF_STEP[dtype] + 2 * loose + tiny, name)
                if not rotary or name == "values":
                    assert torch.equal(now, want)
        if e8:
            _, exponents = to_e4m3(v[:total])
            assert torch.equal(c.value_exponents[pages, :, slots], exponents)
            codes = c.values.view(torch.uint8)[pages, :, slots].view(E4M3)
            assert torch.equal(codes.float(), to_e4m3(v[:total])[0].float())
    # everything else is as it was
    for name in ("keys", "values"):
        now, then = getattr(c, name), old[name]
        now, then = (x.view(torch.uint8).clone() if e8 else x.clone() for x in (now, then))
        now[pages, :, slots] = 0
        then[pages, :, slots] = 0
        assert torch.equal(now, then)
    if bounds:
        want = Cache.__new__(Cache)
        want.__dict__.update(c.__dict__)
        want.bounds = old["bounds"].clone()
        touched = {}
        for s in range(len(new)):
            for at in range(before[s], lengths[s]):
                touched[int(c.table[s, at // page])] = min(page, lengths[s] - at // page * page)
        for p, count in touched.items():
            want.set_bounds(p, count)
        assert torch.equal(c.bounds, want.bounds)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("e8", [False, True])
@pytest.mark.parametrize("layout", ["tokens", "features"])
@pytest.mark.parametrize("dim,page,rotary,interleaved", [(128, 64, 128, False), (64, 16, 64, True), (256, 32, 256, False), (128, 16, 32, True), (64, 256, 0, False),
                                                         (128, 128, 64, False), (256, 16, 128, True)])
def test_append_one_token_each(ops, dev, dtype, e8, layout, dim, page, rotary, interleaved):
    check_append(ops, dev, [1] * 6, [0, 1, page - 1, page, 3 * page + 5, 15], 2, 6, dim, page, dtype, e8, rotary, interleaved, True, layout, single=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("e8", [False, True])
@pytest.mark.parametrize("layout", ["tokens", "features"])
@pytest.mark.parametrize("dim,page,rotary,interleaved,bounds", [(128, 64, 128, False, True), (64, 16, 64, True, True), (256, 32, 256, False, True), (128, 16, 32, True, False),
                                                                (64, 256, 0, False, True), (256, 16, 64, False, True), (128, 128, 112, False, False)])
def test_append_prompts(ops, dev, dtype, e8, layout, dim, page, rotary, interleaved, bounds):
    new = [1, 0, 130, 17, page, 65, 3, 0]
    before = [0, 9, 3, page - 1, page, 0, 2 * page - 1, 0]
    check_append(ops, dev, new, before, 2, 4, dim, page, dtype, e8, rotary, interleaved, bounds, layout, extra=5)


def test_append_many_sequences_and_strided_pages(ops, dev):
    """More sequences than a wavefront has lanes; keys and values side by side in one array; odd head counts."""
    new = [i % 4 for i in range(200)]
    before = [i * 7 % 50 for i in range(200)]
    check_append(ops, dev, new, before, 3, 5, 64, 16, BF16, False, 64, False, True, "tokens", strided=True)
    check_append(ops, dev, new, before, 1, 1, 128, 16, F16, True, 128, True, True, "features", strided=True)


def test_append_without_queries_or_tokens(ops, dev):
    c = Cache(dev, [5, 3], 2, 64, 16, F16, poison=False)
    k = torch.randn(2, 2, 64, device=dev).half()
    assert append(ops, c, k, k) is None
    assert torch.equal(c.keys[c.table[0, 0], :, 4], k[0]) and torch.equal(c.keys[c.table[1, 0], :, 2], k[1])
    before = c.keys.clone()
    assert append(ops, c, k[:0], k[:0], torch.zeros(3, dtype=torch.int32, device=dev)) is None
    empty = append(ops, c, k[:0], k[:0], torch.zeros(3, dtype=torch.int32, device=dev), q=k[:0])
    assert empty.shape == (0, 2, 64) and torch.equal(before, c.keys)


@pytest.mark.parametrize("layout", ["tokens", "features"])
def test_append_passes_over_what_has_no_place(ops, dev, layout):
    """Lengths beyond the table, short of the new tokens or negative; pages outside the cache; tokens behind the last sequence."""
    shape = feature_major if layout == "features" else lambda x: x
    c = Cache(dev, [40, 40, 40, 40, 40], 2, 64, 16, F16, poison=False, bounds=True)
    c.lengths = torch.tensor([40, 1000, 2, -3, 40], dtype=torch.int32, device=dev)
    c.table[4, 1], c.table[4, 2] = -1, c.pages
    k = torch.randn(20, 2, 64, device=dev).half()
    q = torch.randn(20, 4, 64, device=dev).half()
    old_k, old_v, old_b = c.keys.clone(), c.values.clone(), c.bounds.clone()
    offsets = torch.tensor([0, 3, 6, 9, 12, 15], dtype=torch.int32, device=dev)
    out = append(ops, c, shape(k), shape(k), offsets, shape(q))
    assert torch.equal(out[:3], q[:3]) and torch.equal(out[12:15], q[12:15])
    assert (out[3:12] == 0).all() and (out[15:] == 0).all()
    page = int(c.table[0, 2])
    assert torch.equal(c.keys[page, :, 5:8], k[:3].transpose(0, 1))
    old_k[page, :, 5:8] = old_v[page, :, 5:8] = k[:3].transpose(0, 1)
    assert torch.equal(c.keys, old_k) and torch.equal(c.values, old_v)
    old_b[page] = c.bounds[page]
    assert torch.equal(c.bounds, old_b)
    # offsets that nobody has checked
    wild = torch.tensor([5, -9, 40, 2, 100, 7], dtype=torch.int32, device=dev)
    append(ops, c, shape(k), shape(k), wild, shape(q))
    torch.cuda.synchronize()


@pytest.mark.parametrize("e8", [False, True])
def test_append_in_pieces_is_append_at_once(ops, dev, e8):
    """The cache after a prompt does not depend on how it came: bit for bit, bounds included."""
    n, page = 150, 64
    make = lambda: Cache(dev, [n, n], 2, 128, page, BF16, e8=e8, bounds=True, seed=5, poison=False)  # noqa: E731
    whole, pieces = make(), make()
    for c in (whole, pieces):
        c.bounds.fill_(7.0)
    rotation = rotation_table(whole.width * page, 128, dev)
    k, v, q = (torch.randn(2, n, h, 128, device=dev).to(BF16) for h in (2, 2, 4))
    flat = lambda x, a, b: x[:, a:b].reshape(-1, *x.shape[2:])  # noqa: E731
    out = append(ops, whole, flat(k, 0, n), flat(v, 0, n), torch.tensor([0, n, 2 * n], dtype=torch.int32, device=dev), flat(q, 0, n), rotation)
    out = out.view(2, n, 4, 128)
    for a, b in ((0, 1), (1, 63), (63, 64), (64, 70), (70, 149), (149, 150)):
        pieces.lengths.fill_(b)
        offsets = torch.tensor([0, b - a, 2 * (b - a)], dtype=torch.int32, device=dev) if b - a > 1 else None
        part = append(ops, pieces, flat(k, a, b), flat(v, a, b), offsets, flat(q, a, b), rotation)
        assert torch.equal(part.view(2, b - a, 4, 128), out[:, a:b])
    used = whole.table.long().flatten()
    for name in ("keys", "values", "key_exponents", "value_exponents"):
        x, y = getattr(whole, name), getattr(pieces, name)
        if x is not None:
            x, y = (t.view(torch.uint8) if t.dtype == E4M3 else t for t in (x, y))
            assert torch.equal(x, y), name
    assert torch.equal(whole.bounds[used], pieces.bounds[used])


def test_append_rows_with_infinities_and_nan(ops, dev):
    """16 bits keep them; e4m3, which has no infinity, has NaN in their place and the row's finite values beside them; bounds show NaN."""
    x = torch.randn(4, 1, 64, device=dev).half()
    x[0, 0, 3], x[1, 0, 7], x[2, 0, 9], x[3] = math.inf, -math.inf, math.nan, 0.0
    for e8 in (False, True):
        c = Cache(dev, [9, 9, 9, 9], 1, 64, 16, F16, e8=e8, bounds=True, poison=False)
        c.bounds.zero_()
        append(ops, c, x, x)
        for s in range(4):
            page = int(c.table[s, 0])
            row = c.stored("keys", page)[0, 8]
            want = x[s, 0].double()
            if e8:
                want = torch.where(want.isfinite(), want, math.nan)
                assert torch.equal(row.isnan(), want.isnan())
            else:
                assert torch.equal(row.nan_to_num(5e5, 6e5, 7e5), want.nan_to_num(5e5, 6e5, 7e5))
            low, high = c.bounds[page, 0].double()
            zero = torch.zeros_like(row)
            assert torch.equal(low.nan_to_num(5e5), torch.minimum(zero, row).nan_to_num(5e5)) and torch.equal(high.nan_to_num(5e5), torch.maximum(zero, row).nan_to_num(5e5))


# ---- attention ------------------------------------------------------------------------------------------------------
def attend(ops, c, q, scale=None, pages=None):
    return ops.paged_attention(q, c.keys, c.values, c.table, c.lengths, scale, pages, *c.exponents())


def queries(dev, seqs, heads, dim, dtype, layout="tokens", seed=3, size=1.0):
    q = torch.randn(seqs, heads, dim, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).mul(size).to(dtype)
    return feature_major(q) if layout == "features" else q


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("e8", [False, True])
@pytest.mark.parametrize("dim,page,kv_heads,heads,layout", [(128, 64, 2, 8, "tokens"), (64, 16, 3, 3, "features"), (256, 32, 1, 6, "tokens"), (128, 16, 1, 17, "features"),
                                                            (64, 256, 2, 2, "tokens"), (256, 128, 2, 40, "features")])
def test_attention(ops, dev, dtype, e8, dim, page, kv_heads, heads, layout):
    lengths = [0, 1, 15, 16, 17, 33, 127, 128, 129, 300, 700]
    c = Cache(dev, lengths, kv_heads, dim, page, dtype, e8=e8)
    q = queries(dev, len(lengths), heads, dim, dtype, layout, size=2.0)
    scale = 1 / math.sqrt(dim)
    got = attend(ops, c, q)
    assert got.stride() == q.stride()
    assert (got[0] == 0).all()
    within(got, *c.attend(q, scale), "attention")
    assert torch.equal(attend(ops, c, q, scale), got)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [[77, 130, 200, 65], [129, 64, 1, 190], [5, 3, 376]])
def test_append_columns_of_sequences_off_the_chunk(ops, dev, dim, new):
    """Features of whole chunks of tokens whose sequences begin anywhere, in tiles of 64 and what is left of them."""
    check_append(ops, dev, new, [0] * len(new), 2, 3, dim, 64, BF16, False, dim, False, True, "features", extra=-sum(new) % 8)
    check_append(ops, dev, new, [64] + [63] * (len(new) - 1), 1, 2, dim, 16, F16, True, 64, True, False, "features", extra=8 - sum(new) % 8)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("e8", [False, True])
@pytest.mark.parametrize("dim,kv_heads,heads,layout", [(64, 2, 6, "tokens"), (128, 1, 17, "features"), (256, 3, 3, "tokens"), (256, 1, 20, "features")])
def test_attention_of_short_tables(ops, dev, dtype, e8, dim, kv_heads, heads, layout):
    """Tables of up to 64 tokens, and one page more."""
    for page, lengths in ((16, [0, 1, 15, 16]), (16, [3, 17, 33, 47, 48, 49, 63, 64]), (32, [31, 32, 33, 64, 0]), (64, [1, 64, 30]), (16, [65, 64, 80]), (64, [128, 7])):
        c = Cache(dev, lengths, kv_heads, dim, page, dtype, e8=e8)
        q = queries(dev, len(lengths), heads, dim, dtype, layout, size=2.0)
        within(attend(ops, c, q), *c.attend(q, dim ** -0.5), f"{page} {lengths}")


@pytest.mark.parametrize("e8", [False, True])
@pytest.mark.parametrize("lengths,kv_heads,heads,dim,page", [([9000], 2, 4, 128, 64), ([5000, 3, 0, 1700], 1, 2, 64, 16), ([2500] * 3, 1, 5, 256, 256)])
def test_attention_in_parts(ops, dev, e8, lengths, kv_heads, heads, dim, page):
    c = Cache(dev, lengths, kv_heads, dim, page, BF16, e8=e8)
    q = queries(dev, len(lengths), heads, dim, BF16, size=3.0)
    got = attend(ops, c, q, 0.1)
    within(got, *c.attend(q, 0.1), "in parts")
    for _ in range(3):
        assert torch.equal(attend(ops, c, q, 0.1), got)      # (the parts meet in one order)


def test_attention_of_more_sequences_than_lanes(ops, dev):
    lengths = [(i * 37) % 400 for i in range(150)]
    c = Cache(dev, lengths, 1, 64, 16, F16)
    q = queries(dev, 150, 2, 64, F16)
    within(attend(ops, c, q), *c.attend(q, 1 / 8), "many sequences")


@pytest.mark.parametrize("e8", [False, True])
def test_attention_over_strided_pages_and_tables(ops, dev, e8):
    c = Cache(dev, [70, 300], 2, 128, 32, BF16, e8=e8, width=16, strided=True)
    wide = torch.full((2, 40), 10 ** 6, dtype=torch.int32, device=dev)
    wide[:, 3:19] = c.table
    c.table = wide[:, 3:19]
    q = queries(dev, 2, 4, 128, BF16)[:, :, ::1]
    padded = torch.zeros(2, 9, 200, dtype=BF16, device=dev)
    padded[:, 2:6, 7:135] = q
    got = attend(ops, c, padded[:, 2:6, 7:135])
    within(got, *c.attend(q, 128 ** -0.5), "strided")


def test_attention_passes_over_pages_that_were_given_back(ops, dev):
    c = Cache(dev, [200, 64, 40], 2, 64, 16, F16)
    c.table[0, 0], c.table[0, 5], c.table[0, 12] = -1, c.pages, 2 ** 31 - 1
    c.table[1] = -7
    c.lengths[2] = 10 ** 9      # cut to what the table holds, whose entries there are -1
    q = queries(dev, 3, 4, 64, F16)
    got = attend(ops, c, q)
    within(got, *c.attend(q, 1 / 8), "given back")
    assert (got[1] == 0).all()
    c.lengths[0] = -5
    assert (attend(ops, c, q)[0] == 0).all()


@pytest.mark.parametrize("e8", [False, True])
def test_attention_over_listed_pages(ops, dev, e8):
    c = Cache(dev, [1000, 37, 0, 500], 2, 128, 16, F16, e8=e8)
    q = queries(dev, 4, 6, 128, F16)
    pages = torch.randint(-2, 70, (4, 2, 11), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    pages[0, 0] = torch.tensor([0, 5, 5, 62, 61, 3, -1, 63, 2 ** 31 - 1, -2 ** 31, 62])      # twice, past the end, out of order
    pages[3, 1] = -1
    pages = pages.to(dev)
    got = attend(ops, c, q, pages=pages)
    within(got, *c.attend(q, 128 ** -0.5, pages), "listed")
    assert (got[2] == 0).all() and (got[3, 3:] == 0).all()
    assert (attend(ops, c, q, pages=pages[:, :, :0].contiguous()) == 0).all()
    every = torch.arange(c.width, dtype=torch.int32, device=dev).expand(4, 2, -1).contiguous()
    within(attend(ops, c, q, pages=every), *c.attend(q, 128 ** -0.5), "all listed")


def test_attention_shows_what_it_attends_to(ops, dev):
    """Infinities and NaN among the attended keys and values come out as the formula has it."""
    c = Cache(dev, [60] * 6, 1, 64, 16, F16, poison=False)
    q = queries(dev, 6, 1, 64, F16).abs() + 0.1
    put = lambda s, t, x, what: getattr(c, what)[c.table[s, t // 16], 0, t % 16].fill_(x)  # noqa: E731
    for t in range(60):
        put(1, t, -math.inf, "keys")      # scores of -infinity only: NaN
    put(2, 7, -math.inf, "keys")          # one: no trace
    put(3, 7, math.inf, "keys")           # +infinity: NaN
    put(4, 7, math.nan, "keys")
    put(5, 7, math.inf, "values")
    got = attend(ops, c, q)
    want, allowed = c.attend(q, 1 / 8)
    assert got[1].isnan().all() and got[3].isnan().all() and got[4].isnan().all() and torch.isposinf(got[5]).all()
    within(got[[0, 2]], want[[0, 2]], allowed[[0, 2]], "beside them")


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_of_infinite_values(ops, dev, dtype, dim):
    """Infinities among the values come out with their sign whatever the bits of their weight (one, a power of two, any) and wherever
    the token is; both signs in a feature, and NaN, are NaN."""
    lengths = [1, 2, 4, 17, 60, 333, 1500, 60] + list(range(3, 43))
    c = Cache(dev, lengths, 2, dim, 16, dtype, poison=False, seed=7)
    q = queries(dev, len(lengths), 8, dim, dtype) * 0.25   # (weights of a row within a factor of 2^16)
    q[:3] = 0.0                                            # equal weights: 1, 1/2, 1/4
    for s, n in enumerate(lengths):
        for h in range(2):
            for d, (token, x) in enumerate(((0, math.inf), (n - 1, -math.inf), (n // 2, math.inf), (n // 3, math.nan))):
                c.values[c.table[s, token // 16], h, token % 16, d * 9 + h] = x
    c.values[c.table[7, 0], :, :2, 50] = torch.tensor([math.inf, -math.inf], device=dev, dtype=dtype)
    want, allowed = c.attend(q, dim ** -0.5)
    assert want[:, :, 9].isinf().any() and want[7, :, 50].isnan().all()
    within(attend(ops, c, q), want, allowed, "infinite values")


def test_scores_of_large_magnitude(ops, dev):
    """A score far above the rest after many small ones, and below: maxima that grow late and never."""
    c = Cache(dev, [400, 400], 1, 64, 16, BF16, poison=False)
    q = queries(dev, 2, 1, 64, BF16)
    for s, (token, factor) in enumerate(((399, 40.0), (0, 40.0))):
        c.keys[c.table[s, token // 16], 0, token % 16] = (q[s, 0].float() * factor).to(BF16)
    got = attend(ops, c, q, 1.0)
    within(got, *c.attend(q, 1.0), "large")


# ---- selection ------------------------------------------------------------------------------------------------------
def select(ops, c, q, count, first=1, last=1):
    return ops.select_pages(q, c.bounds, c.table, c.lengths, c.page, count, first, last)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,page,kv_heads,heads,layout", [(128, 16, 2, 8, "tokens"), (64, 16, 3, 3, "features"), (256, 32, 1, 6, "tokens"), (128, 64, 1, 20, "features")])
@pytest.mark.parametrize("count,first,last", [(1, 0, 0), (2, 1, 1), (7, 0, 3), (40, 1, 1)])
def test_select(ops, dev, dtype, dim, page, kv_heads, heads, layout, count, first, last):
    c = Cache(dev, [0, 1, 16, 17, 333, 1000, 1600], kv_heads, dim, page, dtype, bounds=True)
    q = queries(dev, 7, heads, dim, dtype, layout)
    got = select(ops, c, q, count, first, last)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), c.select(q, count, first, last))


def test_select_ties_unsound_pages_and_nan(ops, dev):
    c = Cache(dev, [640, 640, 640, 640], 1, 64, 16, BF16, bounds=True, poison=False)
    q = queries(dev, 4, 2, 64, BF16)
    c.bounds[c.table[0].long()] = c.bounds[c.table[0, 0].long()].clone()      # all alike: the lowest numbers
    c.table[1, 3], c.table[1, 39], c.table[1, 0] = -1, c.pages + 5, -2 ** 31   # never selected, not as first or last either
    c.bounds[c.table[2, 17].long(), 0, 1, 5] = math.nan                        # NaN comes first
    c.bounds[c.table[2, 9].long()] = math.inf
    c.bounds[c.table[3].long()] = 0.0                                          # zeros of either sign are equal
    c.bounds[c.table[3, 20].long()] = -0.0
    for count, first, last in ((5, 0, 0), (5, 1, 2), (39, 0, 1), (64, 1, 1)):
        got = select(ops, c, q, count, first, last).cpu()
        assert torch.equal(got, c.select(q, count, first, last)), (count, first, last)
    assert select(ops, c, q, 3, 0, 0)[0].tolist() == [[0, 1, 2]]


@pytest.mark.parametrize("tokens,page,count", [(200000, 16, 100), (16 * 12288, 16, 5000), (16 * 12289 + 1, 16, 12289)])
def test_select_of_many_pages(ops, dev, tokens, page, count):
    """More pages than fit in LDS, and just as many; scores in 64 bits of all pages at once."""
    pages = -(-tokens // page)
    bounds = torch.randn(pages, 1, 2, 64, device=dev).sort(2)[0].half()
    table = torch.randperm(pages, device=dev).to(torch.int32)[None]
    lengths = torch.tensor([tokens], dtype=torch.int32, device=dev)
    q = queries(dev, 1, 2, 64, F16)
    got = ops.select_pages(q, bounds, table, lengths, page, count, 1, 1)[0, 0].long()
    x = q[0].double()
    b = bounds[table[0].long(), 0].double()
    score = (b[:, 1] * x.clamp(min=0).sum(0) + b[:, 0] * x.clamp(max=0).sum(0)).sum(1).float()
    score[0] = score[-1] = math.inf
    want = torch.sort(score, descending=True, stable=True)[1][:count].sort()[0]
    assert torch.equal(got, want)
