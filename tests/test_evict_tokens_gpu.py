"""Tokens that got least attention leave a paged cache: which ones, where the others go, and what stays as it was."""
import math

import pytest
import torch

from _paged import Cache
from intrasm_engine_amd import _lib

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(dev):
    return torch.ops.iex_ops


def evict(ops, c, weights, keep, recent, first=0, bounds=None):
    return ops.evict_tokens_(c.keys, c.values, c.table, c.lengths, weights, keep, recent, first, bounds, *c.exponents())


def row_of(c, name, s, h, places):
    """What sequence s's key head h holds at some places, as bits."""
    places = torch.as_tensor(places, device=c.table.device)
    rows = getattr(c, name)
    rows = rows.view(torch.uint8) if c.e8 and name in ("keys", "values") else rows
    return rows[c.table[s, places // c.page].long(), h, places % c.page]


def plain(weights, length, keep, recent, first):
    """The kept tokens of one row, ascending."""
    if length <= keep:
        return list(range(length))
    w = weights[:length].double().cpu().tolist()
    rank = [(-math.inf, 0) if i < first or i >= length - recent else (-1.0, 0) if math.isnan(w[i]) else (0.0, -w[i]) for i in range(length)]
    return sorted(sorted(range(length), key=lambda i: (rank[i], i))[:keep])


def random_weights(c, seed=1, zeros=0.3):
    gen = torch.Generator(device=c.table.device).manual_seed(seed)
    w = torch.randn(c.lengths.numel(), c.kv_heads, c.width * c.page, generator=gen, device=c.table.device).mul(3).exp()
    return torch.where(torch.rand(w.shape, generator=gen, device=w.device) < zeros, 0.0, w)


def check(ops, c, weights, keep, recent, first=0, bounds=None, passed_over=()):
    names = [n for n in ("keys", "values", "key_exponents", "value_exponents") if getattr(c, n) is not None]
    old = Cache.__new__(Cache)
    old.__dict__.update(c.__dict__)
    for n in names:
        setattr(old, n, getattr(c, n).view(torch.uint8).clone().view(getattr(c, n).dtype) if c.e8 else getattr(c, n).clone())
    before, lengths, old_bounds = weights.clone(), c.lengths.clone(), None if bounds is None else bounds.clone()
    kept = evict(ops, c, weights, keep, recent, first, bounds)
    assert kept.shape == (c.lengths.numel(), c.kv_heads, keep) and kept.dtype == torch.int32
    touched = torch.zeros(c.pages, c.kv_heads, c.page, dtype=torch.bool, device=c.table.device)
    paged = torch.zeros(c.pages, dtype=torch.bool, device=c.table.device)
    for s in range(c.lengths.numel()):
        n = min(max(0, int(lengths[s])), c.width * c.page)
        cut = n > keep and s not in passed_over
        assert int(c.lengths[s]) == (keep if cut else int(lengths[s])), s
        for h in range(c.kv_heads):
            want = [] if s in passed_over else plain(before[s, h], n, keep, recent, first)
            assert kept[s, h].tolist() == want + [-1] * (keep - len(want)), (s, h)
            if not cut:
                assert torch.equal(weights[s, h].view(torch.int32), before[s, h].view(torch.int32))
                continue
            for name in names:
                assert torch.equal(row_of(c, name, s, h, range(keep)), row_of(old, name, s, h, want)), (s, h, name)
            assert torch.equal(weights[s, h, :keep].view(torch.int32), before[s, h, want].view(torch.int32))
            assert (weights[s, h, keep:n] == 0).all() and torch.equal(weights[s, h, n:], before[s, h, n:])
            places = torch.arange(keep, device=c.table.device)
            touched[c.table[s, places // c.page].long(), h, places % c.page] = True
        if cut:
            paged[c.table[s, :-(-keep // c.page)].long()] = True
    for name in names:   # everything else is as it was
        now, then = (x.view(torch.uint8) if c.e8 else x for x in (getattr(c, name), getattr(old, name)))
        now, then = now[~touched], then[~touched]
        assert torch.equal(now.view(torch.uint8), then.view(torch.uint8)), name
    if bounds is not None:
        plain_bounds = Cache.__new__(Cache)
        plain_bounds.__dict__.update(c.__dict__)
        plain_bounds.bounds = old_bounds
        for s in range(c.lengths.numel()):
            if min(int(lengths[s]), c.width * c.page) > keep and s not in passed_over:
                for i in range(-(-keep // c.page)):
                    plain_bounds.set_bounds(int(c.table[s, i]), min(c.page, keep - i * c.page))
        assert torch.equal(bounds, plain_bounds.bounds)


@pytest.mark.parametrize("dtype,e8", [(F16, False), (BF16, True)])
@pytest.mark.parametrize("dim,page,kv_heads,keep,recent,first", [(64, 16, 2, 100, 20, 4), (128, 64, 1, 1, 0, 0), (256, 32, 3, 33, 33, 0), (128, 256, 2, 300, 0, 7), (64, 128, 2, 129, 64, 65),
                                                                 (256, 16, 1, 64, 1, 1), (128, 16, 2, 2, 1, 1)])
def test_short_rows(ops, dev, dtype, e8, dim, page, kv_heads, keep, recent, first):
    c = Cache(dev, [0, 1, keep - 1, keep, keep + 1, keep + 63, 2 * keep + 5, 700, 513], kv_heads, dim, page, dtype, e8=e8, bounds=True, width=max(-(-(2 * keep + 5) // page), -(-700 // page)) + 1)
    check(ops, c, random_weights(c), keep, recent, first, c.bounds)


@pytest.mark.parametrize("dtype,e8,dim", [(F16, False, 64), (BF16, False, 128), (F16, False, 256), (BF16, True, 64), (F16, True, 128), (BF16, True, 256)])
def test_many_chunks(ops, dev, dtype, e8, dim):
    """Rows of many chunks, some nearly all of which move far and some where only the end does; LDS and not."""
    for width, seed in ((50, 1), (200, 2)):
        c = Cache(dev, [3000, 2999, 2300, 12800 if width == 200 else 1700], 2, dim, 64, dtype, e8=e8, width=width, spare=500 if width == 200 else 3, poison=False)
        weights = random_weights(c, seed)
        weights[1, 0, :1500] += 1e6          # the first half stays where it is
        weights[1, 1, 1500:2999] += 1e6      # the second half moves to the front
        weights[2, 0, ::2] += 1e6
        check(ops, c, weights, 1500, 100, 3)


@pytest.mark.parametrize("keep,recent,first", [(1, 0, 0), (16383, 300, 2), (8192, 8192, 0), (20000, 0, 19000), (33000, 1, 1)])
def test_rows_in_slices(ops, dev, keep, recent, first):
    """Tables of more than 32768 tokens: lengths that end a slice, are short of one, fill the table; equal keys over slices' ends, and rows of nothing else."""
    lengths = [34000, 8192, 8193, 16384, 0, 5, 33024, 1 << 30, 33001]
    c = Cache(dev, [min(n, 34048) for n in lengths], 2, 64, 256, F16, poison=False, width=133, bounds=True)
    c.lengths[7] = lengths[7]
    weights = random_weights(c)
    weights[2, 0] = 0.5
    weights[3, :, 8000:8400] = 7e4
    weights[3, 1, 8100:16300] = 7e4
    weights[0, 0], weights[0, 0, 5000:30000:7] = -0.0, 1e-30
    weights[7, 1, ::3] = math.nan
    check(ops, c, weights, keep, recent, first, c.bounds)
    assert "evict_slice_kernel" in _lib.last_kernels()


def test_ties_and_values_that_are_not_numbers(ops, dev):
    """Equal weights: the earlier ones; negative ones, infinities, zeros of both signs; NaN is larger than everything."""
    c = Cache(dev, [200] * 6, 1, 64, 16, F16, poison=False)
    weights = torch.zeros(6, 1, c.width * 16, device=dev)
    weights[1, 0, ::3] = 1.0
    weights[2, 0, 50:60], weights[2, 0, 70] = math.nan, math.inf
    weights[3, 0] = -torch.arange(c.width * 16, device=dev).float()
    weights[4, 0, :150], weights[4, 0, 150:] = -math.inf, -0.0
    weights[5, 0, 1::2] = -0.0
    check(ops, c, weights, 60, 5, 2)


def test_sequences_passed_over(ops, dev):
    """Pages given back (in a sequence that would lose tokens), lengths beyond the table, lengths below zero."""
    c = Cache(dev, [200, 200, 30, 200, 200], 2, 64, 16, BF16, width=13, poison=False, bounds=True)
    c.table[0, 12], c.table[1, 0], c.table[2, 1] = -1, c.pages, -1
    c.lengths[3], c.lengths[4] = 1 << 30, -3
    check(ops, c, random_weights(c), 90, 10, 2, None, passed_over=(0, 1))


@pytest.mark.parametrize("e8", [False, True])
def test_strided_pages_tables_and_other_streams(ops, dev, e8):
    c = Cache(dev, [900, 333, 77], 3, 128, 32, F16, e8=e8, strided=True, poison=False)
    wide = torch.full((3, 2 * c.width), -1, dtype=torch.int32, device=dev)
    wide[:, :c.width] = c.table
    c.table = wide[:, :c.width]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        check(ops, c, random_weights(c), 128, 16, 4)
    torch.cuda.current_stream().wait_stream(stream)


def test_again_and_again(ops, dev):
    """What is left is cut again, down to one token, and a second call with the same budget changes nothing."""
    c = Cache(dev, [500, 40], 2, 64, 16, F16, poison=False, bounds=True)
    weights = random_weights(c, 9)
    for keep in (300, 299, 64, 63, 17, 1):
        check(ops, c, weights, keep, min(10, keep), 0, c.bounds)
        check(ops, c, weights, keep, min(10, keep), 0, c.bounds)


def test_replays_follow_what_is_there(ops, dev):
    c = Cache(dev, [500, 400], 2, 64, 16, F16, poison=False, width=40)
    weights, rows = random_weights(c), [x.clone() for x in (c.keys, c.values, c.lengths)]
    start = weights.clone()
    def restore():
        for x, y in zip((c.keys, c.values, c.lengths), rows):
            x.copy_(y)
        weights.copy_(start)
    evict(ops, c, weights, 200, 20, 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = evict(ops, c, weights, 200, 20, 2)
    for step in range(4):
        restore()
        c.lengths.copy_(torch.tensor([500 - 101 * step, 199 + step], device=dev))
        weights.add_(random_weights(c, 50 + step))
        state = [x.clone() for x in (c.keys, c.values, c.lengths, weights)]
        graph.replay()
        got = [x.clone() for x in (kept, c.keys, c.values, c.lengths, weights)]
        for x, y in zip((c.keys, c.values, c.lengths, weights), state):
            x.copy_(y)
        want = [evict(ops, c, weights, 200, 20, 2), c.keys, c.values, c.lengths, weights]
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_two_streams_and_threads(ops, dev):
    """Passes that keep account over one cache, each with an account of its own, and evictions of different sequences of it, at once on two streams."""
    import threading

    c = Cache(dev, [3000, 900, 2500, 1400], 2, 64, 16, F16, poison=False)
    halves = [slice(0, 2), slice(2, 4)]
    q = torch.randn(2, 2, 4, 64, generator=torch.Generator(device=dev).manual_seed(1), device=dev).half()

    def pass_over(i, cache, lengths, weights):
        out = [ops.paged_attention_accumulate_(q[i], cache.keys, cache.values, cache.table[halves[i]], lengths, weights, 0.2) for _ in range(5)]
        kept = ops.evict_tokens_(cache.keys, cache.values, cache.table[halves[i]], lengths, weights, 700, 100, 4)
        return [out[-1], kept, ops.paged_attention(q[i], cache.keys, cache.values, cache.table[halves[i]], lengths, 0.2)]

    def copy():
        new = Cache.__new__(Cache)
        new.__dict__.update(c.__dict__)
        new.keys, new.values = c.keys.clone(), c.values.clone()
        return new, [c.lengths[h].clone() for h in halves], [torch.zeros(2, 2, c.width * 16, device=dev) for _ in halves]

    alone, lengths, weights = copy()
    want = [pass_over(i, alone, lengths[i], weights[i]) for i in range(2)]
    both, lengths2, weights2 = copy()
    torch.cuda.synchronize()
    got, streams = [None, None], [torch.cuda.Stream() for _ in range(2)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            got[i] = pass_over(i, both, lengths2[i], weights2[i])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i])) and torch.equal(weights[i], weights2[i]) and torch.equal(lengths[i], lengths2[i])
    assert torch.equal(both.keys, alone.keys) and torch.equal(both.values, alone.values)


def test_a_budget_beyond_the_table(ops, dev):
    """Nothing ever leaves: the list is the tokens, whatever the budget; a length beyond the table stays as it is."""
    c = Cache(dev, [48, 20, 0], 2, 64, 16, F16, width=3, poison=False, bounds=True)
    c.lengths[0] = 1 << 20
    weights = random_weights(c)
    for keep in (48, 49, 100000):
        check(ops, c, weights, keep, 10, 2, c.bounds)
    assert c.lengths.tolist() == [1 << 20, 20, 0]


def test_offsets_beyond_32_bits(ops, dev):
    """A cache of more than 2^31 elements, the sequence in its last pages."""
    pages, page, kv, dim = 140000, 64, 2, 128
    keys = torch.empty(pages, kv, page, dim, dtype=F16, device=dev)
    values = torch.empty_like(keys)
    table = torch.arange(pages - 1, pages - 11, -1, dtype=torch.int32, device=dev)[None]
    for x in (keys, values):
        x[-10:] = torch.randn(10, kv, page, dim, generator=torch.Generator(device=dev).manual_seed(2), device=dev).half()
    c = Cache.__new__(Cache)
    lengths = torch.tensor([640], dtype=torch.int32, device=dev)
    c.__dict__.update(table=table, lengths=lengths, page=page, dim=dim, kv_heads=kv, pages=pages, dtype=F16, e8=False, width=10, keys=keys, values=values, key_exponents=None,
                      value_exponents=None, bounds=None)
    weights = random_weights(c)
    old = keys[-10:].clone(), values[-10:].clone()
    kept = evict(ops, c, weights, 100, 10)
    for h in range(kv):
        for name, rows in (("keys", old[0]), ("values", old[1])):
            want = rows.flip(0)[:, h].reshape(-1, dim)[kept[0, h].long()]      # (the table counts down)
            assert torch.equal(row_of(c, name, 0, h, range(100)), want)


def test_attention_over_what_is_left(ops, dev):
    """Attention, account and eviction in turn: the tokens left are those that a plain account of the passes names, and what is attended to then is theirs."""
    c = Cache(dev, [300, 90], 2, 64, 16, F16, poison=False)
    weights = torch.zeros(2, 2, c.width * 16, device=dev)
    total = [[torch.zeros(n, dtype=torch.float64, device=dev) for _ in range(2)] for n in (300, 90)]
    for step in range(6):
        q = torch.randn(2, 4, 64, generator=torch.Generator(device=dev).manual_seed(step), device=dev).half() * 2
        ops.paged_attention_accumulate_(q, c.keys, c.values, c.table, c.lengths, weights, 0.3)
        for s in range(2):
            for h in range(2):
                k, _ = c.rows(s, h)
                total[s][h] += torch.softmax((k @ q[s, 2 * h:2 * h + 2].double().T).T * 0.3, -1).sum(0)
    kept = evict(ops, c, weights, 120, 30, 4)
    for h in range(2):
        middle = total[0][h][4:270]
        order = middle.sort(descending=True)[0]
        assert order[85] - order[86] > 1e-4 * order[85]      # (the account's roundings do not decide)
        want = sorted([0, 1, 2, 3] + [int(i) + 4 for i in middle.topk(86)[1]] + list(range(270, 300)))
        assert kept[0, h].tolist() == want
    q = torch.randn(2, 4, 64, generator=torch.Generator(device=dev).manual_seed(77), device=dev).half()
    want, allowed = c.attend(q, 0.3)
    assert c.lengths.tolist() == [120, 90]
    assert ((ops.paged_attention(q, c.keys, c.values, c.table, c.lengths, 0.3).double() - want).abs() <= allowed).all()


def test_kernels_and_changes_are_noted(ops, dev):
    c = Cache(dev, [100], 1, 64, 16, F16, poison=False, bounds=True)
    weights = random_weights(c)
    versions = [x._version for x in (c.keys, c.values, c.lengths, weights, c.bounds)]
    evict(ops, c, weights, 50, 10, 0, c.bounds)
    for name in ("evict_select_kernel", "evict_move_kernel<64, 16>", "evict_bounds_kernel<f16, 64, 16>"):
        assert name in _lib.last_kernels()
    assert all(x._version > v for x, v in zip((c.keys, c.values, c.lengths, weights, c.bounds), versions))


def test_refusals(ops, dev):
    c = Cache(dev, [48, 20], 2, 64, 16, F16, width=3, poison=False)
    weights = torch.zeros(2, 2, 48, device=dev)
    old = c.keys.clone()
    for keep, recent, first in ((0, 0, 0), (-3, 0, 0), (10, 11, 0), (10, 5, 6), (10, -1, 0), (10, 0, -1), (1 << 31, 0, 0)):
        with pytest.raises(RuntimeError, match="at least one token|too large"):
            evict(ops, c, weights, keep, recent, first)
    for bad in (weights[:1], weights.half(), weights.cpu(), torch.zeros(2, 2, 96, device=dev)[..., ::2], weights.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="weights must be|no gradient"):
            evict(ops, c, bad, 10, 0)
    with pytest.raises(RuntimeError, match="bounds must be"):
        evict(ops, c, weights, 10, 0, 0, torch.zeros(c.pages, 2, 2, 64, device=dev))
    with pytest.raises(RuntimeError, match="exponents"):
        ops.evict_tokens_(c.keys, c.values, c.table, c.lengths, weights, 10, 0, 0, None, torch.zeros(c.pages, 2, 16, dtype=torch.uint8, device=dev))
    with pytest.raises(RuntimeError, match="int32"):
        ops.evict_tokens_(c.keys, c.values, c.table, c.lengths.long(), weights, 10, 0)
    with pytest.raises(RuntimeError, match="fp16 or bf16"):
        ops.evict_tokens_(c.keys.float(), c.values.float(), c.table, c.lengths, weights, 10, 0)
    assert torch.equal(c.keys, old) and c.lengths.tolist() == [48, 20]
    kept = ops.evict_tokens_(c.keys, c.values, c.table[:0], c.lengths[:0], weights[:0], 5, 0)
    assert kept.shape == (0, 2, 5)
    kept = ops.evict_tokens_(c.keys[:0], c.values[:0], c.table, c.lengths, weights, 30, 0)      # every page is outside the cache
    assert (kept[0] == -1).all() and kept[1, 0].tolist() == list(range(20)) + [-1] * 10 and c.lengths.tolist() == [48, 20]
