"""The paged cache as a program uses it: prompts, then tokens one at a time, captured and not, on several streams, with selection; and
the calls that the operators refuse."""
import math

import pytest
import torch

from _paged import E4M3, HALF_STEP, Cache, feature_major, rotated, rotation_table
from intrasm_engine_amd import workloads as W
from intrasm_engine_amd.decoder_layer import SparseDecoderLayer
from intrasm_engine_amd.pytorch import paged_attention as PA
from intrasm_engine_amd.pytorch.utils import sparse_to_dense

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(dev):
    return torch.ops.iex_ops


def tables(dev, counts, spare=2, seed=0):
    """A table of pages in no order for sequences of so many pages, and how many pages there are."""
    order = torch.randperm(sum(counts) + spare, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return table.to(dev), sum(counts) + spare


def plain_step(q, keys, values, scale):
    """(heads, dim) queries over (n, kv_heads, dim) keys and values, in 64 bits."""
    group = q.shape[0] // keys.shape[1]
    k, v = (x.double().repeat_interleave(group, 1) for x in (keys, values))
    p = torch.softmax((k * q.double()).sum(-1) * scale, 0)
    return (p[..., None] * v).sum(0)


@pytest.mark.parametrize("dtype,kv_heads,heads,dim,page,interleaved", [(F16, 2, 4, 64, 16, False), (BF16, 1, 8, 128, 32, True), (F16, 3, 3, 256, 64, False)])
@pytest.mark.parametrize("eight_bits", [False, True])
def test_prompts_then_tokens(dev, dtype, kv_heads, heads, dim, page, interleaved, eight_bits):
    """Ragged prompts in one call, then steps: every step's result against all keys and values so far, kept plainly beside the cache."""
    gen = torch.Generator(device=dev).manual_seed(7)
    prompts, steps = [5, 40, 1, 17], 6
    table, pages = tables(dev, [-(-(n + steps) // page) for n in prompts])
    cache = PA.KVCache(pages, page, kv_heads, dim, dtype, dev, eight_bits)
    rotation = PA.rotation_table(table.shape[1] * page, dim, device=dev)
    assert torch.equal(rotation, rotation_table(table.shape[1] * page, dim, dev))
    lengths = torch.tensor(prompts, dtype=torch.int32, device=dev)
    offsets = torch.tensor([0] + prompts, device=dev).cumsum(0).to(torch.int32)
    draw = lambda n, h: torch.randn(n, h, dim, generator=gen, device=dev).to(dtype)  # noqa: E731
    k, v = draw(sum(prompts), kv_heads), draw(sum(prompts), kv_heads)
    cache.append_(k, v, table, lengths, offsets, None, rotation, interleaved)
    keys, values, at = [], [], 0
    for n in prompts:
        keys.append(rotated(k[at:at + n], torch.arange(n, device=dev), rotation, interleaved)[0])
        values.append(v[at:at + n].double())
        at += n
    for _ in range(steps):
        lengths += 1
        k, v, q = draw(4, kv_heads), draw(4, kv_heads), draw(4, heads)
        q = cache.append_(k, v, table, lengths, None, q, rotation, interleaved)
        out = cache.attend(q, table, lengths)
        for s in range(4):
            position = torch.tensor([len(keys[s])], device=dev)
            keys[s] = torch.cat([keys[s], rotated(k[s:s + 1], position, rotation, interleaved)[0]])
            values[s] = torch.cat([values[s], v[s:s + 1].double()])
            want = plain_step(q[s], keys[s], values[s], dim ** -0.5)
            # a key is a half step of its stored type off (codes below e4m3's normal ones 2^-10 of a scale that is at most the row's largest
            # / 224: 2^-17 of it, well under 2^-10 of sum |q k|), which moves a score by at most sum |q k| of that, a probability by
            # twice as much; a value likewise; the result is rounded once
            step = HALF_STEP[E4M3] + 2.0 ** -10 if eight_bits else HALF_STEP[dtype]
            group = heads // kv_heads
            magnitude = (keys[s].repeat_interleave(group, 1) * q[s].double()).abs().sum(-1).max() * dim ** -0.5
            largest = values[s].abs().max()
            allowed = want.abs() * HALF_STEP[dtype] + largest * (step + math.expm1(2 * step * float(magnitude)) + 2.0 ** -12)
            assert ((out[s].double() - want).abs() <= allowed).all()


@pytest.mark.parametrize("eight_bits", [False, True])
def test_selected_pages_are_where_the_keys_are(dev, eight_bits):
    """The bounds that appending keeps, read by the selection, read by the attention: each against its plain form on what the
    cache holds, over steps that end pages and begin them."""
    page, kv_heads, heads, dim, steps = 16, 2, 6, 64, 20
    prompts = [300, 33, 1]
    table, pages = tables(dev, [-(-(n + steps) // page) for n in prompts])
    cache = PA.KVCache(pages, page, kv_heads, dim, BF16, dev, eight_bits, bounds=True)
    for t in (cache.keys, cache.values):
        t.view(torch.uint8).zero_()
    plain = Cache.__new__(Cache)
    plain.__dict__.update(table=table, page=page, dim=dim, kv_heads=kv_heads, pages=pages, dtype=BF16, e8=eight_bits, width=table.shape[1], keys=cache.keys,
                          values=cache.values, key_exponents=cache.key_exponents, value_exponents=cache.value_exponents, bounds=torch.zeros_like(cache.bounds))
    rotation = PA.rotation_table(table.shape[1] * page, dim, device=dev)
    lengths = torch.tensor(prompts, dtype=torch.int32, device=dev)
    plain.lengths = lengths
    gen = torch.Generator(device=dev).manual_seed(3)
    draw = lambda n, h: torch.randn(n, h, dim, generator=gen, device=dev).to(BF16)  # noqa: E731
    offsets = torch.tensor([0] + prompts, device=dev).cumsum(0).to(torch.int32)
    cache.append_(draw(sum(prompts), kv_heads), draw(sum(prompts), kv_heads), table, lengths, offsets, None, rotation)
    for step in range(steps):
        lengths += 1
        q = cache.append_(draw(3, kv_heads), draw(3, kv_heads), table, lengths, None, draw(3, heads), rotation)
        chosen = cache.select(q, table, lengths, 5, 1, 2)
        out = cache.attend(q, table, lengths, 0.2, chosen)
        for s in range(3):
            n = int(lengths[s])
            for i in range(-(-n // page)):
                plain.set_bounds(int(table[s, i]), min(page, n - i * page))
                assert torch.equal(plain.bounds[table[s, i]], cache.bounds[table[s, i]])
        if step % 6 == 0 or step == steps - 1:
            assert torch.equal(chosen.cpu(), plain.select(q, 5, 1, 2))
            want, allowed = plain.attend(q, 0.2, chosen)
            assert ((out.double() - want).abs() <= allowed).all()


def layer(dev, hidden=256, heads=4, mlp=512):
    weights = {name: W.pruned_weight(100 + i, hidden, hidden, "2:4", sigma=0.06) for i, name in enumerate(("q", "k", "v", "o"))}
    weights |= {"gate": W.pruned_weight(104, mlp, hidden, 0.80, sigma=0.06), "up": W.pruned_weight(105, mlp, hidden, 0.80, sigma=0.06),
                "down": W.pruned_weight(106, hidden, mlp, 0.80, sigma=0.06)}
    return SparseDecoderLayer(weights, hidden, heads, mlp, dev), weights


def test_layer_generates(dev):
    """prompt() and decode() of the decoder layer against dense 32-bit matrices and plain attention with the same rotation."""
    made, weights = layer(dev)
    dense = {n: sparse_to_dense(c.m, c.k, torch.from_numpy(c.values).to(dev).half().float(), torch.from_numpy(c.row_offsets).to(dev),
                                torch.from_numpy(c.column_indices).to(dev)) for n, c in weights.items()}
    gen = torch.Generator().manual_seed(0)
    prompts, page = [24, 8], 16
    table, pages = tables(dev, [-(-(n + 4) // page) for n in prompts])
    cache = made.new_cache(pages, page, bounds=True)
    rotation = PA.rotation_table(table.shape[1] * page, made.head_dim, device=dev)
    lengths = torch.tensor(prompts, dtype=torch.int32, device=dev)
    x = torch.relu(torch.randn(256, sum(prompts), generator=gen)).half().to(dev)
    made.prompt(x, cache, table, lengths, torch.tensor([0, 24, 32], dtype=torch.int32, device=dev), rotation)
    split = lambda t: t.view(4, 64, -1).permute(2, 0, 1)  # noqa: E731
    turn = lambda t, p: rotated(t, p, rotation, False)[0].float()  # noqa: E731
    keys = [turn(split(dense["k"] @ x[:, a:b].float()), torch.arange(b - a, device=dev)) for a, b in ((0, 24), (24, 32))]
    values = [split(dense["v"] @ x[:, a:b].float()) for a, b in ((0, 24), (24, 32))]
    for step in range(4):
        lengths += 1
        x = torch.relu(torch.randn(256, 2, generator=gen)).half().to(dev)
        y = made.decode(x, cache, table, lengths, rotation, pages=8 if step % 2 else 0)      # (more pages than there are: all of them)
        q, k, v = (split(dense[n] @ x.float()) for n in ("q", "k", "v"))
        attended = []
        for s in range(2):
            at = torch.tensor([keys[s].shape[0]], device=dev)
            keys[s] = torch.cat([keys[s], turn(k[s:s + 1], at)])
            values[s] = torch.cat([values[s], v[s:s + 1]])
            attended.append(plain_step(turn(q[s:s + 1], at)[0], keys[s], values[s], 1 / 8).float())
        h = x.float() + dense["o"] @ torch.stack(attended).permute(1, 2, 0).reshape(256, 2)
        want = h + dense["down"] @ (torch.nn.functional.silu(dense["gate"] @ h) * (dense["up"] @ h))
        assert y.shape == x.shape and (y.float() - want).abs().max() <= 2e-2 * want.abs().max()      # (the layer's own measure: a chain of fp16 operators)


def test_captured_steps_follow_lengths_and_tables(dev):
    """One captured step of the layer, replayed over positions that end pages, against the eager step on a copy of the cache; then with
    another table."""
    made, _ = layer(dev)
    page, n0, steps = 16, 13, 9
    rotation = PA.rotation_table(4 * page, 64, device=dev)
    table, pages = tables(dev, [4, 4, 4])
    other, _ = tables(dev, [4, 4, 4], seed=5)
    gen = torch.Generator().manual_seed(0)
    prompt = torch.randn(256, 3 * n0, generator=gen).half().to(dev)
    xs = [torch.randn(256, 3, generator=gen).half().to(dev) for _ in range(steps)]
    for selected in (0, 2):
        caches = [made.new_cache(pages, page, bounds=True) for _ in range(2)]
        lengths, eager_lengths = (torch.full((3,), n0, dtype=torch.int32, device=dev) for _ in range(2))
        offsets = torch.tensor([0, n0, 2 * n0, 3 * n0], dtype=torch.int32, device=dev)
        live = table.clone()
        for c in caches:
            made.prompt(prompt, c, live, lengths, offsets, rotation)
        x = xs[0].clone()
        made.decode(x, made.new_cache(pages, page, bounds=True), live, lengths + 1, rotation, selected)      # (weights laid out, patterns looked at)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lengths += 1
            y = made.decode(x, caches[0], live, lengths, rotation, selected)
        for i, given in enumerate(xs):
            if i == steps - 2:      # somebody moves the sequences to other pages
                for c in caches:
                    for t in (c.keys, c.values, c.bounds):
                        moved = t.clone()
                        moved[other.flatten().long()] = t[table.flatten().long()]
                        t.copy_(moved)
                live.copy_(other)
            x.copy_(given)
            graph.replay()
            eager_lengths += 1
            want = made.decode(given, caches[1], live, eager_lengths, rotation, selected)
            torch.cuda.synchronize()
            # (the captured projections may be by another form of the weights: sums in another order)
            assert (y.float() - want.float()).abs().max() <= 2e-2 * want.float().abs().max(), i
            assert torch.equal(lengths, eager_lengths)


def test_replays_are_the_eager_bits(dev, ops):
    """Append, selection and attention captured together, rows in parts, replayed several times between eager work: bit for bit."""
    c = Cache(dev, [3000, 70, 1, 1500], 2, 128, 64, BF16, bounds=True, poison=False)
    k, v = (torch.randn(4, 2, 128, device=dev).to(BF16) for _ in range(2))
    q = torch.randn(4, 8, 128, device=dev).to(BF16)
    rotation = rotation_table(c.width * 64, 128, dev)

    def step():
        turned = ops.kv_append_(k, v, c.keys, c.values, c.table, c.lengths, None, q, rotation, False, c.bounds)
        pages = ops.select_pages(turned, c.bounds, c.table, c.lengths, 64, 6)
        return turned, pages, ops.paged_attention(turned, c.keys, c.values, c.table, c.lengths, None, pages), ops.paged_attention(turned, c.keys, c.values, c.table, c.lengths)

    step()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]      # two that share the cache
    results = []
    for g in graphs:
        with torch.cuda.graph(g):
            results.append(step())
    for i in range(5):
        q.copy_(torch.randn(4, 8, 128, device=dev).to(BF16))
        c.lengths.copy_(torch.tensor([3000 - 700 * i, 70 + i, 1, 1500], dtype=torch.int32))
        want = step()
        for g, got in zip(graphs, results):
            for t in got:
                t.view(torch.uint8).fill_(0x55)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_two_streams_at_once(dev, ops):
    """Calls that overlap on two streams, and from two threads, over one cache: each has its own workspace."""
    import threading

    c = Cache(dev, [20000, 9000], 2, 128, 64, F16, bounds=True)
    qs = [torch.randn(2, 8, 128, device=dev).half() for _ in range(2)]
    want = [ops.paged_attention(q, c.keys, c.values, c.table, c.lengths) for q in qs]
    chosen = [ops.select_pages(q, c.bounds, c.table, c.lengths, 64, 9) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]

    def work(i):
        with torch.cuda.stream(streams[i]):
            got[i] = [(ops.paged_attention(qs[i], c.keys, c.values, c.table, c.lengths), ops.select_pages(qs[i], c.bounds, c.table, c.lengths, 64, 9)) for _ in range(20)]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        for out, pages in got[i]:
            assert torch.equal(out, want[i]) and torch.equal(pages, chosen[i])


def test_caches_beyond_32_bit_offsets(dev, ops):
    """Pages whose elements lie past 2^31 and, 8-bit ones, bytes past 2^32."""
    pages, page, dim = 70000, 256, 128
    for dtype in (F16, E4M3):
        heads = 1 if dtype == F16 else 2
        keys = torch.empty(pages, heads, page, dim, dtype=dtype, device=dev)
        values = torch.empty_like(keys)
        assert keys.numel() > 2 ** 31 and keys.numel() * keys.element_size() > 2 ** 32
        exponents = [torch.full((pages, heads, page), 127, dtype=torch.uint8, device=dev) for _ in range(2)] if dtype == E4M3 else [None, None]
        table = torch.tensor([[pages - 1, pages - 2], [pages - 3, 0]], dtype=torch.int32, device=dev)
        n = 300
        lengths = torch.tensor([n, n], dtype=torch.int32, device=dev)
        k, v = (torch.randn(2 * n, heads, dim, device=dev).half() for _ in range(2))
        ops.kv_append_(k, v, keys, values, table, lengths, torch.tensor([0, n, 2 * n], dtype=torch.int32, device=dev), None, None, False, None, *exponents)
        if dtype == F16:
            assert torch.equal(keys[pages - 1, 0], k[:256, 0]) and torch.equal(values[0, 0, :44], v[n + 256:, 0])
        q = torch.randn(2, heads * 2, dim, device=dev).half()
        got = ops.paged_attention(q, keys, values, table, lengths, None, None, *exponents)
        small = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=dev)
        near = [t[table.flatten().long()].clone() if t.dtype != E4M3 else t.view(torch.uint8)[table.flatten().long()].clone().view(E4M3) for t in (keys, values)]
        near_exponents = [e[table.flatten().long()].clone() if e is not None else None for e in exponents]
        assert torch.equal(got, ops.paged_attention(q, *near, small, lengths, None, None, *near_exponents))
        assert got.abs().max() > 0
        del keys, values, near
        torch.cuda.empty_cache()


def test_what_an_eight_bit_cache_holds_of_infinities(dev, ops):
    """NaN codes come out as NaN where they are attended to and leave no trace where they are not."""
    c = Cache(dev, [20, 20, 20], 1, 64, 16, F16, e8=True)
    c.keys.view(torch.uint8)[c.table[0, 1], 0, 2, 5] = 0x7F
    c.values.view(torch.uint8)[c.table[1, 1], 0, 3, 7] = 0xFF
    q = torch.randn(3, 2, 64, device=dev).half()
    out = ops.paged_attention(q, c.keys, c.values, c.table, c.lengths, None, None, *c.exponents())
    assert out[0].isnan().all() and out[1, :, 7].isnan().all() and out[1].isnan().sum() == 2
    first = torch.zeros(3, 1, 1, dtype=torch.int32, device=dev)
    out = ops.paged_attention(q, c.keys, c.values, c.table, c.lengths, None, first, *c.exponents())
    want, allowed = c.attend(q, 1 / 8, first)
    assert ((out.double() - want).abs() <= allowed).all()


def test_changes_are_counted(dev, ops):
    c = Cache(dev, [5], 1, 64, 16, F16, bounds=True)
    k = torch.randn(1, 1, 64, device=dev).half()
    before = [t._version for t in (c.keys, c.values, c.bounds)]
    ops.kv_append_(k, k, c.keys, c.values, c.table, c.lengths, None, None, None, False, c.bounds)
    assert [t._version for t in (c.keys, c.values, c.bounds)] == [n + 1 for n in before]
    with torch.inference_mode():
        ops.paged_attention(k, c.keys, c.values, c.table, c.lengths)


def test_calls_that_are_refused(dev, ops):
    c = Cache(dev, [20, 30], 2, 64, 16, F16, bounds=True)
    e = Cache(dev, [20, 30], 2, 64, 16, F16, e8=True)
    q = torch.randn(2, 4, 64, device=dev).half()
    k = torch.randn(2, 2, 64, device=dev).half()
    rotation = rotation_table(c.width * 16, 64, dev)

    def attend(match, q=q, keys=c.keys, values=c.values, table=c.table, lengths=c.lengths, **more):
        with pytest.raises(RuntimeError, match=match):
            ops.paged_attention(q, keys, values, table, lengths, **more)

    attend("CUDA tensor", q=q.cpu())
    attend("fp16 or bf16", q=q.float())
    attend("must have 3 dimensions", q=q[0])
    attend("heads of 64, 128 or 256", q=q[..., :32], keys=c.keys[..., :32].contiguous(), values=c.values[..., :32].contiguous())
    attend("pages of 16", keys=c.keys[:, :, :8].contiguous(), values=c.values[:, :, :8].contiguous())
    attend("operands' type", q=q.bfloat16())
    attend("alike", values=c.values[:-1])
    attend("heads of 64 over", keys=torch.zeros(3, 2, 16, 128, device=dev).half(), values=torch.zeros(3, 2, 16, 128, device=dev).half())
    attend("must be contiguous", keys=c.keys.transpose(1, 2).contiguous().transpose(1, 2))
    attend("multiple of key heads", q=q[:, :3])
    attend("one token per sequence", q=q[:1])
    attend("page_table must be int32", table=c.table.long())
    attend("page_table must have contiguous rows", table=c.table.t().contiguous().t())
    attend("lengths must be int32", lengths=c.lengths.float())
    attend("a length for every row", lengths=c.lengths[:1])
    attend("scale", scale=0.0)
    attend("scale", scale=-1.0)
    attend("scale", scale=math.nan)
    attend("pages must be int32", pages=torch.zeros(2, 2, 3, device=dev))
    attend("pages must be contiguous", pages=torch.zeros(2, 1, 3, dtype=torch.int32, device=dev))
    attend("exponents", keys=e.keys, values=e.values)
    attend("exponents", key_exponents=e.key_exponents, value_exponents=e.value_exponents)
    attend("uint8", keys=e.keys, values=e.values, key_exponents=e.key_exponents.int(), value_exponents=e.value_exponents)
    attend("no gradient", q=q.clone().requires_grad_())
    attend("no gradient", values=c.values.clone().requires_grad_())

    def append(match, k=k, v=k, keys=c.keys, values=c.values, table=c.table, lengths=c.lengths, *more, **named):
        with pytest.raises(RuntimeError, match=match):
            ops.kv_append_(k, v, keys, values, table, lengths, *more, **named)

    append("k and v", v=k.bfloat16())
    append("4 heads over a cache of 2", k=q, v=q)
    append("one token per sequence", k=k[:1], v=k[:1])
    append("offsets must be int32", offsets=torch.zeros(3, device=dev))
    append("an entry more", offsets=torch.zeros(2, dtype=torch.int32, device=dev))
    append("q must be", q=q[:1])
    append("rotation must be contiguous float32", rotation=rotation.half())
    append("multiple of 16", rotation=rotation[:, :24].contiguous())
    append("every position", rotation=rotation[:-1])
    append("bounds must be", bounds=c.bounds[:-1])
    append("no gradient", k=k.clone().requires_grad_())
    append("no gradient", keys=c.keys.clone().requires_grad_())
    append("no gradient", rotation=rotation.clone().requires_grad_())

    def select(match, q=q, bounds=c.bounds, count=2, first=1, last=1, page=16):
        with pytest.raises(RuntimeError, match=match):
            ops.select_pages(q, bounds, c.table, c.lengths, page, count, first, last)

    select("at least one page", count=0)
    select("no gradient", bounds=c.bounds.clone().requires_grad_())
    select("among them", count=1)
    select("at least one page", first=-1)
    select("pages of 16", page=17)
    select("bounds must be", bounds=c.bounds.bfloat16())
    select("multiple of key heads", q=q[:, :3])
    with pytest.raises(RuntimeError, match="no bounds"):
        PA.KVCache(4, 16, 2, 64, F16, dev).select(q, c.table, c.lengths, 2)


def test_empty_caches_and_no_sequences(dev, ops):
    c = Cache(dev, [20, 30], 2, 64, 16, F16, bounds=True)
    q = torch.randn(2, 4, 64, device=dev).half()
    none = ops.paged_attention(q, c.keys[:0], c.values[:0], c.table, c.lengths)
    assert (none == 0).all()
    assert (ops.select_pages(q, c.bounds[:0], c.table, c.lengths, 16, 2) == -1).all()
    ops.kv_append_(q[:, :2], q[:, :2], c.keys[:0], c.values[:0], c.table, c.lengths)
    assert (ops.paged_attention(q, c.keys, c.values, c.table[:, :0], c.lengths) == 0).all()
    assert (ops.select_pages(q, c.bounds, c.table[:, :0], c.lengths, 16, 2) == -1).all()
    assert ops.paged_attention(q[:0], c.keys, c.values, c.table[:0], c.lengths[:0]).shape == (0, 4, 64)
    assert ops.select_pages(q[:0], c.bounds, c.table[:0], c.lengths[:0], 16, 2).shape == (0, 2, 2)
    nobody = torch.zeros(1, dtype=torch.int32, device=dev)      # tokens behind the last of no sequences
    rest = ops.kv_append_(q[:, :2], q[:, :2], c.keys, c.values, c.table[:0], c.lengths[:0], nobody, q)
    assert (rest == 0).all()
    alike = feature_major(q)
    assert torch.equal(ops.paged_attention(alike, c.keys, c.values, c.table, c.lengths), ops.paged_attention(q, c.keys, c.values, c.table, c.lengths))
