"""Attention over a paged cache that keeps account of what every token got, against its plain form in 64 bits."""
import math

import pytest
import torch

from _paged import HALF_STEP, Cache, feature_major
from intrasm_engine_amd import _lib

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(dev):
    return torch.ops.iex_ops


def accumulate(ops, c, q, weights, scale):
    return ops.paged_attention_accumulate_(q, c.keys, c.values, c.table, c.lengths, weights, scale, *c.exponents())


def account(c, q, scale):
    """What every token of (sequences, kv_heads, tokens of a table) gets, in 64 bits, and how far 32 bits may be off; -1 where nothing is attended to.

    A score is off by D + 4 roundings of its terms' magnitudes (the products' sum, the scale, the scale's own rounding, the maximum taken off), which
    reaches a weight as relative error, once in the exponential and once in the sum; the exponential itself by 2^-22, the sum of n terms in chains of n / 8
    and the parts behind them, the division, the products and the sum over the heads by a rounding each."""
    seqs, heads, dim = q.shape
    group = heads // c.kv_heads
    room = c.width * c.page
    want = torch.full((seqs, c.kv_heads, room), -1.0, dtype=torch.float64, device=q.device)
    slack = torch.zeros_like(want)
    for s in range(seqs):
        length = min(max(0, int(c.lengths[s])), room)
        at = [t for i in range(-(-length // c.page)) if 0 <= int(c.table[s, i]) < c.pages for t in range(i * c.page, min(length, (i + 1) * c.page))]
        if not at:
            continue
        at = torch.tensor(at, device=q.device)
        for h in range(c.kv_heads):
            k, _ = c.rows(s, h)
            terms = k[None] * q[s, h * group:(h + 1) * group].double()[:, None]
            p = torch.softmax(terms.sum(-1) * scale, -1)
            magnitude = terms.abs().sum(-1).amax(-1, keepdim=True) * scale
            relative = 2.0 ** -21 + 2 * (dim + 4) * 2.0 ** -24 * magnitude + (k.shape[0] / 8 + 64) * 2.0 ** -24
            want[s, h, at] = p.sum(0)
            slack[s, h, at] = (p * (relative + group * 2.0 ** -24)).sum(0)
    return want, slack


def check(ops, c, q, scale, kernels=None, seed=3):
    gen = torch.Generator(device=q.device).manual_seed(seed)
    weights = torch.rand(q.shape[0], c.kv_heads, c.width * c.page, generator=gen, device=q.device)
    before = weights.clone()
    got = accumulate(ops, c, q, weights, scale)
    names = _lib.last_kernels()
    if kernels is not None:
        for name in kernels:
            assert name in names, names
    want, allowed = c.attend(q, scale)
    assert got.stride() == q.stride() and ((got.double() - want).abs() <= allowed).all()
    plain = ops.paged_attention(q, c.keys, c.values, c.table, c.lengths, scale, None, *c.exponents())
    assert torch.equal(got, plain)
    want, slack = account(c, q, scale)
    there = want >= 0
    assert torch.equal(weights[~there], before[~there])
    off = (weights.double() - before.double() - want).abs() - (slack * 1.001 + 2.0 ** -24 * (before.double() + want))
    assert not (off[there] > 0).any(), f"{float(off[there].max()):.3g} beyond"
    again = before.clone()
    accumulate(ops, c, q, again, scale)
    assert torch.equal(again, weights)       # the same bits


def queries(dev, c, heads, layout="tokens", seed=5):
    q = torch.randn(c.lengths.numel(), heads, c.dim, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(c.dtype)
    return feature_major(q) if layout == "features" else q


ONE, TWO = "(scores kept)", "paged_account_kernel"


@pytest.mark.parametrize("dtype,e8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("dim,page,kv_heads,heads,layout", [(128, 64, 2, 2, "features"), (64, 16, 1, 5, "tokens"), (256, 32, 2, 12, "features"), (128, 256, 1, 16, "tokens"),
                                                            (64, 128, 3, 9, "features"), (128, 16, 1, 40, "tokens")])
def test_short_rows(ops, dev, dtype, e8, dim, page, kv_heads, heads, layout):
    c = Cache(dev, [1, 0, 15, 16, 17, 129, 300, page, 513], kv_heads, dim, page, dtype, e8=e8)
    check(ops, c, queries(dev, c, heads, layout), dim ** -0.5, [ONE] + ([TWO] if heads // kv_heads > 16 else []))


@pytest.mark.parametrize("dtype,e8", [(F16, False), (BF16, True)])
@pytest.mark.parametrize("dim,kv_heads,heads", [(64, 2, 2), (128, 1, 7), (256, 1, 3)])
def test_rows_of_one_wavefront(ops, dev, dtype, e8, dim, kv_heads, heads):
    c = Cache(dev, [1, 2, 5, 13, 16, 0, 31, 33, 64], kv_heads, dim, 16, dtype, e8=e8)
    check(ops, c, queries(dev, c, heads), 0.3, [", 1>"])


@pytest.mark.parametrize("e8", [False, True])
@pytest.mark.parametrize("lengths,kv_heads,heads,dim,page", [([5000], 1, 1, 128, 64), ([3000, 1, 0, 1025, 2047], 2, 6, 64, 16), ([2500, 700], 1, 3, 256, 32),
                                                             ([1500, 4097], 1, 33, 128, 256), ([9000], 2, 16, 128, 64)])
def test_rows_in_parts(ops, dev, e8, lengths, kv_heads, heads, dim, page):
    c = Cache(dev, lengths, kv_heads, dim, page, BF16, e8=e8)
    check(ops, c, queries(dev, c, heads), dim ** -0.5, [ONE, TWO])


def test_more_sequences_than_lanes_and_turns(ops, dev):
    """150 sequences in tables of 2304 tokens; and so many rows that one workgroup takes all of a row's tokens."""
    lengths = [(i * 37) % 200 for i in range(149)] + [2300]
    c = Cache(dev, lengths, 1, 64, 16, F16)
    check(ops, c, queries(dev, c, 2), 0.2, [TWO])
    c = Cache(dev, [3000 if i % 70 == 0 else 3 for i in range(300)], 8, 64, 256, BF16)
    check(ops, c, queries(dev, c, 8), 0.2, [TWO])


@pytest.mark.parametrize("width", [9, 90])
def test_pages_given_back(ops, dev, width):
    """Some, and all of a sequence's: nothing is added there, zeros come out, whatever a row's other scores are."""
    c = Cache(dev, [130, 144, 77, 16], 2, 64, 16, F16, width=width, poison=False)
    c.table[0, 2], c.table[0, 8], c.table[1, :] = -1, c.pages, -1
    c.table[2, 0] = -7
    check(ops, c, queries(dev, c, 4), 0.4)


@pytest.mark.parametrize("width", [9, 90])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_scores_that_are_not_numbers(ops, dev, bad, width):
    """A NaN or infinite score shows in the tokens attended to as in the formula (all of that query's are NaN; with a score of -inf just this one is 0) and
    not in those behind the length or in a page given back, nor in other key heads or sequences."""
    c = Cache(dev, [100, 50], 2, 64, 16, BF16, width=width, poison=False)
    c.table[0, 3] = -1
    q = queries(dev, c, 4)
    q[0, :2, 0] = 1.0
    c.keys[int(c.table[0, 1]), 0, 5, 0] = bad
    weights = torch.zeros(2, 2, width * 16, device=dev)
    out = accumulate(ops, c, q, weights, 0.4)
    attended = torch.ones(100, dtype=torch.bool, device=dev)
    attended[48:64] = False
    if bad == -math.inf:
        assert weights[0, 0, 21] == 0 and abs(float(weights[0, 0].sum()) - 2) < 1e-4 and not out.isnan().any()
    else:
        assert weights[0, 0, :100][attended].isnan().all() and out[0, :2].isnan().all()
        assert not out[0, 2:].isnan().any() and not out[1].isnan().any()
    assert (weights[0, 0, :100][~attended] == 0).all() and (weights[0, :, 100:] == 0).all() and (weights[1, :, 50:] == 0).all()
    assert not weights[0, 1].isnan().any() and not weights[1].isnan().any()


def test_weights_sum_to_the_heads(ops, dev):
    """Every pass adds one per query head, over many passes (32 bits: a rounding of each pass and token)."""
    c = Cache(dev, [33, 1400], 2, 128, 64, F16)
    weights = torch.zeros(2, 2, c.width * 64, device=dev)
    for step in range(20):
        accumulate(ops, c, queries(dev, c, 6, seed=step), weights, 0.1)
    for s, n in enumerate((33, 1400)):
        assert ((weights[s].double().sum(-1) - 60).abs() < 60 * 2.0 ** -18).all() and (weights[s, :, n:] == 0).all()


@pytest.mark.parametrize("poison", [True, False])
def test_replays_streams_and_strided_pages(ops, dev, poison):
    """A captured pass follows lengths, tables and weights; replayed between eager passes; on another stream; pages with others between them.  (Bits: the
    lengths reach into what is poisoned.)"""
    c = Cache(dev, [40, 1900, 700], 2, 64, 16, F16, width=130, strided=True, poison=poison)
    q = queries(dev, c, 4)
    weights = torch.zeros(3, 2, 130 * 16, device=dev)
    static_q = q.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = accumulate(ops, c, static_q, weights, 0.2)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = accumulate(ops, c, static_q, weights, 0.2)
    for step in range(3):
        c.lengths.copy_(torch.tensor([41 + step, 1900 - 300 * step, 2080 - step], device=dev))
        c.table[2, :] = c.table[1].flip(0) if step else c.table[1]
        static_q.copy_(queries(dev, c, 4, seed=20 + step))
        eager = torch.rand(3, 2, 130 * 16, generator=torch.Generator(device=dev).manual_seed(step), device=dev)
        weights.copy_(eager)
        graph.replay()
        want = accumulate(ops, c, static_q, eager, 0.2)
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)) and torch.equal(weights.view(torch.int32), eager.view(torch.int32))
        assert out.isnan().any() == poison


def test_lengths_cut_to_the_table_and_changes_counted(ops, dev):
    c = Cache(dev, [48, 20], 1, 64, 16, F16, width=3)
    q = queries(dev, c, 2)
    a, b = torch.zeros(2, 1, 48, device=dev), torch.zeros(2, 1, 48, device=dev)
    want = accumulate(ops, c, q, a, 0.2)
    c.lengths[0], version = 1 << 30, b._version
    assert torch.equal(accumulate(ops, c, q, b, 0.2), want) and torch.equal(a, b) and b._version > version
    c.lengths[:] = -5
    assert (accumulate(ops, c, q, b, 0.2) == 0).all() and torch.equal(a, b)


def test_refusals(ops, dev):
    c = Cache(dev, [48, 20], 2, 64, 16, F16, width=3)
    q = queries(dev, c, 4)
    good = torch.zeros(2, 2, 48, device=dev)
    for weights, text in [(good[:1], "weights must be"), (good[:, :1], "weights must be"), (good.half(), "weights must be"), (torch.zeros(2, 2, 64, device=dev), "weights must be"),
                          (torch.zeros(2, 2, 96, device=dev)[..., ::2], "weights must be"), (good[0], "3 dimensions"), (good.cpu(), "CUDA tensor"),
                          (torch.zeros(193, device=dev)[1:].view(2, 2, 48), "16-byte aligned"), (good.clone().requires_grad_(), "no gradient")]:
        with pytest.raises(RuntimeError, match=text):
            accumulate(ops, c, q, weights, 0.2)
    for bad, text in [(q[:1], "one token per sequence"), (q[:, :3], "multiple of key heads"), (q.float(), "fp16 or bf16"), (q.clone().requires_grad_(), "no gradient")]:
        with pytest.raises(RuntimeError, match=text):
            accumulate(ops, c, bad, good, 0.2)
    for scale in (0.0, -1.0, math.nan):
        with pytest.raises(RuntimeError, match="scale"):
            accumulate(ops, c, q, good, scale)
    with pytest.raises(RuntimeError, match="4096 query heads"):
        one = Cache(dev, [3], 1, 64, 16, F16)
        accumulate(ops, one, torch.zeros(1, 4097, 64, dtype=F16, device=dev), torch.zeros(1, 1, 16, device=dev), 0.2)
    assert (good == 0).all()
    empty = torch.zeros(0, 2, 64, dtype=F16, device=dev)
    assert ops.paged_attention_accumulate_(empty, c.keys, c.values, c.table[:0], c.lengths[:0], good[:0]).shape == (0, 2, 64)
    nothing = ops.paged_attention_accumulate_(q, c.keys[:0], c.values[:0], c.table, c.lengths, good)
    assert (nothing == 0).all() and (good == 0).all()
