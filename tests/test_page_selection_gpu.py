"""Selection of pages by bounds that reach the ends of their type."""
import math

import pytest
import torch

from _paged import Cache, feature_major
from intrasm_engine_amd import _lib
from intrasm_engine_amd.pytorch import paged_attention as PA

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def by_definition(c, q, count, first, last):
    """Pages by the sum over heads and features of max(q lo, q hi) in 64 bits, rounded once; a feature whose query is zero adds nothing
    (NaN if a bound is)."""
    group = q.shape[1] // c.kv_heads
    out = torch.full((q.shape[0], c.kv_heads, count), -1, dtype=torch.int32)
    for s in range(q.shape[0]):
        used = -(-int(c.lengths[s]) // c.page)
        rows = c.table[s, :used].long()
        for h in range(c.kv_heads):
            x = q[s, h * group:(h + 1) * group].double()[:, None]
            low, high = c.bounds[rows, h].double().unbind(1)
            term = torch.maximum(x * low, x * high)
            zero = torch.where(low.isnan() | high.isnan(), math.nan, 0.0).expand_as(term)
            score = torch.where(x == 0, zero, term).sum((0, 2)).float()
            score = torch.where(score.isnan(), math.inf, score).cpu()      # (first, beside those that are infinite: the tests have no ties of the two)
            rank = torch.arange(used)
            score[(rank < first) | (rank >= used - last)] = math.inf
            out[s, h, :min(count, used)] = torch.sort(score, descending=True, stable=True)[1][:count].sort()[0].to(torch.int32)
    return out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kv_heads,heads", [(64, 1, 2), (128, 2, 8), (256, 1, 1)])
@pytest.mark.parametrize("pages", [40, 300])
def test_infinite_bounds(dev, dtype, dim, kv_heads, heads, pages):
    """A bound that no query reaches leaves no trace: an infinite smallest key under a positive query, an infinite largest one under a negative
    query, any under a query of zero.  (300 pages: scores in a launch of their own.)"""
    ops = torch.ops.iex_ops
    c = Cache(dev, [pages * 16, 333], kv_heads, dim, 16, dtype, bounds=True, poison=False)
    gen = torch.Generator(device=dev).manual_seed(1)
    sign = torch.where(torch.rand(dim, generator=gen, device=dev) < 0.5, -1.0, 1.0)
    q = (torch.randn(2, heads, dim, generator=gen, device=dev).abs() + 0.1) * sign      # (all heads of a feature have its sign)
    q[:, :, 7] = 0.0
    q = q.to(dtype)
    hit = torch.rand(c.pages, kv_heads, dim, generator=gen, device=dev) < 0.3
    c.bounds[:, :, 0][hit & (sign > 0)] = -math.inf
    c.bounds[:, :, 1][hit & (sign < 0)] = math.inf
    c.bounds[:, :, 0, 7], c.bounds[:, :, 1, 7] = -math.inf, math.inf
    for count, first, last in ((5, 0, 0), (17, 1, 2)):
        got = ops.select_pages(q, c.bounds, c.table, c.lengths, 16, count, first, last)
        assert torch.equal(got.cpu(), by_definition(c, q, count, first, last))
    # what a query does reach: infinities of one sign come first or last, of both signs together (and NaN) first
    c.bounds[c.table[0, 11].long(), :, 0, 0] = c.bounds[c.table[0, 11].long(), :, 1, 0] = math.inf * float(sign[0])
    c.bounds[c.table[0, 23].long(), :, :, 1] = -math.inf * float(sign[1])
    got = ops.select_pages(q, c.bounds, c.table, c.lengths, 16, 3, 0, 0)
    assert torch.equal(got.cpu(), by_definition(c, q, 3, 0, 0)) and (got[0] == 11).any(-1).all()
    got = ops.select_pages(q, c.bounds, c.table, c.lengths, 16, pages - 1, 0, 0)
    assert not (got[0] == 23).any()


def test_a_key_that_eight_bits_round_past_fp16(dev):
    """65504 becomes 65536 in an e4m3 row, whose bound in fp16 is infinite: queries that are negative there do not see it."""
    page, dim = 16, 64
    cache = PA.KVCache(40, page, 1, dim, F16, dev, eight_bits=True, bounds=True)
    n = 30 * page
    gen = torch.Generator(device=dev).manual_seed(2)
    k = torch.randn(n, 1, dim, generator=gen, device=dev).half()
    k[5 * page + 3, 0, 9] = 65504.0
    table = torch.randperm(40, device=dev)[None, :30].to(torch.int32)
    lengths = torch.tensor([n], dtype=torch.int32, device=dev)
    cache.append_(k, k, table, lengths, torch.tensor([0, n], dtype=torch.int32, device=dev))
    assert torch.isposinf(cache.bounds[table[0, 5], 0, 1, 9])
    plain = Cache.__new__(Cache)
    plain.__dict__.update(table=table, page=page, kv_heads=1, lengths=lengths, bounds=cache.bounds)
    q = torch.randn(1, 2, dim, generator=gen, device=dev).half()
    for sign in (-1.0, 1.0):
        q[:, :, 9] = sign * q[:, :, 9].abs()
        assert torch.equal(cache.select(q, table, lengths, 4, 0, 0).cpu(), by_definition(plain, q, 4, 0, 0))
    q[:, :, 9] = -0.001
    assert not (cache.select(q, table, lengths, 4, 0, 0) == 5).any()


def test_many_rows(dev):
    """More sequences and key heads than a launch has in its second dimension, where a workgroup selects a row."""
    seqs, kv_heads, dim, page = 4100, 16, 64, 16
    pages = 50
    gen = torch.Generator(device=dev).manual_seed(3)
    bounds = torch.randn(pages, kv_heads, 2, dim, generator=gen, device=dev).sort(2)[0].half()
    table = torch.randint(0, pages, (seqs, 6), generator=gen, device=dev, dtype=torch.int32)
    lengths = torch.randint(0, 6 * page + 1, (seqs,), generator=gen, device=dev, dtype=torch.int32)
    q = torch.randn(seqs, kv_heads, dim, generator=gen, device=dev).half()
    got = torch.ops.iex_ops.select_pages(q, bounds, table, lengths, page, 2, 0, 1)
    assert _lib.last_kernels().startswith("page_select_kernel<f16, 64>")
    b = bounds[table.long()].double()                                               # (seqs, 6, kv_heads, 2, dim)
    score = torch.maximum(q.double()[:, None] * b[:, :, :, 0], q.double()[:, None] * b[:, :, :, 1]).sum(-1).float().transpose(1, 2)
    used = (-(-lengths // page)).long()[:, None, None]
    number = torch.arange(6, device=dev)
    score = torch.where(number < used, torch.where(number == used - 1, math.inf, score), -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :2]
    best = torch.where(best < used, best, 6).sort(-1)[0]
    assert torch.equal(got.long(), torch.where(best < 6, best, -1))
