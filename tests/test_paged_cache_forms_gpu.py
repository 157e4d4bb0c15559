"""The forms that a call's size chooses, each named by the kernels that ran: listed pages in parts, whole rows by four wavefronts, one and two
rounds of parts, prompts by four heads a workgroup, selection in one launch and in two."""
import math

import pytest
import torch

from _paged import E4M3, HALF_STEP, power
from intrasm_engine_amd import _lib
from test_paged_cache_gpu import check_append

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(dev):
    return torch.ops.iex_ops


class Pool:
    """Pages that sequences share at random (nothing is appended), some entries of their tables outside the cache."""

    def __init__(self, dev, lengths, width, kv_heads, dim, page, dtype, e8=False, seed=0, pages=400):
        gen = torch.Generator(device=dev).manual_seed(seed)
        self.page, self.dim, self.kv_heads, self.dtype = page, dim, kv_heads, dtype
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=dev)
        self.table = torch.randint(0, pages, (len(lengths), width), generator=gen, device=dev, dtype=torch.int32)
        gone = torch.rand(self.table.shape, generator=gen, device=dev) < 0.02
        self.table[gone] = torch.tensor([-1, pages, 2 ** 31 - 1], dtype=torch.int32, device=dev)[torch.randint(0, 3, (int(gone.sum()),), generator=gen, device=dev)]
        keys, values = (torch.randn(pages, kv_heads, page, dim, generator=gen, device=dev).to(dtype) for _ in range(2))
        self.exponents = (None, None)
        if e8:
            self.exponents = tuple(torch.randint(118, 122, (pages, kv_heads, page), generator=gen, device=dev, dtype=torch.uint8) for _ in range(2))
            keys, values = (x.float().mul(64).to(E4M3) for x in (keys, values))
        self.keys, self.values, self.gen = keys, values, gen
        self.pages = pages

    def q(self, heads, size=1.0):
        return torch.randn(self.lengths.numel(), heads, self.dim, generator=self.gen, device=self.table.device).mul(size).to(self.dtype)

    def stored(self, rows, exponents):
        x = rows.float().double()
        return x if exponents is None else x * power(exponents)[..., None]

    def attend(self, q, scale, listed=None):
        """(result, allowed error) in 64 bits, a sequence at a time.  Allowed: half a step of the result; weights to 2^-21 (22 of 24 bits in fp16, the
        exponential); scores to dim + 4 roundings, twice, of their terms' magnitudes; sums of n terms in chains of n / 8 and their parts."""
        seqs, heads, _ = q.shape
        kv, group, page = self.kv_heads, heads // self.kv_heads, self.page
        out, slack = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
        keys, values = self.stored(self.keys, self.exponents[0]), self.stored(self.values, self.exponents[1])
        slots, head = torch.arange(page, device=q.device), torch.arange(kv, device=q.device)[:, None]
        for s in range(seqs):
            length = int(self.lengths[s].clamp(0, self.table.shape[1] * page))
            number = torch.arange(self.table.shape[1], device=q.device).expand(kv, -1) if listed is None else listed[s].long()      # (kv, count)
            inside = (number >= 0) & (number < self.table.shape[1])
            at = torch.where(inside, self.table[s].long()[number.clamp(0, self.table.shape[1] - 1)], -1)
            there = ((at >= 0) & (at < self.pages))[..., None] & (number[..., None] * page + slots < length)
            k, v = (x[at.clamp(0, self.pages - 1), head].reshape(kv, -1, self.dim) for x in (keys, values))                          # (kv, tokens, dim)
            there = there.reshape(kv, 1, -1)
            x = q[s].double().view(kv, group, self.dim)
            score = torch.matmul(x, k.transpose(1, 2).contiguous()) * scale
            magnitude = (torch.matmul(x.abs(), k.abs().transpose(1, 2).contiguous()) * scale * there).amax(-1, keepdim=True)
            weight = torch.softmax(torch.where(there, score, -math.inf), -1).nan_to_num(0.0)
            n = there.sum(-1, keepdim=True)
            relative = 2.0 ** -21 + 2 * (self.dim + 4) * 2.0 ** -24 * magnitude + (n / 8 + 64) * 2.0 ** -24
            out[s] = torch.matmul(weight, v).view(heads, -1)
            slack[s] = (relative * torch.matmul(weight, v.abs())).view(heads, -1)
        half = HALF_STEP[q.dtype]
        return out, out.abs() * half + slack * (1 + half) + (2.0 ** -25 if q.dtype == F16 else 0.0)

    def check(self, ops, q, kernels, listed=None):
        got = ops.paged_attention(q, self.keys, self.values, self.table, self.lengths, self.dim ** -0.5, listed, *self.exponents)
        ran = _lib.last_kernels()
        assert all(name in ran for name in kernels), ran
        want, allowed = self.attend(q, self.dim ** -0.5, listed)
        beyond = float(((got.double() - want).abs() - allowed).max())
        assert beyond <= 0, f"{beyond} beyond what is allowed"
        for _ in range(2):
            assert torch.equal(ops.paged_attention(q, self.keys, self.values, self.table, self.lengths, self.dim ** -0.5, listed, *self.exponents), got)
        return got


def lists(pool, count):
    """Pages in order, out of order, twice, with holes and tails of -1, past the end; fewer pages than entries."""
    seqs, kv, dev = pool.lengths.numel(), pool.kv_heads, pool.table.device
    width = pool.table.shape[1]
    out = torch.randint(-2, width + 3, (seqs, kv, count), generator=pool.gen, device=dev, dtype=torch.int32)
    for s in range(seqs):
        used = -(-int(pool.lengths[s].clamp(0, width * pool.page)) // pool.page)
        if s % 4 == 0:      # as a selection leaves them
            n = min(count, used)
            out[s] = -1
            for h in range(kv):
                out[s, h, :n] = torch.randperm(max(1, used), generator=pool.gen, device=dev)[:n].sort()[0]
        elif s % 4 == 1:
            out[s, :, count // 3:] = -1
        elif s % 4 == 2:
            out[s, :, :count // 2] = -1
    return out.contiguous()


@pytest.mark.parametrize("dtype,e8", [(BF16, False), (F16, True)])
@pytest.mark.parametrize("dim,kv_heads,heads,page,count", [(128, 2, 8, 16, 64), (128, 2, 8, 16, 65), (64, 1, 3, 64, 64), (256, 2, 2, 32, 129), (128, 1, 20, 128, 33)])
def test_listed_pages_in_parts(ops, dev, dtype, e8, dim, kv_heads, heads, page, count):
    """Lists of 1024 tokens stay whole, longer ones are cut by their length."""
    pool = Pool(dev, [30000, 0, 1, 700, 5000, 16, 2049, 0], -(-30000 // page), kv_heads, dim, page, dtype, e8)
    join = ["paged_join_kernel"] if count * page > 1024 else []
    got = pool.check(ops, pool.q(heads, 2.0), ["paged_attention_kernel", *join], lists(pool, count))
    assert (got[1] == 0).all() and (got[7] == 0).all()
    assert ("paged_join_kernel" in _lib.last_kernels()) == bool(join)


def test_listed_pages_in_parts_of_many_entries(ops, dev):
    """Parts of more than 64 entries of a list: as many as a wavefront has lanes are looked up at a time."""
    pool = Pool(dev, [(s * 977) % 12000 for s in range(64)], 750, 8, 64, 16, BF16)
    pool.check(ops, pool.q(8), ["paged_attention_kernel<bf16, 64, 16, 4>", "paged_join_kernel"], lists(pool, 640))


@pytest.mark.parametrize("dtype,e8", [(BF16, False), (F16, False), (BF16, True)])
@pytest.mark.parametrize("seqs,kv_heads,heads,dim,waves", [(128, 4, 4, 128, 4), (127, 4, 12, 128, 8), (520, 1, 1, 64, 4), (65, 8, 8, 256, 4)])
def test_whole_rows(ops, dev, dtype, e8, seqs, kv_heads, heads, dim, waves):
    """Eight wavefronts a row below 512 rows, four from there on; nothing is cut."""
    pool = Pool(dev, [(s * 131) % 900 for s in range(seqs)], 14, kv_heads, dim, 64, dtype, e8)
    pool.check(ops, pool.q(heads, 1.5), [f"paged_attention_kernel<{'bf16' if dtype == BF16 else 'f16'}, {dim}, {'e4m3' if e8 else '16'}, {waves}>"])
    assert "join" not in _lib.last_kernels()


@pytest.mark.parametrize("dtype,e8", [(BF16, False), (F16, True)])
@pytest.mark.parametrize("seqs,kv_heads,heads", [(63, 4, 8), (64, 4, 8), (300, 1, 1), (7, 40, 40)])
def test_rows_in_parts(ops, dev, dtype, e8, seqs, kv_heads, heads):
    """Ragged rows over tables that they do not fill, on either side of 256 rows."""
    pool = Pool(dev, [(s * 613) % 5000 for s in range(seqs)], 400, kv_heads, 64, 16, dtype, e8)
    pool.check(ops, pool.q(heads, 1.5), ["paged_attention_kernel", "paged_join_kernel"])


@pytest.mark.parametrize("layout", ["tokens", "features"])
@pytest.mark.parametrize("dim,page,kv_heads,heads,dtype,e8,bounds", [(64, 16, 6, 18, BF16, False, True), (64, 64, 5, 21, F16, True, True), (128, 32, 3, 27, F16, False, False),
                                                                     (64, 16, 7, 1, BF16, True, False)])
def test_prompts_by_several_heads_a_workgroup(ops, dev, layout, dim, page, kv_heads, heads, dtype, e8, bounds):
    """Spans times heads of 4096 and more: four heads a workgroup (keys one, where there are bounds), the last group of fewer."""
    new = [601, 1, 640, 0, 583, 64, 700, 129, 511, 77, 900, 3, 611, 640, 580, 599] * (2 if heads > 1 else 5)
    before = [(i * 37) % 100 for i in range(len(new))]
    span = max(64, page)
    assert (sum(new) // span) * (2 * kv_heads + heads) >= 4096
    check_append(ops, dev, new, before, kv_heads, heads, dim, page, dtype, e8, dim // 2, heads % 2 == 1, bounds, layout, extra=-sum(new) % 8)
    assert _lib.last_kernels().startswith("kv_append_" + ("columns_" if layout == "features" else "") + "kernel<") and "(4 heads a workgroup)" in _lib.last_kernels()


def select_plainly(q, bounds, table, lengths, page, count, first, last):
    seqs, kv, width = q.shape[0], bounds.shape[1], table.shape[1]
    number = torch.arange(width, device=q.device)
    used = (-(-lengths.clamp(0, width * page) // page)).long()[:, None, None]
    there = (table >= 0) & (table < bounds.shape[0])
    score = torch.empty(seqs, kv, width, device=q.device)
    for s in range(seqs):
        x = q[s].double().view(kv, -1, 1, q.shape[2])
        low, high = bounds[table[s].clamp(0, bounds.shape[0] - 1).long()].double().permute(1, 2, 0, 3).unbind(1)      # (kv, width, dim)
        score[s] = torch.maximum(x * low[:, None], x * high[:, None]).sum((1, 3)).float()
    score = torch.where((number < first) | (number >= used - last), math.inf, score)
    score = torch.where((number < used) & there[:, None], score, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :count]
    best = torch.where(torch.gather(score, 2, best) > -math.inf, best, width).sort(-1)[0]
    best = torch.where(best < width, best, -1).to(torch.int32)
    return torch.nn.functional.pad(best, (0, count - best.shape[-1]), value=-1)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,seqs,kv_heads,heads,width,kernels", [
    (64, 3, 2, 2, 300, 2), (128, 3, 2, 6, 300, 2), (256, 2, 3, 3, 300, 2),                                    # scores in a launch of their own
    (64, 64, 2, 4, 1100, 2), (128, 16, 4, 8, 2100, 2), (256, 8, 4, 4, 2100, 2),                               # ... two chunks a wavefront
    (64, 40, 8, 8, 400, 1), (128, 64, 4, 16, 777, 1), (256, 256, 1, 2, 300, 1), (128, 255, 1, 1, 300, 2),     # rows enough for one launch
    (128, 300, 1, 1, 256, 1)])
def test_selection(ops, dev, dtype, dim, seqs, kv_heads, heads, width, kernels):
    pages, page = 500, 16
    gen = torch.Generator(device=dev).manual_seed(5)
    bounds = torch.randn(pages, kv_heads, 2, dim, generator=gen, device=dev).sort(2)[0].to(dtype)
    table = torch.randint(-4, pages + 4, (seqs, width), generator=gen, device=dev, dtype=torch.int32)
    lengths = torch.tensor([(s * 7919) % (width * page + 1) if s else width * page for s in range(seqs)], dtype=torch.int32, device=dev)
    q = torch.randn(seqs, heads, dim, generator=gen, device=dev).to(dtype)
    for count, first, last in ((4, 1, 1), (129, 0, 2)):
        got = ops.select_pages(q, bounds, table, lengths, page, count, first, last)
        ran = _lib.last_kernels()
        assert ("page_score_kernel" in ran) == (kernels == 2) and "page_select_kernel" in ran, ran
        assert torch.equal(got, select_plainly(q, bounds, table, lengths, page, count, first, last))
