"""An eviction whose waits give up (they are not waited for at all here): what is left says so, in the list and in the cache."""
import ctypes

import pytest
import torch

from _paged import Cache
from intrasm_engine_amd import _lib
from test_evict_tokens_gpu import plain, random_weights, row_of

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
CHUNK = {(64, 2): 256, (128, 2): 128, (256, 2): 64, (64, 1): 256, (128, 1): 256, (256, 1): 128}      # tokens, by head_dim and bytes of an element


def evict(c, weights, keep, recent, first, tries, bounds=None):
    pointer = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    cache = _lib.PagedCache(dtype=_lib.BF16 if c.dtype == BF16 else _lib.F16, eight_bits=int(c.e8), pages=c.pages, page_size=c.page, kv_heads=c.kv_heads, head_dim=c.dim,
                            key_page_stride=c.keys.stride(0), value_page_stride=c.values.stride(0), keys=pointer(c.keys), values=pointer(c.values),
                            key_exponents=pointer(c.key_exponents), value_exponents=pointer(c.value_exponents), bounds=pointer(bounds), table=pointer(c.table),
                            seqs=c.table.shape[0], table_width=c.width, table_stride=c.table.stride(0), lengths=pointer(c.lengths))
    lib = _lib.load()
    size = lib.iex_evict_tokens_workspace_bytes(ctypes.byref(cache), keep)
    workspace = torch.empty(size, dtype=torch.uint8, device=c.table.device)
    kept = torch.empty(c.table.shape[0], c.kv_heads, keep, dtype=torch.int32, device=c.table.device)
    _lib.check(lib.iex_evict_tokens_within(ctypes.byref(cache), pointer(c.lengths), pointer(weights), keep, recent, first, pointer(kept), tries, pointer(workspace), size,
                                           torch.cuda.current_stream().cuda_stream), "evict_tokens")
    torch.cuda.synchronize()      # (the workspace is the call's until then)
    return kept


def made(dev, dtype, e8, dim):
    c = Cache(dev, [2000, 1990, 700, 30], 2, dim, 64, dtype, e8=e8, poison=False, bounds=True)
    weights = random_weights(c)
    weights[1, 0, :1500] += 1e6          # all of them are where they belong
    weights[1, 1, 1000:] += 1e6          # the second half moves to the front
    return c, weights


@pytest.mark.parametrize("dtype,e8,dim", [(F16, False, 64), (BF16, False, 128), (F16, False, 256), (BF16, True, 64), (F16, True, 128), (BF16, True, 256)])
def test_what_is_left(dev, dtype, e8, dim):
    c, weights = made(dev, dtype, e8, dim)
    old, _ = made(dev, dtype, e8, dim)
    before, lengths, keep, size = weights.clone(), c.lengths.tolist(), 600, CHUNK[dim, 1 if e8 else 2]
    kept = evict(c, weights, keep, 100, 3, 0, c.bounds)
    abandoned = 0
    for s, length in enumerate(lengths):
        for h in range(2):
            want = plain(before[s, h], length, keep, 100, 3)
            if length <= keep:
                assert kept[s, h].tolist() == want + [-1] * (keep - length)
                continue
            told = list(want)
            for begin in range(0, keep, size):
                end = min(keep, begin + size)
                waits = any(begin <= t < begin + size for t in want[:begin]) or any(begin <= t < begin + size for t in want[end:])
                if want[end - 1] != end - 1 and waits:
                    told[begin:end] = [-2] * (end - begin)
            assert kept[s, h].tolist() == told, (s, h)
            gone = torch.tensor([t == -2 for t in told], device=dev)
            abandoned += int(gone.sum())
            for name in ("keys", "values"):
                now, then = (row_of(x, name, s, h, at) for x, at in ((c, range(keep)), (old, want)))
                ones = (now.view(torch.uint8) == 0xFF).all(-1)
                assert ones[gone].all() and (ones | (now.view(torch.uint8) == then.view(torch.uint8)).all(-1)).all(), (s, h, name)
                behind = range(keep, length)
                assert torch.equal(row_of(c, name, s, h, behind).view(torch.uint8), row_of(old, name, s, h, behind).view(torch.uint8))
            assert torch.equal(weights[s, h, :keep], before[s, h, want]) and (weights[s, h, keep:length] == 0).all()
    assert abandoned > 0 and c.lengths.tolist() == [keep, keep, keep, 30]
    # and attention shows it
    out = torch.ops.iex_ops.paged_attention(torch.ones(4, 2, dim, dtype=dtype, device=dev), c.keys, c.values, c.table, c.lengths, None, None, *c.exponents())
    for s in range(4):
        for h in range(2):
            assert out[s, h].isnan().all() if (kept[s, h] == -2).any() else not out[s, h].isnan().any(), (s, h)


@pytest.mark.parametrize("e8", [False, True])
def test_waits_that_end(dev, e8):
    """The longest wait: the operator's own result."""
    (c, weights), (other, same) = (made(dev, BF16, e8, 128) for _ in range(2))
    kept = evict(c, weights, 600, 100, 3, 1 << 20, c.bounds)
    want = torch.ops.iex_ops.evict_tokens_(other.keys, other.values, other.table, other.lengths, same, 600, 100, 3, other.bounds, *other.exponents())
    assert torch.equal(kept, want) and not (kept == -2).any()
    for a, b in ((c.keys, other.keys), (c.values, other.values), (c.lengths, other.lengths), (weights, same), (c.bounds, other.bounds)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
