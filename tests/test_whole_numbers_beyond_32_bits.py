"""Whole numbers that a caller gives and 32 bits do not hold: refused, on both sides, not wrapped to others that would be taken."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import intrasm_engine_amd  # noqa: F401
from _paged import Cache, rotation_table

BELOW, ABOVE = -(1 << 32), 1 << 32


def test_sections_of_a_rotation():
    """Without a GPU: tensors without memory."""
    with FakeTensorMode():
        x, table, positions = torch.empty(0, 2, 64, device="cuda"), torch.empty(0, 64, device="cuda"), torch.empty(2, 0, dtype=torch.int32, device="cuda")
        for off, text in ((BELOW, "too small"), (ABOVE, "too large")):
            with pytest.raises(RuntimeError, match=text):
                torch.ops.iex_ops.rotate(x, table, positions, [off + 16, 16])


@pytest.mark.gpu
def test_operators_of_the_cache(dev):
    ops = torch.ops.iex_ops
    c = Cache(dev, [60, 40], 2, 64, 16, torch.float16, poison=False, bounds=True)
    q = torch.randn(2, 2, 64, generator=torch.Generator(device=dev).manual_seed(1), device=dev).half()
    weights = torch.rand(2, 2, c.width * 16, generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    table, positions = rotation_table(70, 64, dev), torch.zeros(2, 2, dtype=torch.int32, device=dev)
    held = [c.keys, c.values, c.bounds, c.lengths, weights]
    before = [t.clone() for t in held]
    calls = [lambda off: ops.evict_tokens_(c.keys, c.values, c.table, c.lengths, weights, 30, off + 5, 2),
             lambda off: ops.evict_tokens_(c.keys, c.values, c.table, c.lengths, weights, 30, 5, off + 2),
             lambda off: ops.rotate(q, table, positions, [off + 16, 16]),
             lambda off: ops.kv_append_(q, q, c.keys, c.values, c.table, c.lengths, None, q, table, False, c.bounds, None, None, positions, [16, off + 16]),
             lambda off: ops.select_pages(q, c.bounds, c.table, c.lengths, off + 16, 2),
             lambda off: ops.select_pages(q, c.bounds, c.table, c.lengths, 16, 2, off + 1, 1),
             lambda off: ops.select_pages(q, c.bounds, c.table, c.lengths, 16, 2, 1, off + 1)]
    for call in calls:
        for off, text in ((BELOW, "too small"), (ABOVE, "too large")):
            with pytest.raises(RuntimeError, match=text):
                call(off)
    assert all(torch.equal(a, b) for a, b in zip(held, before))
    for call in calls:
        call(0)
