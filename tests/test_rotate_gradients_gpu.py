"""A rotation's gradient where other operands than x could have one."""
import pytest
import torch
import torch.autograd.forward_ad as forward

from _paged import Cache, rotation_table

pytestmark = pytest.mark.gpu


@pytest.fixture
def operands(dev):
    gen = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(20, 2, 64, generator=gen, device=dev)
    return x, rotation_table(50, 64, dev), torch.randint(0, 50, (20,), generator=gen, device=dev, dtype=torch.int32)


def test_a_table_that_requires_a_gradient(operands):
    """Refused with x or without; of a detached one x has its gradient, and the gradient one of its own."""
    x, table, positions = operands
    rotate = torch.ops.iex_ops.rotate
    learned = table.clone().requires_grad_()
    for given in (x, x.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="the table has no gradient"):
            rotate(given, learned, positions)
    with torch.no_grad():
        want = rotate(x, learned, positions)
    given, g = x.clone().requires_grad_(), x.flip(0).contiguous().requires_grad_()
    out = rotate(given, learned.detach(), positions)
    assert torch.equal(out.detach(), want)
    grad, = torch.autograd.grad(out, given, g, create_graph=True)
    assert torch.equal(grad.detach(), rotate(g.detach(), table, positions, back=True))
    again, = torch.autograd.grad(grad, g, x)
    assert torch.equal(again, want)


def test_forward_mode_is_refused(dev, operands):
    """By the rotation and by the operators of the paged cache, for every operand that could be differentiated; nothing has been written then."""
    x, table, positions = operands
    ops = torch.ops.iex_ops
    c = Cache(dev, [20, 5], 2, 64, 16, torch.float16, poison=False, bounds=True)
    q = torch.randn(2, 2, 64, generator=torch.Generator(device=dev).manual_seed(1), device=dev).half()
    weights = torch.rand(2, 2, c.width * 16, generator=torch.Generator(device=dev).manual_seed(2), device=dev)
    at = positions[:2].contiguous()
    calls = {
        "rotate": (lambda t: ops.rotate(t["x"], t["table"], positions), dict(x=x, table=table)),
        "kv_append_": (lambda t: ops.kv_append_(t["k"], t["v"], t["keys"], t["values"], c.table, c.lengths, None, t["q"], t["table"], False, t["bounds"], None, None, at),
                       dict(k=q, v=q, keys=c.keys, values=c.values, q=q, table=table, bounds=c.bounds)),
        "paged_attention": (lambda t: ops.paged_attention(t["q"], t["keys"], t["values"], c.table, c.lengths), dict(q=q, keys=c.keys, values=c.values)),
        "paged_attention_accumulate_": (lambda t: ops.paged_attention_accumulate_(t["q"], t["keys"], t["values"], c.table, c.lengths, t["weights"]),
                                        dict(q=q, keys=c.keys, values=c.values, weights=weights)),
        "select_pages": (lambda t: ops.select_pages(t["q"], t["bounds"], c.table, c.lengths, 16, 2), dict(q=q, bounds=c.bounds)),
        "evict_tokens_": (lambda t: ops.evict_tokens_(t["keys"], t["values"], c.table, c.lengths, t["weights"], 10, 2, 0, t["bounds"]),
                          dict(keys=c.keys, values=c.values, weights=weights, bounds=c.bounds)),
    }
    held = [c.keys, c.values, c.bounds, c.lengths, weights]
    before = [t.clone() for t in held]
    with forward.dual_level():
        for op, (call, operands_of) in calls.items():
            for name, t in operands_of.items():
                with torch.no_grad(), pytest.raises(RuntimeError, match=f"{op} has no forward-mode derivative"):
                    call({**operands_of, name: forward.make_dual(t, torch.ones_like(t))})
    assert all(torch.equal(a, b) for a, b in zip(held, before))
    for op, (call, operands_of) in calls.items():
        call(operands_of)
