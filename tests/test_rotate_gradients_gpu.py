"""A rotation's gradient where other operands than x could have one."""
import pytest
import torch

from _paged import rotation_table

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
