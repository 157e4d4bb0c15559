"""Which gradients a rotation has, without a GPU: tensors of a device that nothing stands behind (a call that passes the checks ends at their memory)."""
import pytest
import torch
import torch.autograd.forward_ad as forward
from torch._subclasses.fake_tensor import FakeTensorMode

import intrasm_engine_amd  # noqa: F401

PASSED = "data is not allocated"


@pytest.fixture
def operands():
    with FakeTensorMode():
        yield torch.empty(4, 2, 64, device="cuda"), torch.empty(9, 64, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("learned", [False, True])
@pytest.mark.parametrize("trained", [False, True])
def test_a_table_that_requires_a_gradient(operands, trained, learned):
    """It gets none, so the call is refused, whether x requires one or not; without gradients it is a table like any other."""
    x, table, positions = operands
    x.requires_grad_(trained), table.requires_grad_(learned)
    with pytest.raises(RuntimeError, match="the table has no gradient" if learned else PASSED):
        torch.ops.iex_ops.rotate(x, table, positions)
    with torch.no_grad(), pytest.raises(RuntimeError, match=PASSED):
        torch.ops.iex_ops.rotate(x, table, positions)


@pytest.mark.parametrize("dual", ["x", "table"])
@pytest.mark.parametrize("trained", [False, True])
def test_forward_mode(operands, trained, dual):
    """No result without the tangent that it should have: a dual operand is refused, gradients or not; what is not differentiated passes."""
    x, table, positions = operands
    x.requires_grad_(trained)
    rotate = torch.ops.iex_ops.rotate
    with forward.dual_level():
        given = [forward.make_dual(t, t.detach()) if name == dual else t for name, t in (("x", x), ("table", table))]
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                rotate(*given, positions)
        with pytest.raises(RuntimeError, match=PASSED):
            rotate(*(forward.unpack_dual(t).primal for t in given), positions)
