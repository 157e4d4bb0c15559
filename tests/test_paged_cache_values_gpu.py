"""What weights, sums and stored rows of the paged cache hold: bits of the weights, values at the ends of the type's range, rows with infinities."""
import math

import pytest
import torch

from _paged import E4M3, HALF_STEP, Cache

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops(dev):
    return torch.ops.iex_ops


def attend(ops, c, q, scale=1.0, pages=None):
    return ops.paged_attention(q, c.keys, c.values, c.table, c.lengths, scale, pages, *c.exponents())


def fill(c, s, h, keys, values):
    """Rows of sequence s's first tokens (n, dim): 16 bits as they are, in an 8-bit cache with the exponent of 1 (values it holds exactly)."""
    for name, rows in (("keys", keys), ("values", values)):
        for t in range(rows.shape[0]):
            page, slot = int(c.table[s, t // c.page]), t % c.page
            if c.e8:
                getattr(c, name).view(torch.uint8)[page, h, slot] = rows[t].float().to(E4M3).view(torch.uint8)
                getattr(c, name[:-1] + "_exponents")[page, h, slot] = 127
            else:
                getattr(c, name)[page, h, slot] = rows[t].to(c.dtype)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,e8", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
def test_bits_of_the_weights(ops, dev, dtype, e8, dim):
    """Values of 1 and -1 with scores 0 and -x: (1 - e^-x) / (1 + e^-x), the difference of two weights near 1, shows every bit of them.

    Allowed beside the result's rounding, of a pair's weights whose sum is 1.9 at least: the exponential of one (2^-23; its argument is below
    2^-2, whose roundings are nothing beside that), a lowest bit that is set in each (2^-23) and, with two parts of 11 bits in fp16, 2^-22
    of each; the sum of the weights and of three parts' products, n terms each, rounded at 2^-24 of n."""
    parts = 2.0 ** -22 if dtype == F16 and not e8 else 0.0
    xs = [0.015625, 0.0078125, 0.001953125, 0.0625] if e8 else [0.0117, 0.0039, 0.0007, 0.0521, 0.0003, 0.0313]
    for n in (2, 40):
        c = Cache(dev, [n] * len(xs), 2, dim, 16, dtype, e8=e8, poison=False)
        q = torch.zeros(len(xs), 4, dim, dtype=dtype, device=dev)
        q[..., 0] = 1.0
        want = torch.zeros(len(xs), 4, dim, dtype=torch.float64, device=dev)
        for s, x in enumerate(xs):
            for h in range(2):
                x_h = float(torch.tensor(-x * (1 + h), dtype=dtype))
                keys, values = torch.zeros(n, dim, device=dev), torch.ones(n, dim, device=dev)
                keys[1::2, 0] = x_h
                values[1::2] = -1.0
                fill(c, s, h, keys, values)
                want[s, 2 * h:2 * h + 2] = math.tanh(-x_h / 2)
        got = attend(ops, c, q).double()
        allowed = want.abs() * HALF_STEP[dtype] + (3 * 2.0 ** -23 + 2 * parts + 4 * 2.0 ** -23) / 1.9
        assert ((got - want).abs() <= allowed).all(), f"{n}: {float(((got - want).abs() - allowed).max()):.3g} beyond {float(allowed.min()):.3g}"
