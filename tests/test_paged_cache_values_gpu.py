"""What weights, sums and stored rows of the paged cache hold: bits of the weights, values at the ends of the type's range, rows with infinities."""
import math

import pytest
import torch

from _paged import E4M3, HALF_STEP, Cache, feature_major, power

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


@pytest.mark.parametrize("dim,e8", [(64, False), (128, False), (256, False), (128, True)])
@pytest.mark.parametrize("n", [1, 2, 3, 33, 300, 1500, 9000])
def test_values_at_the_ends_of_the_range(ops, dev, dim, e8, n):
    """softmax . v of values near bf16's largest is no larger than they are, however many there are; of its smallest normal ones no smaller
    (e4m3: of exponents from 48 on).

    Allowed: as in _paged.Cache.attend, and for the smallest the sums' own smallest step over a weight of 1 / (2 n)."""
    c = Cache(dev, [n, n, n, n], 1, dim, 64, BF16, e8=e8, poison=False)
    largest = float(torch.finfo(BF16).max)
    for s, (size, exponent) in enumerate(((2e38, 247), (1.3 * 2.0 ** 127 if e8 else largest, 247), (2.0 ** -73 if e8 else 2.0 ** -110, 48), (2.0 ** -71 if e8 else 2.0 ** -126, 48))):
        rows = torch.full((n, dim), size, device=dev)
        rows[:, 1::2] *= -1
        if s == 2:
            rows *= 1 + torch.rand(n, dim, device=dev)
        pages = c.table[s, :-(-n // 64)].long()
        rows = torch.cat([rows, torch.zeros(-n % 64, dim, device=dev)]).view(-1, 1, 64, dim).to(BF16)
        if e8:
            c.values.view(torch.uint8)[pages] = (rows.double() / power(torch.tensor(exponent))).float().to(E4M3).view(torch.uint8)
            c.value_exponents[pages] = exponent
        else:
            c.values[pages] = rows
    q = torch.randn(4, 3, dim, device=dev).to(BF16)
    q[0] = 0.0
    scale = dim ** -0.5
    want, allowed = c.attend(q, scale)
    assert want[:2].abs().max() <= largest * (1 + 2.0 ** -40)
    allowed[2:] += 2 * n * 2.0 ** -149
    got = attend(ops, c, q, scale).double()
    for s in range(4):
        beyond = float(((got[s] - want[s]).abs() - allowed[s]).max())
        assert beyond <= 0, (s, float(got[s].abs().max()), beyond / float(allowed[s].max()))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout,single", [("tokens", True), ("features", True), ("tokens", False), ("features", False)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_eight_bit_rows_keep_what_is_finite(ops, dev, dtype, layout, single, dim):
    """Infinities and NaN of a row become NaN; its other features are stored by the least power of two that brings the largest finite one to
    448, as in a row without them."""
    n = 6 if single else 70
    gen = torch.Generator(device=dev).manual_seed(4)
    c = Cache(dev, [1] * n if single else [n], 2, dim, 16, dtype, e8=True, bounds=True, poison=False)
    x = torch.randn(n, 2, dim, generator=gen, device=dev).to(dtype)
    bad = torch.zeros(n, 2, dim, dtype=torch.bool, device=dev)
    for i, value in enumerate((math.inf, -math.inf, math.nan)):
        bad[i, 0, 5 + i] = True
        x[i, 0, 5 + i] = value
    bad[3, 1], bad[4, 0, 1:] = True, True
    x[3, 1], x[4, 0, 1:] = math.inf, math.nan
    shape = feature_major if layout == "features" else lambda t: t
    offsets = None if single else torch.tensor([0, n], dtype=torch.int32, device=dev)
    ops.kv_append_(shape(x), shape(x), c.keys, c.values, c.table, c.lengths, offsets, None, None, False, c.bounds, *c.exponents())
    finite = torch.where(bad, 0.0, x.double())
    top = finite.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)
    exponent = torch.where(top == 0, 1, (exponent + 118 + (mantissa > 0.875)).clamp(1, 254))
    step = torch.maximum(finite.abs() * HALF_STEP[E4M3], 2.0 ** -10 * power(exponent)[..., None])
    for name, exponents in (("keys", c.key_exponents), ("values", c.value_exponents)):
        for i in range(n):
            page, slot = (int(c.table[i, 0]), 0) if single else (int(c.table[0, i // 16]), i % 16)
            got = c.stored(name, page)[:, slot]
            assert torch.equal(got.isnan(), bad[i]) and torch.equal(exponents[page, :, slot].long(), exponent[i])
            assert ((got - finite[i]).abs()[~bad[i]] <= step[i][~bad[i]]).all()
