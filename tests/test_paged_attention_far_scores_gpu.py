"""Finite operands with scores as large as their types allow: the softmax of far scores is its limit, a share for each of the largest."""
import pytest
import torch

from _paged import Cache

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


# scale * score from below where the fused step is given up (2^16) to fp16's largest, 128 * 65504^2 / sqrt(128), and bf16's
@pytest.mark.parametrize("dtype,size", [(F16, 90.0), (F16, 200.0), (F16, 1100.0), (F16, 2500.0), (F16, 9000.0), (F16, 61000.0), (BF16, 1100.0), (BF16, 3e4), (BF16, 1e9), (BF16, 1e17)])
@pytest.mark.parametrize("e8", [False, True])
@pytest.mark.parametrize("lengths,width", [([1, 40, 700], None), ([3000, 5, 129], None), ([12], 2)])
def test_shares_of_the_largest(dev, dtype, size, e8, lengths, width):
    """Keys are a direction times 1 / 16 .. 3 / 4, but for one, two or four tokens with all of it: by the 16 features' size each a gap of at least
    2^10 in scale * score, so the others get nothing and those the same.  Their values are whole numbers of up to 15, their means have 6 bits: a result is its mean, or off by the roundings of a few products in
    32 bits where the weights before the division are 2^(up to 2^-8) and not 1."""
    dim, kv, heads = 128, 2, 4
    c = Cache(dev, lengths, kv, dim, 64 if width is None else 16, dtype, e8=e8, poison=False, width=width)
    gen = torch.Generator(device=dev).manual_seed(9)
    signs = torch.where(torch.rand(dim, generator=gen, device=dev) < 0.5, -1.0, 1.0)
    keys = torch.randint(1, 13, (c.pages, kv, c.page, 1), generator=gen, device=dev) / 16 * signs * size
    values = torch.randint(-15, 16, (c.pages, kv, c.page, dim), generator=gen, device=dev).float()
    first = [[[0] if n < 5 else [n - 1, n // 2] if h else [1, 3, n // 3, n - 2] for h in range(kv)] for n in lengths]
    for s in range(len(lengths)):
        for h in range(kv):
            first[s][h] = sorted(set(first[s][h]))
            for t in first[s][h]:
                keys[int(c.table[s, t // c.page]), h, t % c.page] = signs * size
    if e8:      # (a power of two of what e4m3 has: whole numbers of up to 4 bits)
        codes = lambda x, top: ((x / top).float().to(torch.float8_e4m3fn), torch.full(x.shape[:3], int(torch.log2(torch.tensor(top))) + 127, dtype=torch.uint8, device=dev))  # noqa: E731
        power = 2.0 ** round(float(torch.log2(torch.tensor(size / 16))))
        c.keys, c.key_exponents = codes(keys / size * 16 * power, power)
        c.values, c.value_exponents = codes(values, 1.0)
    else:
        c.keys, c.values = keys.to(dtype), values.to(dtype)
    q = (signs * size).to(dtype).expand(len(lengths), heads, dim) * torch.tensor([1, 1, 1, 0.5], device=dev, dtype=dtype)[:, None]
    weights = torch.zeros(len(lengths), kv, c.width * c.page, device=dev)
    scale = dim ** -0.5
    assert c.keys.isfinite().all() if not e8 else c.keys.float().isfinite().all()
    got = torch.ops.iex_ops.paged_attention_accumulate_(q, c.keys, c.values, c.table, c.lengths, weights, scale, *c.exponents())
    plain = torch.ops.iex_ops.paged_attention(q, c.keys, c.values, c.table, c.lengths, scale, None, *c.exponents())
    assert torch.equal(got, plain)
    for s in range(len(lengths)):
        for h in range(heads):
            k, v = c.rows(s, h // 2)
            scores = (k @ q[s, h].double()) * scale
            at = torch.tensor(first[s][h // 2], device=dev)
            others = torch.ones(lengths[s], dtype=torch.bool, device=dev)
            others[at] = False
            assert (scores[at] == scores.max()).all() and (not others.any() or scores.max() - scores[others].max() > 150)
            assert (got[s, h].double() - v[at].mean(0)).abs().max() <= 4 * 15 * 2.0 ** -22, (s, h)
        for h in range(kv):
            want = torch.zeros(c.width * c.page, device=dev)
            want[first[s][h]] = 2.0 / len(first[s][h])
            assert (weights[s, h] - want).abs().max() <= 2.0 ** -20 and (weights[s, h][want == 0] == 0).all(), (s, h)
