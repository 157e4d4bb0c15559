"""Ragged prompts and then steps over caches of both widths, at tolerances that nothing but the right result meets: what the cache holds against the
tokens that went in, and the attention against what it holds."""
import pytest
import torch

from _paged import E4M3, HALF_STEP, Cache, rotated
from intrasm_engine_amd.pytorch import paged_attention as PA

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def view_of(cache, table, lengths):
    """The cache for _paged's plain forms."""
    plain = Cache.__new__(Cache)
    plain.__dict__.update(table=table, lengths=lengths, page=cache.page_size, dim=cache.head_dim, kv_heads=cache.kv_heads, pages=cache.keys.shape[0], dtype=cache.dtype,
                          e8=cache.key_exponents is not None, width=table.shape[1], keys=cache.keys, values=cache.values, key_exponents=cache.key_exponents,
                          value_exponents=cache.value_exponents)
    return plain


@pytest.mark.parametrize("dtype,kv_heads,heads,dim,page,interleaved", [(F16, 2, 4, 64, 16, False), (BF16, 1, 8, 128, 32, True), (F16, 3, 3, 256, 64, False), (BF16, 2, 6, 128, 16, True)])
@pytest.mark.parametrize("eight_bits", [False, True])
def test_prompts_then_tokens(dev, dtype, kv_heads, heads, dim, page, interleaved, eight_bits):
    gen = torch.Generator(device=dev).manual_seed(11)
    prompts, steps = [5, 40, 1, 17], 6
    counts = [-(-(n + steps) // page) for n in prompts]
    order = torch.randperm(sum(counts) + 2, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(dev)
    table = torch.full((4, max(counts)), -1, dtype=torch.int32, device=dev)
    for s, n in enumerate(counts):
        table[s, :n] = order[sum(counts[:s]):sum(counts[:s + 1])]
    cache = PA.KVCache(sum(counts) + 2, page, kv_heads, dim, dtype, dev, eight_bits)
    rotation = PA.rotation_table(table.shape[1] * page, dim, device=dev)
    lengths = torch.tensor(prompts, dtype=torch.int32, device=dev)
    offsets = torch.tensor([0] + prompts, device=dev).cumsum(0).to(torch.int32)
    draw = lambda n, h: torch.randn(n, h, dim, generator=gen, device=dev).to(dtype)  # noqa: E731
    k, v = draw(sum(prompts), kv_heads), draw(sum(prompts), kv_heads)
    cache.append_(k, v, table, lengths, offsets, None, rotation, interleaved)
    went_in = [(k[a:b], v[a:b]) for a, b in zip([0, 5, 45, 46], [5, 45, 46, 63])]
    for step in range(steps):
        lengths += 1
        k, v, q = draw(4, kv_heads), draw(4, kv_heads), draw(4, heads)
        turned = cache.append_(k, v, table, lengths, None, q, rotation, interleaved)
        out = cache.attend(turned, table, lengths).double()
        went_in = [(torch.cat([a, k[s:s + 1]]), torch.cat([b, v[s:s + 1]])) for s, (a, b) in enumerate(went_in)]
        plain = view_of(cache, table, lengths)
        for s, (k_in, v_in) in enumerate(went_in):
            n = k_in.shape[0]
            positions = torch.arange(n, device=dev)
            want_q, loose = rotated(q[s:s + 1], positions[-1:], rotation, interleaved)
            assert ((turned[s:s + 1].double() - want_q).abs() <= want_q.abs() * HALF_STEP[dtype] + 2 * loose + 2.0 ** -25).all()
            want_k, loose = rotated(k_in, positions, rotation, interleaved)
            for h in range(kv_heads):
                held = plain.rows(s, h)
                for got, want, rounding in ((held[0], want_k[:, h], 2 * loose[:, h]), (held[1], v_in[:, h].double(), 0.0)):
                    # (e4m3: half a step of a normal code, or of the smallest ones 2^-10 of a scale that is at most the largest / 224)
                    allowed = want.abs() * HALF_STEP[E4M3] + 2.0 ** -10 / 224 * want.abs().amax(-1, keepdim=True) if eight_bits else want.abs() * HALF_STEP[dtype] + 2.0 ** -25
                    assert got.shape[0] == n and ((got - want).abs() <= allowed + rounding).all()
        want, allowed = plain.attend(turned, dim ** -0.5)
        assert ((out - want).abs() <= allowed).all()
        # neither nothing, nor a neighbour's result, nor the values' mean passes for it
        for other in (torch.zeros_like(want), want.roll(1, 0), torch.stack([torch.stack([plain.rows(s, h * kv_heads // heads)[1].mean(0) for h in range(heads)]) for s in range(4)])):
            assert ((other - want).abs() > allowed).any(-1).all()
