"""Two layers' caches over one table and one tensor of lengths, each with an account of its own: steps, and evictions by a copy of the lengths each but the last."""
import pytest
import torch

from intrasm_engine_amd.pytorch import paged_attention as PA

pytestmark = pytest.mark.gpu
PAGE, KV, HEADS, DIM, KEEP = 16, 2, 4, 64, 40


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_two_layers(dev, dtype):
    """Every layer keeps what got most of its own attention, its own rows; lengths are cut once; and steps go on over what each has."""
    gen = torch.Generator(device=dev).manual_seed(6)
    draw = lambda n, h: torch.randn(n, h, DIM, generator=gen, device=dev).to(dtype)  # noqa: E731
    caches = [PA.KVCache(12, PAGE, KV, DIM, dtype, dev) for _ in range(2)]
    table = torch.randperm(12, generator=gen, device=dev).to(torch.int32).view(2, 6)
    accounts = [c.new_weights(table) for c in caches]
    prompts = [60, 30]
    lengths = torch.tensor(prompts, dtype=torch.int32, device=dev)
    offsets = torch.tensor([0, 60, 90], dtype=torch.int32, device=dev)
    rows = []      # of a layer and sequence: keys and values, (tokens, heads, features)
    for c in caches:
        k, v = draw(90, KV), draw(90, KV)
        c.append_(k, v, table, lengths, offsets)
        rows.append([[k[:60], v[:60]], [k[60:], v[60:]]])
    for step in range(16):
        lengths += 1
        for c, account, mine in zip(caches, accounts, rows):
            k, v, q = draw(2, KV), draw(2, KV), draw(2, HEADS)
            c.append_(k, v, table, lengths)
            out = c.attend(q, table, lengths, weights=account)
            for s in range(2):
                mine[s] = [torch.cat([a, b[s:s + 1]]) for a, b in zip(mine[s], (k, v))]
                for h in range(HEADS):
                    keys, values = (x[:, h // 2].double() for x in mine[s])
                    p = torch.softmax(keys @ q[s, h].double() * DIM ** -0.5, 0)
                    want = p @ values
                    # the result's half step; probabilities to 2^-16, scores to 68 roundings of up to 24 (terms' magnitudes, twice), sums of 80 terms
                    slack = (2.0 ** -16 + 2 * 68 * 2.0 ** -24 * 24 + 80 * 2.0 ** -24) * (p @ values.abs())
                    assert ((out[s, h].double() - want).abs() <= want.abs() * torch.finfo(dtype).eps / 2 + slack + 2.0 ** -25).all(), (step, s, h)
        if step in (3, 12):
            before = [a.clone() for a in accounts]
            kept = [c.evict_(table, n, a, KEEP, 8, 2) for c, n, a in zip(caches, (lengths.clone(), lengths), accounts)]
            for layer in range(2):
                for s in range(2):
                    n = rows[layer][s][0].shape[0]
                    if n <= KEEP:
                        continue
                    for h in range(KV):
                        middle = before[layer][s, h, 2:n - 8]
                        want = sorted([0, 1] + (middle.sort(descending=True, stable=True)[1][:KEEP - 10] + 2).tolist() + list(range(n - 8, n)))
                        assert kept[layer][s, h].tolist() == want, (layer, s, h)
                        assert torch.equal(accounts[layer][s, h, :KEEP], before[layer][s, h, want])
                    heads = torch.arange(KV, device=dev)
                    rows[layer][s] = [x[kept[layer][s].T.long(), heads] for x in rows[layer][s]]
            assert not torch.equal(*kept) and lengths.tolist() == [rows[0][s][0].shape[0] for s in range(2)]
