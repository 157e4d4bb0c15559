"""The decoder layer generating with a bounded cache: steps that keep account, evictions between them, positions that are given."""
import pytest
import torch

from _paged import rotated
from intrasm_engine_amd import workloads as W
from intrasm_engine_amd.decoder_layer import SparseDecoderLayer
from intrasm_engine_amd.pytorch import paged_attention as PA
from intrasm_engine_amd.pytorch.utils import sparse_to_dense

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, MLP, PAGE = 256, 4, 512, 16


@pytest.fixture(scope="module")
def made(dev):
    weights = {name: W.pruned_weight(100 + i, HIDDEN, HIDDEN, "2:4", sigma=0.06) for i, name in enumerate(("q", "k", "v", "o"))}
    weights |= {"gate": W.pruned_weight(104, MLP, HIDDEN, 0.80, sigma=0.06), "up": W.pruned_weight(105, MLP, HIDDEN, 0.80, sigma=0.06),
                "down": W.pruned_weight(106, HIDDEN, MLP, 0.80, sigma=0.06)}
    dense = {n: sparse_to_dense(c.m, c.k, torch.from_numpy(c.values).to(dev).half().float(), torch.from_numpy(c.row_offsets).to(dev),
                                torch.from_numpy(c.column_indices).to(dev)) for n, c in weights.items()}
    return SparseDecoderLayer(weights, HIDDEN, HEADS, MLP, dev), dense


@pytest.mark.parametrize("eight_bits", [False, True])
def test_layer_with_a_budget(dev, made, eight_bits):
    """Against dense 32-bit matrices, plain attention over what the evictions left, and a plain account of it."""
    layer, dense = made
    gen = torch.Generator().manual_seed(0)
    prompts, keep = [50, 20], 30
    table = torch.randperm(12, generator=gen).to(torch.int32).view(2, 6)[:, :5].contiguous().to(dev)
    cache = layer.new_cache(12, PAGE, eight_bits=eight_bits)
    account = cache.new_weights(table)
    rotation = PA.rotation_table(100, layer.head_dim, device=dev)
    lengths = torch.tensor(prompts, dtype=torch.int32, device=dev)
    x = torch.relu(torch.randn(HIDDEN, sum(prompts), generator=gen)).half().to(dev)
    places = torch.cat([torch.arange(n) for n in prompts]).to(dev, torch.int32)
    layer.prompt(x, cache, table, lengths, torch.tensor([0, 50, 70], dtype=torch.int32, device=dev), rotation, positions=places)
    split = lambda t: t.view(HEADS, 64, -1).permute(2, 0, 1)  # noqa: E731
    turn = lambda t, at: rotated(t, at.long(), rotation, False)[0].float()  # noqa: E731
    parts = ((0, 50), (50, 70))
    keys = [turn(split(dense["k"] @ x[:, a:b].float()), torch.arange(b - a, device=dev)) for a, b in parts]
    values = [split(dense["v"] @ x[:, a:b].float()) for a, b in parts]
    got = [torch.zeros(n, HEADS, device=dev) for n in prompts]
    position = torch.tensor(prompts, dtype=torch.int32, device=dev)
    heads = torch.arange(HEADS, device=dev)
    for step in range(9):
        lengths += 1
        x = torch.relu(torch.randn(HIDDEN, 2, generator=gen)).half().to(dev)
        before = account.clone()
        y = layer.decode(x, cache, table, lengths, rotation, positions=position, weights=account)
        q, k, v = (split(dense[n] @ x.float()) for n in ("q", "k", "v"))
        attended = []
        for s in range(2):
            at = position[s:s + 1]
            keys[s], values[s] = torch.cat([keys[s], turn(k[s:s + 1], at)]), torch.cat([values[s], v[s:s + 1]])
            p = torch.softmax((keys[s] * turn(q[s:s + 1], at)).sum(-1) / 8, 0)      # (tokens, heads)
            got[s] = torch.cat([got[s], torch.zeros(1, HEADS, device=dev)]) + p
            attended.append((p[..., None] * values[s]).sum(0))
            mine = account[s, :, :got[s].shape[0]]
            assert (mine - got[s].T).abs().max() <= 2e-2 * (step + 1) and (account[s, :, got[s].shape[0]:] == 0).all()
        # what a pass adds is one per head and sequence (the account's own sum may differ from the plain one's behind an eviction: what left took with it what
        # roundings of e4m3 had moved to it): weights to 2^-18, and each token's sum, nine in all at most, rounded to 2^-24 of itself, before and now
        assert ((account.double() - before.double()).sum(-1) - 1).abs().max() <= 2.0 ** -18 + 2 * 9 * 2.0 ** -24
        h = x.float() + dense["o"] @ torch.stack(attended).permute(1, 2, 0).reshape(HIDDEN, 2)
        want = h + dense["down"] @ (torch.nn.functional.silu(dense["gate"] @ h) * (dense["up"] @ h))
        # (the layer's own measure: a chain of fp16 operators; a value in e4m3 is 2^-4 off)
        assert y.shape == x.shape and (y.float() - want).abs().max() <= (5e-2 if eight_bits else 2e-2) * want.abs().max()
        position += 1
        if step in (2, 5):
            kept = cache.evict_(table, lengths, account, keep, 6, 2)
            for s in range(2):
                if keys[s].shape[0] <= keep:
                    assert kept[s, 0].tolist() == list(range(keys[s].shape[0])) + [-1] * (keep - keys[s].shape[0])
                    continue
                at = kept[s].T.long()      # (keep, heads)
                keys[s], values[s], got[s] = keys[s][at, heads], values[s][at, heads], got[s][at, heads]
            assert lengths.tolist() == [keys[0].shape[0], keys[1].shape[0]]


def test_refused_before_anything_is_written(dev, made):
    layer, _ = made
    cache = layer.new_cache(4, PAGE, bounds=True)
    for t in (cache.keys, cache.values):
        t.zero_()
    table, lengths = torch.zeros(1, 2, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    x = torch.ones(HIDDEN, 1, dtype=torch.float16, device=dev)
    good = cache.new_weights(table)
    for weights, pages, match in ((good, 1, "selected"), (good[..., :16], 0, "weights must be"), (good.half(), 0, "weights must be"), (good.cpu(), 0, "weights must be")):
        with pytest.raises(ValueError, match=match):
            layer.decode(x, cache, table, lengths, pages=pages, weights=weights)
    with pytest.raises(ValueError, match="listed"):
        cache.attend(torch.zeros(1, HEADS, 64, dtype=torch.float16, device=dev), table, lengths, None, torch.zeros(1, HEADS, 1, dtype=torch.int32, device=dev), good)
    assert not cache.keys.any() and not cache.values.any() and not good.any()


def test_a_captured_step_keeps_account(dev, made):
    """Positions, lengths, account and evictions between replays, against eager steps on a copy."""
    layer, _ = made
    gen = torch.Generator().manual_seed(3)
    rotation = PA.rotation_table(60, 64, device=dev)
    table = torch.arange(6, dtype=torch.int32, device=dev).view(2, 3)
    caches = [layer.new_cache(6, PAGE) for _ in range(2)]
    prompt = torch.randn(HIDDEN, 40, generator=gen).half().to(dev)
    lengths = [torch.tensor([25, 15], dtype=torch.int32, device=dev) for _ in range(2)]
    accounts = [caches[0].new_weights(table) for _ in range(2)]
    position = torch.tensor([[25, 15], [3, 4]], dtype=torch.int32, device=dev)
    for c in caches:
        for t in (c.keys, c.values):
            t.zero_()
        places = torch.cat([torch.arange(25), torch.arange(15)]).to(dev, torch.int32).expand(2, -1).contiguous()
        layer.prompt(prompt, c, table, lengths[0], torch.tensor([0, 25, 40], dtype=torch.int32, device=dev), rotation, places, [20, 12], True)
    x = torch.randn(HIDDEN, 2, generator=gen).half().to(dev)
    step = lambda i, given: layer.decode(given, caches[i], table, lengths[i], rotation, positions=position, sections=[20, 12], in_turn=True, weights=accounts[i])  # noqa: E731
    layer.decode(x, layer.new_cache(6, PAGE), table, lengths[0], rotation, positions=position, sections=[20, 12], in_turn=True, weights=accounts[0].clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lengths[0] += 1
        y = step(0, x)
    for i in range(8):
        x.copy_(torch.randn(HIDDEN, 2, generator=gen).half())
        graph.replay()
        lengths[1] += 1
        want = step(1, x.clone())
        torch.cuda.synchronize()
        assert (y.float() - want.float()).abs().max() <= 2e-2 * want.float().abs().max(), i
        assert (accounts[0] - accounts[1]).abs().max() <= 2e-2 * (i + 1) and torch.equal(lengths[0], lengths[1])
        position += 1
        if i in (2, 5):
            accounts[1].copy_(accounts[0])      # (the captured projections may be by another form of the weights: the same tokens are to go)
            kept = [c.evict_(table, n, w, 18, 4, 1) for c, n, w in zip(caches, lengths, accounts)]
            assert torch.equal(*kept) and torch.equal(*accounts)
