"""Generation by the decoder layer: what decode() refuses it refuses before the cache has changed."""
import pytest
import torch

from intrasm_engine_amd import workloads as W
from intrasm_engine_amd.decoder_layer import SparseDecoderLayer
from intrasm_engine_amd.pytorch import paged_attention as PA

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, MLP, PAGE = 256, 4, 512, 16


@pytest.fixture(scope="module")
def layer(dev):
    weights = {name: W.pruned_weight(100 + i, HIDDEN, HIDDEN, "2:4", sigma=0.06) for i, name in enumerate(("q", "k", "v", "o"))}
    weights |= {"gate": W.pruned_weight(104, MLP, HIDDEN, 0.80, sigma=0.06), "up": W.pruned_weight(105, MLP, HIDDEN, 0.80, sigma=0.06),
                "down": W.pruned_weight(106, HIDDEN, MLP, 0.80, sigma=0.06)}
    return SparseDecoderLayer(weights, HIDDEN, HEADS, MLP, dev)


def begun(layer, dev, tokens, bounds=True):
    """A cache with prompts of ``tokens`` tokens, and what decode() takes beside x."""
    width = [-(-(n + 4) // PAGE) for n in tokens]
    table = torch.full((len(tokens), max(width)), -1, dtype=torch.int32, device=dev)
    order = torch.randperm(sum(width), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(dev)
    for s, n in enumerate(width):
        table[s, :n] = order[sum(width[:s]):sum(width[:s + 1])]
    cache = layer.new_cache(sum(width), PAGE, bounds=bounds)
    for t in (cache.keys, cache.values, cache.bounds):
        if t is not None:
            t.zero_()
    lengths = torch.tensor(tokens, dtype=torch.int32, device=dev)
    rotation = PA.rotation_table(table.shape[1] * PAGE, HIDDEN // HEADS, device=dev)
    offsets = torch.tensor([0] + tokens, device=dev).cumsum(0).to(torch.int32)
    gen = torch.Generator().manual_seed(2)
    layer.prompt(torch.relu(torch.randn(HIDDEN, sum(tokens), generator=gen)).half().to(dev), cache, table, lengths, offsets, rotation)
    x = torch.relu(torch.randn(HIDDEN, len(tokens), generator=gen)).half().to(dev)
    return cache, table, lengths, rotation, x


def test_one_page_is_the_newest(layer, dev):
    """pages=1: the page that holds the new token, whatever the scores of the others."""
    cache, table, lengths, rotation, x = begun(layer, dev, [40, 8, 16])
    lengths += 1
    got = layer.decode(x, cache, table, lengths, rotation, pages=1)
    split = lambda name: layer._tokens(layer.proj(name, x))  # noqa: E731
    q = cache.append_(split("k"), split("v"), table, lengths, None, split("q"), rotation)
    newest = ((lengths - 1) // PAGE).view(-1, 1, 1).expand(-1, HEADS, 1).contiguous()
    attended = cache.attend(q, table, lengths, None, newest)
    h = layer._proj_with("o", attended.permute(1, 2, 0).reshape(HIDDEN, 3), x, 1)
    want = layer.mlp_block(h).float()
    assert (got.float() - want).abs().max() <= 2e-2 * want.abs().max()      # (the layer's own measure: a chain of fp16 operators)


def test_refused_before_anything_is_written(layer, dev):
    for bounds, pages, match in ((True, -1, "pages"), (False, 2, "bounds")):
        cache, table, lengths, rotation, x = begun(layer, dev, [20, 5], bounds)
        before = [t.clone() for t in (cache.keys, cache.values)]
        lengths += 1
        with pytest.raises((RuntimeError, ValueError), match=match):
            layer.decode(x, cache, table, lengths, rotation, pages=pages)
        assert torch.equal(cache.keys, before[0]) and torch.equal(cache.values, before[1])
