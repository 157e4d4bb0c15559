"""Rotation by positions on one to four axes, its gradient, and keys appended so, against plain forms in 64 bits."""
import math

import pytest
import torch

from _paged import E4M3, HALF_STEP, Cache, feature_major, rotation_table
from intrasm_engine_amd import _lib
from intrasm_engine_amd.pytorch import paged_attention as PA

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
STEP = {**HALF_STEP, F32: 2.0 ** -24}
TINY = {F16: 2.0 ** -25, BF16: 0.0, F32: 0.0}


@pytest.fixture(scope="module")
def ops(dev):
    return torch.ops.iex_ops


def axes_of(sections, in_turn):
    left, out = list(sections), []
    if not in_turn:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    while sum(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


def turned(x, table, positions, sections=None, in_turn=False, interleaved=False, back=False):
    """In 64 bits, and how far 32-bit products and sums may be off: a product's and the sum's half steps."""
    r = table.shape[1]
    places = positions if positions.dim() == 2 else positions[None]
    axes = axes_of(sections if sections is not None else [r // 2], in_turn)
    rows = torch.stack([places[a] for a in axes], 1).long().clamp(min=0)
    wide = torch.cat([table.double(), torch.full((1, r), math.nan, dtype=torch.float64, device=x.device)])
    rows = rows.clamp(max=table.shape[0])
    plane = torch.arange(r // 2, device=x.device)
    c, s = wide[rows, plane][:, None], wide[rows, plane + r // 2][:, None]
    s = -s if back else s
    out, slack = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    x0, x1 = out[..., a].clone(), out[..., b].clone()
    out[..., a], out[..., b] = x0 * c - x1 * s, x1 * c + x0 * s
    slack[..., a] = slack[..., b] = 2 * 2.0 ** -24 * (x0.abs() + x1.abs())
    return out, slack


def close(got, want, slack, what=""):
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    off = (got.double() - want).abs() - (want.abs() * STEP[got.dtype] + slack * (1 + STEP[got.dtype]) + TINY[got.dtype])
    assert not (torch.where(want.isnan(), -1.0, off) > 0).any(), what


def inputs(dev, tokens, heads, dim, r, axes, dtype, rows=97, seed=1):
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=gen, device=dev).to(dtype)
    positions = torch.randint(0, rows, (axes, tokens), generator=gen, device=dev, dtype=torch.int32)
    return x, rotation_table(rows, r, dev), positions if axes > 1 else positions[0]


LAYOUTS = {
    "tokens": lambda x: x,
    "features": feature_major,
    "features_apart": lambda x: torch.stack([x, x], -1).flatten(-2)[..., ::2],
    "rows_apart": lambda x: torch.cat([x, x.flip(2)], 1)[:, :x.shape[1]],
    "features_off_the_chunk": lambda x: torch.cat([x.permute(1, 2, 0), torch.zeros_like(x.permute(1, 2, 0)[..., :3])], -1)[..., 1:1 + x.shape[0]].permute(2, 0, 1) if x.shape[0] > 1 else x,
}


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tokens,heads,dim,r,sections,in_turn,interleaved", [
    (1, 2, 64, 64, None, False, False), (130, 3, 128, 128, [16, 24, 24], False, False), (67, 5, 128, 64, [12, 10, 10], True, True), (200, 1, 256, 256, [100, 1, 20, 7], True, False),
    (33, 9, 80, 80, [15, 25], False, True), (9, 2, 48, 32, [0, 16], False, False), (64, 2, 72, 36, [7, 11], True, False), (50, 3, 7, 4, [1, 1], False, True),
    (1, 3, 5, 2, None, False, False), (71, 2, 96, 96, [48], True, False)])
def test_rotate(ops, dev, dtype, layout, tokens, heads, dim, r, sections, in_turn, interleaved):
    x, table, positions = inputs(dev, tokens, heads, dim, r, len(sections) if sections and len(sections) > 1 else 1, dtype)
    given = LAYOUTS[layout](x)
    # (the values that the layout shows; what lies between them does not matter)
    x = given.contiguous()
    for back in (False, True):
        got = ops.rotate(given, table, positions, sections, in_turn, interleaved, back)
        assert got.shape == x.shape and got.dtype == dtype
        want, slack = turned(x, table, positions, sections, in_turn, interleaved, back)
        close(got, want, slack, f"back {back}")
        assert torch.equal(got[..., r:], x[..., r:])


@pytest.mark.parametrize("dtype,layout,tokens,heads,dim,kernel", [(F16, "tokens", 300, 4, 128, "rotate_rows_kernel<f16>"), (F32, "features", 64, 4, 128, "rotate_columns_kernel<f32>"),
                                                                  (BF16, "features", 65, 4, 64, "rotate_tokens_kernel<bf16>"), (BF16, "tokens", 65, 4, 66, "rotate_single_kernel<bf16>"),
                                                                  (F16, "features", 7, 4, 64, "rotate_single_kernel<f16>")])
def test_kernels(ops, dev, dtype, layout, tokens, heads, dim, kernel):
    x, table, positions = inputs(dev, tokens, heads, dim, dim, 1, dtype)
    ops.rotate(LAYOUTS[layout](x), table, positions)
    assert kernel in _lib.last_kernels()


def test_many_heads_and_tokens(ops, dev):
    """Threads that take several heads, one after the other, and more tokens than one workgroup's."""
    for layout in ("tokens", "features"):
        for heads, tokens in ((67, 2001), (40, 8192)):
            x, table, positions = inputs(dev, tokens, heads, 64, 64, 3, BF16)
            got = ops.rotate(LAYOUTS[layout](x), table, positions, [10, 11, 11])
            want, slack = turned(x, table, positions, [10, 11, 11])
            close(got, want, slack)


def test_positions_outside_the_table(ops, dev):
    """Below zero: as zero.  Behind the table: NaN, in the planes of that axis only."""
    for layout, dim in (("tokens", 64), ("features", 64), ("tokens", 36)):
        x, table, positions = inputs(dev, 40, 2, dim, dim, 2, F16, rows=20)
        positions[0, 3], positions[1, 5], positions[0, 7], positions[1, 9], positions[0, 11] = -1, -(1 << 31), 20, (1 << 31) - 1, 19
        got = ops.rotate(LAYOUTS[layout](x), table, positions, [dim // 4, dim // 4], False, True)
        want, slack = turned(x, table, positions, [dim // 4, dim // 4], False, True)
        close(got, want, slack)
        assert got[7, :, :dim // 2].isnan().all() and not got[7, :, dim // 2:].isnan().any() and got[9, :, dim // 2:].isnan().all() and not got[:7].isnan().any()


@pytest.mark.parametrize("layout", ["tokens", "features"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(ops, dev, layout, interleaved):
    """Against the formula's gradient, against differences (the map is linear: f(x + d) - f(x) is its exact difference), and of the gradient again."""
    x, table, positions = inputs(dev, 37, 3, 64, 48, 3, F32)
    sections = [5, 9, 10]
    given = LAYOUTS[layout](x).detach().requires_grad_()
    out = ops.rotate(given, table, positions, sections, True, interleaved)
    assert torch.equal(out.detach(), ops.rotate(given.detach(), table, positions, sections, True, interleaved))
    g = torch.randn(x.shape, generator=torch.Generator(device=dev).manual_seed(4), device=dev).requires_grad_()
    grad, = torch.autograd.grad(out, given, g, create_graph=True)
    want, slack = turned(g.detach(), table, positions, sections, True, interleaved, back=True)
    close(grad.detach(), want, slack)
    d = torch.randn(x.shape, generator=torch.Generator(device=dev).manual_seed(5), device=dev)
    f = [(turned(x + e * d, table, positions, sections, True, interleaved)[0] * g.detach()).sum() for e in (1.0, -1.0)]
    # x + d is rounded (2^-24 of it), as is every element of the gradient (2^-24 and 2 * 2^-24 of the pair)
    allowed = 2.0 ** -23 * float(((x.abs() + d.abs()).sum() + (grad.detach().abs() * d.abs()).sum()) * 8)
    assert abs(float((f[0] - f[1]) / 2 - (grad.detach().double() * d).sum())) <= allowed
    again, = torch.autograd.grad(grad, g, d)
    want, slack = turned(d, table, positions, sections, True, interleaved)
    close(again, want, slack)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_gradients_of_other_layouts(ops, dev, dtype):
    """A gradient that is the same everywhere (no memory of its own), one that lies another way than x, an x that several uses share."""
    x, table, positions = inputs(dev, 24, 2, 64, 64, 1, dtype)
    x.requires_grad_()
    out = ops.rotate(x, table, positions)
    grad, = torch.autograd.grad(out.sum(), x, retain_graph=True)
    want, slack = turned(torch.ones_like(x), table, positions, back=True)
    close(grad, want, slack)
    g = torch.randn(x.shape, generator=torch.Generator(device=dev).manual_seed(8), device=dev).to(dtype)
    grad, = torch.autograd.grad(out, x, feature_major(g))
    want, slack = turned(g, table, positions, back=True)
    close(grad, want, slack)
    wide = x[:, :1].expand(-1, 2, -1)      # one head for two
    grad, = torch.autograd.grad(ops.rotate(wide, table, positions), x, g)
    want, slack = turned(g, table, positions, back=True)
    rounded = want[:, :1].abs() + want[:, 1:].abs()
    off = (grad[:, :1].double() - want.sum(1, keepdim=True)).abs() - 3 * STEP[dtype] * rounded - slack.sum(1, keepdim=True) * 2 - 3 * TINY[dtype]
    assert not (off > 0).any() and (grad[:, 1:] == 0).all()


def test_there_and_back(ops, dev):
    """Back turns what was turned, up to both roundings."""
    x, table, positions = inputs(dev, 100, 4, 128, 128, 3, BF16)
    there = ops.rotate(x, table, positions, [20, 22, 22])
    back = ops.rotate(there, table, positions, [20, 22, 22], back=True)
    length = torch.cat([x[..., :64].double() ** 2 + x[..., 64:].double() ** 2] * 2, -1).sqrt()
    # both roundings (2^-8 of an element, at most of its plane's length, the first one turned: of two elements), the table's 2^-24
    assert ((back.double() - x.double()).abs() <= length * (2 * 2.0 ** -8 + 2.0 ** -8 * 1.01 + 2.0 ** -20)).all()


def test_replays_and_streams(ops, dev):
    """Captured forward and backward follow positions and operands; between the replays eager passes and other work."""
    x, table, positions = inputs(dev, 90, 4, 64, 64, 2, F16)
    x, g = x.requires_grad_(), torch.randn(90, 4, 64, device=dev).half()
    eager_out = ops.rotate(x, table, positions, [16, 16])     # an eager graph of the same leaf lives on
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(ops.rotate(x, table, positions, [16, 16]), x, g)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotate(x, table, positions, [16, 16])
        grad, = torch.autograd.grad(out, x, g)
    for step in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(90, 4, 64, generator=torch.Generator(device=dev).manual_seed(step), device=dev))
            positions.copy_(torch.randint(0, 97, (2, 90), generator=torch.Generator(device=dev).manual_seed(step), device=dev))
        graph.replay()
        want, slack = turned(x.detach(), table, positions, [16, 16])
        close(out.detach(), want, slack)
        fresh = x.detach().clone().requires_grad_()
        eager = ops.rotate(fresh, table, positions, [16, 16])
        eager_grad, = torch.autograd.grad(eager, fresh, g)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(grad, eager_grad)
    assert eager_out.shape == x.shape


def test_an_in_place_change_is_found(ops, dev):
    x, table, positions = inputs(dev, 8, 1, 64, 64, 1, F32)
    x.requires_grad_()
    out = ops.rotate(x, table, positions)
    positions.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), x)


def test_refusals(ops, dev):
    x, table, positions = inputs(dev, 8, 2, 64, 64, 3, F16)
    good = [10, 11, 11]
    for arguments, text in [((x, table, positions), "need sections"), ((x, table, positions, [10, 11, 10]), "sections of 31"), ((x, table, positions, [43, -11, 0]), "a section of -11"),
                            ((x, table, positions, [32, 0]), "a section for each"), ((x, table, positions[:, :7], good), "positions must be"), ((x, table, positions.long(), good), "int32"),
                            ((x, table.double(), positions, good), "rotation must be"), ((x, table.t().contiguous().t(), positions, good), "rotation must be"),
                            ((x, rotation_table(9, 66, dev), positions[0]), "even number"), ((x, torch.zeros(9, 3, device=dev), positions[0]), "even number"),
                            ((x, table[:0], positions, good), "must have a row"), ((x, table[:, :0], positions[0]), "without a rotation"), ((x.double(), table, positions, good), "fp32, fp16 or bf16"),
                            ((x[0], table, positions, good), "3 dimensions"), ((x.cpu(), table, positions, good), "CUDA tensor"), ((x, table.cpu(), positions, good), "CUDA tensor"),
                            ((x, table, positions.cpu(), good), "CUDA tensor"), ((x, table, positions.t().contiguous().t(), good), "contiguous rows"),
                            ((x, table, torch.zeros(5, 8, dtype=torch.int32, device=dev), [7, 7, 7, 7, 4]), "one to four axes"), ((x, table.clone().requires_grad_(), positions, good), "no gradient")]:
        with pytest.raises(RuntimeError, match=text):
            ops.rotate(*arguments)
    wide = torch.zeros(2, 1, 320, dtype=F16, device=dev)
    with pytest.raises(RuntimeError, match="up to 256"):
        ops.rotate(wide, torch.zeros(5, 320, device=dev), torch.zeros(2, 2, dtype=torch.int32, device=dev), [80, 80])
    assert ops.rotate(x[:0], table, positions[:, :0], good).shape == (0, 2, 64) and ops.rotate(x[:, :0], table, positions, good).shape == (8, 0, 64)
    nothing = torch.zeros(0, 2, 64, dtype=F16, device=dev, requires_grad=True)      # (tensors without memory)
    out = ops.rotate(nothing, table, torch.zeros(3, 0, dtype=torch.int32, device=dev), good)
    assert torch.autograd.grad(out.sum(), nothing)[0].shape == (0, 2, 64)
    one = inputs(dev, 5, 1, 320, 320, 1, F16)      # (one axis: any number of features)
    want, slack = turned(*one)
    close(ops.rotate(*one), want, slack)


# ---- appending by given positions ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,e8", [(F16, False), (BF16, True)])
@pytest.mark.parametrize("layout", ["tokens", "features"])
@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("dim,page,kv_heads,heads,r,sections,in_turn,interleaved", [(128, 64, 2, 4, 128, [16, 24, 24], False, False), (64, 16, 3, 3, 32, None, False, True),
                                                                                   (256, 32, 1, 5, 256, [40, 43, 40, 5], True, False), (128, 16, 2, 2, 64, [0, 32], False, True)])
def test_append(ops, dev, dtype, e8, layout, single, dim, page, kv_heads, heads, r, sections, in_turn, interleaved):
    """Keys and queries turned by their given positions; where they lie goes by the lengths as ever."""
    new, before = ([1] * 5 if single else [5, 0, 70, 1, 33]), [0, 3, page - 1, page, 2 * page + 5]
    lengths = [a + b for a, b in zip(new, before)]
    c = Cache(dev, lengths, kv_heads, dim, page, dtype, e8=e8, poison=False, bounds=True)
    c.bounds.zero_()
    n = sum(new)
    k, table, positions = inputs(dev, n, kv_heads, dim, r, len(sections) if sections else 1, dtype, rows=50, seed=2)
    v, q = inputs(dev, n, kv_heads, dim, r, 1, dtype, seed=3)[0], inputs(dev, n, heads, dim, r, 1, dtype, seed=4)[0]
    positions[..., 1] = -3
    offsets = None if single else torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    lay = LAYOUTS[layout]
    got = ops.kv_append_(lay(k), lay(v), c.keys, c.values, c.table, c.lengths, offsets, lay(q), table, interleaved, c.bounds, *c.exponents(), positions, sections, in_turn)
    assert "(positions given)" in _lib.last_kernels()
    want, slack = turned(q, table, positions, sections, in_turn, interleaved)
    close(got, want, slack, "q")
    want, slack = turned(k, table, positions, sections, in_turn, interleaved)
    places = [(int(c.table[s, at // page]), at % page) for s in range(5) for at in range(before[s], lengths[s])]
    pages, slots = (torch.tensor(x, device=dev) for x in zip(*places))
    for name, want, slack in (("keys", want, slack), ("values", v.double(), torch.zeros_like(slack))):
        now = c.stored(name, pages)[torch.arange(n, device=dev), :, slots]
        if e8:
            scale = want.abs().amax(-1, keepdim=True) / 224
            assert ((now - want).abs() <= want.abs() * HALF_STEP[E4M3] + 2.0 ** -10 * scale + 2 * slack).all(), name
        else:
            close(now.to(dtype), want, slack, name)
    for s in range(5):      # pages that began with this call have their bounds
        for i in range(-(-before[s] // page), -(-lengths[s] // page)):
            p = int(c.table[s, i])
            x = c.stored("keys", p)[:, :min(page, lengths[s] - i * page)]
            assert torch.equal(c.bounds[p, :, 0], x.amin(1).to(dtype)) and torch.equal(c.bounds[p, :, 1], x.amax(1).to(dtype))


@pytest.mark.parametrize("layout", ["tokens", "features"])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(8, 2, 3000), (4, 4, 200)])
def test_append_is_rotate_and_append(ops, dev, layout, heads, kv_heads, tokens):
    """The same bits as the rotation by itself, and, at the places' own positions, as without positions given."""
    c = Cache(dev, [tokens, tokens - 7], kv_heads, 128, 32, F16, poison=False)
    offsets = torch.tensor([0, tokens, 2 * tokens - 7], dtype=torch.int32, device=dev)
    k, table, positions = inputs(dev, 2 * tokens - 7, kv_heads, 128, 128, 3, F16, rows=5000)
    v, q = inputs(dev, 2 * tokens - 7, kv_heads, 128, 128, 1, F16, seed=3)[0], inputs(dev, 2 * tokens - 7, heads, 128, 128, 1, F16, seed=4)[0]
    k, v, q = (LAYOUTS[layout](x) for x in (k, v, q))

    def append(k, q, rotation=None, positions=None, sections=None, in_turn=False):
        got = ops.kv_append_(k, v, c.keys, c.values, c.table, c.lengths, offsets, q, rotation, False, None, None, None, positions, sections, in_turn)
        return got, c.keys.clone()

    by_three = append(k, q, table, positions, [20, 22, 22], True)
    plain = append(*(ops.rotate(x, table, positions, [20, 22, 22], True) for x in (k, q)))
    assert all(torch.equal(a, b) for a, b in zip(by_three, plain))
    own = torch.cat([torch.arange(tokens), torch.arange(tokens - 7)]).to(dev, torch.int32)
    given, places = append(k, q, table, own), append(k, q, table)
    assert all(torch.equal(a, b) for a, b in zip(given, places))


def test_append_refusals(ops, dev):
    c = Cache(dev, [5], 1, 64, 16, F16, poison=False)
    k, table, positions = inputs(dev, 1, 1, 64, 64, 2, F16)
    append = lambda *more: ops.kv_append_(k, k, c.keys, c.values, c.table, c.lengths, None, k, *more)  # noqa: E731
    for more, text in [((None, False, None, None, None, positions, [16, 16]), "without a rotation"), ((table, False, None, None, None, None, [32]), "sections without positions"),
                       ((table, False, None, None, None, positions), "need sections"), ((table[:, :36].contiguous(), False, None, None, None, positions, [9, 9]), "multiple of 16"),
                       ((table[:0], False, None, None, None, positions, [16, 16]), "must have a row")]:
        with pytest.raises(RuntimeError, match=text):
            append(*more)
    none = torch.zeros(0, 1, 64, dtype=F16, device=dev)
    got = ops.kv_append_(none, none, c.keys, c.values, c.table, c.lengths, torch.zeros(2, dtype=torch.int32, device=dev), none, table, False, None, None, None,
                         torch.zeros(2, 0, dtype=torch.int32, device=dev), [16, 16])
    assert got.shape == (0, 1, 64)
    append(table[:2], False, None, None, None, positions.clamp(max=1), [16, 16])      # (a table shorter than the cache's)
    with pytest.raises(RuntimeError, match="every position"):
        append(table[:2], False)


def test_generation_behind_an_eviction(ops, dev):
    """Prompt, steps that keep account, eviction, steps at positions of their own: every result against all keys and values that are left, kept plainly."""
    page, kv, heads, dim, keep = 16, 2, 4, 64, 40
    cache = PA.KVCache(8, page, kv, dim, F16, dev)
    table = torch.arange(8, dtype=torch.int32, device=dev).flip(0)[None].contiguous()
    rotation = PA.rotation_table(300, dim, device=dev)
    gen = torch.Generator(device=dev).manual_seed(6)
    draw = lambda n, h: torch.randn(n, h, dim, generator=gen, device=dev).half()  # noqa: E731
    k, v = draw(70, kv), draw(70, kv)
    lengths = torch.tensor([70], dtype=torch.int32, device=dev)
    weights = torch.zeros(1, kv, 128, device=dev)
    at = torch.arange(70, dtype=torch.int32, device=dev)
    ops.kv_append_(k, v, cache.keys, cache.values, table, lengths, torch.tensor([0, 70], dtype=torch.int32, device=dev), None, rotation, positions=at)
    keys, values = [turned(k, rotation, at)[0][:, h] for h in range(kv)], [v[:, h].double() for h in range(kv)]
    position = 70
    for step in range(12):
        if step == 6:
            kept = ops.evict_tokens_(cache.keys, cache.values, table, lengths, weights, keep, 8, 2)
            keys, values = [keys[h][kept[0, h].long()] for h in range(kv)], [values[h][kept[0, h].long()] for h in range(kv)]
        lengths += 1
        at = torch.tensor([position], dtype=torch.int32, device=dev)
        k, v, q = draw(1, kv), draw(1, kv), draw(1, heads)
        q = ops.kv_append_(k, v, cache.keys, cache.values, table, lengths, None, q, rotation, positions=at)
        out = ops.paged_attention_accumulate_(q, cache.keys, cache.values, table, lengths, weights, dim ** -0.5)
        for h in range(kv):
            keys[h] = torch.cat([keys[h], turned(k, rotation, at)[0][:, h]])
            values[h] = torch.cat([values[h], v[:, h].double()])
            for i in range(2):
                score = keys[h] @ q[0, 2 * h + i].double() * dim ** -0.5
                want = torch.softmax(score, 0) @ values[h]
                # keys are a half step off, which moves a score by that of sum |q k| and a probability by twice as much; the result is rounded
                magnitude = float((keys[h] * q[0, 2 * h + i].double()).abs().sum(1).max() * dim ** -0.5)
                allowed = want.abs() * 2.0 ** -11 + values[h].abs().max() * (math.expm1(2 * 2.0 ** -11 * magnitude) + 2.0 ** -12)
                assert ((out[0, 2 * h + i].double() - want).abs() <= allowed).all(), (step, h)
        position += 1
    assert lengths.tolist() == [keep + 6]
