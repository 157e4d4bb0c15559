"""A paged cache for the tests, and the operators over it written plainly in 64 bits."""
import math

import torch

E4M3 = torch.float8_e4m3fn
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, E4M3: 2.0 ** -4}


def power(exponents):
    """2 ** (exponent - 127) in 64 bits."""
    return torch.exp2(exponents.double() - 127.0)


def to_e4m3(x):
    """Codes and exponents of rows: the least power of two that brings the largest magnitude to 448 (written apart from the kernel: by frexp)."""
    top = x.double().abs().amax(-1)
    mantissa, exponent = torch.frexp(top)                       # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent + 118 + (mantissa > 0.875).to(exponent.dtype)   # 448 = 0.875 * 2^9
    e = torch.where(top == 0, 1, e).clamp(1, 254)
    return (x.double() / power(e)[..., None]).float().to(E4M3), e.to(torch.uint8)


class Cache:
    """pages of random keys and values, a table of pages in no order, and what is beyond the lengths poisoned."""

    def __init__(self, dev, lengths, kv_heads, dim, page, dtype, e8=False, width=None, spare=3, seed=0, poison=True, bounds=False, strided=False):
        gen = torch.Generator(device=dev).manual_seed(seed)
        used = [-(-max(0, n) // page) for n in lengths]
        self.width = max(used + [1]) if width is None else width
        pages = sum(used) + spare
        order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
        self.table = torch.full((len(lengths), self.width), -1, dtype=torch.int32, device=dev)
        at = 0
        for s, n in enumerate(used):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=dev)
        self.page, self.dim, self.kv_heads, self.pages, self.dtype, self.e8 = page, dim, kv_heads, pages, dtype, e8
        keys = torch.randn(pages, kv_heads, page, dim, generator=gen, device=dev).to(dtype)
        values = torch.randn(pages, kv_heads, page, dim, generator=gen, device=dev).to(dtype)
        if poison:   # what no sequence has written
            written = torch.zeros(pages, page, dtype=torch.bool, device=dev)
            for s, n in enumerate(lengths):
                for i in range(used[s]):
                    written[self.table[s, i], :max(0, n - i * page)] = True
            bad = torch.tensor([math.nan, math.inf, -math.inf], device=dev).to(dtype)
            junk = bad[torch.randint(0, 3, keys.shape, generator=gen, device=dev)]
            keys, values = (torch.where(written[:, None, :, None], x, junk) for x in (keys, values))
        self.key_exponents = self.value_exponents = self.bounds = None
        if e8:
            keys, self.key_exponents = to_e4m3(keys)
            values, self.value_exponents = to_e4m3(values)
        if strided:   # keys and values side by side in one array
            both = torch.stack([keys.view(torch.uint8) if e8 else keys, values.view(torch.uint8) if e8 else values], 1)
            keys, values = (x.view(E4M3) if e8 else x for x in both.unbind(1))
        self.keys, self.values = keys, values
        if bounds:
            self.bounds = torch.zeros(pages, kv_heads, 2, dim, dtype=dtype, device=dev)
            for s, n in enumerate(lengths):
                for i in range(used[s]):
                    self.set_bounds(int(self.table[s, i]), min(page, n - i * page))

    def exponents(self):
        return (self.key_exponents, self.value_exponents)

    def stored(self, name, page):
        """What a page (kv_heads, page, dim) stands for, in 64 bits."""
        rows, exponents = (self.keys, self.key_exponents) if name == "keys" else (self.values, self.value_exponents)
        if not self.e8:
            return rows[page].double()
        return rows.view(torch.uint8)[page].view(E4M3).float().double() * power(exponents[page])[..., None]

    def set_bounds(self, page, count):
        x = self.stored("keys", page)[:, :count]
        self.bounds[page, :, 0] = x.amin(1).to(self.dtype)
        self.bounds[page, :, 1] = x.amax(1).to(self.dtype)

    def rows(self, s, head, listed=None):
        """Keys and values (n, dim) in 64 bits that key head ``head`` of sequence ``s`` attends to."""
        length = min(max(0, int(self.lengths[s])), self.width * self.page)
        numbers = range(-(-length // self.page)) if listed is None else [int(x) for x in listed]
        ks, vs = [], []
        for i in numbers:
            page = int(self.table[s, i]) if 0 <= i < self.width else -1
            n = min(self.page, length - i * self.page)
            if 0 <= page < self.pages and n > 0:
                ks.append(self.stored("keys", page)[head, :n])
                vs.append(self.stored("values", page)[head, :n])
        empty = torch.zeros(0, self.dim, dtype=torch.float64, device=self.table.device)
        return torch.cat(ks + [empty]), torch.cat(vs + [empty])

    def attend(self, q, scale, pages=None):
        """(result, allowed error) in 64 bits.

        The error of a call: half a step of the result's type; scores to D + 4 roundings of their terms' magnitudes (the sum of the
        products in 32 bits, the scale, the maximum taken off), which reach a probability as relative error; probabilities to 2^-16 (two
        16-bit parts, 2^-17 between them for bf16, and the exponential); sums of n terms in 32 bits, in chains of at most n / 8 and
        the parts behind them."""
        seqs, heads, dim = q.shape
        group = heads // self.kv_heads
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        slack = torch.zeros_like(out)
        for s in range(seqs):
            for h in range(heads):
                k, v = self.rows(s, h // group, None if pages is None else pages[s, h // group])
                if k.shape[0] == 0:
                    continue
                x = q[s, h].double()
                p = torch.softmax((k * x).sum(1) * scale, 0)
                out[s, h] = (p[:, None] * v).sum(0)
                magnitude = (k * x).abs().sum(1).max() * scale
                relative = 2.0 ** -16 + 2 * (dim + 4) * 2.0 ** -24 * magnitude + (k.shape[0] / 8 + 64) * 2.0 ** -24
                slack[s, h] = relative * (p[:, None] * v.abs()).sum(0)
        tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
        return out, out.abs() * HALF_STEP[q.dtype] + slack * (1 + HALF_STEP[q.dtype]) + tiny

    def select(self, q, count, first=1, last=1):
        """The selected pages as lists, by sums in 64 bits rounded once to 32."""
        seqs, heads, dim = q.shape
        group = heads // self.kv_heads
        out = torch.full((seqs, self.kv_heads, count), -1, dtype=torch.int32)
        for s in range(seqs):
            length = min(max(0, int(self.lengths[s])), self.width * self.page)
            used = -(-length // self.page)
            for h in range(self.kv_heads):
                scores = []
                for i in range(used):
                    page = int(self.table[s, i])
                    if not 0 <= page < self.pages:
                        continue
                    low, high = self.bounds[page, h].double()
                    x = q[s, h * group:(h + 1) * group].double()
                    score = float((x.clamp(min=0).sum(0) * high + x.clamp(max=0).sum(0) * low).sum().float())
                    rank = 2 if i < first or i >= used - last else 1 if math.isnan(score) else 0
                    scores.append((-rank, 0.0 if rank else -score, i))
                chosen = sorted(i for _, _, i in sorted(scores)[:count])
                out[s, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        return out


def feature_major(x):
    """The same (rows, heads, dim) values as a projection W @ X leaves them: rows next to each other."""
    return x.permute(1, 2, 0).contiguous().permute(2, 0, 1)


def rotated(x, positions, table, interleaved):
    """x (tokens, heads, dim) turned by the table's rows, in 64 bits, and how far 32-bit products and sums may be off."""
    x = x.double().clone()
    slack = torch.zeros_like(x)
    if table is None:
        return x, slack
    r = table.shape[1]
    c, s = (t[:, None] for t in table[positions].double().chunk(2, 1))
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    x0, x1 = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = x0 * c - x1 * s, x1 * c + x0 * s
    slack[..., a] = slack[..., b] = 2 * 2.0 ** -24 * (x0.abs() + x1.abs())   # a product's and the sum's half step
    return x, slack


def rotation_table(positions, r, dev):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * torch.arange(r // 2, dtype=torch.float64) / r)
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(dev)
