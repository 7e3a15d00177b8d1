"""Plain 64-bit forms of the operators on a paged cache, row by row from their definitions, and how far a kernel may be off."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Case:
    """Sequences over a cache whose pages lie in random order, with garbage (NaN, infinities) wherever nothing may be read."""

    def __init__(self, dtype, new, lens, heads=2, group=3, dim=64, page=16, prefix=0, seed=0, layout="slots", starts=True, garbage=True, width=None, device="cpu",
                 behind=0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.new, self.lens, self.heads, self.group, self.dim, self.page, self.prefix = dtype, new, lens, heads, group, dim, page, prefix
        per = [-(-n // page) for n in lens]
        shared = -(-prefix // page)
        pages = sum(per) + shared + 2
        self.order = torch.randperm(pages, generator=g).int()
        width = max(per + [1]) + 1 if width is None else width
        table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32)  # entries past the keys are never read
        at = shared
        for b, n in enumerate(per):
            table[b, :n] = self.order[at:at + n]
            at += n
        self.table, self.prefix_table = table, self.order[:shared].clone()
        shape = (pages, page, heads, dim)
        self.k, self.v = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
        if garbage:
            live = torch.zeros(pages, page, dtype=torch.bool)
            for rows, n in [(self.prefix_table, prefix)] + [(table[b], n) for b, n in enumerate(lens)]:
                for j in range(n):
                    live[rows[j // page], j % page] = True
            self.k[~live], self.v[~live] = math.nan, math.inf
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.tokens = self.starts[-1] + behind
        self.q = torch.randn(self.tokens, heads * group, dim, generator=g).to(dtype) * 2
        self.layout, self.device = layout, device
        self.q_starts = torch.tensor(self.starts, dtype=torch.int32) if starts else None

    def pool(self, t):
        """The pool on the device, laid out as asked: [page][slot][head], [page][head][slot], or every other row of a larger one."""
        t = t.to(self.device)
        if self.layout == "heads":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if self.layout == "gaps":
            big = torch.full((t.shape[0], t.shape[1], 2, t.shape[2], t.shape[3]), math.nan, dtype=t.dtype, device=self.device)
            big[:, :, 1] = t
            return big[:, :, 1]
        return t.contiguous()

    def on(self, t):
        return None if t is None else t.to(self.device)

    def keys(self, b, pool):
        """[prefix + own, heads, dim] of sequence b in 64 bits."""
        def rows(table, n):
            j = torch.arange(n)
            return pool[table[j // self.page].long(), j % self.page].double()
        return torch.cat((rows(self.prefix_table, self.prefix), rows(self.table[b], self.lens[b])))

    def want(self, causal=True, scale=None):
        """(result, how far each value may be off): sum p |v| times the relative errors of p and of the sums, and the result's rounding."""
        scale = self.dim ** -0.5 if scale is None else scale
        u = HALF_STEP[self.dtype]
        out = torch.zeros(self.tokens, self.heads * self.group, self.dim, dtype=torch.float64)
        tol = torch.zeros_like(out)
        for b in range(len(self.lens)):
            k, v = self.keys(b, self.k), self.keys(b, self.v)
            for i in range(self.new[b]):
                n = self.prefix + (max(0, min(self.lens[b], self.lens[b] - self.new[b] + i + 1)) if causal else self.lens[b])
                if n == 0:
                    continue
                row = self.starts[b] + i
                for h in range(self.heads * self.group):
                    q = self.q[row, h].double()
                    kk, vv = k[:n, h // self.group], v[:n, h // self.group]
                    p = torch.softmax(scale * (kk @ q), 0)
                    out[row, h] = p @ vv
                    # A score's error: products of 16-bit values are exact, those of split fp32 values lose 3 * 2^-21; at most 49 additions that
                    # cut off 2^-23 each; 2^-22 for the scale.  It moves a power of two by its own size, the row's sum by as much.
                    ds = float((scale * (kk.abs() @ q.abs())).max()) * ((3 * 2.0 ** -21 if self.dtype is torch.float32 else 0.0) + 51 * 2.0 ** -23)
                    dp = 2 * (ds + 2.0 ** -21)  # (2^-22 of the hardware's power of two, as much for its argument's rounding)
                    sums = (n / 4 + 64) * 2.0 ** -24  # additions of 32 bits, rounded or cut off, in at most n / 8 steps
                    products = 3 * 2.0 ** -21 if self.dtype is torch.float32 else u  # of p and v: split in two, or p rounded to 16 bits
                    tol[row, h] = (p @ vv.abs()) * (dp + sums + products) * 1.01 + out[row, h].abs() * u * 1.01 + 2.0 ** -25 * (self.dtype is torch.float16)
        return out, tol

    def check(self, got, causal=True, scale=None):
        want, tol = self.want(causal, scale)
        n = self.starts[-1]
        off = (got[:n].double().cpu() - want[:n]).abs()
        assert torch.isfinite(got[:n]).all(), "not finite"
        assert (off <= tol[:n]).all(), f"off by {float((off / tol[:n].clamp_min(1e-30)).max()):.3g} of what is allowed"

    def attend(self, ctx, causal=True, scale=None, out=None, q=None):
        q = self.on(self.q) if q is None else q
        k, v, t, n, s = self.pool(self.k), self.pool(self.v), self.on(self.table), self.on(torch.tensor(self.lens, dtype=torch.int32)), self.on(self.q_starts)
        if self.prefix or self.prefix_table.numel():
            return ctx.attention_prefix(q, k, v, self.on(self.prefix_table), self.prefix, t, n, q_starts=s, causal=causal, scale=scale, out=out)
        return ctx.attention_paged(q, k, v, t, n, q_starts=s, causal=causal, scale=scale, out=out)


def rotated(x, angle, interleaved):
    """x [heads, dim] in 64 bits turned by angle [pairs]; and |x1| + |x2| of each value's pair (0 where it is not turned)."""
    x, pairs = x.double(), len(angle)
    y, size = x.clone(), torch.zeros_like(x)
    for j in range(pairs):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
        c, s = math.cos(angle[j]), math.sin(angle[j])
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
        size[:, a] = size[:, b] = x[:, a].abs() + x[:, b].abs()
    return y, size
