"""Plain 64-bit forms of the paged cache operators, and caches to try them on."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def inverse_frequencies(d, theta=1e6):
    return theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)


class Pool:
    """Pages in random order; slots that no sequence uses hold NaN."""

    def __init__(self, lens, kv_heads, page, d, dtype, *, seed=0, spare=2, extra_columns=0, fill=1.0, joint=False):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.d, self.kv_heads, self.dtype = list(lens), page, d, kv_heads, dtype
        counts = [-(-n // page) for n in lens]
        pages = sum(counts) + spare
        order = torch.randperm(pages, generator=g).int()
        width = max(1, max(counts, default=1)) + extra_columns
        self.table = torch.full((len(lens), width), -(1 << 30), dtype=torch.int32)  # unused entries lead nowhere
        shape = (pages, kv_heads, page, d)
        self.k = torch.full(shape, math.nan, dtype=torch.float64)
        self.v = torch.full(shape, math.nan, dtype=torch.float64)
        at = 0
        for b, c in enumerate(counts):
            held = order[at:at + c]
            self.table[b, :c] = held
            at += c
            for x in (self.k, self.v):
                data = torch.randn(kv_heads, c * page, d, generator=g, dtype=torch.float64) * fill
                data[:, lens[b]:] = math.nan
                x[held.long()] = data.view(kv_heads, c, page, d).transpose(0, 1)
        self.k, self.v = self.k.to(dtype), self.v.to(dtype)
        self.joint = joint

    def device_cache(self, dev, cls):
        if self.joint:  # one pool of [pages, 2, ...]: page stride twice a page
            pool = torch.stack((self.k, self.v), dim=1).to(dev)
            k, v = pool[:, 0], pool[:, 1]
        else:
            k, v = self.k.to(dev), self.v.to(dev)
        return cls(k, v, self.table.to(dev), torch.tensor(self.lens, dtype=torch.int32, device=dev))

    def rows(self, pages, b, n):
        """[kv_heads, n, d] of sequence b in 64 bits."""
        held = self.table[b, : -(-n // self.page)].long()
        return pages[held].double().transpose(0, 1).reshape(self.kv_heads, -1, self.d)[:, :n]


def attention(pool, q, owners, scale=None):
    """(out, tolerance) in 64 bits of q [tokens, heads, d]; ``owners``: for
    each row (sequence, number of visible slots).

    Tolerance, by row and element, u = half a step of the type:
      u |o|               the output's rounding
      u sum p |v|         each weight rounded to the type before the product
      2 e sum p |v|       weights off by a factor e^(+-e), e the scores'
                          error: (d + 4) fp32 roundings of sum |q k| scale,
                          and 2^-21 for the exponential
      n 2^-22 sum p |v|   fp32 sums over n keys (n the steps of a running
                          sum: at most keys / 16 per matrix product step),
                          taken as 2^-13 at most for these lengths
    """
    t, heads, d = q.shape
    group = heads // pool.kv_heads
    scale = d ** -0.5 if scale is None else scale
    u = HALF_STEP[pool.dtype]
    out = torch.zeros(t, heads, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i, (b, n) in enumerate(owners):
        if b is None or n <= 0:
            continue
        k, v = pool.rows(pool.k, b, n), pool.rows(pool.v, b, n)
        qq = q[i].double().view(pool.kv_heads, group, d)
        x = torch.matmul(qq, k.transpose(1, 2)) * scale
        p = torch.softmax(x, -1)
        o = torch.matmul(p, v)
        mass = torch.matmul(p, v.abs())
        size = (torch.matmul(qq.abs(), k.abs().transpose(1, 2)) * abs(scale)).amax(-1, keepdim=True)
        e = (d + 4) * 2.0 ** -24 * size + 2.0 ** -21
        sums = min(max(n / 16, 8) * 2.0 ** -22, 2.0 ** -13)
        out[i] = o.reshape(heads, d)
        tol[i] = (u * o.abs() + (u + 2 * e + sums) * mass).reshape(heads, d)
    return out, tol


def rotated(x, positions, theta=1e6):
    """(rotation in 64 bits, tolerance): half a step of the type, and the fp32
    table's and arithmetic's 4 roundings of |x_j| + |x_j+d/2|."""
    d = x.shape[-1]
    ang = positions.double()[:, None] * inverse_frequencies(d, theta)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x.double().chunk(2, -1)
    y = torch.cat((a * c - b * s, b * c + a * s), -1)
    mass = (a.abs() + b.abs()).repeat(1, 1, 2)
    return y, HALF_STEP[x.dtype] * y.abs() + 4 * 2.0 ** -24 * mass
