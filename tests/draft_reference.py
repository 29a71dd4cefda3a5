"""Plain forms of the drafted-tree operators, row by row in 64 bits, and trees to try them on."""
import random

import torch

from .paged_reference import HALF_STEP, inverse_frequencies


def random_tree(n, seed, roots=1):
    """Parents of n rows: the first ``roots`` have none, every other any row before it."""
    r = random.Random(seed)
    return [-1 if i < roots else r.randrange(i) for i in range(n)]


def chain(n):
    return list(range(-1, n - 1))


def path_to(parents, i):
    """Row i's ancestors and itself, from the top; the way up ends at a parent that does not come before its child."""
    out = []
    while i >= 0:
        out.append(i)
        up = parents[i]
        i = up if up < i else -1
    return out[::-1]


def visible_slots(parents, i, length):
    """Slots that row i of n sees in a sequence of ``length``."""
    before = length - len(parents)
    return list(range(max(0, before))) + [before + a for a in path_to(parents, i) if before + a >= 0]


def attention_over(pool, q, rows, scale=None):
    """(out, tolerance) of q [tokens, heads, d]; ``rows``: for each row (sequence, the slots it sees) or None.

    Tolerance by row and element as in ``paged_reference.attention``, u half a
    step of the type, over the slots seen:
      u |o|               the output's rounding
      u sum p |v|         each weight rounded to the type before the product
      2 e sum p |v|       weights off by a factor e^(+-e): (d + 4) fp32 roundings
                          of the scores' size and 2^-21 for the exponential
      n 2^-22 / 16 ...    fp32 sums, 8 to n / 16 steps of 2^-22, 2^-13 at most
    A piece's rows are rescaled and joined in fp32: within the last term.
    """
    t, heads, d = q.shape
    group = heads // pool.kv_heads
    scale = d ** -0.5 if scale is None else scale
    u = HALF_STEP[pool.dtype]
    out = torch.zeros(t, heads, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    held = {}
    for i, row in enumerate(rows):
        if row is None or not row[1]:
            continue
        b, slots = row
        if b not in held:
            held[b] = pool.rows(pool.k, b, pool.lens[b]), pool.rows(pool.v, b, pool.lens[b])
        k, v = (x[:, slots] for x in held[b])
        qq = q[i].double().view(pool.kv_heads, group, d)
        p = torch.softmax(torch.matmul(qq, k.transpose(1, 2)) * scale, -1)
        o = torch.matmul(p, v)
        mass = torch.matmul(p, v.abs())
        size = (torch.matmul(qq.abs(), k.abs().transpose(1, 2)) * abs(scale)).amax(-1, keepdim=True)
        e = (d + 4) * 2.0 ** -24 * size + 2.0 ** -21
        sums = min(max(len(slots) / 16, 8) * 2.0 ** -22, 2.0 ** -13)
        out[i] = o.reshape(heads, d)
        tol[i] = (u * o.abs() + (u + 2 * e + sums) * mass).reshape(heads, d)
    return out, tol


def rotated_by(x, positions, sections, theta=1e6):
    """(rotation in 64 bits, tolerance) of x [tokens, heads, d] by positions [axes, tokens]: half a step of the type, and
    the fp32 table's and arithmetic's 4 roundings of |x_j| + |x_j+d/2|."""
    d = x.shape[-1]
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    ang = positions.double()[axis].T * inverse_frequencies(d, theta)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x.double().chunk(2, -1)
    y = torch.cat((a * c - b * s, b * c + a * s), -1)
    mass = (a.abs() + b.abs()).repeat(1, 1, 2)
    return y, HALF_STEP[x.dtype] * y.abs() + 4 * 2.0 ** -24 * mass


def accepted(parents, ids, answers):
    """(path, next token) of one tree."""
    depth = []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            depth.append(0)
        elif p == -1:
            depth.append(1)
        else:
            depth.append(depth[p] + 1 if depth[p] and ids[i] == answers[p] else 0)
    if not depth or max(depth) == 0:
        return [], -1
    best = depth.index(max(depth))
    return path_to(parents, best), answers[best]


def packed(lists):
    """(boundaries, one flat list)."""
    cu, flat = [0], []
    for x in lists:
        flat += x
        cu.append(len(flat))
    return cu, flat


def i32(x, dev=None):
    return torch.tensor(x, dtype=torch.int32, device=dev)
