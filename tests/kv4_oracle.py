"""The 4-bit key / value cache in 64 bits, from its definition: pages, nearest codes, rotation by one or
several axes, and softmax attention row by row, with how far an implementation may be off.  Written
apart from the package's own reference."""
import math
from fractions import Fraction

import torch

NUMBERS = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
EXPONENTS = {torch.bfloat16: (-120, 125), torch.float16: (-22, 13), torch.float32: (-120, 125)}


def nearest(x, dtype):
    """(values, scale exponents per block of 32) of x [.., d] in 64 bits: by distance, ties to the even code."""
    b = x.double().reshape(-1, 32)
    lo, hi = EXPONENTS[dtype]
    e = []
    for most in b.abs().amax(1).tolist():
        if most == 0:
            e.append(lo)
            continue
        m, k = math.frexp(min(most, 2.0 ** 200))              # most = m 2^k, m in [1/2, 1)
        e.append(min(max(k - 3 + (m > 0.875), lo), hi))
    e = torch.tensor(e, dtype=torch.float64)
    a = (b / 2 ** e[:, None]).abs()
    off = (a[..., None] - NUMBERS).abs()
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])            # an even code keeps a tie
    code = order[off[..., order].argmin(-1)]
    return (NUMBERS[code] * b.sign() * 2 ** e[:, None]).view(x.shape), e.view(*x.shape[:-1], -1)


def rotate(x, cos, sin):
    a, b = x.double().chunk(2, -1)
    return torch.cat([a * cos.double() - b * sin.double(), b * cos.double() + a * sin.double()], -1)


def cos_sin_rows(table, positions, sections=None):
    """cos, sin [T, 1, d/2], pair by pair."""
    half = table.shape[1] // 2
    if sections is None:
        c = table[positions]
        return c[:, None, :half], c[:, None, half:]
    axis = sum(([a] * n for a, n in enumerate(sections)), [])
    cos = torch.stack([table[positions[a].clamp(0, len(table) - 1), i] for i, a in enumerate(axis)], 1)
    sin = torch.stack([table[positions[a].clamp(0, len(table) - 1), half + i] for i, a in enumerate(axis)], 1)
    return cos[:, None], sin[:, None]


def token(cache, slot, head, d):
    """One token's row of one kv head, from the bytes."""
    bs = cache.shape[2]
    page = cache[slot // bs, head].flatten()
    row = page[(slot % bs) * (d // 2):][:d // 2]
    scales = page[bs * d // 2 + (slot % bs) * (d // 32):][:d // 32]
    code = torch.stack([row & 15, row >> 4], 1).flatten().long()
    v = NUMBERS[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    return (v.view(-1, 32) * 2 ** (scales.double() - 127)[:, None]).flatten()


def rows(cache, table, n, head, d):
    """[n, d] of a sequence's first n tokens."""
    bs = cache.shape[2]
    page = cache[table[: -(-n // bs)].long(), head].flatten(1)
    data = page[:, :bs * d // 2].reshape(-1, d // 2)[:n]
    scales = page[:, bs * d // 2:].reshape(-1, d // 32)[:n]
    code = torch.stack([data & 15, data >> 4], 2).flatten(1).long()
    v = NUMBERS[code & 7] * torch.where(code >= 8, -1.0, 1.0)
    return (v.view(n, -1, 32) * 2 ** (scales.double() - 127)[..., None]).flatten(1)


def attend(q, k, v, scale, seen, dtype):
    """(softmax(q k^T scale) v, how far off) for q [m, d], k, v [n, d], seen [m, n] bool; rows that see
    nothing are zero.

    With u = eps / 2 of ``dtype`` and r = 2^-24, A = sum p |v| / sum p:
      scores   d products summed in fp32 in any order, then scaled: (d + 2) r scale sum |q k|, relative on p
               (with the largest score's error, since p is relative to it): twice that; in log2 units the
               subtraction's own rounding 2 r |s - m| log2(e), |s - m| below 130 where p matters
      exp2     2 r relative, for p and for every rescale of a running sum: n / 32 + 1 of them
      p        rounded to ``dtype``: u relative, or for fp16 half its smallest step, 2^-25, absolute; and 0 below
               fp32's smallest normal number, 2^-126 absolute (a weight of e^-190 = 10^-83 is none in 32 bits)
      sums     n terms of fp32 in any order: n r A
      result   u |o|"""
    u, r = torch.finfo(dtype).eps / 2, 2.0 ** -24
    n, d = k.shape
    s = (q.double() @ k.double().T) * scale
    big = ((q.double().abs() @ k.double().abs().T) * scale)
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(1, keepdim=True)
    p = torch.where(seen, (s - torch.where(m > -math.inf, m, 0)).exp(), 0)
    total = p.sum(1, keepdim=True)
    safe = torch.where(total > 0, total, 1)
    o, mag = p @ v.double() / safe, p @ v.double().abs() / safe
    ds = 2 * (d + 2) * r * torch.where(seen, big, 0).amax(1, keepdim=True) + 4 * r * 130 * 1.45
    rel = u + 2 * (ds + 4 * r * (n / 32 + 2)) + 2 * (n + 4) * r
    tol = 1.01 * rel * mag + 1.01 * u * o.abs() + r * mag + 2.0 ** -126 * (seen.double() @ v.double().abs())
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (seen.double() @ v.double().abs()) + 2.0 ** -25
    return o, tol


def random_cache(g, nb, nkv, bs, d, dtype, size=1.0):
    """Random pages with blocks of unequal size."""
    lo, hi = EXPONENTS[dtype]
    out = torch.randint(0, 256, (nb, nkv, bs, d // 2 + d // 32), generator=g, dtype=torch.uint8)
    e = torch.randint(-4, 1, (nb, nkv, bs * d // 32), generator=g) + round(math.log2(size))
    out.view(nb, nkv, -1)[..., bs * d // 2:] = (e.clamp(lo, hi) + 127).to(torch.uint8)
    return out


def tables(g, totals, bs, spare=2):
    """Block tables [n, width] of scattered pages (page 0 is nobody's), and how many pages there are; the
    entries behind a sequence's pages name page 0."""
    width = max(-(-max(totals) // bs), 1) + spare
    need = [-(-t // bs) for t in totals]
    order = (torch.randperm(sum(need), generator=g) + 1).tolist()
    bt = torch.zeros(len(totals), width, dtype=torch.int32)
    for i, n in enumerate(need):
        bt[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    return bt, sum(need) + 1


def _nearest_fractions(block):
    """e2m1 numbers of 32 fractions and their exponent, in rational arithmetic."""
    most, e = max(abs(x) for x in block), EXPONENTS[torch.float32][0]
    while most > 7 * Fraction(2) ** e:
        e += 1
    out = []
    for x in block:
        a = abs(x) / Fraction(2) ** e
        n = min((0.0, 1.0, 2.0, 4.0, .5, 1.5, 3.0, 6.0), key=lambda n: abs(a - Fraction(n)))   # an even code keeps a tie
        out.append(math.copysign(n * 2.0 ** e, x))
    return out, e


def keys_beside_borders():
    """Keys [T, 64] and a row of cos / sin whose rotations lie 2^-60 beside the borders of two codes, on both sides,
    and beside 7 times the scale: sums of two products that no 64-bit float holds.
    -> keys, table [1, 64], values [T, 64], exponents [T, 2]."""
    ties, tiny = [.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0], 2.0 ** -20
    a = torch.tensor([6.0] + ties * 4 + [0.0] * 3)
    a[15:29] *= -1
    b = torch.tensor([0.0] + [-tiny] * 7 + [tiny] * 14 + [-tiny] * 7 + [0.0] * 3)
    x = torch.stack([a, b]).repeat(4, 1, 1)
    x[1, :, 0], x[2, :, 0] = torch.tensor([7.0, -tiny]), torch.tensor([7.0, tiny])
    x[3] = x[3].flip(0)                                       # the small ones first: b + a sin
    x[3, 0] *= -1
    table = torch.cat([torch.ones(32), torch.full((32,), 2.0 ** -40)])[None]
    f = lambda t: [Fraction(v) for v in t.double().tolist()]   # noqa: E731
    cos, sin = f(table[0, :32]), f(table[0, 32:])
    v, e = [], []
    for p, q in ((f(r[0]), f(r[1])) for r in x):
        one = _nearest_fractions([i * c - j * s for i, j, c, s in zip(p, q, cos, sin)])
        two = _nearest_fractions([j * c + i * s for i, j, c, s in zip(p, q, cos, sin)])
        v.append(one[0] + two[0])
        e.append([one[1], two[1]])
    return x.view(4, 64), table, torch.tensor(v, dtype=torch.float64), torch.tensor(e, dtype=torch.float64)
