"""AdamW's update in 64 bits, from the formulas, for the tests."""
import math

import torch

BLOCK = 128
TYPES_8 = {'m': torch.float8_e4m3fn, 'v': torch.float8_e5m2}
LARGEST = {'m': 448., 'v': 57344.}
LEAST_TOP = 2. ** -100
MASK = 0xffffffff


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & MASK
    x = x ^ (x >> 15)
    x = (x * 0xB504F333) & MASK
    return x ^ (x >> 16)


def words(n, seed, step, index, first=0):
    """The random words of elements first ... first + n - 1 (first: a multiple of 8) of tensor `index` of the list."""
    key = mix((mix((mix(seed & MASK) + step) & MASK) + index) & MASK)
    unit = torch.arange(first // 8, first // 8 + -(-n // 8), dtype=torch.int64)
    rows = [mix((unit + key) & MASK)]
    for _ in range(7):
        x = rows[-1]
        x = x ^ ((x << 13) & MASK)
        x = x ^ (x >> 17)
        rows.append(x ^ ((x << 5) & MASK))
    return torch.stack(rows, 1).view(-1)[:n]


def numbers(kind):
    """All numbers >= 0 of the 8-bit type, in order"""
    t = torch.arange(128, dtype=torch.uint8).view(TYPES_8[kind]).double()
    return t[torch.isfinite(t)]


def blocks_top(x):
    """Largest finite |x| of every block of a flat tensor"""
    x = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    whole = torch.zeros(-(-x.numel() // BLOCK) * BLOCK, dtype=torch.float64)
    whole[:x.numel()] = x
    return whole.view(-1, BLOCK).amax(1)


def spread(per_block, n):
    return per_block.repeat_interleave(BLOCK)[:n]


def encode(x, kind, random16):
    """(what a flat state in 64 bits becomes in units of its scales, scales, the two neighbours' distance)"""
    top = blocks_top(x)
    scale = torch.where(top >= LEAST_TOP, top / LARGEST[kind], torch.zeros_like(top))
    each = spread(scale, x.numel())
    a = torch.where(each > 0, x.abs() / each, torch.zeros_like(x)).clamp_(max=LARGEST[kind])
    table = numbers(kind)
    at = (torch.searchsorted(table, a, right=True) - 1).clamp_(max=table.numel() - 2)
    low, high = table[at], table[at + 1]
    up = (a - low) / (high - low) + random16.double() / 65536 >= 1
    q = torch.where(up, high, low)
    if kind == 'v':
        q = torch.where((a > 0) & (q == 0), table[1], q)
    return q * torch.sign(x), scale, high - low


def decode(q, scale):
    return q.detach().cpu().float().double().reshape(-1) * spread(scale.detach().cpu().double(), q.numel())


class Update(object):
    """One update of a tensor: inputs as they are (flat, 64 bits), results and the sizes of their terms."""

    def __init__(self, p, g, m, v, step, lr, betas, eps, weight_decay):
        b1, b2 = betas
        self.m = b1 * m + (1 - b1) * g
        self.v = b2 * v + (1 - b2) * g * g
        self.m_size = b1 * m.abs() + (1 - b1) * g.abs()
        root = (self.v / -math.expm1(step * math.log(b2)) if b2 > 0 else self.v).sqrt()
        size = lr / (-math.expm1(step * math.log(b1)) if b1 > 0 else 1.)
        self.p = (1 - lr * weight_decay) * p - size * self.m / (root + eps)
        self.p_size = p.abs()
        self.u_size = size * self.m_size / (root + eps)


def flat(t):
    """The elements of a tensor in the order of its memory, in 64 bits on the host"""
    t = t.detach()
    order = sorted(range(t.dim()), key=lambda d: -t.stride(d))
    t = t.permute(order)
    return t.contiguous().view(-1).cpu().double() if t.dtype not in TYPES_8.values() \
        else t.contiguous().view(-1).cpu().float().double()


def check_m(got, u):
    """b1, 1 - b1, their product and the sum: four roundings of 2^-24 at most of the terms' sizes."""
    assert bool(((got - u.m).abs() <= 2. ** -22 * u.m_size + 2. ** -149).all())


def check_v(got, u):
    """b2, 1 - b2, two products and the sum of positive terms: five roundings (and what leaves float32 below)."""
    assert bool(((got - u.v).abs() <= 5 * 2. ** -24 * u.v + 4 * 2. ** -149).all())


def check_p(got, u, dtype):
    """Half a step of the type; the product with 1 - lr wd, that number itself and the sum, 2^-24 each of their size; and of the
    second term m (2^-22), half of v's 5 2^-24, the root and the reciprocal, 2^-23 each, the correction, the sum, the size and
    two products, 2^-24 each: 16 2^-24 of it."""
    info = torch.finfo(dtype)
    bound = (info.eps / 2) * (1 + 2. ** -10) * u.p.abs() + info.smallest_normal * info.eps \
        + 3 * 2. ** -24 * (u.p_size + u.u_size) + 16 * 2. ** -24 * u.u_size
    error = (got - u.p).abs()
    assert bool((error <= bound).all()), (error / bound).max().item()


def check_8(q, scale, want, kind, random16):
    """An 8-bit state (numbers, scales) of what is `want` in 64 bits.

    The scale is a quotient of the block's largest number, which is off by at most 5 2^-24: 2^-21 of it.  A number a in units
    of the scale is off by as much, twice (the reciprocal is rounded too), 2^-20: at most 16 steps of the type make that
    2^-16 of a step, so one number in 2^15 may be the other neighbour, and no other one."""
    n = want.numel()
    expect, scales, step = encode(want, kind, random16)
    got_scale = scale.detach().cpu().double()
    assert got_scale.shape == scales.shape
    assert bool(((got_scale - scales).abs() <= 2. ** -21 * scales).all())
    got = flat(q)
    off = (got - expect).abs()
    assert bool((off <= step * (1 + 1e-9) * 2).all())              # (a neighbour's own step may be the wider one)
    other = int((off > 0).sum())
    assert other <= 6 + n * 2. ** -14, (other, n)
