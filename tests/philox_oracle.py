"""Philox4x32-10 masks of large tensors: 32 x 32 bit products from 16-bit limbs
in int64, checked against the plain Python form where the tests use it."""

import torch

_LOW = (1 << 32) - 1


def _product(m, t):
    """Upper and lower word of m * t (m, t below 2^32)."""
    lo = m * (t & 0xFFFF)
    hi = m * (t >> 16) + (lo >> 16)
    return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)


def words(first, count, seed, offset=0, device="cuda"):
    """Word e % 4 of block offset + e // 4 for first <= e < first + count (first a multiple of 4), as int64."""
    block = torch.arange(first // 4, -(-(first + count) // 4), device=device)
    low = (block & _LOW) + (offset & _LOW)
    high = ((block >> 32) + (offset >> 32) + (low >> 32)) & _LOW
    x = [low & _LOW, high, torch.zeros_like(block), torch.zeros_like(block)]
    for r in range(10):
        k0, k1 = (seed + r * 0x9E3779B9) & _LOW, ((seed >> 32) + r * 0xBB67AE85) & _LOW
        h0, l0 = _product(0xD2511F53, x[0])
        h1, l1 = _product(0xCD9E8D57, x[2])
        x = [h1 ^ x[1] ^ k0, l1, h0 ^ x[3] ^ k1, l0]
    return torch.stack(x, 1).view(-1)[:count]


def keep(shape, p, seed, offset=0, device="cuda"):
    n = 1
    for s in shape:
        n *= s
    out = torch.empty(n, dtype=torch.bool, device=device)
    step = 1 << 24
    for at in range(0, n, step):
        m = min(step, n - at)
        out[at:at + m] = words(at, m, seed, offset, device) >= int(p * 2**32)
    return out.view(shape)
