"""Microscaled rows in 64 bits, for the tests: the definition by exact arithmetic on float64 tensors of any device."""
import math

import torch

E4M3, E2M1 = 1, 2
LEAST = {E4M3: -6, E2M1: 0}  # exponent of the smallest normal element
BITS = {E4M3: 3, E2M1: 1}    # stored mantissa bits
MOST = {E4M3: 448.0, E2M1: 6.0}


def pow2(e):
    """2^e in float64, from its bits (torch.ldexp goes through pow, whose last bit may be off on a GPU)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def scale_bytes(top, fmt):
    """Scale byte of blocks whose largest magnitudes are top (float64): the least power of two s for which top / s is at most
    464 (e4m3; it ties to 448) or below 7 (e2m1); at least 2^-127; 255 for an infinity or NaN."""
    m, e = torch.frexp(top)
    e = e.long() - 1
    s = e - (8 if fmt == E4M3 else 2)
    up = 2 * m > 464 / 256 if fmt == E4M3 else 2 * m >= 7 / 4
    b = torch.where(top > 0, s + up.long() + 127, torch.zeros_like(s)).clamp(min=0)
    return torch.where(torch.isfinite(top), b, torch.full_like(b, 255))


def scale_values(b):
    v = pow2(b.long() - 127)
    return torch.where(b == 255, torch.full_like(v, math.nan), v)


def nearest(v, fmt):
    """Elements nearest to v, halves to the even one."""
    _, e = torch.frexp(v.abs())
    step = pow2((e.long() - 1).clamp(min=LEAST[fmt]) - BITS[fmt])
    return (torch.round(v / step) * step).clamp(-MOST[fmt], MOST[fmt])


def quantize(x, fmt):
    """(elements float64 [n,k], scale bytes int64 [n,k/32]) of x [n,k]."""
    x = x.double()
    n, k = x.shape
    b = x.view(n, k // 32, 32)
    top = b.abs().amax(2) if n else b.abs().sum(2)
    byte = scale_bytes(top, fmt)
    q = nearest(torch.where((byte == 255)[:, :, None], torch.zeros_like(b), b / scale_values(byte.clamp(max=254))[:, :, None]), fmt)
    return q.view(n, k), byte


def values(q, byte):
    n, k = q.shape
    return (q.view(n, k // 32, 32) * scale_values(byte)[:, :, None]).view(n, k)


def elements(codes, fmt):
    """float64 elements that the code bytes are."""
    if fmt == E4M3:
        return codes.view(torch.float8_e4m3fn).double()
    c = torch.stack((codes & 15, codes >> 4), 2).view(codes.shape[0], -1).long()
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)
    return torch.where(c >= 8, -table[c % 8], table[c % 8])


def half_step(v, s, fmt):
    """Half the distance between elements around |v| (float64) under scale s: how far a rounding may be off."""
    a = (v / s).abs()
    _, e = torch.frexp(a)
    return 0.5 * s * pow2((e.long() - 1).clamp(min=LEAST[fmt]) - BITS[fmt])
