"""The formats of a cache with block scales, by their definitions, in 64 bits on the CPU.

A block of 32 values y with largest magnitude a: the smallest e >= -127 with
a <= M 2^e (M = 448, 6); codes are the nearest multiples of 2^e, ties to the even code.
"""
import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def e4m3_table():
    i = torch.arange(128, dtype=torch.float64)
    e, m = (i / 8).floor(), i % 8
    v = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))
    v[127] = float("nan")
    return v


E4M3 = e4m3_table()


def half_bytes(heads, dim, bits):
    n = heads * dim
    return -(-(n * bits // 8 + n // 32) // 16) * 16


def last_of(dtype, bits):
    """The last magnitude that does not round past the largest of its type."""
    return (1.875 if bits == 8 else 1.5) * 2.0 ** (15 if dtype == torch.float16 else 127)


def quantise(y, bits, dtype):
    """(codes [.., n], one a byte; scale bytes [.., n / 32]) of y [.., n] (64-bit numbers)
    that come from `dtype`."""
    table, most = (E4M3[:127], 448.0) if bits == 8 else (E2M1, 6.0)
    y = y.double().unflatten(-1, (-1, 32))
    finite = torch.isfinite(y).all(-1)
    last = last_of(dtype, bits)
    x = torch.where(torch.isfinite(y), y, 0.0).clamp(-last, last)
    a = x.abs().amax(-1)
    e = torch.full(a.shape, -127, dtype=torch.int64)
    for k in range(-127, 128):                        # the smallest that holds the largest
        e = torch.where(a > most * 2.0 ** k, k + 1, e)
    x = x / (2.0 ** e.double())[..., None]
    mid = (table[1:] + table[:-1]) / 2
    m = x.abs()
    up = torch.searchsorted(mid, m, right=False)      # midpoints below m
    tie = mid[up.clamp(max=mid.numel() - 1)] == m
    code = torch.where(tie & (up % 2 == 1), up + 1, up)
    code = code + torch.signbit(y) * (128 if bits == 8 else 8)
    return code.flatten(-2).to(torch.uint8), torch.where(finite, e + 127, 255).to(torch.uint8)


def pack(codes, bits):
    return codes if bits == 8 else codes[..., 0::2] | codes[..., 1::2] << 4


def unpack(half, heads, dim, bits):
    """(codes [.., heads, dim], scale bytes [.., heads, dim / 32]) of half records."""
    n = heads * dim
    c = half[..., : n * bits // 8]
    if bits == 4:
        c = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    s = half[..., n * bits // 8:][..., : n // 32]
    return c.unflatten(-1, (heads, dim)), s.unflatten(-1, (heads, dim // 32))


def values(half, heads, dim, bits):
    """Values [.., heads, dim] of half records."""
    c, s = unpack(half, heads, dim, bits)
    table = torch.cat([E4M3, -E4M3]) if bits == 8 else torch.cat([E2M1, -E2M1])
    power = torch.where(s == 255, float("nan"), torch.exp2(s.double() - 127))
    return (table[c.long()].unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)
