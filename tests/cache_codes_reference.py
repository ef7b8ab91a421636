"""A cache in 8 bits in 64 bits on the CPU: codes by search in the list of what codes stand for, a block at a time."""

from __future__ import annotations

import torch

E4M3 = torch.tensor([m / 512 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127],
                    dtype=torch.float64)
INT8 = torch.arange(128, dtype=torch.float64)


def book(dtype):
    return E4M3 if dtype == torch.uint8 else INT8


def power(byte):
    """2^(byte - 127), NaN for 255."""
    table = torch.tensor([2.0 ** (b - 127) for b in range(255)] + [float("nan")], dtype=torch.float64)
    return table[byte.long()]


def values(codes):
    """What codes stand for, before their scale."""
    c = codes.long()
    magnitude, negative = (c & 127, c > 127) if codes.dtype == torch.uint8 else (c.abs(), c < 0)
    v = book(codes.dtype)[magnitude.clamp(max=126 if codes.dtype == torch.uint8 else 127)]
    v = torch.where((magnitude == 127) & (codes.dtype == torch.uint8), torch.nan, v)
    return torch.where(negative, -v, v)


def encode(x, dtype):
    """Nearest codes of x (float64, magnitudes in range), ties to the even one."""
    b, y = book(dtype), x.abs()
    hi = torch.searchsorted(b, y).clamp(max=b.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = y - b[lo], b[hi] - y
    pick = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    if dtype == torch.uint8:
        return torch.where(torch.signbit(x), pick + 128, pick).to(torch.uint8)
    return torch.where(x < 0, -pick, pick).to(torch.int8)


def exponent(top, dtype):
    """The least e with top <= largest * 2^e as a byte; 255 for what is not finite."""
    if not top < float("inf"):
        return 255
    largest = float(book(dtype)[-1])
    e = -127
    while e < 127 and top > largest * 2.0 ** e:
        e += 1
    return e + 127


def append(x, codes, scales, table, starts, context):
    """x [heads, tokens, D] in float64 into codes and scales, in place, a block after the other."""
    pages, heads, page, _ = codes.shape
    block = page // scales.shape[2]
    for b in range(table.shape[0]):
        s, n, c = int(starts[b]), int(starts[b + 1]) - int(starts[b]), int(context[b])
        first = max(c - n, 0)
        for lo in range(first // block * block, c if n else 0, block):
            if lo // page >= table.shape[1]:
                continue
            at = int(table[b, lo // page])
            if not 0 <= at < pages:
                continue
            slot = lo % page
            new = slice(max(lo, first), min(lo + block, c))
            rows = x[:, s + new.start - (c - n):s + new.stop - (c - n)]
            for h in range(heads):
                r = rows[h]
                top = float(r.abs().max()) if torch.isfinite(r).all() else float("inf")
                e, kept = exponent(top, codes.dtype), int(scales[at, h, slot // block])
                if lo < first:
                    e = max(e, kept)
                    old = codes[at, h, slot:slot + first - lo]
                    if kept < e < 255:
                        old.copy_(encode(values(old) * 2.0 ** (kept - e), codes.dtype))
                scales[at, h, slot // block] = e
                unit = 2.0 ** (e - 127)
                codes[at, h, slot + new.start - lo:slot + new.stop - lo] = (
                    encode(r / unit, codes.dtype) if e < 255 else 0)


def cache(codes, scales):
    """A whole cache as values in float64."""
    block = codes.shape[2] // scales.shape[2]
    return values(codes) * power(scales).repeat_interleave(block, 2)[..., None]


def held(seed, pages, heads, page, d, block, dtype, spread=1.0):
    """A random cache as (codes, scales), its blocks of different sizes."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(pages, heads, page, d, generator=g, dtype=torch.float64)
    size = torch.exp2(spread * torch.randn(pages, heads, page // block, generator=g, dtype=torch.float64))
    x = x * size.repeat_interleave(block, 2)[..., None]
    tops = x.abs().reshape(pages, heads, page // block, -1).amax(3)
    scales = torch.tensor([exponent(float(t), dtype) for t in tops.flatten()], dtype=torch.uint8).reshape(tops.shape)
    return encode(x / power(scales).repeat_interleave(block, 2)[..., None], dtype), scales
