"""4-bit KV cache oracle (CPU, float64): the groups' codes and pairs, the layout of a cache's blocks, and the values it stands
for, written out from the definition. With :mod:`oracle.paged` on those values it is the oracle of the 4-bit operators. Test
infrastructure only (see ``oracle/__init__.py``).
"""

from __future__ import annotations

import torch

GROUP, BLOCK = 32, 16


def quantise(x):
    """Codes [..., hd] (int64), s and m [..., hd / 32] (float64, values of bf16) of bf16 rows x [..., hd]."""
    x = x.double()
    x = torch.where(x.isnan(), torch.zeros_like(x), x.clamp(-(2.0 ** 63), 2.0 ** 63)).unflatten(-1, (-1, GROUP))
    m, high = x.amin(-1), x.amax(-1)
    s = ((high - m) / 15).float().bfloat16().double()
    s = torch.where(s < 2.0 ** -100, torch.zeros_like(s), s)
    safe = torch.where(s > 0, s, torch.ones_like(s))[..., None]
    c = torch.where(s[..., None] > 0, torch.floor((x - m[..., None]) / safe + 0.5).clamp(0, 15), torch.zeros_like(x))
    return c.long().flatten(-2), s, m


def stands_for(codes, s, m):
    """Values [..., hd] (float64); a pair that is not finite, or of 2^64 and more, counts as zeros."""
    s, m = s.repeat_interleave(GROUP, -1), m.repeat_interleave(GROUP, -1)
    none = ~((s.abs() < 2.0 ** 64) & (m.abs() < 2.0 ** 64))
    return torch.where(none, torch.zeros_like(s), m + s * codes.double())


def _places(hd):
    """(byte of a row, shift in it) of every element."""
    places = []
    for d in range(hd):
        g, t, e = d // 32, d % 32 // 8, d % 8
        nibble = e // 2 + 4 * (e % 2)
        places.append((4 * (t * (hd // 32) + g) + nibble // 2, 4 * (nibble % 2)))
    return places


def _parts(hd, value):
    return (8 if value else 0) * hd, (18 if value else 16) * hd


def store(cache, page, row, head, x, value):
    """A bf16 row x [hd] as key or value of head ``head`` in row ``row`` of page ``page`` of a cache [pages, Hkv, blocks, 20 hd]."""
    hd = x.shape[-1]
    codes, s, m = quantise(x)
    at, pairs = _parts(hd, value)
    block = cache[page, head, row // BLOCK]
    inside = at + (row % BLOCK) * (hd // 2)
    block[inside:inside + hd // 2] = 0
    for d, (byte, shift) in enumerate(_places(hd)):
        block[inside + byte] |= int(codes[d]) << shift
    inside = pairs + (row % BLOCK) * (hd // 8)
    block[inside:inside + hd // 8] = torch.stack([s, m], -1).flatten().bfloat16().view(torch.uint8)


def store_all(k, v):
    """A cache that holds keys and values [pages, page_size, Hkv, hd] (bf16)."""
    pages, page_size, Hkv, hd = k.shape
    cache = torch.zeros(pages, Hkv, page_size // BLOCK, 20 * hd, dtype=torch.uint8)
    places = _places(hd)
    for value, x in enumerate((k, v)):
        at, pairs = _parts(hd, value)
        codes, s, m = quantise(x.unflatten(1, (-1, BLOCK)).permute(0, 3, 1, 2, 4))  # [pages, Hkv, blocks, 16, hd]
        rows = torch.zeros(*codes.shape[:-1], hd // 2, dtype=torch.int64)
        for d, (byte, shift) in enumerate(places):
            rows[..., byte] |= codes[..., d] << shift
        cache[..., at:at + 8 * hd] = rows.to(torch.uint8).flatten(-2)
        both = torch.stack([s, m], -1).flatten(-2).bfloat16().contiguous()
        cache[..., pairs:pairs + 2 * hd] = both.view(torch.uint8).flatten(-2)
    return cache


def read(cache):
    """Keys and values [pages, page_size, Hkv, hd] (float64) that a cache stands for."""
    hd = cache.shape[-1] // 20
    found = []
    for value in range(2):
        at, pairs = _parts(hd, value)
        rows = cache[..., at:at + 8 * hd].unflatten(-1, (BLOCK, hd // 2)).long()
        codes = torch.stack([(rows[..., byte] >> shift) & 15 for byte, shift in _places(hd)], -1)
        both = cache[..., pairs:pairs + 2 * hd].contiguous().view(torch.bfloat16).unflatten(-1, (BLOCK, hd // 32, 2)).double()
        x = stands_for(codes, both[..., 0], both[..., 1])  # [pages, Hkv, blocks, 16, hd]
        found.append(x.permute(0, 2, 3, 1, 4).flatten(1, 2))
    return found[0], found[1]
