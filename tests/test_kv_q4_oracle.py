"""The 4-bit cache's oracle against itself and the definition (CPU): the layout's round trip, the bounds of what 4 bits keep, the
rules for values that are not finite, and the plain forms of the measured cases."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import paged, paged_q4


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_round_trip_and_error_bound(hd):
    """A group's elements come back within half a step, s / 2, and s is range / 15 within its rounding, 2^-8."""
    gen = torch.Generator().manual_seed(hd)
    k, v = (torch.randn(3, 32, 2, hd, generator=gen).bfloat16() * 2 ** i for i in range(2))
    cache = paged_q4.store_all(k, v)
    for x, y in zip((k, v), paged_q4.read(cache)):
        g = x.double().unflatten(-1, (-1, 32))
        step = (g.amax(-1) - g.amin(-1)) / 15 * (1 + 2.0 ** -8)
        assert ((x.double() - y).abs() <= step.repeat_interleave(32, -1) / 2).all()
    one = torch.zeros_like(cache)
    for page in range(3):
        for row in range(32):
            for head in range(2):
                paged_q4.store(one, page, row, head, k[page, row, head], False)
                paged_q4.store(one, page, row, head, v[page, row, head], True)
    assert torch.equal(one, cache)


def test_words_hold_pairs_of_elements():
    """(word >> 4 i) & 0x000f000f is elements 2 i and 2 i + 1 of 8; word t * groups + g holds dims 32 g + 8 t .."""
    x = torch.arange(64).bfloat16()
    x = (x % 32 // 2).bfloat16() + torch.where(torch.arange(64) < 32, 0, 100).bfloat16()
    cache = torch.zeros(1, 1, 1, 20 * 64, dtype=torch.uint8)
    paged_q4.store(cache, 0, 3, 0, x, False)
    words = cache[0, 0, 0, 3 * 32:4 * 32].view(torch.int32)
    codes, s, m = paged_q4.quantise(x)
    assert s.tolist() == [1.0, 1.0] and m.tolist() == [0.0, 100.0]
    for t in range(4):
        for g in range(2):
            w = int(words[t * 2 + g]) & 0xFFFFFFFF
            for i in range(4):
                pair = (w >> 4 * i) & 0x000F000F
                assert [pair & 15, pair >> 16] == codes[32 * g + 8 * t + 2 * i:][:2].tolist()


def test_values_that_four_bits_do_not_keep():
    x = torch.zeros(64).bfloat16()
    x[0], x[1], x[2], x[3] = math.nan, math.inf, 1.0, -3.0
    x[32:] = 7.0
    codes, s, m = paged_q4.quantise(x)
    assert m.tolist() == [-3.0, 7.0] and s[1] == 0 and s[0] == torch.tensor((2.0 ** 63 + 3) / 15).bfloat16().double()
    assert codes[1] == 15 and codes[32:].eq(0).all() and codes[0] == 0  # NaN counts as 0, far below a step from -3
    y = paged_q4.stands_for(codes, s, m)
    assert y.isfinite().all() and y[32:].eq(7.0).all()
    for bad in (math.nan, math.inf, -(2.0 ** 64)):
        pair = torch.tensor([bad], dtype=torch.float64)
        one = torch.ones(1, dtype=torch.float64)
        assert paged_q4.stands_for(codes[:32], pair, one).eq(0).all() and paged_q4.stands_for(codes[:32], one, pair).eq(0).all()
    tiny = torch.full((32,), 2.0 ** -101).bfloat16()
    tiny[0] = 0
    assert paged_q4.quantise(tiny)[1].eq(0).all()


def test_halves_go_up():
    """(x - m) / s = k + 1/2 exactly takes code k + 1."""
    x = torch.zeros(32).bfloat16()
    x[31] = 15.0
    x[1:9] = torch.arange(8).bfloat16() + 0.5
    assert paged_q4.quantise(x)[0][1:9].tolist() == list(range(1, 9))


def test_sinks_of_the_attention_oracle():
    """With sinks the softmax runs over the window's keys and the first ones, each once."""
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, 16, 1, 8, generator=gen).double() for _ in range(2))
    q = torch.randn(1, 1, 8, generator=gen).double()
    table, seqlens, cu = torch.tensor([[1, 0]], dtype=torch.int32), torch.tensor([29]), torch.tensor([0, 1])
    keys = torch.cat([k[1], k[0]])[:29, 0]
    values = torch.cat([v[1], v[0]])[:29, 0]
    for window, sinks, at in ((4, 3, [0, 1, 2, 25, 26, 27, 28]), (4, 0, [25, 26, 27, 28]), (27, 9, list(range(29))), (0, 5, list(range(29)))):
        out = paged.chunk(q, k, v, table, seqlens, cu, window=window, sinks=sinks)[0]
        w = torch.softmax(keys[at] @ q[0, 0] / math.sqrt(8), 0)
        assert torch.allclose(out[0, 0], w @ values[at])
