"""GPU: attention over the 4-bit KV cache where one key stands far out above thousands of others and its value is (near) zero, as the
first tokens of long streams do: the output then comes from weights thousands of times smaller than the largest one.

Keys are constant in the first group and zero in the others, so 4 bits hold them exactly (s = 0, m the key) and a score is the key
itself: no rounding of keys is left in the bound. What is left: the output's rounding, 2^-8 |out| <= 2^-8 spread (spread =
sum_j p_j |v_j|); weights and values in fp16, 2^-11 each, s times a weight another 2^-11 of a group's range (at most 4 mean |v| of
these values); weights below fp16's normal range, 2^-25 of 2^7 or more for each key, which is 2^-32 x 8000 keys of a sum that is at least
2^-10 here. Together below 2^-8 + 2^-9, and the bound is the bf16 cache's, 2^-7 (1 + 2^-4) spread."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import paged, paged_q4
from test_gqa_paged_gpu import _batch, _close

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _outstanding(gen, news, caches, Hq, Hkv, hd, page, nats, spread, first=0, values=1.0):
    """A batch whose scores are key values: ``nats`` for key ``first`` of every request, N(0, ``spread``) for the others."""
    table, seqlens, cu, pages = _batch(gen, news, caches, page)
    k = torch.zeros(pages, page, Hkv, hd)
    k[..., :32] = (torch.randn(pages, page, Hkv, 1, generator=gen) * spread)
    v = (torch.randn(pages, page, Hkv, hd, generator=gen) + 0.5) * values
    for b in range(len(news)):
        at = int(table[b, first // page]), first % page
        k[at][..., :32] = nats
        v[at] = 0.0
    cache = paged_q4.store_all(k.bfloat16(), v.bfloat16())
    q = torch.zeros(int(cu[-1]), Hq, hd)
    q[..., 0] = 1.0
    return q.bfloat16(), cache, table, seqlens, cu


def _check(zb, q, cache, table, seqlens, cu, bound=2.0 ** -7 * (1 + 2.0 ** -4), **kw):
    lse = torch.full(q.shape[:2], 7.0, device=DEV)
    out = zb.ops.gqa_chunk_q4(*(t.to(DEV) for t in (q, cache, table, seqlens, cu)), softmax_scale=1.0, lse=lse, **kw)
    kw.pop("max_new", None)
    ref, spread, ref_lse, size = paged.chunk(q, *paged_q4.read(cache), table, seqlens, cu, scale=1.0, **kw)
    _close(out, ref, bound * spread)
    _close(lse, ref_lse, 2.0 ** -15 + 2.0 ** -12 + q.shape[-1] * 2.0 ** -23 * size)
    assert zb.ops.device_status() == 0


@pytest.mark.parametrize("hd,Hq,Hkv", [(128, 4, 1), (64, 8, 2), (96, 2, 1), (32, 4, 1)])
@pytest.mark.parametrize("nats,spread", [(10.0, 0.0), (10.5, 1.0), (11.5, 0.0), (12.0, 0.5), (13.0, 1.0)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1000, 5)])
def test_a_first_key_that_stands_out(zb, hd, Hq, Hkv, nats, spread, window, sinks):
    """Single tokens, short drafts and chunks, by every kernel of the operator; the first key among the sinks of a window."""
    gen = torch.Generator().manual_seed(hd + int(nats * 10))
    x = _outstanding(gen, [1, 9, 200, 1], [8000, 3000, 2300, 5000], Hq, Hkv, hd, 16, nats, spread)
    _check(zb, *x, window=window, sinks=sinks)


@pytest.mark.parametrize("news", [[1, 1], [70, 140]])
@pytest.mark.parametrize("first", [1, 127, 130, 1500])
def test_a_key_further_on_stands_out(zb, news, first):
    """Not in the first tile: the accumulator is rescaled when it comes, and what was summed before it counts as little."""
    gen = torch.Generator().manual_seed(first)
    _check(zb, *_outstanding(gen, news, [4000, 2500], 4, 1, 128, 32, 12.0, 0.5, first=first))


@pytest.mark.parametrize("low", [-40.0, -3.0, 3.0, 5.0, 40.0])
def test_a_first_tile_anywhere(zb, low):
    """All scores moved up or down together: the first tile's largest is inside and outside of what needs no new reference."""
    gen = torch.Generator().manual_seed(3)
    q, cache, table, seqlens, cu = _outstanding(gen, [1, 150], [3000, 2000], 4, 1, 64, 16, 11.0, 0.0)
    k, v = paged_q4.read(cache)
    k[..., :32] += low  # 8 bits hold the sums
    _check(zb, q, paged_q4.store_all(k.bfloat16(), v.bfloat16()), table, seqlens, cu)


@pytest.mark.parametrize("sigma,nats", [(2.0 ** -10, 14.0), (2.0 ** -9, 14.0), (2.0 ** -10, 16.0), (2.0 ** -7, 16.0), (2.0 ** -5, 16.0), (2.0 ** -5, 20.0),
                                        (2.0 ** -60, 12.0)])
@pytest.mark.parametrize("Hq,hd", [(4, 128), (12, 128), (4, 64)])
def test_small_values_behind_a_key_that_stands_out(zb, sigma, nats, Hq, hd):
    """Single tokens, each unit's keys summed by one or two warps (many requests, over the same pages): small values with weights of
    2^-20 and less of the largest. Bound, where weights and s c are bf16's: 2^-8 for the output, 2 x 2^-8 for the weights above and below
    the fraction bar, 2^-8 of a group's range (4 mean |v|, of random signs: counted as 2)."""
    gen = torch.Generator().manual_seed(Hq + hd)
    keys, requests = 65536, 2400
    q, cache, table, seqlens, cu = _outstanding(gen, [1], [keys - 1], Hq, 1, hd, 256, nats, 0.5, values=sigma)
    many = [q.expand(requests, Hq, hd), cache, table.expand(requests, -1), seqlens.expand(requests)]
    many = [t.contiguous().to(DEV) for t in many]
    out = zb.ops.gqa_chunk_q4(*many, torch.arange(requests + 1, dtype=torch.int32, device=DEV), softmax_scale=1.0, max_new=1)
    ref, spread, *_ = paged.chunk(q, *paged_q4.read(cache), table, seqlens, cu, scale=1.0)
    _close(out, ref.expand_as(out), (5 * 2.0 ** -8 * spread).expand_as(out))
    assert zb.ops.device_status() == 0


@pytest.mark.parametrize("hd,Hq", [(128, 3), (96, 2), (64, 2), (32, 2)])
@pytest.mark.parametrize("nats", [10.0, 11.0, 11.5, 12.0])
def test_many_rows_over_a_long_flat_tail(zb, hd, Hq, nats):
    """Units that several CTAs hold parts of: only the first part sees the key that stands out."""
    gen = torch.Generator().manual_seed(int(nats * 2) + hd)
    _check(zb, *_outstanding(gen, [40], [17000], Hq, 1, hd, 64, nats, 0.0))
