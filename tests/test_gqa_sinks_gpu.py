"""GPU: windows with first keys that stay visible over the bf16 cache (zb_gqa_chunk_sinks) through ops.gqa_chunk against the float64
oracle, at the tolerances of tests/test_gqa_paged_gpu.py; the count of the keys seen (queries of zero: lse is its logarithm)."""

from __future__ import annotations

import math

import pytest
import torch

from test_gqa_paged_gpu import CHUNKS, _check_chunk, _chunk_inputs

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("case", CHUNKS)
@pytest.mark.parametrize("window,sinks", [(37, 4), (1, 200), (130, 1)])
def test_sinks_match_oracle(zb, case, window, sinks):
    news, caches, Hq, Hkv, hd, page = case
    gen = torch.Generator().manual_seed(CHUNKS.index(case))
    _check_chunk(zb, *_chunk_inputs(gen, news, caches, Hq, Hkv, hd, page), window=window, sinks=sinks)


@pytest.mark.parametrize("page", [1, 7, 8, 16, 128])
@pytest.mark.parametrize("window,sinks", [(1, 1), (128, 128), (500, 4), (3, 300), (200, 130), (1 << 40, 1 << 40)])
def test_sinks_count_their_keys(zb, page, window, sinks):
    gen = torch.Generator().manual_seed(page)
    for spread in (1.0, 0.0):
        _check_chunk(zb, *_chunk_inputs(gen, [40, 1, 130, 5], [260, 700, 0, 900], 8, 2, 64, page, spread), window=window, sinks=sinks)


@pytest.mark.parametrize("keys,Hq,hd", [(20000, 16, 128), (9001, 4, 64)])
def test_sinks_far_behind(zb, keys, Hq, hd):
    """Windows split over CTAs, the first tile's keys among the parts."""
    gen = torch.Generator().manual_seed(keys)
    _check_chunk(zb, *_chunk_inputs(gen, [1, 3, 70], [keys - 1, keys // 3, keys // 2], Hq, Hq // 4, hd, 64), window=4000, sinks=4)


@pytest.mark.parametrize("hd,page", [(128, 16), (64, 24), (96, 1), (128, 128)])
def test_sinks_ignore_what_they_do_not_see(zb, hd, page):
    """NaN and infinities between the first keys and the windows, past the keys and in free pages leave every row as it was; in a
    first key they reach all rows, in a key that some windows have left only those that see it."""
    gen = torch.Generator().manual_seed(hd + page)
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [9, 1, 40], [200, 130, 0], 8, 2, hd, page)
    kw = dict(window=64, sinks=3)
    clean = _check_chunk(zb, q, k, v, table, seqlens, cu, **kw)
    used = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b in range(3):
        n, keys = int(cu[b + 1] - cu[b]), int(seqlens[b])
        for j in [*range(min(3, keys)), *range(max(0, keys - n + 1 - 64), keys)]:
            used[int(table[b, j // page]), j % page] = True
    junk = torch.tensor([math.nan, math.inf, -math.inf])
    pick = torch.randint(0, 3, k.shape, generator=gen)
    k[~used], v[~used] = junk[pick].bfloat16()[~used], junk[pick.flip(0)].bfloat16()[~used]
    assert torch.equal(clean, _check_chunk(zb, q, k, v, table, seqlens, cu, **kw))
    # request 0's tokens stand at 200 .. 208: the first two see key 138, the others' windows begin behind it
    where = int(table[0, 138 // page]), 138 % page
    v[where][0, 3] = math.nan
    got = zb.ops.gqa_chunk(*(t.to(DEV) for t in (q, k, v, table, seqlens, cu)), **kw)
    assert got[:2, :4, 3].isnan().all() and torch.equal(got[2:], clean[2:])
    v[where][0, 3] = 0.0
    where = int(table[0, 2 // page]), 2 % page
    v[where][1, 5] = math.inf
    got = zb.ops.gqa_chunk(*(t.to(DEV) for t in (q, k, v, table, seqlens, cu)), **kw)
    assert got[:9, 4:, 5].eq(math.inf).all() and torch.equal(got[9:], clean[9:])


def test_sinks_that_change_nothing_give_equal_results(zb):
    gen = torch.Generator().manual_seed(21)
    x = [t.to(DEV) for t in _chunk_inputs(gen, [1, 40], [500, 300], 8, 2, 128, 16)]
    plain = zb.ops.gqa_chunk(*x)
    assert torch.equal(plain, zb.ops.gqa_chunk(*x, sinks=7)) and torch.equal(plain, zb.ops.gqa_chunk(*x, window=600, sinks=7))


def test_sinks_in_a_graph_follow_the_lengths(zb):
    gen = torch.Generator().manual_seed(22)
    d = [t.to(DEV) for t in _chunk_inputs(gen, [30, 1, 2], [40, 3000, 600], 8, 2, 128, 16)]
    out = torch.empty_like(d[0])
    zb.ops.gqa_chunk(*d, out=out, window=200, sinks=4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        zb.ops.gqa_chunk(*d, out=out, window=200, sinks=4)
    d[4].copy_(torch.tensor([700, 1500, 17], dtype=torch.int32))
    d[5].copy_(torch.tensor([0, 20, 22, 33], dtype=torch.int32))
    graph.replay()
    expected = zb.ops.gqa_chunk(*d, window=200, sinks=4)
    torch.cuda.synchronize()
    assert torch.equal(out, expected)
