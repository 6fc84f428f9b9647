"""GPU: the 4-bit KV cache (zb_gqa_append_q4, zb_kv_read_q4, zb_gqa_chunk_q4) through the package's ops against the float64
oracles (oracle.paged, oracle.paged_q4): head dims 32 .. 128, query groups 1 .. 16, pages of 16 to 256 rows, requests with no, one,
a few and hundreds of new tokens, caches from empty to many tiles, windows with first tokens kept, masked pages, strides.

Tolerances, derived from the operators' rounding points (bf16 rounds by at most 2^-8 of a value):
* codes and pairs of bf16 rows stored as they come follow from exact comparisons: the cache's bytes are equal. Behind the norm and
  the rotation a key x is off by 2^-18 of its pair's magnitude and 2^-8 |x| (its rounding) before it is quantised; then by half a
  step, s / 2, with s = range / 15 within 2^-8 of it, the range from elements that are off as much.
* kv_read rounds m + s c once: equal to the oracle's rounding.
* chunk sees keys and values rounded to bf16 at most: values 2^-8 sum_j p_j |v_j|; scores 2^-8 size each (size = max_j scale sum_d
  |q_d k_jd|), so weights, numerator and denominator, e^(2 2^-8 size) - 1. Its own roundings as for the bf16 cache: weights and
  output 2^-8 each, the rest below 2^-4 of those two.
* lse: 2^-8 size for the keys, hd 2^-23 size for the products' sums, 2^-15 for the exponentials and their sum. With queries of zero
  it is the logarithm of the number of keys seen, to 2^-15."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import paged, paged_q4
from test_gqa_paged_gpu import _batch, _close

pytestmark = pytest.mark.gpu

DEV = "cuda"


# ------------------------------------------------------------------------------------------------------- append

APPENDS = [
    # news, caches, heads, kv_heads, hd, page, rotary, interleaved
    ([1], [877], 16, 4, 128, 16, 128, True),
    ([1, 1, 0, 1], [0, 15, 3, 16], 16, 4, 128, 16, 128, True),
    ([40, 3], [5, 70], 8, 2, 128, 48, 128, False),
    ([13, 1, 30], [100, 2, 0], 14, 2, 64, 32, 32, False),
    ([7, 9], [1, 33], 6, 2, 96, 64, 48, False),
    ([7, 9], [1, 33], 5, 5, 96, 64, 96, True),
    ([5, 6], [0, 1000000], 8, 2, 32, 20000, 32, True),
    ([5, 2], [3, 4], 3, 1, 32, 16, 0, True),
]


def _append_inputs(gen, case, pad=0):
    news, caches, heads, kv, hd, page, rotary, interleaved = case
    table, seqlens, cu, pages = _batch(gen, news, caches, page)
    proj = torch.randn(int(cu[-1]), (heads + 2 * kv) * hd + pad, generator=gen).bfloat16()
    cache = torch.randint(0, 256, (pages, kv, page // 16, 20 * hd), generator=gen, dtype=torch.uint8)
    temp = (1 + 0.3 * torch.randn(heads, generator=gen)).bfloat16()
    return proj, cache, table, seqlens, cu, temp


def _slots(table, seqlens, cu, page, pages):
    """(row of proj, page, row in it) of every new token that has a page."""
    for b, first, rows, keys in paged.requests(cu, seqlens):
        for i in range(rows):
            slot = paged._slot(table, pages, page, b, keys - rows + i)
            if slot is not None:
                yield first + i, *slot


@pytest.mark.parametrize("case", APPENDS)
def test_rows_stored_as_they_come(zb, case):
    """k | v alone, without norm and rotation: the cache's bytes, those of rows that were not written among them."""
    news, caches, _, kv, hd, page, *_ = case
    gen = torch.Generator().manual_seed(APPENDS.index(case))
    proj, cache, table, seqlens, cu, _ = _append_inputs(gen, (news, caches, 0, *case[3:]))
    proj[0, :40] = 1.25  # a group of equal elements, and halves of a step
    proj[-1, 32 * (kv * hd // 32 - 1):][:8] = torch.tensor([0.0, 15.0, 0.5, 1.5, 2.5, 7.5, 13.5, 14.5])
    proj[-1, 32 * (kv * hd // 32 - 1) + 8:][:24] = 3.0
    got = cache.to(DEV)
    assert zb.ops.gqa_append_q4(proj.to(DEV), got, table.to(DEV), seqlens.to(DEV), cu.to(DEV), heads=0, kv_heads=kv, eps=None,
                                rotary_dim=0) is None
    for t, p, row in _slots(table, seqlens, cu, page, cache.shape[0]):
        rows = proj[t, : 2 * kv * hd].view(2, kv, hd)
        for h in range(kv):
            paged_q4.store(cache, p, row, h, rows[0, h], False)
            paged_q4.store(cache, p, row, h, rows[1, h], True)
    assert torch.equal(got.cpu(), cache)


def _check_append(zb, case, proj, cache, table, seqlens, cu, views=None, **kw):
    news, caches, heads, kv, hd, page, rotary, interleaved = case
    d = {n: t.to(DEV) for n, t in dict(proj=proj, cache=cache, table=table, seqlens=seqlens, cu=cu).items()}
    d.update(views or {})
    extra = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    q = zb.ops.gqa_append_q4(d["proj"], d["cache"], d["table"], d["seqlens"], d["cu"], heads=heads, kv_heads=kv,
                             rotary_dim=rotary, interleaved=interleaved, **extra)
    pages = cache.shape[0]
    k64 = torch.full((pages, page, kv, hd), math.nan, dtype=torch.float64)
    v64 = k64.clone()
    q64, q_mag, k_mag = paged.append(proj, k64, v64, table, seqlens, cu, heads=heads, kv_heads=kv, rotary=rotary,
                                     interleaved=interleaved, **{n: t for n, t in kw.items() if n != "q_out"})
    _close(q, q64, 2.0 ** -8 * q64.abs() + 2.0 ** -18 * q_mag)
    k, v = paged_q4.read(d["cache"].cpu())
    k_old, v_old = paged_q4.read(cache)
    written = ~k64.isnan().any(-1).any(-1)  # [pages, page]
    assert torch.equal(k[~written], k_old[~written]) and torch.equal(v[~written], v_old[~written])
    exact, mag = k64[written], k_mag[written]
    off = 2.0 ** -8 * exact.abs() * (1 + 2.0 ** -8) + 2.0 ** -18 * mag
    groups = exact.unflatten(-1, (-1, 32))
    step = (groups.amax(-1) - groups.amin(-1) + 2 * off.unflatten(-1, (-1, 32)).amax(-1)) / 15 * (1 + 2.0 ** -8)
    _close(k[written], exact, off + step.repeat_interleave(32, -1) / 2)
    codes, s, m = paged_q4.quantise(v64[written].bfloat16())
    assert torch.equal(v[written], paged_q4.stands_for(codes, s, m))
    return q, d["cache"]


@pytest.mark.parametrize("case", APPENDS)
def test_append_matches_oracle(zb, case):
    gen = torch.Generator().manual_seed(100 + APPENDS.index(case))
    proj, cache, table, seqlens, cu, temp = _append_inputs(gen, case)
    _check_append(zb, case, proj, cache, table, seqlens, cu, temp=temp)


@pytest.mark.parametrize("pad", [1, 6, 24])
def test_append_strides_and_positions(zb, pad):
    """Projection rows at 2-, 4- and 16-byte alignment, a cache that is a slice of a larger pool, q as a slice, positions given."""
    case = APPENDS[2]
    gen = torch.Generator().manual_seed(pad)
    proj, cache, table, seqlens, cu, temp = _append_inputs(gen, case, pad=pad)
    pages, kv, blocks, block = cache.shape
    pool = torch.full((pages, 2, kv + 1, blocks, block), 7, dtype=torch.uint8, device=DEV)
    view = pool[:, 1, 1:]
    view.copy_(cache)
    wide = torch.full((proj.shape[0], 8 * 128 + 8), 5.0, dtype=torch.bfloat16, device=DEV)
    positions = torch.randint(0, 50000, (proj.shape[0],), generator=gen, dtype=torch.int32)
    _check_append(zb, case, proj, cache, table, seqlens, cu, views={"cache": view}, temp=temp, positions=positions,
                  q_out=wide[:, :1024].unflatten(1, (8, 128)))
    assert wide[:, 1024:].eq(5.0).all() and pool[:, 0].eq(7).all() and pool[:, 1, 0].eq(7).all()


def test_append_without_pages_and_rows_of_no_request(zb):
    case = ([6, 20, 3], [30, 0, 40], 8, 2, 64, 16, 64, True)
    gen = torch.Generator().manual_seed(3)
    proj, cache, table, seqlens, cu, temp = _append_inputs(gen, case)
    table[1, 0], table[2] = -1, cache.shape[0]
    seqlens[0] = 4  # two of its six tokens stand before the first position
    proj = torch.cat([proj[:2], proj, proj[:5]])
    q, _ = _check_append(zb, case, proj, cache, table, seqlens, cu + 2, temp=temp)
    assert q[:2].eq(0).all() and q[-5:].eq(0).all()


def test_append_of_values_that_four_bits_do_not_keep(zb):
    """NaN, infinities and magnitudes beyond 2^63, in one group of keys and one of values: the others are as without them."""
    case = ([4], [9], 0, 2, 64, 16, 0, True)
    gen = torch.Generator().manual_seed(4)
    proj, cache, table, seqlens, cu, _ = _append_inputs(gen, case)
    proj[1, 3], proj[1, 40], proj[2, 70], proj[2, 128 + 5], proj[3, 200] = math.nan, math.inf, -3e38, -math.inf, 2.0 ** 63
    proj[0, 64:96] = 2.0 ** -120
    got = cache.to(DEV)
    zb.ops.gqa_append_q4(proj.to(DEV), got, table.to(DEV), seqlens.to(DEV), cu.to(DEV), heads=0, kv_heads=2, eps=None, rotary_dim=0)
    for t, p, row in _slots(table, seqlens, cu, 16, cache.shape[0]):
        rows = proj[t].view(2, 2, 64)
        for h in range(2):
            paged_q4.store(cache, p, row, h, rows[0, h], False)
            paged_q4.store(cache, p, row, h, rows[1, h], True)
    assert torch.equal(got.cpu(), cache)
    k, v = zb.ops.kv_read_q4(got, table.to(DEV), seqlens.to(DEV), cu.to(DEV), 4)
    assert k.isfinite().all() and v.isfinite().all()


# --------------------------------------------------------------------------------------------------------- read


def _q4_cache(gen, pages, page, kv, hd, spread=1.0):
    k, v = (torch.randn(pages, page, kv, hd, generator=gen) * spread for _ in range(2))
    return paged_q4.store_all(k.bfloat16(), v.bfloat16())


@pytest.mark.parametrize("hd,kv,page", [(128, 4, 16), (64, 2, 48), (96, 3, 32), (32, 1, 256), (128, 1, 64), (32, 5, 16)])
def test_read_matches_oracle(zb, hd, kv, page):
    """Ragged tails, whole requests, none, and rows of no request; equal to m + s c rounded once."""
    gen = torch.Generator().manual_seed(hd + kv + page)
    news, caches = [40, 0, 1, 130, 17], [0, 9, 300, 61, 16]
    table, seqlens, cu, pages = _batch(gen, news, caches, page)
    cache = _q4_cache(gen, pages, page, kv, hd)
    table[3, 0] = -1
    k64, v64 = paged_q4.read(cache)
    rows = int(cu[-1]) + 7
    cu = cu + 3
    k, v = zb.ops.kv_read_q4(*(t.to(DEV) for t in (cache, table, seqlens, cu)), rows)
    k_ref, v_ref = (torch.zeros(rows, kv, hd, dtype=torch.float64) for _ in range(2))
    for t, p, row in _slots(table, seqlens, cu, page, pages):
        k_ref[t], v_ref[t] = k64[p, row], v64[p, row]
    assert torch.equal(k.cpu(), k_ref.bfloat16()) and torch.equal(v.cpu(), v_ref.bfloat16())
    whole = torch.cat([torch.zeros(1, dtype=torch.int32), seqlens.cumsum(0).to(torch.int32)])
    n = int(whole[-1])
    wide = torch.full((2, n, kv * hd + 8), 9.0, dtype=torch.bfloat16, device=DEV)
    views = [w[:, : kv * hd].unflatten(1, (kv, hd)) for w in wide]
    zb.ops.kv_read_q4(*(t.to(DEV) for t in (cache, table, seqlens, whole)), n, k_out=views[0], v_out=views[1])
    k_ref, v_ref = (torch.zeros(n, kv, hd, dtype=torch.float64) for _ in range(2))
    for t, p, row in _slots(table, seqlens, whole, page, pages):
        k_ref[t], v_ref[t] = k64[p, row], v64[p, row]
    assert torch.equal(views[0].cpu(), k_ref.bfloat16()) and torch.equal(views[1].cpu(), v_ref.bfloat16())
    assert wide[..., kv * hd:].eq(9.0).all()


def test_read_many_rows_and_pairs_that_are_none(zb):
    """Enough rows that a warp takes several, of requests that end inside a run; pairs that stand for zeros."""
    gen = torch.Generator().manual_seed(8)
    news = [int(n) for n in torch.randint(0, 40, (3000,), generator=gen)]
    table, seqlens, cu, pages = _batch(gen, news, [int(c) for c in torch.randint(0, 9, (3000,), generator=gen)], 16)
    cache = _q4_cache(gen, 50, 16, 2, 64)
    bad = torch.tensor([math.nan, math.inf, -(2.0 ** 64), 1.0]).bfloat16().view(torch.uint8)
    cache[7, 1, 0, 18 * 64 + 16:18 * 64 + 24] = bad  # a row's (NaN, inf), (-2^64, 1)
    table = torch.where(table >= 0, table % 50, table)
    k64, v64 = paged_q4.read(cache)
    assert v64[7, 2, 1].eq(0).all()
    k, v = zb.ops.kv_read_q4(*(t.to(DEV) for t in (cache, table, seqlens, cu)), int(cu[-1]))
    where = torch.tensor(list(_slots(table, seqlens, cu, 16, 50)))
    assert len(where) == len(k)
    assert torch.equal(k.cpu(), k64[where[:, 1], where[:, 2]].bfloat16())
    assert torch.equal(v.cpu(), v64[where[:, 1], where[:, 2]].bfloat16())


# --------------------------------------------------------------------------------------------------------- chunk


def _chunk_inputs(gen, news, caches, Hq, Hkv, hd, page, spread=1.0):
    table, seqlens, cu, pages = _batch(gen, news, caches, page)
    cache = _q4_cache(gen, pages, page, Hkv, hd)
    q = (torch.randn(int(cu[-1]), Hq, hd, generator=gen) * spread).bfloat16()
    return q, cache, table, seqlens, cu


def _check_chunk(zb, q, cache, table, seqlens, cu, gate=None, views=None, **kw):
    d = {n: t.to(DEV) for n, t in dict(q=q, cache=cache, table=table, seqlens=seqlens, cu=cu).items()}
    d.update(views or {})
    N, Hq, hd = q.shape
    lse = torch.full((N, Hq), 7.0, device=DEV)
    out = zb.ops.gqa_chunk_q4(d["q"], d["cache"], d["table"], d["seqlens"], d["cu"], lse=lse,
                              gate=None if gate is None else gate.to(DEV), out=d.get("out"), **kw)
    kw.pop("max_new", None)
    kw = {**kw, "scale": kw.pop("softmax_scale", None)}
    ref, spread, ref_lse, size = paged.chunk(q, *paged_q4.read(cache), table, seqlens, cu, gate=gate, **kw)
    weights = torch.expm1(2 * 2.0 ** -8 * size)[..., None]
    _close(out, ref, (2.0 ** -7 * (1 + 2.0 ** -4) + 2.0 ** -8 + weights) * spread)
    empty = ref_lse == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty)
    _close(lse.cpu()[~empty], ref_lse[~empty], (2.0 ** -15 + (hd * 2.0 ** -23 + 2.0 ** -8) * size)[~empty])
    assert zb.ops.device_status() == 0
    return out


CHUNKS = [
    # news, caches, Hq, Hkv, hd, page
    ([1], [0], 16, 4, 128, 16),
    ([1, 1, 1, 1], [0, 126, 127, 128], 16, 4, 128, 16),
    ([5, 0, 1, 33], [0, 9, 300, 95], 16, 4, 128, 16),
    ([2, 4, 3, 1], [700, 14, 0, 15], 8, 2, 128, 32),
    ([31, 32, 33, 64, 65], [0, 1, 127, 128, 129], 8, 2, 128, 32),
    ([150, 1], [0, 700], 4, 1, 128, 48),
    ([70, 3], [60, 258], 8, 8, 128, 32),
    ([17, 1, 0], [130, 5, 40], 14, 2, 64, 48),
    ([1, 1, 2], [130, 5, 40], 14, 2, 64, 48),
    ([129, 2], [3, 255], 6, 2, 64, 128),
    ([9, 40, 1], [77, 0, 1000], 16, 1, 64, 208),
    ([20, 1], [33, 140], 8, 2, 32, 16),
    ([11, 7], [150, 0], 6, 2, 96, 64),
]


@pytest.mark.parametrize("case", CHUNKS)
@pytest.mark.parametrize("mode", ["causal", "window", "sinks", "full", "gate", "count"])
def test_chunk_matches_oracle(zb, case, mode):
    news, caches, Hq, Hkv, hd, page = case
    gen = torch.Generator().manual_seed(CHUNKS.index(case))
    x = _chunk_inputs(gen, news, caches, Hq, Hkv, hd, page, spread=0.0 if mode == "count" else 1.0)
    gate = torch.randn(x[0].shape[0], Hq, generator=gen).bfloat16() if mode == "gate" else None
    kw = {"window": dict(window=37), "sinks": dict(window=37, sinks=5), "full": dict(causal=False),
          "count": dict(window=100, sinks=3)}.get(mode, {})
    for max_new in (None, max(news)):
        _check_chunk(zb, *x, gate=gate, max_new=max_new, **kw)


FEW = [
    # news, caches, Hq, Hkv, hd, page: rows of up to 8 and of up to 16 heads of tokens
    ([1, 1, 0, 1, 1], [0, 15, 3, 16, 17], 8, 1, 128, 16),
    ([2, 1, 2, 0, 2], [0, 300, 127, 5, 1000], 16, 4, 64, 32),
    ([8, 3, 1], [5, 77, 640], 4, 4, 128, 64),
    ([4, 1, 3], [130, 0, 2000], 16, 4, 128, 48),
    ([1, 1], [33, 700], 16, 1, 64, 16),
    ([16, 7, 2], [0, 9, 250], 2, 2, 128, 16),
    ([1, 1, 1], [1, 900, 31], 12, 1, 128, 256),
]


@pytest.mark.parametrize("case", FEW)
@pytest.mark.parametrize("mode", ["causal", "sinks", "full", "gate", "count"])
def test_chunk_of_few_rows_matches_oracle(zb, case, mode):
    """Batches whose every request has few rows, known to have them: the kernel of few rows alone. Its scores and weights are
    nearer to the oracle's than the bound for rounded keys: without the keys' rounding it is the bf16 cache's."""
    news, caches, Hq, Hkv, hd, page = case
    gen = torch.Generator().manual_seed(200 + FEW.index(case))
    x = _chunk_inputs(gen, news, caches, Hq, Hkv, hd, page, spread=0.0 if mode == "count" else 1.0)
    gate = torch.randn(x[0].shape[0], Hq, generator=gen).bfloat16() if mode == "gate" else None
    kw = {"sinks": dict(window=37, sinks=5), "full": dict(causal=False), "count": dict(window=100, sinks=3)}.get(mode, {})
    before = zb._lib.launch_count()
    out = _check_chunk(zb, *x, gate=gate, max_new=max(news), **kw)
    assert zb._lib.launch_count() - before == 1
    _, spread, _, _ = ref = paged.chunk(x[0], *paged_q4.read(x[1]), *x[2:], gate=gate, **kw)
    _close(out, ref[0], 2.0 ** -7 * (1 + 2.0 ** -4) * spread)


def test_chunk_of_more_new_tokens_than_said(zb):
    """A status bit; the other requests are as they are without it."""
    gen = torch.Generator().manual_seed(20)
    x = [t.to(DEV) for t in _chunk_inputs(gen, [1, 3, 1], [500, 300, 90], 16, 4, 128, 16)]
    expected = zb.ops.gqa_chunk_q4(*x)
    assert zb.ops.device_status() == 0
    out = zb.ops.gqa_chunk_q4(*x, max_new=1)
    assert zb.ops.device_status() == 256
    assert torch.equal(out[0], expected[0]) and torch.equal(out[4], expected[4])


@pytest.mark.parametrize("news", [[1, 2], [40, 3]])
@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -20, 2.0 ** -12, 2.0 ** 12, 2.0 ** 20, 2.0 ** 59])
def test_chunk_values_of_all_magnitudes(zb, news, scale):
    """Values outside fp16's range, all of them and every third group alone: as precise as any."""
    gen = torch.Generator().manual_seed(21)
    for alone in (False, True):
        table, seqlens, cu, pages = _batch(gen, news, [100, 300], 16)
        k, v = (torch.randn(pages, 16, 2, 128, generator=gen) for _ in range(2))
        v *= torch.where(torch.rand(pages, 16, 2, 4, 1, generator=gen).lt(0.3) if alone else torch.ones(1).bool(), scale,
                         1.0).expand(pages, 16, 2, 4, 32).flatten(-2)
        cache = paged_q4.store_all(k.bfloat16(), v.bfloat16())
        q = torch.randn(int(cu[-1]), 8, 128, generator=gen).bfloat16()
        _check_chunk(zb, q, cache, table, seqlens, cu)


@pytest.mark.parametrize("news", [[1, 2], [40, 3], [130, 17]])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 48), (96, 32), (32, 64)])
def test_chunk_blocks_of_different_magnitudes(zb, news, hd, page):
    """Blocks of 16 keys whose values fp16 holds beside blocks that it does not hold: for their size, and for a group's step of 0."""
    gen = torch.Generator().manual_seed(hd + news[0])
    for window, sinks in ((0, 0), (90, 5)):
        table, seqlens, cu, pages = _batch(gen, news, [300, 700], page)
        k, v = (torch.randn(pages, page, 2, hd, generator=gen) for _ in range(2))
        kind = torch.randint(0, 4, (pages, page // 16, 1, 2, 1), generator=gen)
        v = v.unflatten(1, (-1, 16))
        v = torch.where(kind == 0, v * 2.0 ** 14, torch.where(kind == 1, v.clone().mul_(2.0 ** 11), v * 2.0 ** 12))
        v[..., :32] = torch.where(kind == 3, torch.tensor(2.0 ** 13), v[..., :32])
        cache = paged_q4.store_all(k.bfloat16(), v.flatten(1, 2).bfloat16())
        q = torch.randn(int(cu[-1]), 8, hd, generator=gen).bfloat16()
        _check_chunk(zb, q, cache, table, seqlens, cu, window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(1, 1), (2, 0), (128, 128), (500, 4), (3, 300), (130, 17), (1 << 40, 1 << 40)])
def test_chunk_windows_and_sinks(zb, window, sinks):
    gen = torch.Generator().manual_seed(sinks)
    for spread in (1.0, 0.0):
        _check_chunk(zb, *_chunk_inputs(gen, [40, 1, 130, 3], [260, 511, 0, 700], 8, 2, 64, 16, spread), window=window, sinks=sinks)


@pytest.mark.parametrize("keys,Hq,hd", [(20000, 16, 128), (9001, 4, 64), (5000, 32, 96)])
@pytest.mark.parametrize("max_new", [None, 3])
def test_chunk_few_rows_over_a_long_cache(zb, keys, Hq, hd, max_new):
    """One and three tokens over a long cache: the key axis is split and joined."""
    gen = torch.Generator().manual_seed(keys)
    _check_chunk(zb, *_chunk_inputs(gen, [1, 3], [keys - 1, keys // 3], Hq, Hq // 4, hd, 64), max_new=max_new)


@pytest.mark.parametrize("Hq,Hkv,hd", [(8, 8, 64), (14, 2, 64), (6, 2, 64), (8, 8, 128), (6, 2, 128)])
@pytest.mark.parametrize("max_new", [None, 1])
def test_chunk_odd_rows_over_a_long_cache(zb, Hq, Hkv, hd, max_new):
    """An odd number of rows, whose parts are joined in more than one step: a warp's lanes do not all have an element of them."""
    gen = torch.Generator().manual_seed(Hq + hd)
    _check_chunk(zb, *_chunk_inputs(gen, [1, 1, 1], [9000, 700, 5001], Hq, Hkv, hd, 48), max_new=max_new)


@pytest.mark.parametrize("max_new", [None, 3])
def test_chunk_many_requests(zb, max_new):
    """More requests than CTAs, with and without new tokens; requests of few and of many rows."""
    gen = torch.Generator().manual_seed(9)
    news = [(b * 7) % 4 for b in range(700)]
    if max_new is None:
        news[5], news[600] = 90, 33
    caches = [(b * 13) % 50 for b in range(700)]
    _check_chunk(zb, *_chunk_inputs(gen, news, caches, 4, 2, 64, 16), max_new=max_new)


def test_chunk_long_prompt(zb):
    gen = torch.Generator().manual_seed(8)
    _check_chunk(zb, *_chunk_inputs(gen, [700], [0], 4, 1, 128, 16))


@pytest.mark.parametrize("hd", [64, 128])
def test_chunk_masked_pages_and_short_caches(zb, hd):
    """Pages outside the cache mask their keys; more new tokens than keys; no keys; more keys than the table has columns."""
    gen = torch.Generator().manual_seed(5)
    news = [20, 9, 4, 30, 6, 8, 3, 1, 1, 2]
    q, cache, table, seqlens, cu = _chunk_inputs(gen, news, [150, 140, 60, 0, 0, 200, 90, 100, 60, 0], 8, 2, hd, 16)
    pages = cache.shape[0]
    table[0, 0], table[0, 5], table[1, -2:] = -1, pages, -7
    table[2] = table[8] = -1
    table[7, 0], table[7, 3] = -1, pages
    seqlens[3], seqlens[4], seqlens[5], seqlens[9] = 12, 0, 16 * table.shape[1] + 3, 1
    seqlens[6] = -4
    table[5] = torch.randint(0, pages, (table.shape[1],), generator=gen, dtype=torch.int32)
    out = _check_chunk(zb, q, cache, table, seqlens, cu)
    rows = slice(int(cu[2]), int(cu[3]))
    assert out[rows].eq(0).all() and out[int(cu[3]):int(cu[3]) + 18].eq(0).all()


@pytest.mark.parametrize("max_new", [None, 1])
def test_chunk_rows_of_no_request(zb, max_new):
    gen = torch.Generator().manual_seed(6)
    q, cache, table, seqlens, cu = _chunk_inputs(gen, [1, 1] if max_new else [10, 25], [100, 7], 8, 2, 128, 16)
    n = q.shape[0]
    padded = torch.cat([torch.randn(3, 8, 128, generator=gen).bfloat16(), q, torch.randn(40, 8, 128, generator=gen).bfloat16()])
    out = _check_chunk(zb, padded, cache, table, seqlens, cu + 3, max_new=max_new)
    assert out[:3].eq(0).all() and out[3 + n:].eq(0).all()


@pytest.mark.parametrize("news", [[9, 1, 40], [1, 1, 2]])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 48), (96, 32)])
def test_chunk_ignores_what_no_token_wrote(zb, news, hd, page):
    """Anything at all in rows past a request's keys, in free pages and before the windows leaves the result as it was, bit by
    bit; a pair that is not finite stands for zeros where it is seen."""
    gen = torch.Generator().manual_seed(hd + page)
    q, cache, table, seqlens, cu = _chunk_inputs(gen, news, [200, 130, 0], 8, 2, hd, page)
    clean = _check_chunk(zb, q, cache, table, seqlens, cu, window=64, sinks=2)
    used = torch.zeros(cache.shape[0], page, dtype=torch.bool)
    for b in range(3):
        n, keys = int(cu[b + 1] - cu[b]), int(seqlens[b])
        for j in [*range(min(2, keys)), *range(max(0, keys - n + 1 - 64), keys)]:
            used[int(table[b, j // page]), j % page] = True
    junk = torch.randint(0, 256, cache.shape, generator=gen, dtype=torch.uint8)
    for value in range(2):
        for at, width in ((8 * value * hd, hd // 2), ((16 + 2 * value) * hd, hd // 8)):
            to = cache[..., at:at + 16 * width].unflatten(-1, (16, width)).permute(0, 2, 3, 1, 4)  # [pages, blocks, 16, Hkv, width]
            bad = junk[..., at:at + 16 * width].unflatten(-1, (16, width)).permute(0, 2, 3, 1, 4).clone()
            if width == hd // 8:
                bad[..., 1::2] = 0xFF  # NaN
            to[~used.unflatten(1, (-1, 16))] = bad[~used.unflatten(1, (-1, 16))]
    assert torch.equal(clean, _check_chunk(zb, q, cache, table, seqlens, cu, window=64, sinks=2))
    j = int(seqlens[0]) - 1  # the last key of request 0, values of head 1: a pair that is infinite
    p, row = int(table[0, j // page]), j % page
    at = 18 * hd + row % 16 * (hd // 8)
    cache[p, 1, row // 16, at:at + 4] = torch.tensor([math.inf, 1.0]).bfloat16().view(torch.uint8)
    _check_chunk(zb, q, cache, table, seqlens, cu, window=64, sinks=2)


@pytest.mark.parametrize("news", [[6, 1], [1, 2]])
def test_chunk_rising_and_extreme_scores(zb, news):
    """Scores that rise along the keys by hundreds (the running maximum keeps moving) and that fall by hundreds: the keys are 15
    steps of one size apart, so 4 bits hold them."""
    gen = torch.Generator().manual_seed(12)
    for sign in (1.0, -1.0):
        q, cache, table, seqlens, cu = _chunk_inputs(gen, news, [500, 900], 8, 2, 128, 16)
        for b in range(2):
            for j in range(int(seqlens[b])):
                for h in range(2):
                    x = torch.zeros(128).bfloat16()
                    x[:32] = sign * (j // 16)
                    paged_q4.store(cache, int(table[b, j // 16]), j % 16, h, x, False)
        q[..., 1:32] = 0.0
        q[..., 0] = 16.0
        _check_chunk(zb, q, cache, table, seqlens, cu)


def test_chunk_large_values(zb):
    """Values near 2^63, cancelling and not, do not overflow."""
    gen = torch.Generator().manual_seed(13)
    for news in ([1, 2], [40, 3]):
        table, seqlens, cu, pages = _batch(gen, news, [100, 300], 16)
        k, v = (torch.randn(pages, 16, 2, 64, generator=gen) for _ in range(2))
        cache = paged_q4.store_all(k.bfloat16(), (v.clamp(-2, 2) * 2.0 ** 62).bfloat16())
        q = torch.randn(int(cu[-1]), 8, 64, generator=gen).bfloat16()
        _check_chunk(zb, q, cache, table, seqlens, cu)


@pytest.mark.parametrize("news", [[12, 1, 50], [1, 2, 1]])
def test_chunk_layouts(zb, news):
    """A cache that is a slice of a larger pool, heads outermost; q, out and gate as slices of wider rows; a wider page table."""
    gen = torch.Generator().manual_seed(14)
    q, cache, table, seqlens, cu = _chunk_inputs(gen, news, [90, 300, 0], 8, 2, 64, 16)
    gate = torch.randn(q.shape[0], 8, generator=gen).bfloat16()
    N, (pages, kv, blocks, block) = q.shape[0], cache.shape
    pool = torch.full((kv, 2, pages, blocks, block), 255, dtype=torch.uint8, device=DEV)
    view = pool[:, 1].transpose(0, 1)
    view.copy_(cache)
    wide_q = torch.full((N, 8 * 64 + 24), math.nan, dtype=torch.bfloat16, device=DEV)
    wide_q[:, :512] = q.reshape(N, -1).to(DEV)
    wide_out = torch.full((N, 8 * 64 + 16), 3.0, dtype=torch.bfloat16, device=DEV)
    wide_table = torch.full((3, table.shape[1] + 5), 1 << 30, dtype=torch.int32, device=DEV)
    wide_table[:, : table.shape[1]] = table.to(DEV)
    views = {"cache": view, "q": wide_q[:, :512].unflatten(1, (8, 64)), "out": wide_out[:, :512].unflatten(1, (8, 64)),
             "table": wide_table[:, : table.shape[1]]}
    _check_chunk(zb, q, cache, table, seqlens, cu, gate=gate, views=views)
    assert wide_out[:, 512:].eq(3.0).all()
    wide_gate = torch.full((N, 20), math.nan, dtype=torch.bfloat16, device=DEV)
    wide_gate[:, 3:11] = gate.to(DEV)
    got = zb.ops.gqa_chunk_q4(views["q"], view, views["table"], seqlens.to(DEV), cu.to(DEV), gate=wide_gate[:, 3:11])
    assert torch.equal(got, views["out"])


def test_offsets_past_32_bits(zb):
    """Pages whose offsets pass 2^32 bytes: append, attention and reading back."""
    case = ([30, 1], [200, 90], 8, 2, 128, 16, 128, True)
    gen = torch.Generator().manual_seed(15)
    proj, _, table, seqlens, cu, temp = _append_inputs(gen, case)
    pages = int(table.max()) + 4
    cache = _q4_cache(gen, pages, 16, 2, 128)
    stride = ((3 << 31) // (pages - 1) + 16) // 16 * 16
    pool = torch.empty(cache[0].numel() + (pages - 1) * stride, dtype=torch.uint8, device=DEV)
    view = pool.as_strided(cache.shape, (stride, 2560, 2560, 1))
    view.copy_(cache)
    q, _ = _check_append(zb, case, proj, cache, table, seqlens, cu, views={"cache": view}, temp=temp)
    cache = view.cpu().contiguous()
    _check_chunk(zb, q.cpu(), cache, table, seqlens, cu, views={"cache": view})
    _check_chunk(zb, q.cpu()[-1:], cache, table[1:], seqlens[1:], torch.tensor([0, 1], dtype=torch.int32), max_new=1,
                 views={"cache": view})
    k, v = zb.ops.kv_read_q4(view, table.to(DEV), seqlens.to(DEV), cu.to(DEV), 31)
    k64, v64 = paged_q4.read(cache)
    for t, p, row in _slots(table, seqlens, cu, 16, pages):
        assert torch.equal(k[t].cpu(), k64[p, row].bfloat16()) and torch.equal(v[t].cpu(), v64[p, row].bfloat16())


@pytest.mark.parametrize("max_new", [None, 4])
def test_chunk_repeats_bit_for_bit_and_runs_on_another_stream(zb, max_new):
    gen = torch.Generator().manual_seed(16)
    x = [t.to(DEV) for t in _chunk_inputs(gen, [1, 4 if max_new else 40, 1], [9000, 300, 2000], 16, 4, 128, 16)]
    first = zb.ops.gqa_chunk_q4(*x, max_new=max_new)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [zb.ops.gqa_chunk_q4(*x, max_new=max_new) for _ in range(5)]
    again = [zb.ops.gqa_chunk_q4(*x, max_new=max_new) for _ in range(5)]  # at the same time, on the current stream
    side.synchronize()
    assert all(torch.equal(first, o) for o in outs + again)


def test_append_chunk_and_read_in_a_graph_follow_the_lengths(zb):
    """A captured step: the new tokens into the cache, their attention, and both read back, with other lengths at each replay."""
    case = ([30, 1, 2], [40, 3000, 600], 8, 2, 128, 16, 128, True)
    gen = torch.Generator().manual_seed(17)
    proj, cache, table, seqlens, cu, temp = (t.to(DEV) for t in _append_inputs(gen, case))
    cache.copy_(_q4_cache(gen, cache.shape[0], 16, 2, 128))
    start = cache.clone()

    def step():
        q = zb.ops.gqa_append_q4(proj, cache, table, seqlens, cu, heads=8, kv_heads=2, temp=temp)
        return zb.ops.gqa_chunk_q4(q, cache, table, seqlens, cu), *zb.ops.kv_read_q4(cache, table, seqlens, cu, 33)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for lengths, bounds in (([70, 1500, 17], [0, 20, 22, 33]), ([33, 0, 0], [0, 33, 33, 33]), ([1, 2, 3], [0, 1, 2, 3])):
        seqlens.copy_(torch.tensor(lengths, dtype=torch.int32))
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        cache.copy_(start)
        graph.replay()
        got = [t.clone() for t in captured]
        cache.copy_(start)
        expected = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_chunk_refuses_bounds_out_of_order(zb):
    """cu_seqlens_q that decreases or leaves [0, N]: a status bit, and nothing is written."""
    gen = torch.Generator().manual_seed(18)
    q, cache, table, seqlens, cu = (t.to(DEV) for t in _chunk_inputs(gen, [4, 1, 30], [9, 70, 0], 8, 2, 64, 16))
    for bad in ([0, 5, 4, 35], [-1, 4, 5, 35], [0, 4, 5, 36]):
        for max_new in (None, 1):
            out = torch.full_like(q, 3.0)
            zb.ops.gqa_chunk_q4(q, cache, table, seqlens, torch.tensor(bad, dtype=torch.int32, device=DEV), out=out, max_new=max_new)
            assert out.eq(3.0).all() and zb.ops.device_status() & 128


def test_a_window_as_long_as_the_keys_and_sinks_alone_change_nothing(zb):
    gen = torch.Generator().manual_seed(19)
    x = [t.to(DEV) for t in _chunk_inputs(gen, [1, 40], [500, 300], 8, 2, 128, 16)]
    plain = zb.ops.gqa_chunk_q4(*x)
    assert torch.equal(plain, zb.ops.gqa_chunk_q4(*x, window=600)) and torch.equal(plain, zb.ops.gqa_chunk_q4(*x, sinks=7))
    assert torch.equal(plain, zb.ops.gqa_chunk_q4(*x, window=100, sinks=500))


def test_batches_without_rows(zb):
    cache = torch.zeros(2, 2, 1, 1280, dtype=torch.uint8, device=DEV)
    table, seqlens, cu = (torch.zeros(*s, dtype=torch.int32, device=DEV) for s in ((3, 2), (3,), (4,)))
    q = torch.zeros(0, 8, 64, dtype=torch.bfloat16, device=DEV)
    assert zb.ops.gqa_chunk_q4(q, cache, table, seqlens, cu).shape == (0, 8, 64)
    assert zb.ops.gqa_append_q4(q.new_zeros(0, 12 * 64), cache, table, seqlens, cu, heads=8, kv_heads=2).shape == (0, 8, 64)
    assert zb.ops.kv_read_q4(cache, table, seqlens, cu, 0)[0].shape == (0, 2, 64)
