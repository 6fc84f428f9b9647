"""GPU: the paged-cache operators (zb_gqa_append, zb_gqa_chunk) through the package's ops against the float64 oracle
(oracle.paged), over head dims 8 .. 128, query groups 1 .. 16, pages of 1 to 200 rows, requests with no, one, a few and
hundreds of new tokens, caches from empty to many tiles, sliding windows, masked pages, strided and permuted layouts.

Tolerances, derived from the operators' rounding points:
* append rounds once to bf16 (8 significant bits, half a unit in the last place: at most 2^-8 of the value); its fp32 steps before that (norm, two
  products and a sum a rotation) stay below 2^-18 of the rotation pair's magnitude. v is a copy.
* chunk rounds each probability to bf16 (2^-8 each, so at most 2^-8 sum_j p_j |v_j|) and the output once (2^-8 of it, no
  more than of that sum); scores are fp32 sums of exact products, exponentials good to 2^-16, so the rest stays below
  2^-4 of the two. Together 2^-7 (1 + 2^-4) sum_j p_j |v_j|, the sum from the oracle.
* lse: the error of a score, hd 2^-23 sum_d |q_d k_d| scale, and 2^-15 for the exponentials and their fp32 sum."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _batch(gen, news, caches, page, extra=3):
    """(page table, cache_seqlens, cu_seqlens_q, pages): every request's pages scattered over a pool."""
    keys = [n + c for n, c in zip(news, caches)]
    need = [-(-k // page) for k in keys]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((len(news), max(max(need), 1) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    return table, torch.tensor(keys, dtype=torch.int32), torch.tensor(cu, dtype=torch.int32), pages


def _chunk_inputs(gen, news, caches, Hq, Hkv, hd, page, spread=1.0):
    table, seqlens, cu, pages = _batch(gen, news, caches, page)
    k = torch.randn(pages, page, Hkv, hd, generator=gen).bfloat16()
    v = torch.randn(pages, page, Hkv, hd, generator=gen).bfloat16()
    q = (torch.randn(int(cu[-1]), Hq, hd, generator=gen) * spread).bfloat16()
    return q, k, v, table, seqlens, cu


def _check_chunk(zb, q, k, v, table, seqlens, cu, gate=None, views=None, **kw):
    """Runs ops.gqa_chunk on copies of the CPU tensors (``views`` overrides device tensors) and holds the result to
    the oracle. Returns the device output."""
    d = {n: t.to(DEV) for n, t in dict(q=q, k=k, v=v, table=table, seqlens=seqlens, cu=cu).items()}
    d.update(views or {})
    N, Hq, hd = q.shape
    lse = torch.full((N, Hq), 7.0, device=DEV)
    out = zb.ops.gqa_chunk(d["q"], d["k"], d["v"], d["table"], d["seqlens"], d["cu"], lse=lse,
                           gate=None if gate is None else gate.to(DEV), out=d.get("out"), **kw)
    kw = {**kw, "scale": kw.pop("softmax_scale", None)}
    ref, scale, ref_lse, size = paged.chunk(q, k, v, table, seqlens, cu, gate=gate, **kw)
    _close(out, ref, 2.0 ** -7 * (1 + 2.0 ** -4) * scale)
    empty = ref_lse == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty)
    _close(lse.cpu()[~empty], ref_lse[~empty], (2.0 ** -15 + hd * 2.0 ** -23 * size)[~empty])
    assert zb.ops.device_status() == 0
    return out


def _close(got, ref, bound):
    got = got.double().cpu()
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst {((got - ref).abs() / bound.clamp_min(1e-30)).max():.3f} of the bound, " \
                          f"first at {tuple(bad.nonzero()[0].tolist())}: {got[bad][0]} against {ref[bad][0]}"


CHUNKS = [
    # news, caches, Hq, Hkv, hd, page
    ([1], [0], 16, 4, 128, 1),
    ([1, 1, 1, 1], [0, 126, 127, 128], 16, 4, 128, 16),
    ([5, 0, 1, 33], [0, 9, 300, 95], 16, 4, 128, 16),
    ([31, 32, 33, 64, 65], [0, 1, 127, 128, 129], 8, 2, 128, 32),
    ([150, 1], [0, 700], 4, 1, 128, 7),
    ([70, 3], [60, 258], 8, 8, 128, 24),
    ([17, 1, 0], [130, 5, 40], 14, 2, 64, 24),
    ([129, 2], [3, 255], 6, 2, 64, 128),
    ([9, 40], [77, 0], 16, 1, 64, 200),
    ([20, 1], [33, 140], 8, 2, 32, 16),
    ([11, 7], [150, 0], 6, 2, 96, 64),
    ([6, 1], [131, 20], 10, 2, 40, 5),
    ([4, 2], [140, 3], 3, 1, 8, 16),
]


@pytest.mark.parametrize("case", CHUNKS)
@pytest.mark.parametrize("mode", ["causal", "window", "full", "gate"])
def test_chunk_matches_oracle(zb, case, mode):
    news, caches, Hq, Hkv, hd, page = case
    gen = torch.Generator().manual_seed(CHUNKS.index(case))
    x = _chunk_inputs(gen, news, caches, Hq, Hkv, hd, page)
    gate = torch.randn(x[0].shape[0], Hq, generator=gen).bfloat16() if mode == "gate" else None
    kw = {"window": dict(window=37), "full": dict(causal=False)}.get(mode, {})
    _check_chunk(zb, *x, gate=gate, **kw)


@pytest.mark.parametrize("window", [1, 2, 128, 500])
def test_chunk_windows(zb, window):
    gen = torch.Generator().manual_seed(window)
    _check_chunk(zb, *_chunk_inputs(gen, [40, 1, 130], [260, 511, 0], 8, 2, 64, 16), window=window)


@pytest.mark.parametrize("keys,Hq,hd", [(20000, 16, 128), (9001, 4, 64)])
def test_chunk_few_rows_over_a_long_cache(zb, keys, Hq, hd):
    """One and three tokens over a long cache: the key axis is split and joined."""
    gen = torch.Generator().manual_seed(keys)
    _check_chunk(zb, *_chunk_inputs(gen, [1, 3], [keys - 1, keys // 3], Hq, Hq // 4, hd, 64))


def test_chunk_long_prompt(zb):
    gen = torch.Generator().manual_seed(8)
    _check_chunk(zb, *_chunk_inputs(gen, [700], [0], 4, 1, 128, 16))


def test_chunk_many_requests(zb):
    """More requests than CTAs, with and without new tokens."""
    gen = torch.Generator().manual_seed(9)
    news = [(b * 7) % 4 for b in range(700)]
    caches = [(b * 13) % 50 for b in range(700)]
    _check_chunk(zb, *_chunk_inputs(gen, news, caches, 4, 2, 64, 16))


@pytest.mark.parametrize("hd", [64, 128])
def test_chunk_masked_pages_and_short_caches(zb, hd):
    """Pages outside the cache mask their keys (a first page, a last one, every one); more new tokens than keys leaves
    the first rows empty; no keys at all; more keys than the table has columns."""
    gen = torch.Generator().manual_seed(5)
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [20, 9, 4, 30, 6, 8, 3], [150, 140, 60, 0, 0, 200, 90], 8, 2, hd, 16)
    pages = k.shape[0]
    table[0, 0], table[0, 5], table[1, -2:] = -1, pages, -7
    table[2] = -1
    seqlens[3], seqlens[4], seqlens[5] = 12, 0, 16 * table.shape[1] + 3
    seqlens[6] = -4
    table[5] = torch.randint(0, pages, (table.shape[1],), generator=gen, dtype=torch.int32)
    out = _check_chunk(zb, q, k, v, table, seqlens, cu)
    rows = slice(int(cu[2]), int(cu[3]))
    assert out[rows].eq(0).all() and out[int(cu[3]):int(cu[3]) + 18].eq(0).all() and out[int(cu[6]):].eq(0).all()


def test_chunk_rows_of_no_request(zb):
    """Rows before cu[0] and from cu[B] on (a padded batch) come back as zeros, the others as if alone."""
    gen = torch.Generator().manual_seed(6)
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [10, 25], [100, 7], 8, 2, 128, 16)
    padded = torch.cat([torch.randn(3, 8, 128, generator=gen).bfloat16(), q, torch.randn(40, 8, 128, generator=gen).bfloat16()])
    out = _check_chunk(zb, padded, k, v, table, seqlens, cu + 3)
    assert out[:3].eq(0).all() and out[38:].eq(0).all()


@pytest.mark.parametrize("hd,page", [(128, 16), (64, 24), (96, 1), (128, 128)])
def test_chunk_ignores_what_it_does_not_see(zb, hd, page):
    """NaN and infinities in keys and values that a row does not see (rows past the request's keys, free pages, keys
    before the window, its own future) leave it as it was; in a key that it sees they reach it."""
    gen = torch.Generator().manual_seed(hd + page)
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [9, 1, 40], [200, 130, 0], 8, 2, hd, page)
    clean = _check_chunk(zb, q, k, v, table, seqlens, cu, window=64)
    used = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b in range(3):
        n, keys = int(cu[b + 1] - cu[b]), int(seqlens[b])
        for j in range(max(0, keys - n + 1 - 64), keys):
            used[int(table[b, j // page]), j % page] = True
    junk = torch.tensor([math.nan, math.inf, -math.inf])
    pick = torch.randint(0, 3, k.shape, generator=gen)
    k[~used], v[~used] = junk[pick].bfloat16()[~used], junk[pick.flip(0)].bfloat16()[~used]
    dirty = _check_chunk(zb, q, k, v, table, seqlens, cu, window=64)
    assert torch.equal(clean, dirty)
    # a token's own future: the value of request 2's token 20 is not finite
    where = int(table[2, 20 // page]), 20 % page
    v[where][0, 3], v[where][1, hd - 1] = math.nan, math.inf
    got = zb.ops.gqa_chunk(*(t.to(DEV) for t in (q, k, v, table, seqlens, cu)), window=64)
    row = int(cu[2]) + 20
    assert torch.equal(got[:row], clean[:row])
    seen = got[row:]
    assert seen[:, :4, 3].isnan().all() and seen[:, 4:, hd - 1].isinf().all()
    seen[:, :4, 3] = clean[row:, :4, 3]
    seen[:, 4:, hd - 1] = clean[row:, 4:, hd - 1]
    torch.testing.assert_close(seen, clean[row:], atol=2e-2, rtol=2e-2)
    # a key that is NaN: the rows that see it are, the rows that do not are not
    v[where] = 0.0
    k[where][1] = math.nan
    got = zb.ops.gqa_chunk(*(t.to(DEV) for t in (q, k, v, table, seqlens, cu)), window=64)
    assert torch.equal(got[:row], clean[:row])
    assert got[row:, 4:].isnan().all() and not got[row:, :4].isnan().any()


def test_chunk_rising_and_extreme_scores(zb):
    """Scores that rise along the keys by hundreds (the running maximum keeps moving) and that fall by hundreds."""
    gen = torch.Generator().manual_seed(12)
    for sign in (1.0, -1.0):
        q, k, v, table, seqlens, cu = _chunk_inputs(gen, [6, 1], [500, 900], 8, 2, 128, 16)
        for b in range(2):
            for j in range(int(seqlens[b])):
                k[int(table[b, j // 16]), j % 16] *= 0.01
                k[int(table[b, j // 16]), j % 16, :, 0] = sign * j / 16
        q[..., 0] = 8.0
        _check_chunk(zb, q, k, v, table, seqlens, cu)


@pytest.mark.parametrize("layout", ["heads_first", "interleaved", "padded", "slots"])
def test_chunk_layouts(zb, layout):
    """Cache views: KV heads before rows, K and V in one pool, padded rows, one token a page as a 3-D cache; q, out and
    gate as slices of wider rows; a page table wider than its columns."""
    gen = torch.Generator().manual_seed(13)
    page = 1 if layout == "slots" else 16
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [12, 1, 50], [90, 300, 0], 8, 2, 64, page)
    gate = torch.randn(q.shape[0], 8, generator=gen).bfloat16()
    N = q.shape[0]
    views = {}
    if layout == "heads_first":
        views["k"], views["v"] = (t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in (k, v))
    elif layout == "interleaved":
        both = torch.stack([k, v], 1).to(DEV)
        views["k"], views["v"] = both[:, 0], both[:, 1]
    elif layout == "padded":
        both = torch.full((2, *k.shape[:3], 96), math.nan, dtype=torch.bfloat16, device=DEV)
        both[..., :64] = torch.stack([k, v]).to(DEV)
        views["k"], views["v"] = both[0, ..., :64], both[1, ..., :64]
    else:
        views["k"], views["v"] = k[:, 0].to(DEV), v[:, 0].to(DEV)
    wide_q = torch.full((N, 8 * 64 + 24), math.nan, dtype=torch.bfloat16, device=DEV)
    wide_q[:, :512] = q.reshape(N, -1).to(DEV)
    views["q"] = wide_q[:, :512].unflatten(1, (8, 64))
    wide_out = torch.full((N, 8 * 64 + 16), 3.0, dtype=torch.bfloat16, device=DEV)
    views["out"] = wide_out[:, :512].unflatten(1, (8, 64))
    wide_table = torch.full((3, table.shape[1] + 5), 1 << 30, dtype=torch.int32, device=DEV)
    wide_table[:, : table.shape[1]] = table.to(DEV)
    views["table"] = wide_table[:, : table.shape[1]]
    _check_chunk(zb, q, k, v, table, seqlens, cu, gate=gate, views=views)
    assert wide_out[:, 512:].eq(3.0).all()
    wide_gate = torch.full((N, 20), math.nan, dtype=torch.bfloat16, device=DEV)
    wide_gate[:, 3:11] = gate.to(DEV)
    got = zb.ops.gqa_chunk(views["q"], views["k"], views["v"], views["table"], seqlens.to(DEV), cu.to(DEV), gate=wide_gate[:, 3:11])
    assert torch.equal(got, views["out"])


def test_chunk_offsets_past_32_bits(zb):
    """Pages whose offsets pass 2^31 and 2^32 elements."""
    gen = torch.Generator().manual_seed(14)
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [3, 1], [200, 90], 8, 2, 128, 16)
    row, pages = 16 * 2 * 128, k.shape[0]
    stride = ((1 << 32) // (pages - 1) + 8) // 8 * 8
    pool = torch.empty(2 * row + (pages - 1) * stride, dtype=torch.bfloat16, device=DEV)
    kd = pool.as_strided((pages, 16, 2, 128), (stride, 256, 128, 1))
    vd = pool.as_strided((pages, 16, 2, 128), (stride, 256, 128, 1), row)
    kd.copy_(k.to(DEV))
    vd.copy_(v.to(DEV))
    _check_chunk(zb, q, k, v, table, seqlens, cu, views={"k": kd, "v": vd})


def test_chunk_repeats_bit_for_bit_and_runs_on_another_stream(zb):
    gen = torch.Generator().manual_seed(15)
    x = [t.to(DEV) for t in _chunk_inputs(gen, [1, 40, 1], [9000, 300, 2000], 16, 4, 128, 16)]
    first = zb.ops.gqa_chunk(*x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [zb.ops.gqa_chunk(*x) for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_chunk_in_a_graph_follows_the_lengths(zb):
    gen = torch.Generator().manual_seed(16)
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [30, 1, 2], [40, 3000, 600], 8, 2, 128, 16)
    d = [t.to(DEV) for t in (q, k, v, table, seqlens, cu)]
    out = torch.empty_like(d[0])
    zb.ops.gqa_chunk(*d, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        zb.ops.gqa_chunk(*d, out=out)
    d[4].copy_(torch.tensor([70, 1500, 17], dtype=torch.int32))
    d[5].copy_(torch.tensor([0, 20, 22, 33], dtype=torch.int32))
    graph.replay()
    expected = zb.ops.gqa_chunk(*d)
    torch.cuda.synchronize()
    assert torch.equal(out, expected)


# ------------------------------------------------------------------------------------------------------- append

APPENDS = [
    # news, caches, heads, kv_heads, hd, page, rotary, interleaved
    ([1], [877], 16, 4, 128, 1, 128, True),
    ([1, 1, 0, 1], [0, 15, 3, 16], 16, 4, 128, 16, 128, True),
    ([40, 3], [5, 70], 8, 2, 128, 24, 128, False),
    ([13, 1, 30], [100, 2, 0], 14, 2, 64, 24, 32, False),
    ([7, 9], [1, 33], 6, 2, 96, 64, 48, False),
    ([7, 9], [1, 33], 6, 2, 96, 64, 96, True),
    ([5, 6], [0, 1000000], 8, 2, 32, 20000, 32, True),
    ([5, 2], [3, 4], 3, 1, 8, 16, 8, True),
    ([5, 2], [3, 4], 3, 1, 40, 2, 0, True),
]


def _append_inputs(gen, case, pad=0):
    news, caches, heads, kv, hd, page, rotary, interleaved = case
    table, seqlens, cu, pages = _batch(gen, news, caches, page)
    proj = torch.randn(int(cu[-1]), (heads + 2 * kv) * hd + pad, generator=gen).bfloat16()
    cache = torch.randn(2, pages, page, kv, hd, generator=gen).bfloat16()
    temp = (1 + 0.3 * torch.randn(heads, generator=gen)).bfloat16()
    return proj, cache[0].clone(), cache[1].clone(), table, seqlens, cu, temp


def _check_append(zb, proj, k, v, table, seqlens, cu, *, heads, kv_heads, views=None, **kw):
    d = {n: t.to(DEV) for n, t in dict(proj=proj, k=k, v=v, table=table, seqlens=seqlens, cu=cu).items()}
    d.update(views or {})
    extra = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in kw.items()}
    got = zb.ops.gqa_append(d["proj"], d["k"], d["v"], d["table"], d["seqlens"], d["cu"], heads=heads, kv_heads=kv_heads,
                            **extra)
    names = dict(rope_theta="theta", rotary_dim="rotary")
    k64, v64 = k.double(), v.double()
    q64, q_mag, k_mag = paged.append(proj, k64, v64, table, seqlens, cu, heads=heads, kv_heads=kv_heads,
                                     **{names.get(n, n): t for n, t in kw.items() if n != "q_out"})
    _close(got, q64, 2.0 ** -8 * q64.abs() + 2.0 ** -18 * q_mag)
    _close(d["k"], k64, torch.where(k_mag > 0, 2.0 ** -8 * k64.abs() + 2.0 ** -18 * k_mag, 0.0))  # untouched rows: equal
    assert torch.equal(d["v"].cpu().double(), v64)
    return got


@pytest.mark.parametrize("case", APPENDS)
@pytest.mark.parametrize("plain", [False, True])
def test_append_matches_oracle(zb, case, plain):
    gen = torch.Generator().manual_seed(APPENDS.index(case))
    proj, k, v, table, seqlens, cu, temp = _append_inputs(gen, case)
    _, _, heads, kv, _, _, rotary, interleaved = case
    kw = dict(temp=None, eps=None, rope_theta=500.0) if plain else dict(temp=temp, eps=1e-5)
    _check_append(zb, proj, k, v, table, seqlens, cu, heads=heads, kv_heads=kv, rotary_dim=rotary, interleaved=interleaved,
                  **kw)


@pytest.mark.parametrize("pad", [0, 2, 3, 8, 16])
def test_append_strides_and_positions(zb, pad):
    """Projection rows of every alignment, rotary positions of their own, strided caches, q into a slice of a wider row."""
    gen = torch.Generator().manual_seed(pad)
    case = ([4, 1, 60], [10, 0, 3], 6, 2, 64, 16, 64, True)
    proj, k, v, table, seqlens, cu, temp = _append_inputs(gen, case, pad)
    positions = torch.randint(0, 100000, (65,), generator=gen, dtype=torch.int32)
    both = torch.stack([k, v], 2).transpose(1, 3).contiguous().to(DEV).transpose(1, 3)
    wide = torch.full((65, 6 * 64 + 8), 5.0, dtype=torch.bfloat16, device=DEV)
    q_out = wide[:, :384].unflatten(1, (6, 64))
    _check_append(zb, proj, k, v, table, seqlens, cu, heads=6, kv_heads=2, temp=temp, positions=positions, q_out=q_out,
                  views={"k": both[:, :, 0], "v": both[:, :, 1]})
    assert wide[:, 384:].eq(5.0).all()


def test_append_skips_what_has_no_page(zb):
    """Tokens whose page is outside the cache or past the table, more new tokens than keys, rows of no request."""
    gen = torch.Generator().manual_seed(3)
    case = ([20, 5, 9, 4], [10, 30, 0, 8], 8, 2, 64, 8, 64, True)
    proj, k, v, table, seqlens, cu, temp = _append_inputs(gen, case)
    table[0, 2], table[1, 4] = -1, k.shape[0]
    seqlens[2], seqlens[3] = 3, 8 * table.shape[1] + 2
    table[3, -1] = table[3, 0]
    proj = torch.cat([proj[:2], proj, proj[:3]])
    got = _check_append(zb, proj, k, v, table, seqlens, cu + 2, heads=8, kv_heads=2, temp=temp)
    assert got[:2].eq(0).all() and got[-3:].eq(0).all()


def test_append_many_tokens_and_offsets_past_32_bits(zb):
    gen = torch.Generator().manual_seed(4)
    case = ([700, 0, 1300], [3, 4, 0], 4, 2, 32, 16, 32, True)
    proj, k, v, table, seqlens, cu, temp = _append_inputs(gen, case)
    row, pages = 16 * 2 * 32, k.shape[0]
    stride = ((1 << 32) // (pages - 1) + 8) // 8 * 8
    pool = torch.empty(2 * row + (pages - 1) * stride, dtype=torch.bfloat16, device=DEV)
    kd = pool.as_strided((pages, 16, 2, 32), (stride, 64, 32, 1))
    vd = pool.as_strided((pages, 16, 2, 32), (stride, 64, 32, 1), row)
    kd.copy_(k.to(DEV))
    vd.copy_(v.to(DEV))
    _check_append(zb, proj, k, v, table, seqlens, cu, heads=4, kv_heads=2, temp=temp, views={"k": kd, "v": vd})


def test_append_agrees_with_the_decode_prologue(zb):
    """At one token a request the operator does what gqa_prologue_decode does, up to that kernel's two further bf16
    roundings (2^-8 each of the pair's magnitude, both elements rounded, beside either's output)."""
    gen = torch.Generator().manual_seed(21)
    B, slots = 9, 400
    proj = torch.randn(B, 24 * 128 + 16, generator=gen).bfloat16().to(DEV)
    temp = (1 + 0.1 * torch.randn(16, generator=gen)).bfloat16().to(DEV)
    table = torch.randperm(slots, generator=gen)[: B * 40].view(B, 40).to(torch.int32).to(DEV)
    seqlens = torch.randint(1, 41, (B,), generator=gen, dtype=torch.int32).to(DEV)
    kc, vc = (torch.zeros(slots, 4, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kc2, vc2 = kc.clone(), vc.clone()
    loc = table.gather(1, (seqlens.long() - 1)[:, None])[:, 0].contiguous()
    old = zb.ops.gqa_prologue_decode(proj, temp, seqlens - 1, kc, vc, loc, heads=16, kv_heads=4)
    new = zb.ops.gqa_append(proj, kc2, vc2, table, seqlens, torch.arange(B + 1, device=DEV, dtype=torch.int32), heads=16,
                            kv_heads=4, temp=temp)
    for a, b in ((old, new), (kc, kc2)):
        pair = b.double().unflatten(-1, (64, 2)).norm(dim=-1, keepdim=True).expand(*b.shape[:-1], 64, 2).flatten(-2)
        assert ((a.double() - b.double()).abs() <= 4 * 2.0 ** -8 * 1.5 * pair).all()
    assert torch.equal(vc, vc2)


# ------------------------------------------------------------------------------------------------------- refusals


def test_refusals(zb):
    gen = torch.Generator().manual_seed(30)
    q, k, v, table, seqlens, cu = (t.to(DEV) for t in _chunk_inputs(gen, [3, 1], [9, 4], 4, 2, 64, 16))
    good = dict(q=q, k_cache=k, v_cache=v, page_table=table, cache_seqlens=seqlens, cu_seqlens_q=cu)
    zb.ops.gqa_chunk(**good)

    def refuses(error=ValueError, **change):
        with pytest.raises(error):
            zb.ops.gqa_chunk(**{**good, **change})

    refuses(q=q.float())
    refuses(q=q.cpu())
    refuses(q=q[:, :3])  # 3 heads over 2
    refuses(q=q.transpose(0, 1))
    refuses(k_cache=k.float())
    refuses(v_cache=v[:-1])
    refuses(k_cache=k[0, 0], v_cache=v[0, 0])
    refuses(page_table=table.long())
    refuses(page_table=table.cpu())
    refuses(page_table=table[:1])
    refuses(page_table=table.t().contiguous().t())
    refuses(cache_seqlens=seqlens[:1])
    refuses(cu_seqlens_q=cu[:-1])
    refuses(cu_seqlens_q=cu.long())
    refuses(softmax_scale=0.0)
    refuses(softmax_scale=-1.0)
    refuses(softmax_scale=math.nan)
    refuses(window=-1)
    refuses(window=4, causal=False)
    refuses(gate=torch.zeros(4, 3, device=DEV, dtype=torch.bfloat16))
    refuses(gate=torch.zeros(4, 4, device=DEV))
    refuses(lse=torch.zeros(4, 3, device=DEV))
    refuses(out=torch.zeros(3, 4, 64, device=DEV, dtype=torch.bfloat16))
    refuses(workspace=torch.zeros(4, device=DEV))
    refuses(RuntimeError, q=q[..., :60].contiguous(), k_cache=k[..., :60], v_cache=v[..., :60])  # head dim 60
    big = torch.zeros(4, 4, 136, device=DEV, dtype=torch.bfloat16)
    cache = torch.zeros(2, 16, 2, 136, device=DEV, dtype=torch.bfloat16)
    refuses(RuntimeError, q=big, k_cache=cache, v_cache=cache)
    odd = torch.zeros(5 * 256, device=DEV, dtype=torch.bfloat16)
    refuses(q=odd.as_strided((4, 4, 64), (257, 64, 1)))  # rows off 16-byte boundaries
    refuses(q=torch.zeros(4 * 256 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(4, 4, 64))
    none = zb.ops.gqa_chunk(q[:0], k, v, table, seqlens, torch.zeros_like(cu))
    assert none.shape == (0, 4, 64)

    proj = torch.zeros(4, 8 * 64, device=DEV, dtype=torch.bfloat16)
    base = dict(proj=proj, k_cache=k, v_cache=v, page_table=table, cache_seqlens=seqlens, cu_seqlens_q=cu, heads=4, kv_heads=2)
    zb.ops.gqa_append(**base)
    for change in (dict(proj=proj.float()), dict(proj=proj[:, :-1]), dict(proj=proj.t()), dict(heads=5), dict(kv_heads=1),
                   dict(rotary_dim=66), dict(rotary_dim=12), dict(rotary_dim=8, interleaved=False), dict(eps=-1.0),
                   dict(rope_theta=0.0), dict(temp=torch.ones(3, device=DEV, dtype=torch.bfloat16)), dict(heads=0),
                   dict(positions=torch.zeros(3, device=DEV, dtype=torch.int32)), dict(q_out=q[:3])):
        with pytest.raises(ValueError):
            zb.ops.gqa_append(**{**base, **change})
    assert zb.ops.gqa_append(**{**base, "proj": proj[:0], "cu_seqlens_q": torch.zeros_like(cu)}).shape == (0, 4, 64)


@pytest.mark.parametrize("Hq, Hkv, hd, page, window", [(16, 4, 128, 16, 0), (16, 1, 128, 1, 0), (14, 2, 64, 24, 300),
                                                       (8, 8, 40, 8, 0), (4, 4, 128, 128, 0)])
def test_units_of_few_rows_keep_their_weights(zb, Hq, Hkv, hd, page, window):
    """Single tokens (up to 16 rows a KV head): the weights' roundings to bf16 are multiplied too, which leaves 2^-16 of a
    weight. Beside that a weight and the sum that divides it are each off by the exponential's 2^-15 and a score's error;
    the output is rounded once (2^-8 of it)."""
    gen = torch.Generator().manual_seed(11)
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [1, 1, 1, 0, 1, 1], [0, 1, 700, 40, 128, 5000], Hq, Hkv, hd, page)
    out = _check_chunk(zb, q, k, v, table, seqlens, cu, window=window)
    ref, spread, _, size = paged.chunk(q, k, v, table, seqlens, cu, window=window)
    _close(out, ref, 2.0 ** -8 * ref.abs() + 2 * spread * (2.0 ** -16 + 2.0 ** -15 + hd * 2.0 ** -23 * size[..., None]))


@pytest.mark.parametrize("new", [1, 3, 40, 200])
def test_a_row_that_sees_one_key_is_its_value(zb, new):
    """A prompt's first token sees its own key alone: its weight is divided by itself, and the output is v."""
    gen = torch.Generator().manual_seed(new)
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [new, new], [0, 0], 8, 2, 128, 16, spread=3.0)
    out = _check_chunk(zb, q, k, v, table, seqlens, cu).cpu()
    for b in range(2):
        first = v[int(table[b, 0]), 0].repeat_interleave(4, 0)
        assert torch.equal(out[b * new], first)


def test_few_rows_over_infinite_values(zb):
    """A value that is infinite and seen makes its dim infinite, of its sign, also where a weight's rounding left nothing."""
    gen = torch.Generator().manual_seed(5)
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, [1, 1], [299, 511], 16, 4, 128, 16)
    for b, key, sign in ((0, 17, 1.0), (1, 500, -1.0)):
        v[int(table[b, key // 16]), key % 16, :, 3] = sign * math.inf
    d = [t.to(DEV) for t in (q, k, v, table, seqlens, cu)]
    out = zb.ops.gqa_chunk(*d).float().cpu()
    assert (out[0, :, 3] == math.inf).all() and (out[1, :, 3] == -math.inf).all()
    rest = torch.cat([out[..., :3], out[..., 4:]], -1)
    assert torch.isfinite(rest).all()
