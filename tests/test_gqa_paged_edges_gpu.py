"""GPU: edges of the paged-cache operators: values near the ends of bf16's range, workspaces that several calls share,
batches whose bounds are wrong, arguments past 32 bits.

Tolerances are those of tests/test_gqa_paged_gpu.py. Where scores are tens of nats large their own error counts beside
the roundings to bf16: a score is off by at most hd 2^-23 scale sum_d |q_d k_d| (``size`` of the oracle) and 2^-15 for its
exponential, and it moves both a weight and the sum that divides it."""

from __future__ import annotations

import pytest
import torch

from oracle import paged
from test_gqa_paged_gpu import DEV, _chunk_inputs, _close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("news, caches", [([1, 1], [700, 130]), ([40, 200], [300, 0]), ([300], [600]), ([1], [6000])])
@pytest.mark.parametrize("offset", [-60.0, -20.0, 0.0, 20.0, 60.0])
@pytest.mark.parametrize("binade", [-100, 0, 100])
def test_chunk_values_of_any_size(zb, news, caches, offset, binade):
    """Values of 2^100 and 2^-100 under scores around ``offset`` nats: the output is a mean of them, so it is neither
    infinite nor 0."""
    gen = torch.Generator().manual_seed(int(offset) + binade + len(news))
    hd = 64 if len(news) == 1 else 128
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, news, caches, 8, 2, hd, 16)
    if offset:  # one dim adds the offset to every score
        q[..., 0] = 8.0
        k[..., 0] = offset * hd ** 0.5 / 8.0
    v = (v.float() * 2.0 ** binade).bfloat16()
    lse = torch.empty(q.shape[:2], device=DEV)
    out = zb.ops.gqa_chunk(*(t.to(DEV) for t in (q, k, v, table, seqlens, cu)), lse=lse)
    ref, spread, ref_lse, size = paged.chunk(q, k, v, table, seqlens, cu)
    score = hd * 2.0 ** -23 * size + 2.0 ** -15
    _close(out, ref, spread * (2.0 ** -7 * (1 + 2.0 ** -4) + 2 * score[..., None]))
    _close(lse, ref_lse, score)
    assert zb.ops.device_status() == 0


FLAG_BYTES = 4096  # of a workspace's start


def _workspace_calls(gen):
    """Calls whose units span CTAs, on grids of 5 CTAs up to all of the GPU's."""
    calls = []
    for news, caches, heads, kv, hd, page in (([1], [383], 1, 1, 64, 16), ([1, 40, 3], [9000, 300, 2000], 16, 4, 128, 16),
                                              ([1], [700], 2, 1, 128, 16), ([3, 1], [4000, 90], 8, 2, 64, 64)):
        calls.append([t.to(DEV) for t in _chunk_inputs(gen, news, caches, heads, kv, hd, page)])
    return calls


def _need(zb, x):
    q, k, _, table, _, _ = x
    return zb.ops.gqa_chunk_workspace_bytes(q.shape[0], q.shape[1], table, k)


def test_chunk_calls_of_different_grids_share_a_workspace(zb):
    """What a call leaves in its parts does not lie where another call has its flags: those are zero after every call, and
    the results are those on a workspace of their own."""
    calls = _workspace_calls(torch.Generator().manual_seed(17))
    needs = [_need(zb, x) for x in calls]
    assert all(n > 0 for n in needs)
    shared = torch.zeros(max(needs), dtype=torch.uint8, device=DEV)
    for i in (0, 1, 2, 0, 3, 1, 2, 1, 0, 3):
        own = torch.zeros(needs[i], dtype=torch.uint8, device=DEV)
        expected = zb.ops.gqa_chunk(*calls[i], workspace=own)
        got = zb.ops.gqa_chunk(*calls[i], workspace=shared)
        assert torch.equal(got, expected)
        assert not shared[:FLAG_BYTES].any() and not own[:FLAG_BYTES].any()
    assert zb.ops.device_status() == 0


def test_chunk_takes_no_notice_of_flags_that_another_call_left(zb):
    """A call whose waits gave up can leave its flags raised. On such a workspace, the caller's and the stream's own, later
    calls wait for their own CTAs all the same."""
    for x in _workspace_calls(torch.Generator().manual_seed(18)):
        workspace = torch.zeros(_need(zb, x), dtype=torch.uint8, device=DEV)
        expected = zb.ops.gqa_chunk(*x, workspace=workspace)
        for _ in range(3):
            workspace[FLAG_BYTES:].random_(0, 256)  # and parts that are not this call's
            workspace[:FLAG_BYTES].view(torch.int32).fill_(1)  # raised by this process's first call
            assert torch.equal(zb.ops.gqa_chunk(*x, workspace=workspace), expected)
        zb.ops.gqa_chunk(*x)
        for own in zb.ops._CHUNK_WS.values():
            own[FLAG_BYTES:].random_(0, 256)
            own[:FLAG_BYTES].view(torch.int32).fill_(1)
        assert torch.equal(zb.ops.gqa_chunk(*x), expected)
    assert zb.ops.device_status() == 0


@pytest.mark.parametrize("cu", [[0, 5, 3, 8], [0, 10, 5, 20], [3, 2, 2, 2], [0, 400, 0, 400], [-1, 2, 3, 8], [0, 2, 5, 9],
                                [0, 2, 1 << 30, 8]])
def test_chunk_refuses_bounds_out_of_order(zb, cu):
    """cu_seqlens_q that decreases, or leaves the rows there are, is the device status's bit 128, and nothing is written."""
    gen = torch.Generator().manual_seed(19)
    N = 8 if cu[-1] == 9 else max(cu[-1], 4)  # [.., 9]: one row more than there is
    q, k, v, table, seqlens, _ = (t.to(DEV) for t in _chunk_inputs(gen, [N, 1, 1], [40, 300, 70], 8, 2, 64, 16))
    out, lse = torch.full_like(q[:N], 3.0), torch.full((N, 8), 7.0, device=DEV)
    zb.ops.device_status()
    zb.ops.gqa_chunk(q[:N], k, v, table, seqlens, torch.tensor(cu, dtype=torch.int32, device=DEV), out=out, lse=lse)
    assert zb.ops.device_status() == 128
    assert out.eq(3.0).all() and lse.eq(7.0).all()


def test_chunk_takes_bounds_at_the_ends(zb):
    """Requests without tokens at either end, and all rows of no request, are in order."""
    gen = torch.Generator().manual_seed(20)
    q, k, v, table, seqlens, _ = (t.to(DEV) for t in _chunk_inputs(gen, [6, 1, 1], [40, 300, 70], 8, 2, 64, 16))
    for cu in ([0, 0, 8, 8], [8, 8, 8, 8], [0, 0, 0, 0], [0, 8, 8, 8]):
        lse = torch.full((8, 8), 7.0, device=DEV)
        bounds = torch.tensor(cu, dtype=torch.int32)
        out = zb.ops.gqa_chunk(q, k, v, table, seqlens, bounds.to(DEV), lse=lse)
        ref, spread, ref_lse, _ = paged.chunk(*(t.cpu() for t in (q, k, v, table, seqlens)), bounds)
        _close(out, ref, 2.0 ** -7 * (1 + 2.0 ** -4) * spread)
        assert torch.equal(lse.cpu() == -torch.inf, ref_lse == -torch.inf)
        assert zb.ops.device_status() == 0


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 40])
def test_chunk_windows_past_32_bits(zb, window):
    """A window longer than any cache is none."""
    gen = torch.Generator().manual_seed(21)
    x = [t.to(DEV) for t in _chunk_inputs(gen, [40, 1], [260, 511], 8, 2, 64, 16)]
    assert torch.equal(zb.ops.gqa_chunk(*x, window=window), zb.ops.gqa_chunk(*x))


@pytest.mark.parametrize("window", [-1, -(2 ** 32) + 5, -(2 ** 31)])
def test_chunk_refuses_negative_windows(zb, window):
    gen = torch.Generator().manual_seed(22)
    x = [t.to(DEV) for t in _chunk_inputs(gen, [40, 1], [260, 511], 8, 2, 64, 16)]
    with pytest.raises(ValueError):
        zb.ops.gqa_chunk(*x, window=window)


@pytest.mark.parametrize("rotary", [2 ** 32, 2 ** 32 + 64, -8, 72])
def test_append_refuses_rotary_dims_outside_the_head(zb, rotary):
    gen = torch.Generator().manual_seed(23)
    q, k, v, table, seqlens, cu = (t.to(DEV) for t in _chunk_inputs(gen, [4, 1], [20, 9], 4, 2, 64, 16))
    proj = torch.zeros(5, 8 * 64, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        zb.ops.gqa_append(proj, k, v, table, seqlens, cu, heads=4, kv_heads=2, rotary_dim=rotary)


def _definition(q, k, v, table, seqlens, cu, b, window, gate=None):
    """(out, spread) of request b in 64 bits on the device, from dense scores; values that are not finite reach no row that
    does not see them."""
    first, last, keys, page = int(cu[b]), int(cu[b + 1]), int(seqlens[b]), k.shape[1]
    at = torch.arange(keys)
    where = table[b, at // page].long().to(DEV), (at % page).to(DEV)
    key, value = k.to(DEV)[where].double(), v.to(DEV)[where].double()  # [keys, Hkv, hd]
    rows = torch.arange(keys - (last - first), keys, device=DEV)[:, None]
    hidden = (at.to(DEV)[None] > rows) | (at.to(DEV)[None] <= rows - window if window else False)
    x = q[first:last].to(DEV).double()
    out, spread = torch.empty_like(x), torch.empty_like(x)
    group = q.shape[1] // k.shape[2]
    for h in range(q.shape[1]):
        s = (x[:, h] @ key[:, h // group].t() * q.shape[2] ** -0.5).masked_fill(hidden, float("-inf"))
        w = torch.softmax(s, -1)
        out[:, h], spread[:, h] = w @ value[:, h // group], w @ value[:, h // group].abs()
    return out, spread


LONG = [
    # news, caches, Hq, Hkv, hd, page, window: units with runs of tiles that every row sees between tiles that hide keys
    ([1747] * 8, [5] * 8, 16, 2, 64, 24, 0),
    ([1400] * 12, [0] * 12, 16, 4, 128, 16, 0),
    ([2000, 900, 3000], [300, 1200, 0], 6, 2, 128, 64, 0),
    ([512, 511, 100], [8192, 6001, 3000], 16, 4, 128, 32, 0),
    ([1, 80, 1, 1, 40, 300] * 8, [5000, 3000, 1856, 4100, 2500, 900] * 8, 8, 8, 128, 16, 1856),
    ([597] * 40, [154] * 40, 8, 2, 128, 64, 964),
    ([1] * 64, [3000] * 64, 14, 2, 64, 128, 1000),
]


@pytest.mark.parametrize("case", LONG)
def test_chunk_long_runs_of_tiles(zb, case):
    """Page copies against 16-byte copies of the same tiles (pages of one row), bit by bit, and against the definition;
    then with values that are not finite in every request, in the future of its first new tokens and, with a window, behind it."""
    news, caches, Hq, Hkv, hd, page, window = case
    gen = torch.Generator().manual_seed(LONG.index(case))
    q, k, v, table, seqlens, cu = _chunk_inputs(gen, news, caches, Hq, Hkv, hd, page)
    # the same rows as pages of one row
    rows = (table.long()[:, :, None] * page + torch.arange(page)).flatten(1).clamp(min=-1).to(torch.int32)

    def both(v):
        slots = [t.reshape(-1, Hkv, hd).to(DEV) for t in (k, v)]
        paged = zb.ops.gqa_chunk(*(t.to(DEV) for t in (q, k, v, table, seqlens, cu)), window=window)
        assert zb.ops.device_status() == 0
        single = zb.ops.gqa_chunk(q.to(DEV), *slots, rows.to(DEV), seqlens.to(DEV), cu.to(DEV), window=window)
        assert zb.ops.device_status() == 0
        return paged, single

    clean, single = both(v)
    assert torch.equal(clean, single)
    for b in {0, len(news) // 2, len(news) - 1}:
        ref, spread = _definition(q, k, v, table, seqlens, cu, b, window)
        got = clean[int(cu[b]):int(cu[b + 1])]
        _close(got, ref.cpu(), 2.0 ** -7 * (1 + 2.0 ** -4) * spread.cpu())
    dirty, unseen = v.clone(), torch.ones(len(q), dtype=torch.bool)
    for b, (n, c) in enumerate(zip(news, caches)):
        for j, bad in ((c + n - 1, torch.nan), (c + n // 2, torch.inf), (c - window if window else -1, -torch.inf)):
            if j < 0:
                continue
            dirty[int(table[b, j // page]), j % page, :, 5] = bad
            seen = torch.arange(n) + c >= j
            if window:
                seen &= torch.arange(n) + c < j + window
            unseen[int(cu[b]):int(cu[b + 1])][seen] = False
    paged, single = both(dirty)
    assert torch.equal(paged[unseen.to(DEV)], clean[unseen.to(DEV)])
    assert torch.equal(paged.isnan(), single.isnan()) and torch.equal(paged.nan_to_num(), single.nan_to_num())
    assert not paged[(~unseen).to(DEV)][..., 5].isfinite().any()


@pytest.mark.parametrize("news, caches, Hq", [([200, 40], [0, 300], 8), ([130], [600], 6), ([5, 1, 1, 3], [700, 300, 20, 0], 8),
                                              ([1, 1, 1], [500, 40, 260], 6)])
def test_chunk_rows_keep_their_bits_whatever_stands_beside_them(zb, news, caches, Hq):
    """Other requests' queries, and keys in a token's own future, leave every bit of its output as it was, also where they
    make other rows' scores thousands of times as large."""
    gen = torch.Generator().manual_seed(24 + len(news))
    x = _chunk_inputs(gen, news, caches, Hq, 2, 128, 16)
    clean = zb.ops.gqa_chunk(*(t.to(DEV) for t in x))
    q, k, v, table, seqlens, cu = x
    for b, n in enumerate(news):
        first, last = int(cu[b]), int(cu[b + 1])
        loud = q.clone()  # every request but b
        loud[:first], loud[last:] = 1000.0 * q[:first], 1000.0 * q[last:]
        got = zb.ops.gqa_chunk(*(t.to(DEV) for t in (loud, k, v, table, seqlens, cu)))
        assert torch.equal(got[first:last], clean[first:last])
        for i in sorted({n - 1, n // 2, n // 3}):
            j = caches[b] + i  # token i's own key: tokens before it do not see it
            loud = k.clone()
            loud[int(table[b, j // 16]), j % 16] *= 1000.0
            got = zb.ops.gqa_chunk(*(t.to(DEV) for t in (q, loud, v, table, seqlens, cu)))
            assert torch.equal(got[first:first + i], clean[first:first + i])
