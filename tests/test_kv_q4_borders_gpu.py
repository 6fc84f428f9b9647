"""GPU: codes next to a border: where x - m has more bits than fp32, the code is that of the exact difference. The cache's bytes are
equal to the oracle's, whose 64 bits hold every difference here."""

from __future__ import annotations

import pytest
import torch

from oracle import paged_q4

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("step", [1.0, 2.0 ** -40, 2.0 ** 40])
def test_codes_beside_a_border(zb, hd, step):
    """m = -(k + 1/2) s and elements of both signs down to 2^-40 s: x - m is (k + 1/2) s, a little less, or a little more."""
    rows = []
    for k in range(15):
        x = torch.zeros(hd)
        x[0::32], x[1::32] = -(k + 0.5), 14.5 - k  # a range of 15 steps: s = 1
        for i in range(2, 32):
            x[i::32] = (-1) ** i * 2.0 ** -(1 + i * 1.3 // 1)
        rows.append(x * step)
    x = torch.stack(rows).bfloat16()
    n = len(x)
    proj = torch.cat([x, x.flip(0)], 1)
    cache = torch.zeros(2, 1, 1, 20 * hd, dtype=torch.uint8)
    table, seqlens, cu = (torch.tensor(t, dtype=torch.int32) for t in ([[1]], [n], [0, n]))
    got = cache.to(DEV)
    zb.ops.gqa_append_q4(proj.to(DEV), got, table.to(DEV), seqlens.to(DEV), cu.to(DEV), heads=0, kv_heads=1, eps=None, rotary_dim=0)
    for t in range(n):
        paged_q4.store(cache, 1, t, 0, proj[t, :hd], False)
        paged_q4.store(cache, 1, t, 0, proj[t, hd:], True)
    assert torch.equal(got.cpu(), cache)
