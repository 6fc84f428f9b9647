"""GPU: kv_read_q4 with more rows than its requests have, as a captured call for other lengths has: zeros, and no search through the
requests for them (one dependent load each: hundreds of microseconds at the largest batch)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _time(call):
    call()
    best = float("inf")
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        call()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("before", [0, 5])
def test_rows_behind_the_last_request(zb, before):
    requests, rows = 16000, 9000
    cache = torch.randint(0, 256, (4, 1, 1, 640), dtype=torch.uint8, device=DEV)
    cache[..., 16 * 32:] = torch.tensor([1.0, -2.0]).bfloat16().view(torch.uint8).repeat(32).to(DEV)
    k, v = torch.empty(2, rows, 1, 32, dtype=torch.bfloat16, device=DEV)

    def call(b):
        table = torch.zeros(b, 1, dtype=torch.int32, device=DEV)
        seqlens = torch.full((b,), 3, dtype=torch.int32, device=DEV)
        cu = torch.full((b + 1,), before + 3, dtype=torch.int32, device=DEV)
        cu[0] = before  # the first request has three rows, the others none
        return lambda: zb.ops.kv_read_q4(cache, table, seqlens, cu, rows, k_out=k, v_out=v)

    one = _time(call(1))
    expected = k.clone(), v.clone()
    k.fill_(7.0), v.fill_(7.0)
    many = _time(call(requests))
    assert torch.equal(k, expected[0]) and torch.equal(v, expected[1])
    assert k[:before].eq(0).all() and k[before + 3:].eq(0).all() and v[before + 3:].eq(0).all()
    assert k[before:before + 3].ne(0).any(2).all()
    assert many < 5 * one + 0.05  # the cost of 16000 loads one after the other is several times that
